"""Dropout in the denoiser's training path (transformer.py:34-72, 302-314): attention with dropped-out probabilities against
its formula in 64 bits, and the whole model, forward and gradients, against a 64-bit restatement that applies the same masks."""
import ctypes as C
import math

import pytest
import torch
import torch.nn.functional as F
import torch.utils.checkpoint

import gpt_amd
from gpt_amd import _lib as L
from oracle import denoiser as od
from tests.cases import gpt_kwargs, make_inputs
from tests.test_hip_parity import plan_of, rel_err
from tests.test_ops import BF, F32, HALF, U, normal, philox_keep, within

DEV = "cuda:0"
gpu = pytest.mark.gpu


def mask(shape, p, seed, offset):
    """keep * scale of a tensor's elements, 64 bits on the CPU."""
    n = math.prod(shape)
    thr = round(65536 * p)
    scale = 0.0 if thr >= 65536 else 65536.0 / (65536.0 - thr)
    return philox_keep(n, p, seed, offset).double().view(shape) * scale


# -------------------------------------------------------------------------------------------------------------- attention
@gpu
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("t", [BF, F32])
@pytest.mark.parametrize("B,T,t_out,H,p", [(3, 26, 26, 2, 0.1), (2, 18, 7, 3, 0.5), (1, 1, 1, 1, 0.5), (5, 32, 32, 1, 0.9), (2, 13, 13, 2, 0.0),
                                          (2, 9, 4, 2, 1.0)])
def test_attention_dropout_and_gradients(B, T, t_out, H, p, hd, t):
    d, seed, offset = H * hd, 0x1234567890AB, (1 << 40) + 3
    qkv, dy = normal(1, B * T, 3 * d, dtype=t), normal(2, B * T, d, dtype=t)
    drop = L.Dropout(p, seed, offset, None)
    y, dqkv = torch.empty(B * t_out, d, device=DEV, dtype=t), torch.full_like(qkv, math.nan)
    code = L.BF16 if t == BF else L.F32
    L.check(L.lib().gpt_attention_dropout(code, L.ptr(qkv), L.ptr(y), B, T, t_out, H, hd, drop, L.stream()), "fwd")
    L.check(L.lib().gpt_attention_dropout_bwd(code, L.ptr(qkv), L.ptr(dy), L.ptr(dqkv), B, T, H, hd, drop, L.stream()), "bwd")
    # the formula, and how far float32 sums, the softmax and one rounding of P~ and dS to the type may take a result from it
    half = 0.0 if t == F32 else HALF[t]
    q, k, v = (x.transpose(1, 2) for x in qkv.cpu().double().view(B, T, 3, H, hd).unbind(2))
    g = dy.cpu().double().view(B, T, H, hd).transpose(1, 2)
    M = mask((B, H, T, 32), p, seed, offset)[..., :T]
    c = hd ** -0.5
    P = torch.softmax(c * q @ k.transpose(-1, -2), -1)
    Pd = M * P
    eP = 2 * (U * (hd + 8) * (c * q.abs() @ k.abs().transpose(-1, -2)).amax(-1, keepdim=True) + 4 * U) + (T + 16) * U
    join = lambda x: x.transpose(1, 2).reshape(B, -1, d)                                                   # noqa: E731
    want = join(Pd @ v)
    tol = join((half + eP + (T + 6) * U) * Pd @ v.abs())
    rounded = lambda x, e: e + HALF[t] * (x.abs() + e)                                                      # noqa: E731
    within(y.cpu().view(B, t_out, d), want[:, :t_out], rounded(want, tol)[:, :t_out], "y")
    absdP, dP = M * (g.abs() @ v.abs().transpose(-1, -2)), M * (g @ v.transpose(-1, -2))
    D = (P * dP).sum(-1, keepdim=True)
    eD = (P * (eP * dP.abs() + (hd + T + 8) * U * absdP)).sum(-1, keepdim=True)
    dS = P * (dP - D)
    n = (T + 8) * U
    edS = P * (eP * (dP - D).abs() + (hd + 8) * U * absdP + eD) + (half + 4 * U + n) * dS.abs()
    grads = [(c * dS @ k, c * edS @ k.abs()), (c * dS.transpose(-1, -2) @ q, c * edS.transpose(-1, -2) @ q.abs()),
             (Pd.transpose(-1, -2) @ g, ((half + eP + n) * Pd).transpose(-1, -2) @ g.abs())]
    for name, got, (w, e) in zip(("dq", "dk", "dv"), dqkv.cpu().view(B, T, 3, d).unbind(2), grads):
        within(got, join(w), rounded(join(w), join(e)), name)


@gpu
def test_attention_dropout_device_counter_and_repeatability():
    B, T, H, hd = 2, 26, 2, 64
    qkv = normal(3, B * T, 3 * H * hd, dtype=BF)
    counter = torch.tensor([5], dtype=torch.int64, device=DEV)

    def run(offset, dev):
        y = torch.empty(B * T, H * hd, device=DEV, dtype=BF)
        drop = L.Dropout(0.4, 9, offset, L.ptr(counter) if dev else None)
        L.check(L.lib().gpt_attention_dropout(L.BF16, L.ptr(qkv), L.ptr(y), B, T, T, H, hd, drop, L.stream()), "fwd")
        return y
    assert torch.equal(run(7, False), run(2, True)) and not torch.equal(run(7, False), run(8, False))


def test_refusals_before_any_launch():
    lib = L.lib()
    one = C.c_void_p(16)
    for drop, args, word in ((None, (L.BF16, 2, 26, 26, 2, 64), "null"), (L.Dropout(1.5, 0, 0, None), (L.BF16, 2, 26, 26, 2, 64), "probability"),
                             (L.Dropout(0.1, 0, 0, None), (L.BF16, 2, 33, 33, 2, 64), "T <= 32"),
                             (L.Dropout(0.1, 0, 0, None), (L.BF16, 2, 26, 27, 2, 64), "stored rows"),
                             (L.Dropout(0.1, 0, 0, None), (L.BF16, 2, 26, 26, 2, 48), "head dim"), (L.Dropout(0.1, 0, 0, None), (7, 2, 26, 26, 2, 64), "dtype"),
                             (L.Dropout(0.1, 0, 0, 4), (L.BF16, 2, 26, 26, 2, 64), "counter")):
        code, B, T, t_out, H, hd = args
        assert lib.gpt_attention_dropout(code, one, one, B, T, t_out, H, hd, drop, None) != 0
        assert word in lib.gpt_last_error().decode(), (word, lib.gpt_last_error())
    assert lib.gpt_attention_dropout_bwd(L.BF16, one, None, one, 2, 26, 2, 64, L.Dropout(0.1, 0, 0, None), None) != 0


# ------------------------------------------------------------------------------------------------------------------ model
PDROP = dict(embd_pdrop=0.15, attn_pdrop=0.3, resid_pdrop=0.2)


def restated(sd, plan, inputs, drop, pruned, pd):
    """od.forward with the masks of one training step; everything in the type of `sd` (64 bits)."""
    x, t, lt, lp, xp = inputs
    B, T, H, d = x.shape[0], plan.T, plan.n_head, plan.n_embd
    hd, To = d // H, len(plan.output_splits)
    site = lambda s, shape, p: mask(shape, p, drop.seed, drop.offset + s)                                   # noqa: E731
    freqs = od.frequencies(plan.num_frequencies, plan.max_freq_log2)
    inp = torch.cat([x.double(), xp.double(), od.freq_embed(t, freqs).double(), od.embed_loss(lt, lp, freqs, plan.absolute).double()], 1)
    h = (od.encode(sd, plan, inp) + sd["decoder.pos_emb"]) * site(0, (B, T, d), pd["embd_pdrop"])
    for l in range(plan.n_layer):
        pre = f"decoder.blocks.{l}."
        w = lambda n: sd[pre + n]                                                                           # noqa: E731,B023
        lin = lambda y, n: F.linear(y, w(n + ".weight"), w(n + ".bias"))                                    # noqa: E731,B023
        a = F.layer_norm(h, (d,), w("ln1.weight"), w("ln1.bias"), 1e-5)
        q, k, v = (lin(a, f"attn.{n}").view(B, T, H, hd).transpose(1, 2) for n in ("query", "key", "value"))
        P = torch.softmax(q @ k.transpose(-1, -2) / math.sqrt(hd), -1) * site(1 + 3 * l, (B, H, T, 32), pd["attn_pdrop"])[..., :T]
        y = (P @ v).transpose(1, 2).reshape(B, T, d)
        if pruned and l == plan.n_layer - 1:
            y, h = y[:, :To], h[:, :To]
        h = h + lin(y, "attn.proj") * site(2 + 3 * l, y.shape, pd["resid_pdrop"])
        y = lin(F.gelu(lin(F.layer_norm(h, (d,), w("ln2.weight"), w("ln2.bias"), 1e-5), "mlp.0")), "mlp.2")
        h = h + y * site(3 + 3 * l, y.shape, pd["resid_pdrop"])
    h = F.layer_norm(h, (d,), sd["decoder.ln_f.weight"], sd["decoder.ln_f.bias"], 1e-5)
    return od.decode(sd, plan, h) + xp.double()


def model(dtype, n_embd, n_head, pd, seed=0, n_layer=2):
    kw = dict(gpt_kwargs("mnist_small"), n_embd=n_embd, n_head=n_head, n_layer=n_layer, **pd)
    base = plan_of("mnist_small")
    plan = od.Plan(kw["parameter_sizes"], 128, 14, True, n_head, n_embd, n_layer, kw["chunk_size"], kw["split_policy"], base.predict_xstart)
    sd = od.random_state_dict(plan, seed=seed)
    m = gpt_amd.Gpt(**kw)
    m.load_state_dict(sd)
    return m.to(DEV).train().set_compute_dtype(dtype), plan, sd


def steps(m, inputs, c, seed):
    """One training forward and backward; the masks' descriptor comes from the same draw."""
    torch.manual_seed(seed)
    drop = m.draw_dropout()
    torch.manual_seed(seed)
    for p in m.parameters():
        p.grad = None
    x, t, lt, lp, xp = (v.to(DEV) for v in inputs)
    out = m(x, t, lt, loss_prev=lp, x_prev=xp)
    (out * c.to(DEV)).sum().backward()
    return drop, out.detach().cpu(), {k: p.grad.float().cpu().clone() for k, p in m.named_parameters()}


@gpu
@pytest.mark.parametrize("pd", [PDROP] + [{k: (v if k == one else 0.0) for k, v in PDROP.items()} for one in PDROP], ids=["all", *PDROP])
@pytest.mark.parametrize("dtype,n_embd,n_head", [("fp32", 192, 2), ("bf16", 192, 2), ("bf16", 256, 4)])
def test_model_forward_and_gradients(dtype, n_embd, n_head, pd):
    """The bars are those of the same path without dropout: float32 2e-4 of the largest output change, 1e-3 of a gradient's largest
    element; bf16 a cosine of 0.99 per parameter (a wrong mask at these rates leaves 0.9 at the most).  256 columns in bf16 take the
    last Block on the decoded tokens alone."""
    m, plan, sd = model(dtype, n_embd, n_head, pd)
    inputs = make_inputs("mnist_small", B=6, seed=11)
    c = normal(7, *inputs[0].shape, device="cpu")
    drop, out, grads = steps(m, inputs, c, seed=5)
    leaves = {k: v.double().requires_grad_() for k, v in sd.items() if k in grads}
    want = restated({**{k: v.double() for k, v in sd.items()}, **leaves}, plan, inputs, drop, dtype == "bf16" and n_embd % 256 == 0, pd)
    (want * c.double()).sum().backward()
    change, xp = (want.detach() - inputs[4].double()), inputs[4].double()
    if dtype == "fp32":
        assert rel_err(out.double() - xp, change) < 2e-4
    else:
        assert float(F.cosine_similarity((out.double() - xp).flatten(), change.flatten(), 0)) > 0.999
    for k, g in grads.items():
        ref = leaves[k].grad
        if k.endswith("attn.key.bias"):
            continue                                     # its gradient is zero without rounding
        if dtype == "fp32":
            assert float((g.double() - ref).abs().max()) < 1e-3 * float(ref.abs().max()) + 1e-9, k
        else:
            assert float(F.cosine_similarity(g.double().flatten(), ref.flatten(), 0)) > 0.99, k


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_model_seeds_modes_and_no_grad(dtype):
    m, plan, sd = model(dtype, 192, 2, PDROP)
    inputs = make_inputs("mnist_small", B=4, seed=13)
    c = normal(8, *inputs[0].shape, device="cpu")
    _, a, ga = steps(m, inputs, c, seed=1)
    _, b, _ = steps(m, inputs, c, seed=1)
    _, other, _ = steps(m, inputs, c, seed=2)
    assert torch.equal(a, b) and not torch.equal(a, other)
    # a forward without gradients draws the same masks (its kernels are the sampling path's)
    torch.manual_seed(1)
    args = [v.to(DEV) for v in inputs]
    with torch.no_grad():
        free = m(args[0], args[1], args[2], loss_prev=args[3], x_prev=args[4]).cpu()
    assert rel_err(free - inputs[4], a - inputs[4]) < (2e-4 if dtype == "fp32" else 2e-2)
    # evaluation mode: exactly the model without dropout, and nothing drawn
    plain = gpt_amd.Gpt(**dict(gpt_kwargs("mnist_small"), n_embd=192, n_head=2, n_layer=2))
    plain.load_state_dict(sd)
    plain = plain.to(DEV).eval().set_compute_dtype(dtype)
    state = torch.get_rng_state()
    with torch.no_grad():
        e = m.eval()(args[0], args[1], args[2], loss_prev=args[3], x_prev=args[4])
        f = plain(args[0], args[1], args[2], loss_prev=args[3], x_prev=args[4])
    assert torch.equal(e, f) and torch.equal(state, torch.get_rng_state())


def test_refuses_to_draw_masks_into_a_captured_graph(monkeypatch):
    m = gpt_amd.Gpt(**dict(gpt_kwargs("mnist_small"), **PDROP)).train()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert isinstance(m.draw_dropout(), L.DenoiserDropout) and m.eval().draw_dropout() is None
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert m.draw_dropout() is None                      # evaluation mode: nothing to draw
    with pytest.raises(L.GptHipError, match="captured graph"):
        m.train().draw_dropout()


@gpu
@pytest.mark.parametrize("dtype,n_embd,n_head", [("fp32", 192, 2), ("bf16", 256, 4)])
def test_train_step_uses_the_masks(dtype, n_embd, n_head):
    """TrainStep.loss_and_grads with dropout: the gradients of the autograd route under the same seed, and other masks every step."""
    from gpt_amd.trainstep import TrainStep
    m, plan, sd = model(dtype, n_embd, n_head, PDROP)
    diff = gpt_amd.create_diffusion(learn_sigma=False, predict_xstart=True, noise_schedule="linear", steps=1000)
    _, t, lt, lp, xp = (v.to(DEV) for v in make_inputs("mnist_small", B=6, seed=17))
    x1 = xp + 0.1 * normal(3, *xp.shape)
    noise = normal(4, *xp.shape)
    torch.manual_seed(3)
    diff.training_losses(m, x1, t, model_kwargs=dict(loss_target=lt, loss_prev=lp, x_prev=xp), noise=noise)["loss"].mean().backward()
    want = {k: p.grad.float().cpu().clone() for k, p in m.named_parameters()}
    for p in m.parameters():
        p.grad = None
    step = TrainStep(m, diff, use_ema=False)
    got = []
    for seed in (3, None):
        if seed is not None:
            torch.manual_seed(seed)
        step.grads.zero_()
        step.loss_and_grads(xp, x1, lp, lt, t, noise=noise)
        got.append({k: v.clone().cpu() for (k, _), v in zip(m.named_parameters(), m.engine(xp.device).arena.views(step.grads, m))})
    for k, w in want.items():
        if k.endswith("attn.key.bias"):
            continue
        assert float((got[0][k].reshape(w.shape) - w).abs().max()) <= 2e-5 * float(w.abs().max()) + 1e-12, k
    k = "decoder.blocks.1.mlp.0.weight"
    assert float(F.cosine_similarity(got[0][k].flatten(), got[1][k].flatten(), 0)) < 0.999


@gpu
@pytest.mark.parametrize("pd", [PDROP, dict(embd_pdrop=0.0, attn_pdrop=0.0, resid_pdrop=0.5)], ids=["all", "resid"])
@pytest.mark.parametrize("B", [1, 5])
def test_one_seed_means_one_set_of_masks_with_and_without_gradients(B, pd):
    """256 columns in bf16: the training forward takes the last Block on the decoded tokens' rows, and so does the forward without gradients
    (activation checkpointing runs both).  The bar is that of 192 columns, where no rows are left out: the two forwards' kernels
    round differently, a mask of other rows changes the output by its own size."""
    m, plan, _ = model("bf16", 256, 4, pd)
    inputs = make_inputs("mnist_small", B=B, seed=19)
    c = normal(8, *inputs[0].shape, device="cpu")
    _, a, grads = steps(m, inputs, c, seed=1)
    args = [v.to(DEV) for v in inputs]
    call = lambda x: m(x, args[1], args[2], loss_prev=args[3], x_prev=args[4])                              # noqa: E731
    torch.manual_seed(1)
    with torch.no_grad():
        free = call(args[0]).cpu()
    assert rel_err(free - inputs[4], a - inputs[4]) < 2e-2
    # checkpointed: a pass without gradients, then one with them under the same generator state
    torch.manual_seed(1)
    for p in m.parameters():
        p.grad = None
    out = torch.utils.checkpoint.checkpoint(call, args[0].clone().requires_grad_(), use_reentrant=True)
    assert rel_err(out.detach().cpu() - inputs[4], a - inputs[4]) < 2e-2
    (out * c.to(DEV)).sum().backward()
    for k, p in m.named_parameters():
        assert torch.equal(p.grad.float().cpu(), grads[k]) or rel_err(p.grad.float().cpu(), grads[k]) < 1e-4, k
