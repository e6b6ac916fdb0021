"""gpt_amd.ops.diff_attention in bfloat16 rounds its results once and nothing else to 8 bits: the softmax weights P and the score
gradients dS enter the matrix products as two bfloat16 operands each, so their error is at most 2^-8 of 2^-8 of them."""
import ctypes as C

import pytest
import torch

from gpt_amd import _lib as L
from gpt_amd import ops
from tests.test_ops import BF, HALF, attention_case, attention_reference, gpu, within

TWO = HALF[BF] ** 2        # what the second operand's rounding leaves of the value


def check_two_operands(B, Tq, Tk, H, hd, lens=None, std=1.0):
    """Every element within the bound of float32 sums, of 2^-16 of P and dS and of the result's one rounding; and over a whole tensor no
    more than 1.1 times the error that rounding the exact result leaves (what is left beside it is 2^-8 of it and some 100 u; one
    more independent rounding of the same size would give 1.4)."""
    _, q, k, v, lam, n, g = attention_case(B, Tq, Tk, H, hd, BF, lens, False, std=std)
    want, tol = attention_reference(q, k, v, lam, H, n, hd ** -0.5, g, TWO)
    leaves = [x.clone().requires_grad_() for x in (q, k, v, lam)]
    out = ops.diff_attention(*leaves, H, n)
    got = dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, g)[:3])))
    for name, x in got.items():
        w = want[name]
        within(x, w, tol[name] + HALF[BF] * (w.abs() + tol[name]), name)
        once = float((w.to(BF).double() - w).norm())
        off = float((x.double() - w).norm())
        assert off <= 1.1 * once + float(tol[name].norm()) * 2.0 ** -8, (name, off, once)


@gpu
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("B,Tq,Tk,lens", [(64, 26, 26, None), (9, 32, 32, [32, 0, 1, 2, 31]), (7, 5, 31, [31, 3, 16]), (3, 17, 1, None), (2, 1, 1, None)])
def test_short_attention_rounds_only_its_results(B, Tq, Tk, lens, hd):
    check_two_operands(B, Tq, Tk, 3, hd, lens)


@gpu
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("B,Tq,Tk,H,lens,std", [
    (2, 130, 130, 3, None, 1.0), (9, 40, 40, 2, [0, 1, 2, 3, 5, 40], 1.0), (2, 96, 200, 2, [200, 77], 2.0),     # few waves per workgroup
    (24, 161, 140, 8, [140, 0, 17, 1, 133], 1.0), (48, 128, 96, 8, None, 1.5),                               # the larger workgroups
    (2, 600, 600, 1, [600, 301], 1.0), (1, 1, 3000, 2, None, 1.0), (2, 20, 900, 1, [900, 1], 1.0)])          # cut into spans and joined
def test_long_attention_rounds_only_its_results(B, Tq, Tk, H, lens, std, hd):
    check_two_operands(B, Tq, Tk, H, hd, lens, std)


@gpu
@pytest.mark.parametrize("T", [20, 70])
def test_rows_of_one_key_have_no_gradient_of_the_scores(T):
    """One key per sample: its weight is 1 whatever the scores are, so dq and dk are 0.  dP - D is what float32 sums of 2 hd products (u each) and,
    on the long path, the outputs to 16 bits leave of 0."""
    B, H, hd = 3, 2, 64
    _, q, k, v, lam, n, g = attention_case(B, T, T, H, hd, BF, [1], False)
    leaves = [x.clone().requires_grad_() for x in (q, k, v, lam)]
    dq, dk, dv, _ = torch.autograd.grad(ops.diff_attention(*leaves, H, n), leaves, g)
    absdP = (g.double().abs().view(B, T, H, -1) * v[:, :1].double().abs().view(B, 1, H, -1)).sum(-1)        # one key: P = 1
    bound = (hd ** -0.5 * (2 * TWO + (4 * hd + 16) * 2.0 ** -24)) * absdP[..., None, None]
    bound = bound * torch.stack([torch.ones(H), lam.cpu().abs()], -1).to(q.device).view(1, 1, H, 2, 1)
    by = lambda x: x.double().abs().view(B, -1, H, 2, hd)                                                    # noqa: E731
    assert bool((by(dq) <= bound * by(k[:, :1]) * (1 + HALF[BF])).all())
    assert bool((by(dk)[:, :1] <= (bound * by(q)).sum(1, keepdim=True) * (1 + HALF[BF])).all()) and bool((dk[:, 1:] == 0).all())


def test_rest_is_refused_where_it_does_not_belong():
    """Before any launch: no GPU is needed."""
    lib, one = L.lib(), 1 << 20

    def call(rest, **kw):
        a = L.DiffAttention(dtype=L.BF16, B=2, Tq=40, Tk=40, n_head=2, hd=64, scale=0.1, q=one, ldq=256, bsq=10240, k=one, ldk=256, bsk=10240,
                            v=one, ldv=256, bsv=10240, lam=one, out=one, ldo=256, bso=10240, lse=one, out2=one)
        for k, v in kw.items():
            setattr(a, k, v)
        g = L.DiffAttentionBwd()
        return [(f(), lib.gpt_last_error().decode()) for f in (lambda: lib.gpt_diff_attention_keep(C.byref(a), rest, None),
                                                                lambda: lib.gpt_diff_attention_bwd_kept(C.byref(a), rest, C.byref(g), None))]
    for rest, kw, word in ((one, dict(dtype=L.F32), "rest"), (one, dict(out2=None), "rest"), (one + 4, {}, "misaligned")):
        assert all(rc < 0 and word in text for rc, text in call(rest, **kw))
