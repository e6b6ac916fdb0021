"""gpt_amd.ops - counter-based dropout, RMS norm with the residual's addition (also in 8 bits), differential attention - against their
formulas in 64 bits, with tolerances counted from the roundings on the way (u = 2^-24 for a float32 operation, half a step of the
type where a value is rounded to it), and their refusals."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import gpt_amd
from gpt_amd import _lib as L
from gpt_amd import ops

DEV = "cuda:0"
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
gpu = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def normal(seed, *shape, dtype=F32, std=1.0, device=DEV):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(device)


def within(got, want, tol, what=""):
    """Every element of `got` within `tol` (tensor or number) of `want`, and finite."""
    got, want = got.detach().double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    off = (got - want).abs() - tol
    if off.numel():
        assert float(off.max()) <= 0, f"{what}: {float(off.max()):.3e} over the tolerance, error {float((got - want).abs().max()):.3e}"


# ---------------------------------------------------------------------------------------------------------------- dropout
def philox_keep(n, p, seed, offset, first=0):
    """Keep mask of elements first .. first + n - 1 (8 | first) from the published Philox4x32-10 (unsigned 64-bit words on the host)."""
    u = np.uint64
    m, s32 = u(0xFFFFFFFF), u(32)
    blk = np.arange(first // 8, first // 8 + (n + 7) // 8, dtype=u)
    c = [blk & m, blk >> s32, np.full_like(blk, offset & 0xFFFFFFFF), np.full_like(blk, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> s32) ^ c[1] ^ u(k0), b & m, (a >> s32) ^ c[3] ^ u(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    halves = np.stack([w >> u(16 * i) & u(0xFFFF) for w in c for i in (0, 1)], 1).reshape(-1)[:n]
    return torch.from_numpy(halves >= round(65536 * p))


def test_philox_known_answer():
    """The generator behind the reference mask: the published known-answer vectors of Philox4x32-10 (counter and key all zeros, and
    the counter / key of the digits of pi)."""
    def words(ctr, key):
        c, (k0, k1) = list(ctr), key
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k0, b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k1, a & 0xFFFFFFFF]
            k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
        return c
    zero = words([0] * 4, (0, 0))
    assert zero == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert words([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], (0xA4093822, 0x299F31D0)) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    halves = [h for w in zero for h in (w & 0xFFFF, w >> 16)]
    for p in (0.1, 0.5, 0.9):
        assert philox_keep(8, p, 0, 0).tolist() == [h >= round(65536 * p) for h in halves]


def factor(p):
    thr = round(65536 * p)
    return float(np.float32(65536 / (65536 - thr))) if thr < 65536 else 0.0


DROP_SHAPES = [(1, 1), (1, 7), (3, 8), (5, 13), (26, 192), (7, 1000), (2, 3, 40), (513, 1536), (1, 70001)]


@gpu
@pytest.mark.parametrize("shape", DROP_SHAPES)
@pytest.mark.parametrize("ht,xt", [(BF, F32), (F32, F32), (BF, BF), (F32, BF)])
def test_dropout_add_and_gradients(shape, ht, xt):
    p, seed, offset = 0.3, 0xFEDCBA9876543210, (1 << 40) + 5
    h, r, g = normal(1, *shape, dtype=ht).requires_grad_(), normal(2, *shape, dtype=xt).requires_grad_(), normal(3, *shape, dtype=xt)
    keep = philox_keep(h.numel(), p, seed, offset).view(shape).to(DEV)
    x = ops.dropout_add(h, r, p, seed, offset)
    # h * s and the sum are float32 operations of their own: the same bits
    want = (r.detach().float() + torch.where(keep, h.detach().float() * factor(p), 0.0)).to(xt)
    assert x.dtype == xt and torch.equal(x.detach(), want)
    dh, dr = torch.autograd.grad(x, (h, r), g)
    assert torch.equal(dr, g) and dh.dtype == ht
    assert torch.equal(dh, torch.where(keep, g.float() * factor(p), 0.0).to(ht))
    y = ops.dropout(h, p, seed, offset)
    assert y.dtype == ht and torch.equal(y.detach(), torch.where(keep, h.detach().float() * factor(p), 0.0).to(ht))


@gpu
@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 2.0 ** -16, 0.5, 1 - 2.0 ** -16, 1.0])
def test_dropout_probabilities(p):
    h, r = normal(1, 64, 520), normal(2, 64, 520)
    keep = philox_keep(h.numel(), p, 7, 3).view_as(h).to(DEV)
    assert torch.equal(ops.dropout_add(h, r, p, 7, 3), r + torch.where(keep, h * factor(p), 0.0))
    if p == 1.0:
        assert torch.equal(ops.dropout(torch.full_like(h, math.inf), p, 7, 3), torch.zeros_like(h))


@gpu
@pytest.mark.parametrize("d", [40, 37])
def test_dropout_strides_and_alignment(d):
    """Strided, offset, transposed and broadcast operands give the contiguous operands' result; NaN and Inf are dropped like the rest."""
    base = normal(1, 30, 3 * d + 5, dtype=BF)
    base[::3, ::2] = math.nan
    base[1::3, 1::2] = math.inf
    r = normal(2, 30, d)
    for h in (base[:, d:2 * d], base[:, 5:5 + d], base[:, 0:2 * d:2], base[::2, :d], base.t()[:30, :30]):
        res = r[:h.shape[0], :h.shape[1]]
        want = ops.dropout_add(h.contiguous(), res.contiguous(), 0.4, 9, 1)
        assert torch.equal(ops.dropout_add(h, res, 0.4, 9, 1).nan_to_num(7.0), want.nan_to_num(7.0))
        keep = philox_keep(h.numel(), 0.4, 9, 1).view(h.shape).to(DEV)
        assert torch.equal(want[~keep], res[~keep])
    row = normal(4, d).requires_grad_()
    x = ops.dropout_add(normal(5, 6, d), row.expand(6, d), 0.2, 1)
    x.sum().backward()
    assert torch.equal(row.grad, torch.full_like(row, 6.0))


@gpu
def test_dropout_in_place_at_the_c_entry():
    """out may be resid or h."""
    h, r = normal(1, 33, 48), normal(2, 33, 48)
    want, alone = ops.dropout_add(h, r, 0.25, 5, 6), ops.dropout(h, 0.25, 5, 6)
    drop = L.Dropout(0.25, 5, 6, None)
    L.check(L.lib().gpt_dropout_add(L.F32, L.ptr(h), 48, L.F32, L.ptr(r), 48, L.ptr(r), 48, 33, 48, C.byref(drop), L.stream()), "x")
    L.check(L.lib().gpt_dropout_add(L.F32, L.ptr(h), 48, L.F32, None, 0, L.ptr(h), 48, 33, 48, C.byref(drop), L.stream()), "x")
    assert torch.equal(r, want) and torch.equal(h, alone)


@gpu
def test_dropout_counter_and_graph_replay():
    """A device counter adds to the offset; a captured step that advances it draws the masks that eager calls draw."""
    h, r = normal(1, 100, 192, dtype=BF), normal(2, 100, 192)
    counter = torch.zeros(1, dtype=torch.int64, device=DEV)
    want = [ops.dropout_add(h, r, 0.5, 11, 100 + i) for i in range(4)]
    assert not torch.equal(want[0], want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.dropout_add(h, r, 0.5, 11, 100, counter)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x = ops.dropout_add(h, r, 0.5, 11, 100, counter)
        counter.add_(1)
    counter.zero_()
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want[i]), i
        assert torch.equal(ops.dropout_add(h, r, 0.5, 11, 100 + i), want[i])
    h = h.requires_grad_()
    x = ops.dropout_add(h, r, 0.5, 11, 100, counter)
    counter.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        x.sum().backward()


@gpu
def test_dropout_beyond_32_bits_of_elements():
    rows, d, last = (1 << 20) + 3, 4104, 5 * 4104
    h = torch.ones(rows, d, dtype=BF, device=DEV)
    y = ops.dropout(h, 0.5, 77, 5)
    n = rows * d
    assert n > 1 << 32
    for first in (0, (1 << 32) - last // 2 // 8 * 8, n - last):
        want = philox_keep(last, 0.5, 77, 5, first).to(BF) * 2
        assert torch.equal(y.view(-1)[first:first + last].cpu(), want), first


@gpu
def test_dropout_masks_differ_and_keep_the_right_share():
    n, p = 1 << 20, 0.1
    ones = torch.ones(1, n, device=DEV)
    masks = [ops.dropout(ones, p, s, o) > 0 for s, o in ((0, 0), (1, 0), (0, 1))]
    for m in masks:      # binomial: 6 standard deviations
        assert abs(float(m.double().mean()) - (1 - round(65536 * p) / 65536)) < 6 * math.sqrt(p * (1 - p) / n)
    for a, b in ((0, 1), (0, 2), (1, 2)):      # independent masks agree with probability p^2 + (1 - p)^2
        agree = float((masks[a] == masks[b]).double().mean())
        want = p * p + (1 - p) ** 2
        assert abs(agree - want) < 6 * math.sqrt(want * (1 - want) / n) + 1e-4


# --------------------------------------------------------------------------------------------------------------- RMS norm
def norm_reference(h, r, w, eps, p, seed, offset, gy=None, gx=None):
    """x as it is stored, y and the gradients in 64 bits, and their tolerances before the output's own rounding."""
    xt = r.dtype
    if h is None:
        keep, s, x = None, 1.0, r
    else:
        keep, s = philox_keep(h.numel(), p, seed, offset).view(h.shape).to(h.device), factor(p)
        x = (r.float() + torch.where(keep, h.float() * s, 0.0)).to(xt)
    X, W = x.double(), w.double()
    d = X.shape[-1]
    rho = (X.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    out = dict(x=x, y=X * rho * W)
    # rho: a sum of d squares (relative d u at most), mean, root, reciprocal; then two products
    e = (d / 2 + 8) * U
    tol = dict(y=e * out["y"].abs())
    if gy is not None:
        G, GX = gy.double(), 0.0 if gx is None else gx.double()
        wg = W * G
        a, b = rho * wg, X * rho ** 3 * (wg * X).mean(-1, keepdim=True)
        dx = GX + a - b
        bb = X.abs() * rho ** 3 * (wg * X).abs().mean(-1, keepdim=True)
        t = 2 * e * a.abs() + (d + 8 + 3 * e / U) * U * bb + 2 * U * dx.abs()
        out["dr"], tol["dr"] = dx, t
        if h is not None:
            out["dh"], tol["dh"] = torch.where(keep, dx * s, 0.0), torch.where(keep, (t + U * dx.abs()) * s, 0.0)
        flat = lambda v: v.reshape(-1, d)                                                                   # noqa: E731
        out["dw"] = flat(G * X * rho).sum(0)
        tol["dw"] = (e + (flat(X).shape[0] + 4) * U) * flat((G * X * rho).abs()).sum(0)
    return out, tol


NORM_SHAPES = [(1, 8), (1, 1), (3, 37), (26, 192), (5, 2, 520), (2049, 512), (2100, 1000), (64, 1536), (2050, 1536), (2048, 2048), (7, 4096), (3, 8192), (2, 8200), (70, 1001)]


@gpu
@pytest.mark.parametrize("shape", NORM_SHAPES)
@pytest.mark.parametrize("ht,xt,p", [(BF, F32, 0.2), (F32, F32, 0.0), (BF, BF, 0.2), (F32, BF, 0.1)])
def test_add_rms_norm_and_gradients(shape, ht, xt, p):
    h, r = normal(1, *shape, dtype=ht).requires_grad_(), normal(2, *shape, dtype=xt, std=2.0).requires_grad_()
    w = (1 + normal(3, shape[-1], std=0.3)).requires_grad_()
    gy, gx = normal(4, *shape, dtype=ht), normal(5, *shape, dtype=xt)
    y, x = ops.add_rms_norm(h, r, w, 1e-5, p, 77, 8)
    dh, dr, dw = torch.autograd.grad((y, x), (h, r, w), (gy, gx))
    want, tol = norm_reference(h.detach(), r.detach(), w.detach(), 1e-5, p, 77, 8, gy, gx)
    assert torch.equal(x.detach(), want["x"]) and y.dtype == ht and x.dtype == xt
    assert dh.dtype == ht and dr.dtype == xt and dw.dtype == F32
    within(y, want["y"], tol["y"] + HALF[ht] * (want["y"].abs() + tol["y"]), "y")
    within(dr, want["dr"], tol["dr"] + HALF[xt] * (want["dr"].abs() + tol["dr"]), "dresid")
    within(dh, want["dh"], tol["dh"] + HALF[ht] * (want["dh"].abs() + tol["dh"]), "dh")
    within(dw, want["dw"], tol["dw"], "dweight")
    again = torch.autograd.grad(ops.add_rms_norm(h, r, w, 1e-5, p, 77, 8), (h, r, w), (gy, gx))
    assert all(torch.equal(a, b) for a, b in zip(again, (dh, dr, dw)))          # fixed order of the sums


@gpu
@pytest.mark.parametrize("xt,yt", [(F32, BF), (F32, F32), (BF, BF), (BF, F32)])
@pytest.mark.parametrize("shape", [(3, 96), (5, 7, 192), (3000, 256), (4, 50)])
def test_rms_norm_alone(shape, xt, yt):
    x, w, gy = normal(1, *shape, dtype=xt, std=3.0).requires_grad_(), (1 + normal(2, shape[-1], std=0.3)).requires_grad_(), normal(3, *shape, dtype=yt)
    y = ops.rms_norm(x, w, 1e-6, yt)
    dx, dw = torch.autograd.grad(y, (x, w), gy)
    want, tol = norm_reference(None, x.detach(), w.detach(), 1e-6, 0.0, 0, 0, gy)
    assert y.dtype == yt and dx.dtype == xt
    within(y, want["y"], tol["y"] + HALF[yt] * (want["y"].abs() + tol["y"]), "y")
    within(dx, want["dr"], tol["dr"] + HALF[xt] * (want["dr"].abs() + tol["dr"]), "dx")
    within(dw, want["dw"], tol["dw"], "dweight")


@gpu
def test_add_rms_norm_gradient_against_differences():
    """The gradient of sum(gy y + gx x) along a direction against central differences of the 64-bit formula: its truncation is the
    third derivative, O(t^2) = 1e-8 relative to values of order 1; the operator's own error is what the test above allows."""
    shape, t = (4, 64), 1e-4
    h, r, w = normal(1, *shape), normal(2, *shape), 1 + normal(3, 64, std=0.3)
    gy, gx = normal(4, *shape), normal(5, *shape)
    leaves = [v.clone().requires_grad_() for v in (h, r, w)]
    y, x = ops.add_rms_norm(*leaves, 1e-5, 0.25, 3, 4)
    grads = torch.autograd.grad((y, x), leaves, (gy, gx))
    keep = philox_keep(h.numel(), 0.25, 3, 4).view(shape).to(DEV)

    def f(h, r, w):
        x = r + keep * h * factor(0.25)
        return (gy.double() * (x * (x.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt() * w) + gx.double() * x).sum()

    base = [v.double() for v in (h, r, w)]
    for i in range(3):
        u = normal(10 + i, *base[i].shape).double()
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + t * u, base[i] - t * u
        want = float((f(*up) - f(*dn)) / (2 * t))
        got = float((grads[i].double() * u).sum())
        assert abs(got - want) < 1e-4 * max(1.0, float((grads[i].double() * u).abs().sum()) * 1e-2)


@gpu
def test_add_rms_norm_partial_gradients_strides_and_empty():
    shape = (26, 200)
    h, r, w = normal(1, *shape, dtype=BF), normal(2, *shape), 1 + normal(3, 200, std=0.3)
    gy, gx = normal(4, *shape, dtype=BF), normal(5, *shape)
    full = [v.clone().requires_grad_() for v in (h, r, w)]
    y, x = ops.add_rms_norm(*full, 1e-5, 0.1, 3, 4)
    want = torch.autograd.grad((y, x), full, (gy, gx), retain_graph=True)
    for i in range(3):                                  # one leaf at a time
        leaves = [v.clone().requires_grad_(j == i) for j, v in enumerate((h, r, w))]
        y1, x1 = ops.add_rms_norm(*leaves, 1e-5, 0.1, 3, 4)
        outs, gs = ((y1, x1), (gy, gx)) if i < 2 else ((y1,), (gy,))
        assert torch.equal(torch.autograd.grad(outs, leaves[i], gs)[0], want[i])
    # only one of the two outputs is used
    zero_y, zero_x = torch.zeros_like(gy), torch.zeros_like(gx)
    for outs, gs, ref in (((y,), (gy,), (gy, zero_x)), ((x,), (gx,), (zero_y, gx))):
        a = torch.autograd.grad(outs, full[:2], gs, retain_graph=True)
        b = torch.autograd.grad((y, x), full[:2], ref, retain_graph=True)
        assert all(torch.equal(s, t) for s, t in zip(a, b))
    # strided and shifted operands, and a weight that is a view
    pad = torch.zeros(26, 403, dtype=BF, device=DEV)
    pad[:, 3:203] = h
    wide = torch.zeros(400, device=DEV)
    wide[::2] = w
    y2, x2 = ops.add_rms_norm(pad[:, 3:203], r.t().contiguous().t(), wide[::2], 1e-5, 0.1, 3, 4)
    assert torch.equal(x2, x.detach())
    within(y2, y.detach().double(), 2 * HALF[BF] * y.detach().double().abs() + 1e-6, "strided")
    for empty in ((0, 64), (3, 0)):
        e = torch.empty(*empty, device=DEV)
        ye, xe = ops.add_rms_norm(e, e, torch.ones(empty[1], device=DEV))
        assert ye.shape == empty and xe.shape == empty


def mx_reference(y):
    """Scale exponents of the blocks of 32: the smallest e >= -127 with amax <= 448 * 2^e."""
    blocks = y.double().reshape(*y.shape[:-1], -1, 32)
    amax = blocks.abs().amax(-1)
    return blocks, amax, torch.ceil(torch.log2(amax.clamp(min=2.0 ** -200) / 448)).clamp(min=-127)


@gpu
@pytest.mark.parametrize("shape", [(1, 32), (5, 96), (52, 1536), (3, 4, 160), (2060, 1536), (2048, 512), (3, 8224)])
@pytest.mark.parametrize("ht,xt", [(BF, F32), (F32, BF)])
def test_add_rms_norm_mx8(shape, ht, xt):
    h, r, w = normal(1, *shape, dtype=ht), normal(2, *shape, dtype=xt, std=2.0), 1 + normal(3, shape[-1], std=0.3)
    w[:32] *= torch.exp2(torch.linspace(-30, 10, 32, device=DEV))           # values down to the format's subnormals and below
    q, s, x = ops.add_rms_norm_mx8(h, r, w, 1e-5, 0.1, 5, 6)
    want, tol = norm_reference(h, r, w, 1e-5, 0.1, 5, 6)
    assert torch.equal(x, want["x"]) and q.dtype == torch.float8_e4m3fn and s.dtype == torch.float8_e8m0fnu
    assert s.shape == (*shape[:-1], shape[-1] // 32)
    blocks, amax, e = mx_reference(want["y"])
    rel = (shape[-1] / 2 + 8) * U
    # an amax within its own error of 448 * 2^e may fall on either side of it
    edge = (torch.log2(amax / 448) - e).abs() <= 2 * rel
    edge |= (torch.log2(amax / 448) - e + 1).abs() <= 2 * rel
    got_e = torch.log2(s.double())
    assert torch.equal(got_e[~edge], e[~edge]) and bool(((got_e - e).abs()[edge] <= 1).all())
    scale = torch.exp2(got_e)[..., None]
    got = q.double().view_as(blocks) * scale
    # half a step: 2^-4 of the value for normal numbers, 2^-10 scales for subnormal ones
    bound = torch.maximum(blocks.abs() * 2.0 ** -4, scale * 2.0 ** -10) + 2 * rel * blocks.abs()
    within(got, blocks, bound, "values")


@gpu
def test_mx8_special_values():
    """Zeros, ties to even, rows with NaN, an infinite weight; no row disturbs another."""
    d = 64
    x = torch.ones(4, d, device=DEV)
    x[0] = 0
    x[2, 5] = math.nan
    w = torch.ones(d, device=DEV)
    w[40] = math.inf
    q, s = ops.rms_norm_mx8(x, w, 0.0 + 1e-30)
    q, sb = q.double(), s.view(torch.uint8)
    assert bool((q[0, :32] == 0).all()) and int(sb[0, 0]) == 0
    assert bool(q[2].isnan().all())
    for row in (1, 3):
        assert torch.equal(q[row, :32] * s.double()[row, 0], torch.ones(32, dtype=torch.float64, device=DEV))
        assert bool(q[row, 40].isnan())
    # ties: y = +-(k + 0.5 steps) at a known scale; with rho = 1 (mean square 1 by construction) y = w
    vals = torch.tensor([1.0, 17 / 16, 19 / 16, 21 / 16, 33 / 32, 448.0] + [1.0] * 26, device=DEV)
    q, s = ops.rms_norm_mx8(torch.ones(1, 32, device=DEV), vals, 0.0)
    assert float(s.double()) == 1.0
    assert q.double()[0, :6].tolist() == [1.0, 1.0, 1.25, 1.25, 1.0, 448.0]


# --------------------------------------------------------------------------------------------- differential attention
def attention_reference(q, k, v, lam, H, lens, scale, g=None, half=0.0):
    """Output and gradients in 64 bits, and tolerances.  half: half a step of the type P, dS and the kept outputs are rounded to."""
    B, Tq, w = q.shape
    Tk, hd = k.shape[1], w // (2 * H)
    if lens is not None:                               # what lies behind the length must not matter
        dead = torch.arange(Tk, device=k.device)[None, :, None] >= lens.clamp(0, Tk)[:, None, None]
        k, v = k.masked_fill(dead, 0.0), v.masked_fill(dead, 0.0)
    split = lambda t: t.double().view(B, -1, H, 2, hd).permute(0, 2, 3, 1, 4)                               # noqa: E731
    heads = lambda t: t.double().view(B, -1, H, 2 * hd).permute(0, 2, 1, 3)                                 # noqa: E731
    join = lambda t: t.permute(0, 2, 1, 3).reshape(B, -1, w)                                                # noqa: E731
    pair = lambda t: t.permute(0, 3, 1, 2, 4).reshape(B, -1, w)                                             # noqa: E731
    Q, K, V, lm = split(q), split(k), heads(v), lam.double().expand(H).view(1, H, 1, 1)
    S = scale * Q @ K.transpose(-1, -2)
    ok = torch.ones(B, 1, 1, 1, Tk, dtype=torch.bool, device=q.device) if lens is None else \
        (torch.arange(Tk, device=q.device) < lens.clamp(0, Tk)[:, None]).view(B, 1, 1, 1, Tk)
    S = S.masked_fill(~ok, -math.inf)
    P = torch.softmax(S.masked_fill(~ok.any(-1, keepdim=True), 0.0), -1).masked_fill(~ok, 0.0)
    A, AA = P[:, :, 0] - lm * P[:, :, 1], P[:, :, 0] + lm.abs() * P[:, :, 1]
    O = A @ V
    # scores: hd products and sums in float32, then scaled and shifted by the row's maximum; a relative error of P follows
    absS = scale * (Q.abs() @ K.abs().transpose(-1, -2)).masked_fill(~ok, 0.0)
    eS = U * (hd + 8) * absS.amax(-1, keepdim=True) + 4 * U
    eP = 2 * eS + (Tk + 16) * U
    eA = eP.amax(2)
    res, tol = dict(out=join(O)), {}
    errO = (half + eA + (Tk + 4) * U) * (AA @ V.abs())
    tol["out"] = join(errO)
    if g is not None:
        G = heads(g)
        dP = (G @ V.transpose(-1, -2)).unsqueeze(2)
        D = (P * dP).sum(-1, keepdim=True)
        sign = torch.stack([torch.ones(H), torch.ones(H)]).to(q.device).double()
        sign[1] = -lam.double().expand(H)
        sign = sign.t().reshape(1, H, 2, 1, 1)
        dS = sign * P * (dP - D)
        res["dq"], res["dk"] = pair(scale * dS @ K), pair(scale * dS.transpose(-1, -2) @ Q)
        res["dv"], res["dlam"] = join(A.transpose(-1, -2) @ G), -D[:, :, 1].sum((0, 2, 3))
        absdP = (G.abs() @ V.abs().transpose(-1, -2)).unsqueeze(2)
        # D_i from the kept outputs: their error times dO (out and out2 each rounded, P_i rounded on the way)
        eD = ((G.abs() * (errO + half * O.abs() + lm.abs() * (half * 2 + eA + (Tk + 4) * U) * (P[:, :, 1] @ V.abs()))).sum(-1, keepdim=True)
              + (2 * hd + 8) * U * (G.abs() * (AA @ V.abs())).sum(-1, keepdim=True) * 4).unsqueeze(2)
        sa = sign.abs()
        edS = sa * P * (eP * (dP - D).abs() + (2 * hd + 8) * U * absdP + eD) + (half + 4 * U) * dS.abs()
        n = (Tk + Tq + 8) * U
        tol["dq"] = pair(scale * (edS + n * dS.abs()) @ K.abs())
        tol["dk"] = pair(scale * (edS + n * dS.abs()).transpose(-1, -2) @ Q.abs())
        tol["dv"] = join(((half + n + eA) * AA).transpose(-1, -2) @ G.abs())
        # dlam: P_2 and dP unrounded; a sum of B Tq Tk terms, its partial sums at most the sum of the absolute terms
        terms = P[:, :, 1] * absdP[:, :, 0]
        depth = 64 * math.sqrt(B * Tq * Tk) + 64            # lanes, waves and blocks: far fewer than the terms in one chain
        tol["dlam"] = ((eA + (2 * hd + 8) * U + depth * U) * terms).sum((0, 2, 3))
    return res, tol


def attention_case(B, Tq, Tk, H, hd, t, lens, fused, seed=0, std=1.0):
    w = 2 * H * hd
    if fused:
        qkv = normal(seed + 1, B, Tq, 3 * w, dtype=t, std=std)
        q, k, v = qkv.chunk(3, -1)
    else:
        qkv = None
        q, k, v = normal(seed + 1, B, Tq, w, dtype=t, std=std), normal(seed + 2, B, Tk, w, dtype=t, std=std), normal(seed + 3, B, Tk, w, dtype=t)
    lam = 0.5 + normal(seed + 4, H, std=0.3)
    if H > 1:
        lam[1] = -0.4
    n = None if lens is None else torch.tensor((lens * B)[:B], dtype=torch.int32, device=DEV)
    return qkv, q, k, v, lam, n, normal(seed + 5, B, Tq, w, dtype=t)


def check_attention(B, Tq, Tk, H, hd, t, lens=None, fused=False, scale=None, std=1.0):
    qkv, q, k, v, lam, n, g = attention_case(B, Tq, Tk, H, hd, t, lens, fused, std=std)
    half = 0.0 if t == F32 else HALF[t]
    c = hd ** -0.5 if scale is None else scale
    want, tol = attention_reference(q, k, v, lam, H, n, c, g, half)
    if fused:
        leaves = [qkv.clone().requires_grad_(), lam.clone().requires_grad_()]
        out = ops.diff_attention_qkv(*leaves, H, n, scale)
        dqkv, dlam = torch.autograd.grad(out, leaves, g)
        grads = (*dqkv.chunk(3, -1), dlam)
        with torch.no_grad():
            plain = ops.diff_attention_qkv(qkv, lam, H, n, scale)
    else:
        leaves = [x.clone().requires_grad_() for x in (q, k, v, lam)]
        out = ops.diff_attention(*leaves, H, n, scale)
        grads = torch.autograd.grad(out, leaves, g)
        with torch.no_grad():
            plain = ops.diff_attention(q, k, v, lam, H, n, scale)
    got = dict(zip(("out", "dq", "dk", "dv", "dlam"), (out, *grads)))
    within(plain, want["out"], tol["out"] + HALF[t] * (want["out"].abs() + tol["out"]), "out (no grad)")
    for name, x in got.items():
        ht = HALF[F32 if name == "dlam" else t]
        within(x, want[name], tol[name] + ht * (want[name].abs() + tol[name]), name)
    if n is not None:
        dead = torch.arange(Tk, device=DEV)[None] >= n.clamp(0, Tk)[:, None]
        assert bool((got["dk"][dead] == 0).all()) and bool((got["dv"][dead] == 0).all())
        empty = n <= 0
        assert bool((got["out"][empty] == 0).all()) and bool((got["dq"][empty] == 0).all())


SHORT = [(1, 1, 1), (3, 2, 2), (2, 5, 31), (4, 26, 26), (2, 32, 32), (3, 17, 1)]
LONG = [(2, 33, 33), (1, 1, 300), (2, 64, 64), (1, 70, 129), (1, 257, 257), (2, 515, 65), (1, 31, 1000), (1, 130, 385)]


@gpu
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("t", [BF, F32])
@pytest.mark.parametrize("B,Tq,Tk", SHORT + LONG)
def test_diff_attention_and_gradients(B, Tq, Tk, hd, t):
    check_attention(B, Tq, Tk, 3 if hd < 128 else 2, hd, t)


@gpu
@pytest.mark.parametrize("t", [BF, F32])
@pytest.mark.parametrize("B,T,H,hd", [(3, 26, 8, 96), (2, 200, 2, 64), (1, 129, 5, 128), (2, 7, 1, 32)])
def test_diff_attention_fused_projection(B, T, H, hd, t):
    check_attention(B, T, T, H, hd, t, fused=True)


@gpu
@pytest.mark.parametrize("t", [BF, F32])
@pytest.mark.parametrize("Tq,Tk", [(26, 26), (5, 32), (40, 40), (100, 300), (1, 700)])
def test_diff_attention_lengths(Tq, Tk, t):
    """Samples without a key, with one, at tile borders, full, and lengths outside the range."""
    check_attention(9, Tq, Tk, 2, 64, t, lens=[0, 1, Tk, Tk - 1, Tk // 2, -3, Tk + 5, min(Tk, 32), min(Tk, 64)])


@gpu
@pytest.mark.parametrize("t", [BF, F32])
@pytest.mark.parametrize("T", [20, 150])
def test_diff_attention_scale_and_peaked_maps(T, t):
    check_attention(2, T, T, 2, 32, t, scale=1.7)
    check_attention(2, T, T, 2, 64, t, std=3.0)


@gpu
@pytest.mark.parametrize("T", [26, 150])
@pytest.mark.parametrize("t", [BF, F32])
def test_diff_attention_garbage_behind_the_lengths(T, t):
    """NaN and Inf in masked keys and values reach neither the output nor a gradient."""
    qkv, q, k, v, lam, n, g = attention_case(4, T, T, 2, 64, t, [T - 3, 1, 0, T // 2], False)
    dead = torch.arange(T, device=DEV)[None, :, None] >= n[:, None, None]
    runs = []
    for fill in (0.0, math.nan, math.inf, torch.finfo(t).min):
        leaves = [x.clone().requires_grad_() for x in (q, k.masked_fill(dead, fill), v.masked_fill(dead, fill), lam)]
        out = ops.diff_attention(*leaves, 2, n)
        runs.append((out.detach(), *torch.autograd.grad(out, leaves, g)))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@gpu
@pytest.mark.parametrize("t", [BF, F32])
@pytest.mark.parametrize("Tq,Tk,gone", [(20, 26, 9), (40, 200, 130), (1, 700, 300), (5, 9000, 8200)])
def test_diff_attention_scores_of_minus_infinity(Tq, Tk, gone, t):
    """Keys whose scores are -inf weigh nothing, also where they fill the first tiles or a whole span of the keys."""
    _, q, k, v, lam, _, _ = attention_case(2, Tq, Tk, 2, 64, t, None, False)
    q, k = q.view(2, Tq, 4, 64), k.view(2, Tk, 4, 64)
    q[..., 7], k[:, :gone, :, 7] = 1.0, -math.inf
    q, k = q.view(2, Tq, -1), k.view(2, Tk, -1)
    want, tol = attention_reference(q, k[:, gone:], v[:, gone:], lam, 2, None, 64 ** -0.5, None, 0.0 if t == F32 else HALF[t])
    got = ops.diff_attention(q, k, v, lam, 2)
    extra = (gone + 4) * U * want["out"].abs()           # the longer sums' adds of zeros round nothing, but their count is counted
    within(got, want["out"], tol["out"] + extra + HALF[t] * (want["out"].abs() + tol["out"]))


@gpu
@pytest.mark.parametrize("t", [BF, F32])
@pytest.mark.parametrize("Tq,Tk,hd", [(600, 600, 64), (40, 2000, 128), (2000, 40, 96), (333, 1025, 32)])
def test_diff_attention_long_sweeps_of_few_heads(Tq, Tk, hd, t):
    """Few (sample, head) pairs: the sweeps over keys and over queries are cut into spans whose sums are joined; lengths end within a
    span, before one, at a tile's edge and at nothing."""
    check_attention(4, Tq, Tk, 1, hd, t, lens=[Tk, 0, Tk // 2 + 1, 32])


@gpu
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("t", [BF, F32])
@pytest.mark.parametrize("B,Tq,Tk,lens", [(24, 70, 70, None), (24, 161, 140, [140, 0, 17, 64, 133]), (96, 40, 33, [33, 1, 32])])
def test_diff_attention_many_heads(B, Tq, Tk, lens, hd, t):
    """Enough (sample, head) pairs to fill the card: the larger workgroups of every kernel."""
    check_attention(B, Tq, Tk, 8, hd, t, lens=lens)


@gpu
@pytest.mark.parametrize("t", [BF, F32])
@pytest.mark.parametrize("Tq,Tk", [(1, 300), (40, 1), (1, 1)])
def test_diff_attention_single_rows_may_have_any_stride_at_the_c_entry(Tq, Tk, t):
    B, H, hd = 2, 2, 64
    w, code = 2 * H * hd, L.BF16 if t == BF else L.F32
    _, q, k, v, lam, _, g = attention_case(B, Tq, Tk, H, hd, t, None, False)
    runs = []
    for one in (w, 0, 32):                              # the stride of what has one row
        ld = lambda T: one if T == 1 else w                                                                # noqa: E731,B023
        out, out2, lse = torch.empty_like(q), torch.empty_like(q), torch.empty(2, B, H, Tq, device=DEV)
        dq, dk, dv, dlam = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty(H, device=DEV)
        n = C.c_int64()
        L.check(L.lib().gpt_diff_attention_workspace(code, B, Tq, Tk, H, hd, C.byref(n)), "workspace")
        ws = torch.empty(max(16, n.value), dtype=torch.uint8, device=DEV)
        f = L.DiffAttention(code, B, Tq, Tk, H, hd, hd ** -0.5, L.ptr(q), ld(Tq), Tq * w, L.ptr(k), ld(Tk), Tk * w, L.ptr(v), ld(Tk), Tk * w,
                            L.ptr(lam), None, L.ptr(out), ld(Tq), Tq * w, L.ptr(lse), L.ptr(out2), L.ptr(ws), ws.numel())
        L.check(L.lib().gpt_diff_attention(C.byref(f), L.stream()), "forward")
        L.check(L.lib().gpt_diff_attention_bwd_workspace(code, B, Tq, Tk, H, hd, C.byref(n)), "workspace")
        ws2 = torch.empty(max(16, n.value), dtype=torch.uint8, device=DEV)
        b = L.DiffAttentionBwd(L.ptr(g), ld(Tq), Tq * w, L.ptr(dq), ld(Tq), Tq * w, L.ptr(dk), ld(Tk), Tk * w, L.ptr(dv), ld(Tk), Tk * w,
                               L.ptr(dlam), L.ptr(ws2), ws2.numel())
        L.check(L.lib().gpt_diff_attention_bwd(C.byref(f), C.byref(b), L.stream()), "backward")
        runs.append([x.clone() for x in (out, dq, dk, dv, dlam)])
    for other in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(runs[0], other))


@gpu
def test_diff_attention_output_changed_in_place():
    """Up to 32 tokens the backward needs nothing of the forward's output, so it may be added to in place; longer ones notice."""
    for T, kept in ((26, False), (60, True)):
        _, q, k, v, lam, _, g = attention_case(2, T, T, 2, 64, BF, None, False)
        leaves = [x.clone().requires_grad_() for x in (q, k, v, lam)]
        want = torch.autograd.grad(ops.diff_attention(*leaves, 2), leaves, g)
        out = ops.diff_attention(*leaves, 2)
        out += 1
        if kept:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(out, leaves, g)
        else:
            assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(out, leaves, g)))


@gpu
@pytest.mark.parametrize("Tq", [1, 40])
def test_diff_attention_rows_beyond_32_bits(Tq):
    """A long cache whose rows lie 512 KiB apart: offsets pass 2^32 bytes, forward and backward, as in a compact cache."""
    Tk, w = 9000, 64
    cache = torch.empty(Tk, 1 << 18, dtype=BF, device=DEV)
    cache[:, :2 * w] = normal(1, Tk, 2 * w, dtype=BF)
    q, lam, g = normal(2, 1, Tq, w, dtype=BF), torch.tensor([0.4], device=DEV), normal(3, 1, Tq, w, dtype=BF)
    runs = []
    for compact in (False, True):
        k, v = (cache[None, :, i * w:(i + 1) * w] for i in (0, 1))
        leaves = [x.detach().requires_grad_() for x in ((q, k.contiguous(), v.contiguous(), lam) if compact else (q, k, v, lam))]
        assert leaves[1].stride(1) == (w if compact else 1 << 18)
        out = ops.diff_attention(*leaves, 1)
        runs.append((out.detach(), *torch.autograd.grad(out, leaves, g)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@gpu
@pytest.mark.parametrize("T", [20, 90])
def test_diff_attention_nan_stays_in_its_sample(T):
    _, q, k, v, lam, n, g = attention_case(3, T, T, 2, 64, BF, None, False)
    q, k = q.clone(), k.clone()
    q[0, 3, 5] = math.nan          # one query row of head 0
    k[1, 2, 70] = math.nan         # every row of sample 1, head 0
    out = ops.diff_attention(q, k, v, lam, 2)
    bad = out.isnan()
    assert bool(bad[0, 3, :128].all()) and not bool(bad[0, :3].any()) and not bool(bad[0, 3, 128:].any())
    assert bool(bad[1, :, :128].all()) and not bool(bad[1, :, 128:].any()) and not bool(bad[2].any())


@gpu
@pytest.mark.parametrize("T,t", [(26, BF), (26, F32), (150, BF), (150, F32)])
def test_diff_attention_is_reproducible_and_takes_any_strides(T, t):
    _, q, k, v, lam, n, g = attention_case(3, T, T, 2, 64, t, [T, T - 1, 3], False)

    def run(q, k, v, g):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, lam)]
        out = ops.diff_attention(*leaves, 2, n)
        return (out.detach(), *torch.autograd.grad(out, leaves, g))

    first = run(q, k, v, g)
    w = q.shape[-1]
    wide = torch.zeros(3, T, 2 * w + 8, dtype=t, device=DEV)
    wide[..., 8:8 + w] = k
    odd = torch.zeros(3, T, w + 3, dtype=t, device=DEV)
    odd[..., 3:] = v
    swap = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)                                          # noqa: E731
    for other in (run(q, k, v, g), run(swap(q), wide[..., 8:8 + w], odd[..., 3:], swap(g)),
                  run(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, g)):
        assert all(torch.equal(a, b) for a, b in zip(first, other))
    shared = run(q, k[:1].expand(3, T, w), v[:1].expand(3, T, w), g)          # one sample's keys for all
    copied = run(q, k[:1].repeat(3, 1, 1), v[:1].repeat(3, 1, 1), g)
    assert all(torch.equal(a, b) for a, b in zip(shared, copied))


@gpu
@pytest.mark.parametrize("T", [12, 48])
def test_diff_attention_gradient_against_differences(T):
    """Along a direction of each leaf: central differences of the 64-bit formula, O(t^2) truncation."""
    H, hd, B, step = 2, 32, 2, 1e-4
    _, q, k, v, lam, n, g = attention_case(B, T, T, H, hd, F32, [T, T - 2], False)
    leaves = [x.clone().requires_grad_() for x in (q, k, v, lam)]
    grads = torch.autograd.grad(ops.diff_attention(*leaves, H, n), leaves, g)

    def f(*x):
        return float((attention_reference(*x[:3], x[3], H, n, hd ** -0.5)[0]["out"] * g.double()).sum())

    base = [x.double() for x in (q, k, v, lam)]
    for i in range(4):
        u = normal(20 + i, *base[i].shape).double()
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + step * u, base[i] - step * u
        want = (f(*up) - f(*dn)) / (2 * step)
        got = float((grads[i].double() * u).sum())
        assert abs(got - want) < 1e-4 * max(1.0, 1e-2 * float((grads[i].double() * u).abs().sum())), i


@gpu
def test_diff_attention_one_lambda_no_grad_inputs_and_empty():
    _, q, k, v, lam, _, g = attention_case(2, 20, 20, 3, 32, BF, None, False)
    one = torch.tensor([0.7], device=DEV, requires_grad=True)
    many = torch.full((3,), 0.7, device=DEV, requires_grad=True)
    a, b = ops.diff_attention(q, k, v, one, 3), ops.diff_attention(q, k, v, many, 3)
    assert torch.equal(a, b)
    d1, d3 = torch.autograd.grad(a, one, g)[0], torch.autograd.grad(b, many, g)[0]
    assert abs(float(d1) - float(d3.double().sum())) <= 4 * U * float(d3.abs().sum())
    n64 = torch.tensor([20, 1 << 40], device=DEV)
    assert torch.equal(ops.diff_attention(q, k, v, many, 3, n64), b)
    e = ops.diff_attention(q[:0], k[:0], v[:0], many, 3)
    assert e.shape == (0, 20, 192)
    assert ops.diff_attention(q[:, :0], k, v, many, 3).shape == (2, 0, 192)
    leaf = q.clone().requires_grad_()
    z = ops.diff_attention(leaf, k[:, :0], v[:, :0], many, 3)
    assert bool((z == 0).all()) and bool((torch.autograd.grad(z, leaf, g)[0] == 0).all())


@gpu
@pytest.mark.parametrize("T", [26, 100])
def test_diff_attention_on_another_stream_and_in_two_graphs(T):
    """A side stream, and two captured graphs replayed in turn with eager work between: every result the eager one's."""
    _, q, k, v, lam, n, _ = attention_case(2, T, T, 2, 64, BF, [T, T - 5], False)
    q2 = normal(50, *q.shape, dtype=BF)
    few, few2 = q[:, :1].contiguous(), q2[:, :1].contiguous()                     # one query: split over the keys through scratch
    kk, vv = normal(51, 2, 2000, q.shape[2], dtype=BF), normal(52, 2, 2000, q.shape[2], dtype=BF)
    call = lambda a, b: (ops.diff_attention(a, k, v, lam, 2, n), ops.diff_attention(b, kk, vv, lam, 2))      # noqa: E731
    want, want2 = call(q, few), call(q2, few2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(q, few)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for args in ((q, few), (q2, few2)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = call(*args)
        graphs.append((gr, res))
    for _ in range(3):
        for (gr, res), ref in zip(graphs, (want, want2)):
            gr.replay()
            call(q2, few)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(res, ref))


# ------------------------------------------------------------------------------------------------ together, as a Block uses them
def block(x, h, p, H, lens, drop, site):
    """norm -> projection -> differential attention -> norm of every head -> projection -> dropout and residual -> norm"""
    y, x = ops.add_rms_norm(h, x, p["n1"], p=drop, seed=9, offset=site)
    qkv = (y.float() @ p["wqkv"]).to(y.dtype)
    o = ops.diff_attention_qkv(qkv, p["lam"], H, lens)
    o = ops.rms_norm(o.view(*o.shape[:2], H, -1), p["nh"]).reshape(o.shape)
    a = (o.float() @ p["wo"]).to(y.dtype)
    return ops.add_rms_norm(a, x, p["n2"], p=drop, seed=9, offset=site + 1)


def block_reference(x, h, p, H, lens, drop, site):
    def norm(v, w):
        return v * (v.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt() * w

    def dropped(v, off):
        return torch.where(philox_keep(v.numel(), drop, 9, off).view(v.shape).to(v.device), v * factor(drop), 0.0)

    x = x + dropped(h, site)
    q, k, v = (norm(x, p["n1"]) @ p["wqkv"]).chunk(3, -1)
    B, T, w = q.shape
    hd = w // (2 * H)
    sh = lambda t: t.view(B, T, H, 2, hd).permute(0, 2, 3, 1, 4)                                             # noqa: E731
    S = sh(q) @ sh(k).transpose(-1, -2) * hd ** -0.5
    ok = (torch.arange(T, device=x.device) < lens[:, None]).view(B, 1, 1, 1, T)
    P = torch.softmax(S.masked_fill(~ok, -math.inf), -1)
    o = (P[:, :, 0] - p["lam"].view(1, H, 1, 1) * P[:, :, 1]) @ v.view(B, T, H, 2 * hd).transpose(1, 2)
    o = norm(o.transpose(1, 2), p["nh"]).reshape(B, T, w)
    x = x + dropped(o @ p["wo"], site + 1)
    return norm(x, p["n2"]), x


@gpu
@pytest.mark.parametrize("t", [F32, BF])
@pytest.mark.parametrize("T", [26, 80])
def test_block_of_the_operators(t, T):
    """Outputs and the gradients of every parameter.  float32: each step is off by a few (d + T) u of its largest value and the norms
    divide by values of order 1: 1e-4 of a tensor's largest value leaves a factor of ten.  bf16: eight roundings of 2^-8 lie between
    the input and the outputs and as many on the way back, none amplified by more than the two norms' factor of order 1: in the
    2-norm, sixteen of them side by side are 16 * 2^-8 / sqrt(3) = 3.6e-2 at the very most."""
    B, H, hd, drop = 3, 2, 64, 0.1
    w = 2 * H * hd
    p = dict(n1=1 + normal(1, w, std=0.1), n2=1 + normal(2, w, std=0.1), nh=1 + normal(3, 2 * hd, std=0.1),
             wqkv=normal(4, w, 3 * w, std=w ** -0.5), wo=normal(5, w, w, std=w ** -0.5), lam=torch.tensor([0.6, 0.3], device=DEV))
    x, h = normal(6, B, T, w), normal(7, B, T, w, dtype=t)
    lens = torch.tensor([T, T - 7, 1], dtype=torch.int32, device=DEV)
    gy, gx = normal(8, B, T, w, dtype=t), normal(9, B, T, w)
    mine = {k: v.clone().requires_grad_() for k, v in dict(p, x=x, h=h).items()}
    y, xo = block(mine["x"], mine["h"], mine, H, lens, drop, 40)
    grads = torch.autograd.grad((y, xo), list(mine.values()), (gy, gx))
    ref = {k: v.detach().double().requires_grad_() for k, v in dict(p, x=x, h=h).items()}
    ry, rx = block_reference(ref["x"], ref["h"], ref, H, lens, drop, 40)
    want = torch.autograd.grad((ry, rx), list(ref.values()), (gy.double(), gx.double()))
    for name, a, b in zip(("y", "x", *mine), (y, xo, *grads), (ry.detach(), rx.detach(), *want)):
        a = a.detach().double()
        if t == F32:
            assert float((a - b).abs().max()) < 1e-4 * float(b.abs().max()), name
        else:
            assert float((a - b).norm()) < 3.6e-2 * float(b.norm()), name


# ---------------------------------------------------------------------------------------------------------------- refusals
def test_refuses_cpu_tensors():
    x, w, lam = torch.zeros(2, 64), torch.ones(64), torch.zeros(1)
    for call in (lambda: ops.dropout(x, 0.1, 0), lambda: ops.dropout_add(x, x, 0.1, 0), lambda: ops.rms_norm(x, w),
                 lambda: ops.add_rms_norm(x, x, w), lambda: ops.add_rms_norm_mx8(x, x, w), lambda: ops.rms_norm_mx8(x, w),
                 lambda: ops.diff_attention(x[None], x[None], x[None], lam, 1), lambda: ops.diff_attention_qkv(torch.zeros(1, 2, 192), lam, 1)):
        with pytest.raises(gpt_amd._lib.GptHipError, match="no CPU fallback"):
            call()


def test_c_entries_refuse_before_any_launch():
    """Every check of the C entries fails with a status and a message; nothing is launched (no GPU is needed)."""
    lib, one = L.lib(), 1 << 20                       # an aligned address that is never used

    def err(rc, text):
        assert rc < 0 and text in lib.gpt_last_error().decode(), (rc, lib.gpt_last_error())

    def drop(h=one, out=one, hd=L.F32, xd=L.F32, rows=4, d=8, ldh=8, ldo=8, p=0.5, counter=None, none=False):
        s = L.Dropout(p, 1, 2, counter)
        return lib.gpt_dropout_add(hd, h, ldh, xd, None, 0, out, ldo, rows, d, None if none else C.byref(s), None)

    err(drop(h=None), "null"), err(drop(out=None), "null"), err(drop(none=True), "null"), err(drop(hd=7), "dtype")
    err(drop(rows=0), "rows"), err(drop(d=-1), "rows"), err(drop(rows=1 << 40, d=1 << 40), "too large"), err(drop(ldo=7), "stride")
    err(drop(p=-0.1), "probability"), err(drop(p=1.5), "probability"), err(drop(p=math.nan), "probability")
    err(drop(h=one + 2), "misaligned"), err(drop(counter=one + 4), "misaligned")

    def norm(**kw):
        a = L.AddRmsNorm(h_dtype=L.BF16, x_dtype=L.F32, y_dtype=L.BF16, h=one, ldh=64, resid=one, ldr=64, x_out=one, ldx=64, weight=one,
                         y=one, ldy=64, rows=3, d=64, eps=1e-5)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.gpt_add_rmsnorm(C.byref(a), None)

    err(lib.gpt_add_rmsnorm(None, None), "null"), err(norm(resid=None), "null"), err(norm(x_out=None), "null"), err(norm(weight=None), "null")
    err(norm(x_dtype=3), "dtype"), err(norm(y_dtype=L.F32), "type of h"), err(norm(rows=0), "size"), err(norm(eps=-1.0), "eps")
    err(norm(y_dtype=L.MXFP8, scales=None), "scales"), err(norm(y_dtype=L.MXFP8, scales=one, d=40), "32"), err(norm(ldy=63), "stride")
    err(norm(resid=one + 2), "misaligned"), err(norm(drop=C.pointer(L.Dropout(2.0, 0, 0, None))), "probability")

    def norm_bwd(**kw):
        a = L.AddRmsNormBwd(h_dtype=L.BF16, x_dtype=L.F32, y_dtype=L.BF16, gy=one, ldgy=64, x=one, ldx=64, weight=one, rho=one, dresid=one,
                            lddr=64, rows=3, d=64)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.gpt_add_rmsnorm_bwd(C.byref(a), None)

    err(norm_bwd(rho=None), "null"), err(norm_bwd(dweight=one), "scratch"), err(norm_bwd(dweight=one, ws=one, ws_bytes=64), "scratch")
    err(norm_bwd(dh=one, lddh=64, h_dtype=L.F32), "type of gy"), err(norm_bwd(lddr=3), "stride"), err(norm_bwd(d=0), "size")

    def att(f=None, **kw):
        a = L.DiffAttention(dtype=L.BF16, B=2, Tq=40, Tk=40, n_head=2, hd=64, scale=0.1, q=one, ldq=256, bsq=10240, k=one, ldk=256, bsk=10240,
                            v=one, ldv=256, bsv=10240, lam=one, out=one, ldo=256, bso=10240)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.gpt_diff_attention(C.byref(a), None) if f is None else f(a)

    err(lib.gpt_diff_attention(None, None), "null"), err(att(dtype=5), "dtype"), err(att(Tk=0), "need B"), err(att(hd=48), "head dim")
    err(att(q=None), "null"), err(att(lam=None), "null"), err(att(scale=0.0), "scale"), err(att(scale=math.nan), "scale")
    err(att(ldk=255), "rows"), err(att(ldv=128), "rows"), err(att(k=one + 8), "rows"), err(att(bso=8), "strides"), err(att(ldo=250), "strides")
    err(att(n_head=5000), "range"), err(att(B=1, Tq=1, Tk=100000), "scratch"), err(att(B=1, Tq=1, Tk=100000, ws=one, ws_bytes=16), "scratch")

    def bwd(a, **kw):
        g = L.DiffAttentionBwd(dout=one, lddo=256, bsdo=10240, dq=one, lddq=256, bsdq=10240, dk=one, lddk=256, bsdk=10240, dv=one, lddv=256,
                               bsdv=10240, dlam=one, ws=one, ws_bytes=1 << 30)
        for k, v in kw.items():
            setattr(g, k, v)
        return lib.gpt_diff_attention_bwd(C.byref(a), C.byref(g), None)

    kept = dict(lse=one, out2=one)
    err(att(lambda a: bwd(a, dout=None), **kept), "null"), err(att(lambda a: bwd(a)), "lse"), err(att(lambda a: bwd(a, ws_bytes=8), **kept), "scratch")
    err(att(lambda a: bwd(a, lddq=100), **kept), "gradient rows"), err(att(lambda a: bwd(a, bsdk=0), **kept), "gradient rows")
    n = C.c_int64()
    assert lib.gpt_diff_attention_workspace(L.BF16, 0, 1, 1, 1, 32, C.byref(n)) < 0
    assert lib.gpt_diff_attention_bwd_workspace(9, 1, 1, 1, 1, 32, C.byref(n)) < 0
    assert lib.gpt_add_rmsnorm_bwd_workspace(0, 4, C.byref(n)) < 0


@gpu
def test_refusals_of_the_python_entries():
    h, w, lam = normal(1, 4, 64), torch.ones(64, device=DEV), torch.zeros(1, device=DEV)
    bad = [
        (lambda: ops.dropout(h.half(), 0.1, 0), "float32 or bfloat16"), (lambda: ops.dropout(h, 1.1, 0), "probability"),
        (lambda: ops.dropout(h, 0.1, 0, 0, torch.zeros(1, device=DEV)), "counter"), (lambda: ops.dropout_add(h, h[:2], 0.1, 0), "same shape"),
        (lambda: ops.dropout(h[0, 0], 0.1, 0), "one dimension"), (lambda: ops.dropout_add(h, h.cpu(), 0.1, 0), "CPU fallback"),
        (lambda: ops.rms_norm(h, w.bfloat16()), "weight"), (lambda: ops.rms_norm(h, w[:32]), "weight"), (lambda: ops.rms_norm(h, w, -1.0), "eps"),
        (lambda: ops.rms_norm(h, w, 1e-5, torch.float16), "out_dtype"), (lambda: ops.rms_norm_mx8(normal(1, 2, 40), torch.ones(40, device=DEV)), "multiple of 32"),
        (lambda: ops.rms_norm_mx8(h.clone().requires_grad_(), w), "no gradient"), (lambda: ops.add_rms_norm(h, h[:1], w), "same shape"),
        (lambda: ops.diff_attention(h[None], h[None], h[None].bfloat16(), lam, 1), "one type"),
        (lambda: ops.diff_attention(h[None], h[None], h[None], lam, 2), "head dim"), (lambda: ops.diff_attention(h, h, h, lam, 1), "need q"),
        (lambda: ops.diff_attention(h[None], h[None], h[None], lam.double(), 1), "lam"),
        (lambda: ops.diff_attention(h[None], h[None], h[None], lam, 1, torch.zeros(2, dtype=torch.int32, device=DEV)), "lengths"),
        (lambda: ops.diff_attention(h[None], h[None], h[None], lam, 1, torch.zeros(1, device=DEV)), "lengths"),
        (lambda: ops.diff_attention(h[None], h[None], h[None], lam, 1, None, -1.0), "scale"),
        (lambda: ops.diff_attention_qkv(h[None], lam, 1), "3 w"),
    ]
    for call, text in bad:
        with pytest.raises(gpt_amd._lib.GptHipError, match=text):
            call()
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate"):
        x = h.clone().requires_grad_()
        g, = torch.autograd.grad(ops.rms_norm(x, w).pow(2).sum(), x, create_graph=True)
        g.sum().backward()


def floating_calls(x):
    """Every entry, with `x` [4, 192] in the place of each floating argument in turn."""
    w, lam, q = torch.ones(192, device=x.device), torch.zeros(1, device=x.device), torch.zeros(4, 192, device=x.device)
    a, b = x[None].narrow(2, 0, 64), q[None].narrow(2, 0, 64)
    return [lambda: ops.dropout(x, 0.1, 0), lambda: ops.dropout_add(x, q, 0.1, 0), lambda: ops.dropout_add(q, x, 0.1, 0), lambda: ops.rms_norm(x, w),
            lambda: ops.rms_norm(q, x[0]), lambda: ops.add_rms_norm(x, q, w), lambda: ops.add_rms_norm(q, x, w), lambda: ops.add_rms_norm(q, q, x[0]),
            lambda: ops.add_rms_norm_mx8(x, q, w), lambda: ops.add_rms_norm_mx8(q, x, w), lambda: ops.rms_norm_mx8(x, w),
            lambda: ops.diff_attention(a, b, b, lam, 1), lambda: ops.diff_attention(b, a, b, lam, 1), lambda: ops.diff_attention(b, b, a, lam, 1),
            lambda: ops.diff_attention(b, b, b, x[0, :1], 1), lambda: ops.diff_attention_qkv(x[None], lam, 1), lambda: ops.diff_attention_qkv(q[None], x[0, :1], 1)]


def check_forward_mode_is_refused(device):
    import torch.autograd.forward_ad as fwd
    x = torch.zeros(4, 192, device=device)
    with fwd.dual_level():
        for call in floating_calls(fwd.make_dual(x, torch.ones_like(x))):
            with pytest.raises(L.GptHipError, match="forward-mode"):
                call()


def test_forward_mode_is_refused():
    """A tangent is an error, not silently dropped (before the check of the device: no GPU is needed)."""
    check_forward_mode_is_refused("cpu")


@gpu
def test_forward_mode_is_refused_on_the_gpu():
    import torch.autograd.forward_ad as fwd
    check_forward_mode_is_refused(DEV)
    with fwd.dual_level():                               # a level without a tangent on any argument is an ordinary call
        assert all(call() is not None for call in floating_calls(normal(1, 4, 192)))
        # nor does a backward pass drop the tangent of its gradient
        x, w, lam = normal(1, 2, 4, 192).requires_grad_(), torch.ones(192, device=DEV), torch.zeros(1, device=DEV)
        for out in (ops.dropout(x, 0.1, 0), ops.rms_norm(x, w), ops.diff_attention_qkv(x, lam, 1)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, x, fwd.make_dual(torch.ones_like(out), torch.ones_like(out)))


def check_tracing_is_refused(device):
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.zeros(4, 192, device=device)
    for i in range(len(floating_calls(x))):
        call = lambda v: floating_calls(v)[i]()                                                               # noqa: E731,B023
        for trace in (lambda: torch.jit.trace(call, (x,), check_trace=False), lambda: make_fx(call)(x), lambda: make_fx(call, pre_dispatch=True)(x),
                      lambda: make_fx(call, tracing_mode="fake")(x), lambda: torch.func.functionalize(call)(x)):
            with pytest.raises(L.GptHipError, match="tracing"):
                trace()
    for transform in (torch.vmap, torch.func.grad):
        with pytest.raises(L.GptHipError, match="tracing"):
            transform(lambda v: ops.dropout(v, 0.1, 0).sum())(x)


def test_tracing_is_refused():
    """A trace would hold an allocation and no launch (before the check of the device: no GPU is needed)."""
    check_tracing_is_refused("cpu")


@gpu
def test_tracing_is_refused_on_the_gpu_and_a_flop_counter_is_not():
    from torch.utils.flop_counter import FlopCounterMode
    check_tracing_is_refused(DEV)
    x = normal(1, 4, 192)
    want = [call() for call in floating_calls(x)]
    with FlopCounterMode(display=False):
        got = [call() for call in floating_calls(x)]
    for a, b in zip(want, got):
        for u, v in zip(a, b) if isinstance(a, tuple) else ((a, b),):
            assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))


@gpu
@pytest.mark.parametrize("T", [5, 40])
def test_gradients_with_a_graph_are_refused_and_never_constants(T):
    """create_graph with a constant incoming gradient: what depends on its own inputs raises; what is linear in the inputs that require a
    gradient has none to keep and is the ordinary gradient."""
    leaf = lambda s, *n: normal(s, *n).requires_grad_()                                                      # noqa: E731
    x, h, w, lam = leaf(1, 1, T, 192), leaf(2, 1, T, 192), leaf(3, 192), torch.rand(1, device=DEV).requires_grad_()
    q, k, v = (leaf(s, 1, T, 64) for s in (4, 5, 6))
    c = lambda t: t.detach()                                                                                 # noqa: E731
    att = ops.diff_attention
    curved = [(ops.rms_norm(x, w), (x, w)), (ops.rms_norm(x, c(w)), (x,)), (ops.rms_norm(x, w), (w,)), (ops.add_rms_norm(h, c(x), c(w))[0], (h,)),
              (ops.add_rms_norm(c(h), x, w)[1], (x,)), (att(q, c(k), c(v), c(lam), 1), (q,)), (att(c(q), k, c(v), c(lam), 1), (k,)),
              (att(c(q), c(k), v, lam, 1), (v, lam)), (att(q, k, v, lam, 1), (v,)), (ops.diff_attention_qkv(x, c(lam), 1), (x,))]
    for out, leaves in curved:
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(out, leaves, torch.ones_like(out), create_graph=True, retain_graph=True)
        assert all(g is not None for g in torch.autograd.grad(out, leaves, torch.ones_like(out)))             # without a graph: as before
    linear = [(ops.dropout_add(h, x, 0.3, 1), (h, x)), (ops.rms_norm(c(x), w), (w,)), (att(c(q), c(k), v, c(lam), 1), (v,)),
              (att(c(q), c(k), c(v), lam, 1), (lam,))]
    for out, leaves in linear:
        g = torch.ones_like(out)
        kept = torch.autograd.grad(out, leaves, g, create_graph=True, retain_graph=True)
        assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(kept, torch.autograd.grad(out, leaves, g, retain_graph=True)))
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(out, leaves, g.requires_grad_(), create_graph=True)


@gpu
@pytest.mark.parametrize("t", [BF, F32])
@pytest.mark.parametrize("Tq,Tk", [(26, 26), (1, 3), (40, 40), (150, 150), (1, 700), (5, 9000), (600, 2000)])
def test_diff_attention_rows_of_nothing_but_minus_infinity(Tq, Tk, t):
    """Scores that are all -inf make their map NaN (0 / 0) at any length - its head's output, dv and that map's dq and dk -, and nothing else:
    the other map's gradients, the other heads and samples, and a sample without a key (zeros) keep their bits."""
    B, H, hd = 3, 2, 64
    _, q, k, v, lam, _, g = attention_case(B, Tq, Tk, H, hd, t, None, False)
    n = torch.tensor([Tk, 0, Tk], dtype=torch.int32, device=DEV)
    q.view(B, Tq, H, 2, hd)[0, :, 0, 0, 7] = 1.0
    runs = []
    for fill in (0.0, -math.inf):
        kk = k.clone()
        kk.view(B, Tk, H, 2, hd)[:2, :, 0, 0, 7] = fill            # head 0, map 0 of sample 0, and of the one without a key
        leaves = [x.detach().clone().requires_grad_() for x in (q, kk, v, lam)]
        out = ops.diff_attention(*leaves, H, n)
        with torch.no_grad():
            assert torch.equal(ops.diff_attention(*leaves, H, n).nan_to_num(7.0), out.nan_to_num(7.0))
        runs.append([x.detach() for x in (out, *torch.autograd.grad(out, leaves, g))])
    (out, dq, dk, dv, dlam), (out0, dq0, dk0, dv0, dlam0) = runs[1], runs[0]
    assert torch.equal(dlam, dlam0)
    for got, ref, maps in ((out, out0, False), (dv, dv0, False), (dq, dq0, True), (dk, dk0, True)):
        got, ref = (x.reshape(B, -1, H, 2, hd) for x in (got, ref))
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[0, :, 0, 0 if maps else slice(None)] = True
        assert bool(got[hit].isnan().all()) and torch.equal(got[~hit], ref[~hit])
    assert bool((out[1] == 0).all()) and bool((dq[1] == 0).all()) and bool((dk[1] == 0).all()) and bool((dv[1] == 0).all())


@gpu
@pytest.mark.parametrize("shape", [(5, 520), (3, 37), (2, 8200), (7, 2048)])
@pytest.mark.parametrize("size", [1e-17, 1e-14, 1e-12, 1e12, 1e14, 1e17])
def test_rms_norm_gradients_of_small_and_large_rows(size, shape):
    """The norm does not depend on its rows' size and the gradients are its reciprocal's: as long as the squares are in float32's range the
    bounds are those of rows around 1 (each scales with the row)."""
    x, w, gy = normal(1, *shape, std=size).requires_grad_(), (1 + normal(2, shape[-1], std=0.3)).requires_grad_(), normal(3, *shape)
    y = ops.rms_norm(x, w, 0.0)
    dx, dw = torch.autograd.grad(y, (x, w), gy)
    want, tol = norm_reference(None, x.detach(), w.detach(), 0.0, 0.0, 0, 0, gy)
    within(y, want["y"], tol["y"] + U * (want["y"].abs() + tol["y"]), "y")
    within(dx, want["dr"], tol["dr"] + U * (want["dr"].abs() + tol["dr"]), "dx")
    within(dw, want["dw"], tol["dw"], "dweight")


@gpu
def test_dropout_counter_advances_by_the_offsets_of_a_step():
    """Sites at offsets 0 .. 2 of a captured step: advanced by three per replay, no mask comes twice; by one (too little, as the documentation
    says), a site draws what its neighbour drew a step before."""
    sites, steps = 3, 4
    h = torch.ones(64, 96, device=DEV)
    counter = torch.zeros(1, dtype=torch.int64, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.dropout(h, 0.5, 21, 0, counter)
    torch.cuda.current_stream().wait_stream(side)
    for advance in (sites, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            masks = [ops.dropout(h, 0.5, 21, s, counter) for s in range(sites)]
            counter.add_(advance)
        counter.zero_()
        seen = []
        for step in range(steps):
            graph.replay()
            torch.cuda.synchronize()
            seen.append([m.clone() for m in masks])
            assert all(torch.equal(m, ops.dropout(h, 0.5, 21, s + advance * step)) for s, m in enumerate(seen[-1]))
        flat = [m for step in seen for m in step]
        same = [(i, j) for i in range(len(flat)) for j in range(i) if torch.equal(flat[i], flat[j])]
        if advance == sites:
            assert not same
        else:
            assert torch.equal(seen[1][0], seen[0][1]) and torch.equal(seen[1][1], seen[0][2])


@gpu
@pytest.mark.parametrize("d", [8, 5])
def test_rms_norm_of_more_rows_than_a_grid_takes(d):
    """2^24 rows and some (a norm over every head has that many): both halves and the last rows are what few rows give, with their masks."""
    rows, p = (1 << 24) + 5, 0.3
    some = torch.cat([torch.arange(3), (1 << 23) + torch.arange(-2, 3), (1 << 24) + torch.arange(-2, 5)]).to(DEV)
    h, r = torch.empty(rows, d, dtype=BF, device=DEV), torch.ones(rows, d, device=DEV)
    h[:], w = torch.arange(d, device=DEV) + 1, 1 + normal(3, d, std=0.3)
    h[some] = normal(1, len(some), d, dtype=BF)
    r[some] = normal(2, len(some), d)
    h.requires_grad_()
    y, x = ops.add_rms_norm(h, r, w, 1e-5, p, 5, 6)
    gy = torch.zeros_like(y)
    gy[some] = normal(4, len(some), d, dtype=BF)
    dh, = torch.autograd.grad(y, h, gy)
    for row in some.tolist():
        base = (row * d) // 8 * 8
        keep = philox_keep(row * d - base + d, p, 5, 6, base)[row * d - base:].to(DEV)
        want = r[row] + torch.where(keep, h.detach()[row].float() * factor(p), 0.0)
        assert torch.equal(x[row], want), row
        ref, tol = norm_reference(None, want[None], w, 1e-5, 0.0, 0, 0, gy[row][None])
        within(y[row][None], ref["y"], tol["y"] + HALF[BF] * (ref["y"].abs() + tol["y"]), "y")
        dhr, t = torch.where(keep, ref["dr"] * factor(p), 0.0), torch.where(keep, (tol["dr"] + U * ref["dr"].abs()) * factor(p), 0.0)
        within(dh[row][None], dhr, t + HALF[BF] * (dhr.abs() + t), "dh")
    assert bool(torch.isfinite(y[:: 1 << 20]).all())


@gpu
@pytest.mark.parametrize("B,T,H,t", [(3, 26, 2, BF), (2, 150, 2, BF), (1, 600, 1, BF), (2, 150, 2, F32)])
def test_a_captured_training_pass(B, T, H, t):
    """Forward and backward of norm, attention and dropout in one graph, warmed up on a side stream as the documentation says: every replay, with
    other data in the same buffers and eager passes between, is the eager pass."""
    hd = 64
    w = 2 * H * hd
    data = [[normal(10 * s + i, B, T, n, dtype=d) for i, (n, d) in enumerate(((w, t), (w, F32), (3 * w, t), (w, t), (w, F32)))] for s in range(3)]
    lens = torch.tensor(([T, T - 3, 1] * B)[:B], dtype=torch.int32, device=DEV)
    weight, lam = 1 + normal(90, w, std=0.2), 0.5 + normal(91, H, std=0.2)

    def step(h, x, qkv, gy, gx):
        leaves = [v.requires_grad_() for v in (h, x, qkv, weight, lam)]
        a = ops.diff_attention_qkv(qkv, lam, H, lens)
        y, s = ops.add_rms_norm(a + h, x, weight, p=0.2, seed=3, offset=1)
        s = ops.dropout_add(y, s, 0.1, 3, 2)
        return [v.detach() for v in (y, s, *torch.autograd.grad((y, s), leaves, (gy, gx)))]

    fresh = lambda d: [v.clone() for v in d]                                                                 # noqa: E731
    want = [step(*fresh(d)) for d in data]
    static = fresh(data[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*static)
    for i in (0, 1, 2, 1, 0):
        with torch.no_grad():
            for dst, src in zip(static, data[i]):
                dst.copy_(src)
        graph.replay()
        other = step(*fresh(data[(i + 1) % 3]))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i])), i
        assert all(torch.equal(a, b) for a, b in zip(other, want[(i + 1) % 3])), i


@gpu
def test_two_threads_at_once():
    """Calls and backward passes from two Python threads on streams of their own: each thread's results are the ones it gets alone."""
    import threading
    work = []
    for s, T in ((1, 26), (2, 300)):
        qkv, lam, g = normal(s, 2, T, 384, dtype=BF).requires_grad_(), torch.rand(1, device=DEV).requires_grad_(), normal(s + 5, 2, T, 128, dtype=BF)
        work.append((qkv, lam, g))

    def run(qkv, lam, g):
        out = ops.diff_attention_qkv(qkv, lam, 1)
        return [out.detach(), *torch.autograd.grad(out, (qkv, lam), g)]

    want = [run(*x) for x in work]
    torch.cuda.synchronize()
    got, failed = [[], []], []

    def thread(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i].append(run(*work[i]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                                                                               # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=thread, args=(i,)) for i in (0, 1)]
    [t.start() for t in threads], [t.join() for t in threads]
    assert not failed and all(len(x) == 20 for x in got)
    assert all(torch.equal(a, b) for i in (0, 1) for r in got[i] for a, b in zip(r, want[i]))
