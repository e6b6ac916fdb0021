"""The gradient of differential attention's lam against 64 bits, with a bound that a missing part of the sum exceeds.

dlam[h] = -sum over samples, queries and keys of P_2 dP, dP = dO V^T.  With dO = P_2 V every row adds |P_2 V|^2: nothing cancels, and each wave's and
each span's share of the sum is a share of dlam itself."""
import math

import pytest
import torch

from gpt_amd import ops
from tests.test_ops import BF, DEV, F32, U, gpu, normal

# (B, Tq, Tk, heads, hd, type, lengths): <= 32 tokens; few waves per workgroup; spans of the sweeps that are joined (over the queries, over the keys,
# both); the larger workgroups
CASES = [(5, 26, 26, 3, 96, BF, None), (4, 32, 17, 2, 64, F32, None), (2, 70, 129, 3, 64, BF, None), (1, 257, 257, 2, 96, F32, None),
         (4, 600, 600, 1, 64, BF, [600, 0, 301, 32]), (4, 40, 2000, 1, 128, BF, None), (4, 2000, 40, 1, 96, F32, None), (4, 333, 1025, 1, 32, BF, [1025, 0, 513, 32]),
         (24, 161, 140, 8, 64, BF, [140, 0, 17, 64, 133, 140]), (24, 161, 140, 8, 128, BF, None), (24, 70, 70, 8, 96, BF, None), (24, 70, 70, 8, 32, F32, None)]


def dlam_case(B, Tq, Tk, H, hd, t, lens, device):
    w = 2 * H * hd
    q, k, v = (normal(s, B, T, w, dtype=t, device=device) for s, T in ((1, Tq), (2, Tk), (3, Tk)))
    lam = 0.5 + normal(4, H, std=0.3, device=device)
    n = torch.tensor((lens * B)[:B] if lens else [Tk] * B, dtype=torch.int32, device=device)
    ok = (torch.arange(Tk, device=device) < n[:, None]).view(B, 1, 1, Tk)
    Q, K = (x.double().view(B, -1, H, 2, hd)[:, :, :, 1].transpose(1, 2) for x in (q, k))
    V = v.double().view(B, Tk, H, 2 * hd).transpose(1, 2)
    c = hd ** -0.5
    S = (c * Q @ K.transpose(-1, -2)).masked_fill(~ok, -math.inf)
    P = torch.softmax(S.masked_fill(~ok.any(-1, keepdim=True), 0.0), -1).masked_fill(~ok, 0.0)
    g = (P @ V).transpose(1, 2).reshape(B, Tq, w).to(t)
    G = g.double().view(B, Tq, H, 2 * hd).transpose(1, 2)
    terms = P * (G @ V.transpose(-1, -2))                                                    # [B, H, Tq, Tk]
    # P from float32 scores (hd products and sums, their size at most absS) and a sum of Tk weights; dP of 2 hd products and sums
    absS = c * Q.abs() @ K.abs().transpose(-1, -2)
    eP = 2 * (U * (hd + 8) * absS.masked_fill(~ok, 0.0).amax(-1, keepdim=True) + 4 * U) + (Tk + 16) * U
    absdP = G.abs() @ V.abs().transpose(-1, -2)
    off = eP * terms.abs() + (2 * hd + 8) * U * P * absdP
    # the sum: 8 terms in float32, tiles of them in 64 bits, one rounding per lane, 6 additions over a wave; then 256 threads with every 256th of the
    # parts - one per 16 keys and span of the queries (five tiles of 32 rows at least in bf16, two in float32) - and 8 additions over those
    parts = B * (math.ceil(Tk / 128) * 8) * math.ceil(Tq / 64)
    depth = 8 + 1 + 6 + math.ceil(parts / 256) + 8 + 2
    tol = (off + depth * U * terms.abs()).sum((0, 2, 3))
    return (q, k, v, lam, n, g), terms, -terms.sum((0, 2, 3)), tol


def check_bound(terms, want, tol):
    assert bool((tol < 0.01 * want.abs()).all()), (tol / want.abs()).max()
    B, H, Tq, Tk = terms.shape
    for axis, size in ((3, 16), (2, 64)):                                # a wave's keys, a short span's queries, of one sample
        shares = torch.stack([s.sum((2, 3)) for s in terms.split(size, axis)])                # [blocks, B, H]
        counted = torch.stack([(s != 0).any(3).any(2) for s in terms.split(size, axis)])
        assert bool((shares > tol).logical_or(~counted).double().mean() > 0.9)
    flipped = torch.stack([s.sum((0, 2, 3)) * (-1) ** i for i, s in enumerate(terms.split(16, 3))]).sum(0)   # every other wave's sign
    assert bool(((want + flipped).abs() > 10 * tol).all())


@pytest.mark.parametrize("case", CASES, ids=str)
def test_the_bound_sees_a_missing_wave_span_or_sign(case):
    _, terms, want, tol = dlam_case(*case, "cpu")
    check_bound(terms, want, tol)


@gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_dlam(case):
    (q, k, v, lam, n, g), terms, want, tol = dlam_case(*case, DEV)
    lens = n if case[-1] else None
    leaves = [x.clone().requires_grad_() for x in (q, k, v, lam)]
    dlam = torch.autograd.grad(ops.diff_attention(*leaves, case[3], lens), leaves, g)[3]
    off = (dlam.double() - want).abs()
    assert bool((off <= tol).all()), (off / tol).max()


@gpu
def test_float32_dlam_of_cancelling_terms():
    """Random dO: dlam is what some thousand rows of either sign leave, and every rounding that a row shares shows.  Per row the kernels round as
    often as the plain formula in float32 does, so over 24 draws of 4 heads their error is no larger; 10 % is the spread of such an estimate
    (1 / sqrt(96))."""
    B, T, H, hd = 4, 257, 4, 96
    w, c = 2 * H * hd, hd ** -0.5

    def plain(q, k, v, g):
        Q, K = (x.view(B, T, H, 2, hd)[:, :, :, 1].transpose(1, 2).contiguous() for x in (q, k))
        V, G = (x.view(B, T, H, 2 * hd).transpose(1, 2).contiguous() for x in (v, g))
        S = c * torch.matmul(Q, K.transpose(-1, -2).contiguous())
        e = torch.exp(S - S.amax(-1, keepdim=True))
        P = e / e.sum(-1, keepdim=True)
        return -(P * torch.matmul(G, V.transpose(-1, -2).contiguous())).sum(-1).sum((0, 2))

    errors = []
    for seed in range(24):
        q, k, v, g = (normal(100 * seed + i, B, T, w) for i in range(4))
        lam = (0.5 + normal(100 * seed + 4, H, std=0.2)).requires_grad_()
        want = plain(*(x.double() for x in (q, k, v, g)))
        got = torch.autograd.grad(ops.diff_attention(q, k, v, lam, H), lam, g)[0]
        errors.append(torch.stack([got.double() - want, plain(q, k, v, g).double() - want]) / want.norm())
    mine, theirs = torch.stack(errors).pow(2).sum((0, 2)).sqrt().tolist()
    assert mine <= 1.1 * theirs, (mine, theirs)
