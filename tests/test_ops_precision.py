"""gpt_amd.ops.diff_attention in bfloat16 rounds its results once and nothing else to 8 bits: the softmax weights P and the score
gradients dS enter the matrix products as two bfloat16 operands each, so their error is at most 2^-8 of 2^-8 of them."""
import pytest
import torch

from gpt_amd import ops
from tests.test_ops import BF, HALF, attention_case, attention_reference, gpu, within

TWO = HALF[BF] ** 2        # what the second operand's rounding leaves of the value


def check_two_operands(B, Tq, Tk, H, hd, lens=None, std=1.0, names=("out", "dq", "dk", "dv")):
    """Every element within the bound of float32 sums, of 2^-16 of P and dS and of the result's one rounding; and over a whole tensor no
    more than 1.1 times the error that rounding the exact result leaves (what is left beside it is 2^-8 of it and some 100 u; one
    more independent rounding of the same size would give 1.4)."""
    _, q, k, v, lam, n, g = attention_case(B, Tq, Tk, H, hd, BF, lens, False, std=std)
    want, tol = attention_reference(q, k, v, lam, H, n, hd ** -0.5, g, TWO)
    leaves = [x.clone().requires_grad_() for x in (q, k, v, lam)]
    out = ops.diff_attention(*leaves, H, n)
    got = dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, g)[:3])))
    for name in names:
        x, w = got[name], want[name]
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
    check_two_operands(B, Tq, Tk, H, hd, lens, std, ("out", "dv"))

