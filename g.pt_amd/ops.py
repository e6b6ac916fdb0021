"""Operators of a differential-attention Block for training and sampling, on hand-written gfx950 kernels (include/gpt_hip.h):

  dropout, dropout_add            counter-based dropout, alone and with the residual's addition; the mask is never stored
  rms_norm, add_rms_norm          RMS norm of the residual stream, alone and with the (dropped-out) residual's addition
  rms_norm_mx8, add_rms_norm_mx8  the same with an 8-bit output (e4m3 values, one power-of-two scale per 32 columns)
  diff_attention(_qkv)            differential attention: (softmax(Q1 K1^T) - lam softmax(Q2 K2^T)) V

All take GPU tensors, run on the current stream of the tensors' device, allocate only their results (and a scratch buffer of their
own), never synchronise, and can be captured into a HIP graph.  The floating-point ones differentiate (once) through torch.autograd;
their gradients do not change from run to run.  bfloat16 results are those of float32 arithmetic, rounded once.  There is no CPU
fallback: what the kernels do not take raises GptHipError, and so do forward-mode differentiation, tracing (jit.trace, make_fx, fake
tensors) and the transforms of torch.func; gradients of gradients raise in the backward pass.

Tensors used on another stream than the one they were made on: as everywhere in torch, the caller orders the streams (and calls
record_stream where an input may be freed early).  Capturing a backward pass into a graph: warm the step up on a side stream first
and let no eager backward graph of the same leaves be alive during the capture, as for any torch operator."""
import importlib.util
import os

from . import _lib as L

_U64 = (1 << 64) - 1
_host = None


def _load():
    """The host side (csrc/ops_binding.cpp), bound to the kernel library that _lib has loaded."""
    global _host
    lib = L.lib()
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "gpt_ops.so")
    if not os.path.exists(path):
        raise L.GptHipError(f"{path} is missing: build it with `make -C g.pt_amd/csrc`")
    spec = importlib.util.spec_from_file_location("gpt_ops", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.init(lib._handle, L.GptHipError)
    _host = mod
    return mod


def dropout_add(h, resid, p, seed, offset=0, counter=None):
    """resid + dropout(h): h [..., d] and resid of the same shape (each float32 or bfloat16); the result has resid's type.

    The mask is a function of (seed, offset, element index): the same pair gives the same mask, so every site of a step takes an
    offset of its own.  `counter`: an int64 GPU tensor of one element that is added to `offset` when the kernel runs; a captured
    step that advances it between replays draws new masks (it must not change between a forward and its backward).  Advance it by the
    number of offsets that a step uses, at least: with sites at offsets 0 .. n - 1 and an advance of less than n, a site draws masks that
    another site drew a step before.  p is realised in steps of 1/65536; kept values are scaled by 1 / (1 - p)."""
    if resid is None:
        raise L.GptHipError("dropout_add: resid is None (use dropout)")
    return (_host or _load()).dropout_add(h, resid, p, seed & _U64, offset & _U64, counter)


def dropout(h, p, seed, offset=0, counter=None):
    """dropout(h) in h's type; see dropout_add."""
    return (_host or _load()).dropout_add(h, None, p, seed & _U64, offset & _U64, counter)


def add_rms_norm(h, resid, weight, eps=1e-5, p=0.0, seed=0, offset=0, counter=None):
    """(y, x): x = resid + dropout(h) (resid's type), y = x / sqrt(mean(x^2) + eps) * weight (h's type; of x as it is stored).

    h, resid [..., d] (float32 or bfloat16 each), weight float32 [d].  p, seed, offset, counter: see dropout_add."""
    return (_host or _load()).add_rms_norm(h, resid, weight, eps, p, seed & _U64, offset & _U64, counter)


def rms_norm(x, weight, eps=1e-5, out_dtype=None):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension, in out_dtype (default: x's type)."""
    return (_host or _load()).rms_norm(x, weight, eps, out_dtype)


def add_rms_norm_mx8(h, resid, weight, eps=1e-5, p=0.0, seed=0, offset=0, counter=None):
    """(q, scales, x): as add_rms_norm, y in 8 bits.  q [..., d] float8_e4m3fn, scales [..., d / 32] float8_e8m0fnu: the values are
    q * scales, one power-of-two scale per 32 columns (the smallest at which no value saturates).  No gradient."""
    if h is None:
        raise L.GptHipError("add_rms_norm_mx8: h is None (use rms_norm_mx8)")
    return (_host or _load()).norm_mx8(h, resid, weight, eps, p, seed & _U64, offset & _U64, counter)


def rms_norm_mx8(x, weight, eps=1e-5):
    """(q, scales) of rms_norm(x) in 8 bits; see add_rms_norm_mx8."""
    return (_host or _load()).norm_mx8(None, x, weight, eps, 0.0, 0, 0, None)[:2]


def diff_attention(q, k, v, lam, n_head, lengths=None, scale=None):
    """Differential attention (non-causal): per head (softmax(scale Q1 K1^T) - lam softmax(scale Q2 K2^T)) V.

    q [B, Tq, w], k and v [B, Tk, w] (float32 or bfloat16; any strides, no copy where rows are 16-byte aligned): head h holds columns
    [2 hd h, 2 hd (h + 1)) with hd = w / (2 n_head) (32, 64, 96 or 128); in q and k the first hd of them belong to the first map, the
    others to the second.  lam: float32 [n_head] or [1], the learned weight.  lengths: int32 (or int64) [B], valid keys per sample
    (clamped to [0, Tk]; a sample without any gives zeros).  scale: default 1 / sqrt(hd).  Returns [B, Tq, w] in q's type; gradients
    for q, k, v and lam."""
    return (_host or _load()).diff_attention(q, k, v, lam, n_head, lengths, scale)


def diff_attention_qkv(qkv, lam, n_head, lengths=None, scale=None):
    """diff_attention on one fused projection qkv [B, T, 3 w] = query | key | value, as the Blocks' fused Linear gives it: one
    gradient tensor, written in place of three."""
    return (_host or _load()).diff_attention_qkv(qkv, lam, n_head, lengths, scale)
