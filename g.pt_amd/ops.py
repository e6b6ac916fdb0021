"""Operators of a differential-attention Block for training and sampling, on hand-written gfx950 kernels (include/gpt_hip.h):

  dropout, dropout_add            counter-based dropout, alone and with the residual's addition; the mask is never stored
  rms_norm, add_rms_norm          RMS norm of the residual stream, alone and with the (dropped-out) residual's addition
  rms_norm_mx8, add_rms_norm_mx8  the same with an 8-bit output (e4m3 values, one power-of-two scale per 32 columns)
  diff_attention(_qkv)            differential attention: (softmax(Q1 K1^T) - lam softmax(Q2 K2^T)) V

All take GPU tensors, run on the current stream of the tensors' device, allocate only their results (and a scratch buffer of their
own), never synchronise, and can be captured into a HIP graph.  The floating-point ones differentiate (once) through torch.autograd;
their gradients do not change from run to run.  There is no CPU fallback: what the kernels do not take raises GptHipError.

Capturing a backward pass into a graph: as for any torch operator, warm the step up on a side stream first and let no eager
backward graph of the same leaves be alive during the capture."""
import ctypes as C
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L

_U64 = (1 << 64) - 1


def _fail(who, msg):
    raise L.GptHipError(f"{who}: {msg}")


def _code(t, who, name):
    if t.dtype == torch.bfloat16:
        return L.BF16
    if t.dtype == torch.float32:
        return L.F32
    _fail(who, f"{name} must be float32 or bfloat16 (got {t.dtype})")


def _same_device(who, *tensors):
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not torch.is_tensor(t) or not t.is_cuda:
            _fail(who, "the HIP path needs GPU tensors; there is no CPU fallback")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            _fail(who, f"tensors on different devices ({dev} and {t.device})")
    return dev


class _On:
    """The tensors' device as the current one for the length of a call."""

    def __init__(self, device):
        self.device, self.guard = device, None

    def __enter__(self):
        if self.device.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _rows(t):
    """`t` [..., d] as rows of d consecutive elements: (tensor that holds them, row stride).  A copy only where the strides do not allow it."""
    d = t.shape[-1]
    if t.is_contiguous():
        return t, d
    if t.stride(-1) == 1 or d == 1:
        shape, stride = t.shape[:-1], t.stride()[:-1]
        dims = [(n, s) for n, s in zip(shape, stride) if n > 1]
        if not dims:
            return t, d
        if all(a[1] == b[0] * b[1] for a, b in zip(dims, dims[1:])):
            return t, dims[-1][1]
    t = t.contiguous()
    return t, d


def _dropout(who, p, seed, offset, counter):
    """The C description of a mask (None: nothing is dropped)."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        _fail(who, f"dropout probability {p} not in [0, 1]")
    if counter is not None and (counter.dtype != torch.int64 or counter.numel() != 1):
        _fail(who, "counter must be an int64 tensor of one element")
    if round(65536 * p) == 0:
        return None
    return L.Dropout(p, int(seed) & _U64, int(offset) & _U64, None if counter is None else counter.data_ptr())


# ------------------------------------------------------------------------------------------------------------------ dropout
def _dropout_add(who, h, resid, out_dtype, drop):
    """out = (resid or 0) + drop(h)"""
    out = torch.empty(h.shape, dtype=out_dtype, device=h.device)
    if h.numel() == 0:
        return out
    d = h.shape[-1]
    hm, ldh = _rows(h)
    rm, ldr = (None, 0) if resid is None else _rows(resid)
    with _On(h.device):
        L.check(L.lib().gpt_dropout_add(_code(h, who, "h"), hm.data_ptr(), ldh, L.BF16 if out_dtype == torch.bfloat16 else L.F32,
                                        None if rm is None else rm.data_ptr(), ldr, out.data_ptr(), d, h.numel() // d, d,
                                        C.byref(drop), L.stream()), "gpt_dropout_add")
    return out


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, resid, counter, p, seed, offset):
        drop = _dropout("dropout", p, seed, offset, counter) or L.Dropout(0.0, 0, 0, None)
        ctx.args, ctx.h_dtype, ctx.has_resid = (p, seed, offset), h.dtype, resid is not None
        # saved, so that a counter advanced between forward and backward is an error and not another mask
        ctx.save_for_backward(*(() if counter is None else (counter,)))
        return _dropout_add("dropout_add", h, resid, h.dtype if resid is None else resid.dtype, drop)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        dh = None
        if ctx.needs_input_grad[0]:
            counter = ctx.saved_tensors[0] if ctx.saved_tensors else None
            drop = _dropout("dropout", *ctx.args, counter) or L.Dropout(0.0, 0, 0, None)
            dh = _dropout_add("dropout_add (backward)", g, None, ctx.h_dtype, drop)
        return dh, g if ctx.has_resid and ctx.needs_input_grad[1] else None, None, None, None, None


def dropout_add(h, resid, p, seed, offset=0, counter=None):
    """resid + dropout(h): h [..., d] and resid of the same shape (each float32 or bfloat16); the result has resid's type.

    The mask is a function of (seed, offset, element index): the same pair gives the same mask, so every site of a step takes an
    offset of its own.  `counter`: an int64 GPU tensor of one element that is added to `offset` when the kernel runs; a captured
    step that advances it between replays draws new masks (it must not change between a forward and its backward).  p is realised
    in steps of 1/65536; kept values are scaled by 1 / (1 - p)."""
    who = "dropout_add"
    _same_device(who, h, resid, counter)
    _code(h, who, "h"), _code(resid, who, "resid")
    if h.dim() == 0 or h.shape != resid.shape:
        _fail(who, f"h and resid must have the same shape, of one dimension at least (got {tuple(h.shape)} and {tuple(resid.shape)})")
    return _DropoutAdd.apply(h, resid, counter, p, seed, offset)


def dropout(h, p, seed, offset=0, counter=None):
    """dropout(h) in h's type; see dropout_add."""
    who = "dropout"
    _same_device(who, h, counter)
    _code(h, who, "h")
    if h.dim() == 0:
        _fail(who, "h must have one dimension at least")
    return _DropoutAdd.apply(h, None, counter, p, seed, offset)


# ----------------------------------------------------------------------------------------------------------------- RMS norm
def _norm_forward(who, h, resid, weight, eps, drop, y_dtype, keep):
    """(y, scales, x, rho); x is resid itself where h is None, rho None unless `keep`."""
    d, mx = resid.shape[-1], y_dtype is None
    rows = resid.numel() // d if d else 0
    dev = resid.device
    y = torch.empty(resid.shape, dtype=torch.float8_e4m3fn if mx else y_dtype, device=dev)
    scales = torch.empty(*resid.shape[:-1], d // 32, dtype=torch.float8_e8m0fnu, device=dev) if mx else None
    x = resid if h is None else torch.empty(resid.shape, dtype=resid.dtype, device=dev)
    rho = torch.empty(rows, dtype=torch.float32, device=dev) if keep else None
    if rows == 0 or d == 0:
        return y, scales, x, rho
    rm, ldr = _rows(resid)
    weight = weight.contiguous()
    a = L.AddRmsNorm()
    yc = L.BF16 if y_dtype == torch.bfloat16 else L.F32
    a.h_dtype, a.x_dtype, a.y_dtype = yc, _code(resid, who, "resid"), L.MXFP8 if mx else yc
    if h is not None:
        hm, a.ldh = _rows(h)
        a.h_dtype, a.h, a.x_out, a.ldx = _code(h, who, "h"), hm.data_ptr(), x.data_ptr(), d
    a.resid, a.ldr, a.weight, a.y, a.ldy = rm.data_ptr(), ldr, weight.data_ptr(), y.data_ptr(), d
    a.scales = scales.data_ptr() if mx else None
    a.rho = rho.data_ptr() if keep else None
    a.rows, a.d, a.eps = rows, d, eps
    if drop is not None:
        a.drop = C.pointer(drop)
    with _On(dev):
        L.check(L.lib().gpt_add_rmsnorm(C.byref(a), L.stream()), "gpt_add_rmsnorm")
    return y, scales, x, rho


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, resid, weight, counter, eps, p, seed, offset, y_dtype):
        keep = any(ctx.needs_input_grad[:3])
        y, _, x, rho = _norm_forward("add_rms_norm", h, resid, weight, eps, _dropout("add_rms_norm", p, seed, offset, counter), y_dtype, keep)
        if keep:
            ctx.set_materialize_grads(False)
            ctx.args, ctx.h_dtype = (p, seed, offset), None if h is None else h.dtype
            ctx.save_for_backward(x, weight, rho, *(() if counter is None else (counter,)))
        return y if h is None else (y, x)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gx=None):
        who = "add_rms_norm (backward)"
        x, weight, rho = ctx.saved_tensors[:3]
        drop = _dropout(who, *ctx.args, ctx.saved_tensors[3] if len(ctx.saved_tensors) > 3 else None)
        if gy is None and gx is None:
            return (None,) * 9
        y_dtype = ctx.h_dtype if gy is None else gy.dtype
        if gy is None:
            gy = torch.zeros(x.shape, dtype=y_dtype, device=x.device)
        d = x.shape[-1]
        need_h, _, need_w = ctx.needs_input_grad[:3]
        need_h = need_h and ctx.h_dtype is not None
        dr = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dh = torch.empty(x.shape, dtype=ctx.h_dtype, device=x.device) if need_h else None
        dw = torch.empty(d, dtype=torch.float32, device=x.device) if need_w else None
        if x.numel() == 0:
            return dh, dr, None if dw is None else dw.zero_(), None, None, None, None, None, None
        a = L.AddRmsNormBwd()
        gm, a.ldgy = _rows(gy)
        xm, a.ldx = _rows(x)
        wm = weight.contiguous()
        a.y_dtype, a.x_dtype = _code(gy, who, "gy"), _code(x, who, "x")
        a.h_dtype = a.y_dtype
        a.gy, a.x, a.weight, a.rho = gm.data_ptr(), xm.data_ptr(), wm.data_ptr(), rho.data_ptr()
        if gx is not None:
            gxm, a.ldgx = _rows(gx)
            a.gx = gxm.data_ptr()
        a.dresid, a.lddr = dr.data_ptr(), d
        if dh is not None:
            a.dh, a.lddh = dh.data_ptr(), d
        a.rows, a.d = x.numel() // d, d
        if drop is not None:
            a.drop = C.pointer(drop)
        with _On(x.device):
            lib = L.lib()
            if dw is not None:
                n = C.c_int64()
                L.check(lib.gpt_add_rmsnorm_bwd_workspace(a.rows, d, C.byref(n)), "gpt_add_rmsnorm_bwd_workspace")
                ws = torch.empty(n.value, dtype=torch.uint8, device=x.device)
                a.dweight, a.ws, a.ws_bytes = dw.data_ptr(), ws.data_ptr(), n.value
            L.check(lib.gpt_add_rmsnorm_bwd(C.byref(a), L.stream()), "gpt_add_rmsnorm_bwd")
        return dh, dr if ctx.needs_input_grad[1] else None, dw, None, None, None, None, None, None


def _check_norm(who, h, resid, weight, eps, counter=None):
    _same_device(who, h, resid, weight, counter)
    _code(resid, who, "the stream")
    if h is not None:
        _code(h, who, "h")
        if h.shape != resid.shape:
            _fail(who, f"h and resid must have the same shape (got {tuple(h.shape)} and {tuple(resid.shape)})")
    if resid.dim() == 0 or weight.dtype != torch.float32 or weight.shape != resid.shape[-1:]:
        _fail(who, f"weight must be float32 of the last dimension's size (got {weight.dtype} {tuple(weight.shape)} for {tuple(resid.shape)})")
    if not (eps >= 0.0 and math.isfinite(eps)):
        _fail(who, f"eps must be finite and not negative (got {eps})")


def add_rms_norm(h, resid, weight, eps=1e-5, p=0.0, seed=0, offset=0, counter=None):
    """(y, x): x = resid + dropout(h) (resid's type), y = x / sqrt(mean(x^2) + eps) * weight (h's type; of x as it is stored).

    h, resid [..., d] (float32 or bfloat16 each), weight float32 [d].  p, seed, offset, counter: see dropout_add."""
    _check_norm("add_rms_norm", h, resid, weight, eps, counter)
    return _AddRmsNorm.apply(h, resid, weight, counter, eps, p, seed, offset, h.dtype)


def rms_norm(x, weight, eps=1e-5, out_dtype=None):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension, in out_dtype (default: x's type)."""
    _check_norm("rms_norm", None, x, weight, eps)
    out_dtype = out_dtype or x.dtype
    if out_dtype not in (torch.float32, torch.bfloat16):
        _fail("rms_norm", f"out_dtype must be float32 or bfloat16 (got {out_dtype})")
    return _AddRmsNorm.apply(None, x, weight, None, eps, 0.0, 0, 0, out_dtype)


def _check_mx(who, d, *tensors):
    if d % 32 or d == 0:
        _fail(who, f"the last dimension must be a multiple of 32 (got {d})")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        _fail(who, "the 8-bit output has no gradient: call it under torch.no_grad()")


def add_rms_norm_mx8(h, resid, weight, eps=1e-5, p=0.0, seed=0, offset=0, counter=None):
    """(q, scales, x): as add_rms_norm, y in 8 bits.  q [..., d] float8_e4m3fn, scales [..., d / 32] float8_e8m0fnu: the values are
    q * scales, one power-of-two scale per 32 columns (the smallest at which no value saturates).  No gradient."""
    who = "add_rms_norm_mx8"
    _check_norm(who, h, resid, weight, eps, counter)
    _check_mx(who, resid.shape[-1], h, resid, weight)
    return _norm_forward(who, h, resid, weight, eps, _dropout(who, p, seed, offset, counter), None, False)[:3]


def rms_norm_mx8(x, weight, eps=1e-5):
    """(q, scales) of rms_norm(x) in 8 bits; see add_rms_norm_mx8."""
    who = "rms_norm_mx8"
    _check_norm(who, None, x, weight, eps)
    _check_mx(who, x.shape[-1], x, weight)
    return _norm_forward(who, None, x, weight, eps, None, None, False)[:2]


# ---------------------------------------------------------------------------------------------------- differential attention
_SHORT = 32     # up to this many queries and keys the backward recomputes the maps and keeps nothing of the forward


def _tokens(t, es):
    """`t` [B, T, w] with rows the kernels take (a copy where the strides or the alignment do not allow it): tensor, token and sample stride."""
    B, T, w = t.shape
    ld, bs = (t.stride(1) if T > 1 else w), (t.stride(0) if B > 1 else 0)
    if (t.stride(2) != 1 and w > 1) or (T > 1 and ld < w) or ld >= 1 << 25 or ld * es % 16 or bs * es % 16 or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        ld, bs = w, T * w
    return t, ld, bs


def _attention_struct(q, k, v, lam, lengths, n_head, scale):
    """The C descriptor without its outputs, and what it points at."""
    es = q.element_size()
    a = L.DiffAttention()
    a.dtype = L.BF16 if q.dtype == torch.bfloat16 else L.F32
    a.B, a.Tq, a.Tk, a.n_head, a.hd = q.shape[0], q.shape[1], k.shape[1], n_head, q.shape[2] // (2 * n_head)
    a.scale = scale
    q, a.ldq, a.bsq = _tokens(q, es)
    k, a.ldk, a.bsk = _tokens(k, es)
    v, a.ldv, a.bsv = _tokens(v, es)
    a.q, a.k, a.v, a.lam = q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr()
    a.lengths = None if lengths is None else lengths.data_ptr()
    return a, (q, k, v, lam, lengths)


def _scratch(fn, name, a, device):
    n = C.c_int64()
    L.check(fn(a.dtype, a.B, a.Tq, a.Tk, a.n_head, a.hd, C.byref(n)), name)
    return (torch.empty(n.value, dtype=torch.uint8, device=device), n.value) if n.value else (None, 0)


def _attention_forward(q, k, v, lam, lengths, n_head, scale, keep):
    B, Tq, w = q.shape
    out = torch.empty(B, Tq, w, dtype=q.dtype, device=q.device)
    lse = out2 = None
    if B == 0 or Tq == 0:
        return out, lse, out2
    if k.shape[1] == 0:
        return out.zero_(), lse, out2
    with _On(q.device):
        a, held = _attention_struct(q, k, v, lam, lengths, n_head, scale)
        a.out, a.ldo, a.bso = out.data_ptr(), w, Tq * w
        if keep and max(a.Tq, a.Tk) > _SHORT:
            lse = torch.empty(2, B, n_head, Tq, dtype=torch.float32, device=q.device)
            out2 = torch.empty_like(out)
            a.lse, a.out2 = lse.data_ptr(), out2.data_ptr()
        lib = L.lib()
        ws, n = _scratch(lib.gpt_diff_attention_workspace, "gpt_diff_attention_workspace", a, q.device)
        if n:
            a.ws, a.ws_bytes = ws.data_ptr(), n
        L.check(lib.gpt_diff_attention(C.byref(a), L.stream()), "gpt_diff_attention")
        del held
    return out, lse, out2


def _attention_backward(g, q, k, v, lam, lengths, out, lse, out2, n_head, scale, dq, dk, dv):
    """Fills dq, dk, dv (views with the kernels' row layout) and returns dlam."""
    dlam = torch.empty(n_head, dtype=torch.float32, device=q.device)
    if q.shape[0] == 0 or q.shape[1] == 0 or k.shape[1] == 0:
        for t in (dq, dk, dv, dlam):
            t.zero_()
        return dlam
    with _On(q.device):
        a, held = _attention_struct(q, k, v, lam, lengths, n_head, scale)
        es = q.element_size()
        a.out, a.ldo, a.bso = out.data_ptr(), out.stride(1), out.stride(0)
        if lse is not None:
            a.lse, a.out2 = lse.data_ptr(), out2.data_ptr()
        b = L.DiffAttentionBwd()
        g, b.lddo, b.bsdo = _tokens(g, es)
        b.dout = g.data_ptr()
        b.dq, b.lddq, b.bsdq = dq.data_ptr(), dq.stride(1), dq.stride(0)
        b.dk, b.lddk, b.bsdk = dk.data_ptr(), dk.stride(1), dk.stride(0)
        b.dv, b.lddv, b.bsdv = dv.data_ptr(), dv.stride(1), dv.stride(0)
        b.dlam = dlam.data_ptr()
        lib = L.lib()
        ws, n = _scratch(lib.gpt_diff_attention_bwd_workspace, "gpt_diff_attention_bwd_workspace", a, q.device)
        b.ws, b.ws_bytes = ws.data_ptr(), n
        L.check(lib.gpt_diff_attention_bwd(C.byref(a), C.byref(b), L.stream()), "gpt_diff_attention_bwd")
        del held
    return dlam


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, lengths, n_head, scale):
        keep = any(ctx.needs_input_grad[:4])
        out, lse, out2 = _attention_forward(q, k, v, lam, lengths, n_head, scale, keep)
        if keep:
            ctx.save_for_backward(q, k, v, lam, lengths, out, lse, out2)
            ctx.args = n_head, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        q, k, v, lam, lengths, out, lse, out2 = ctx.saved_tensors
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        dlam = _attention_backward(g, q, k, v, lam, lengths, out, lse, out2, *ctx.args, dq, dk, dv)
        return dq, dk, dv, dlam, None, None, None


class _DiffAttentionQkv(torch.autograd.Function):
    """The fused projection as one input: its gradient is one tensor too, written in place of three."""

    @staticmethod
    def forward(ctx, qkv, lam, lengths, n_head, scale):
        keep = any(ctx.needs_input_grad[:2])
        out, lse, out2 = _attention_forward(*qkv.chunk(3, -1), lam, lengths, n_head, scale, keep)
        if keep:
            ctx.save_for_backward(qkv, lam, lengths, out, lse, out2)
            ctx.args = n_head, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        qkv, lam, lengths, out, lse, out2 = ctx.saved_tensors
        dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        dlam = _attention_backward(g, *qkv.chunk(3, -1), lam, lengths, out, lse, out2, *ctx.args, *dqkv.chunk(3, -1))
        return dqkv, dlam, None, None, None


def _check_attention(who, q, k, v, lam, n_head, lengths, scale):
    _same_device(who, q, k, v, lam, lengths)
    _code(q, who, "q")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        _fail(who, f"q, k and v must have one type (got {q.dtype}, {k.dtype}, {v.dtype})")
    n_head = int(n_head)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        _fail(who, f"need q [B, Tq, w], k and v [B, Tk, w] (got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)})")
    w = q.shape[2]
    if n_head < 1 or w % (2 * n_head) or w // (2 * n_head) not in (32, 64, 96, 128):
        _fail(who, f"width {w} with {n_head} heads: the head dim w / (2 n_head) must be 32, 64, 96 or 128")
    if lam.dtype != torch.float32 or lam.dim() != 1 or lam.shape[0] not in (1, n_head):
        _fail(who, f"lam must be float32 of 1 or {n_head} elements (got {lam.dtype} {tuple(lam.shape)})")
    if lengths is not None:
        if lengths.dtype not in (torch.int32, torch.int64) or lengths.shape != (q.shape[0],):
            _fail(who, f"lengths must be int32 or int64 [{q.shape[0]}] (got {lengths.dtype} {tuple(lengths.shape)})")
        if lengths.dtype == torch.int64:
            lengths = lengths.clamp(0, k.shape[1]).to(torch.int32)
        lengths = lengths.contiguous()
    scale = 1.0 / math.sqrt(w // (2 * n_head)) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        _fail(who, f"scale must be positive and finite (got {scale})")
    return lam.expand(n_head).contiguous(), lengths, n_head, scale


def diff_attention(q, k, v, lam, n_head, lengths=None, scale=None):
    """Differential attention (non-causal): per head (softmax(scale Q1 K1^T) - lam softmax(scale Q2 K2^T)) V.

    q [B, Tq, w], k and v [B, Tk, w] (float32 or bfloat16; any strides, no copy where rows are 16-byte aligned): head h holds columns
    [2 hd h, 2 hd (h + 1)) with hd = w / (2 n_head) (32, 64, 96 or 128); in q and k the first hd of them belong to the first map, the
    others to the second.  lam: float32 [n_head] or [1], the learned weight.  lengths: int32 (or int64) [B], valid keys per sample
    (clamped to [0, Tk]; a sample without any gives zeros).  scale: default 1 / sqrt(hd).  Returns [B, Tq, w] in q's type; gradients
    for q, k, v and lam."""
    lam, lengths, n_head, scale = _check_attention("diff_attention", q, k, v, lam, n_head, lengths, scale)
    return _DiffAttention.apply(q, k, v, lam, lengths, n_head, scale)


def diff_attention_qkv(qkv, lam, n_head, lengths=None, scale=None):
    """diff_attention on one fused projection qkv [B, T, 3 w] = query | key | value, as the Blocks' fused Linear gives it."""
    if not torch.is_tensor(qkv) or qkv.dim() != 3 or qkv.shape[2] % 3:
        _fail("diff_attention_qkv", "qkv must be a [B, T, 3 w] tensor")
    lam, lengths, n_head, scale = _check_attention("diff_attention_qkv", *qkv.chunk(3, -1), lam, n_head, lengths, scale)
    return _DiffAttentionQkv.apply(qkv, lam, lengths, n_head, scale)
