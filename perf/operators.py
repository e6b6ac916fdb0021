"""The operators of a differential-attention Block as a training or sampling program calls them: sizes, inputs, one pass
in plain torch operations and one through the framework (`own`), the work of a pass, and the result in 64 bits.

Operators: dropout + residual addition, residual addition + RMS norm (output in the compute type or in 8 bits with a scale per
32 values), differential attention.  Training passes return the gradients beside the outputs."""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one residual addition of a short fine-tuning batch: 8 samples of 26 tokens, n_embd 1536
        dict(name="dropout add 8 samples", op="dropout", rows=208, d=1536, type="bf16", stream="fp32", p=0.1, train=False),
        # the training batch of 1024 samples on one GPU, forward and the masked gradient
        dict(name="dropout add training", op="dropout", rows=26624, d=1536, type="bf16", stream="fp32", p=0.1, train=True),
        # residual + norm between two Linears of a Block, training batch of 512 samples at n_embd 2048, with dropout
        dict(name="add norm training", op="norm", rows=13312, d=2048, type="bf16", stream="fp32", p=0.1, train=True),
        # the fp32 (parity) compute mode at an odd batch and a width that is no multiple of a wave
        dict(name="add norm fp32 odd", op="norm", rows=962, d=1000, type="fp32", stream="fp32", p=0.0, train=True),
        # sampling 320 networks: the norm hands 8-bit values to a scaled matrix product
        dict(name="add norm 8 bit", op="norm8", rows=8320, d=1536, type="bf16", stream="fp32", p=0.0, train=False),
        # a prompt of a few samples, latency counts
        dict(name="add norm 8 bit 2 samples", op="norm8", rows=52, d=1536, type="bf16", stream="fp32", p=0.0, train=False),
        # attention over the 26 tokens of a network, sampling 64 of them
        dict(name="attention 26 tokens", op="attention", B=64, Tq=26, Tk=26, H=8, hd=96, type="bf16", ragged=False, train=False),
        # the same in the training batch of 1024
        dict(name="attention 26 tokens training", op="attention", B=1024, Tq=26, Tk=26, H=8, hd=96, type="bf16", ragged=False, train=True),
        # token plans of large networks: thousands of tokens
        dict(name="attention long training", op="attention", B=2, Tq=4096, Tk=4096, H=8, hd=128, type="bf16", ragged=False, train=True),
        # networks of different sizes in one padded batch (an empty one among them)
        dict(name="attention ragged training", op="attention", B=16, Tq=515, Tk=515, H=8, hd=64, type="bf16", ragged=True, train=True),
        # the fp32 (parity) compute mode
        dict(name="attention fp32 training", op="attention", B=4, Tq=257, Tk=257, H=4, hd=96, type="fp32", ragged=False, train=True),
        # one new query token against a long list of parameter tokens
        dict(name="attention single query", op="attention", B=4, Tq=1, Tk=16384, H=8, hd=128, type="bf16", ragged=False, train=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["dropout", "norm", "norm8", "attention", "attention", "attention"])
    kind = rng.choice(["bf16", "bf16", "fp32"])
    train = rng.random() < 0.5
    if op == "attention":
        hd, H = rng.choice([32, 64, 96, 128]), rng.choice([1, 2, 4, 5, 8])
        shape = rng.choice(["tokens", "long", "long", "few"])
        if shape == "tokens":
            Tq = Tk = rng.randint(1, 32)
            B = _log_int(rng, 1, 1024)
        elif shape == "long":
            Tk = _log_int(rng, 33, 4096)
            Tq = Tk if rng.random() < 0.7 else _log_int(rng, 33, 4096)
            B = _log_int(rng, 1, max(1, min(64, 2 * 4096 * 4096 // (Tq * Tk))))
        else:
            Tq, Tk, B, train = rng.randint(1, 8), _log_int(rng, 64, 16384), rng.randint(1, 8), False
        if kind == "fp32":      # the parity mode is run at small sizes
            B = max(1, min(B, 4 * 1024 * 1024 // (Tq * Tk)))
        return dict(op=op, B=B, Tq=Tq, Tk=Tk, H=H, hd=hd, type=kind, ragged=rng.random() < 0.4, train=train)
    rows = _log_int(rng, 1, 26624 if kind == "bf16" else 8192)
    d = 32 * rng.randint(1, 64) if op == "norm8" or rng.random() < 0.7 else rng.randint(1, 2048)
    stream = "fp32" if kind == "fp32" else rng.choice(["fp32", "fp32", "bf16"])
    p = rng.choice([0.0, 0.1, round(rng.uniform(0.01, 0.6), 3)])
    if op == "dropout":
        p = max(p, 0.05)
    if op == "norm8":
        train = False
    return dict(op=op, rows=rows, d=d, type=kind, stream=stream, p=p, train=train)


def _lengths(case):
    """Valid keys per sample: a padded batch from the empty sample to the full one."""
    B, Tk = case["B"], case["Tk"]
    if not case["ragged"]:
        return None
    return [Tk * b // (B - 1) for b in range(B)] if B > 1 else [max(1, (2 * Tk) // 3)]


def work(case):
    es = 2 if case["type"] == "bf16" else 4
    if case["op"] == "attention":
        B, Tq, Tk, H, hd = (case[k] for k in ("B", "Tq", "Tk", "H", "hd"))
        lens = _lengths(case) or [Tk] * B
        keys, w = sum(lens), 2 * H * hd
        flops, nbytes = 8 * hd * H * Tq * keys, es * w * (2 * B * Tq + 2 * keys)
        if case["train"]:
            flops += 16 * hd * H * Tq * keys
            nbytes += es * w * (2 * B * Tq + 2 * B * Tk)
        return {"bytes": nbytes, "flops": flops}
    n = case["rows"] * case["d"]
    xs = 2 if case["stream"] == "bf16" else 4
    if case["op"] == "dropout":
        return {"bytes": n * (es + 2 * xs) + (n * (xs + es) if case["train"] else 0), "flops": 2 * n}
    out = 1 + 1 / 32 if case["op"] == "norm8" else es
    nbytes = n * (es + 2 * xs + out)
    if case["train"]:   # read gy, gx (x is there already), write dh, dresid
        nbytes += n * (2 * es + 2 * xs)
    return {"bytes": nbytes, "flops": 6 * n + (10 * n if case["train"] else 0)}


# ------------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEVICE) * std).to(dtype)

    t, train = TYPES[case["type"]], case["train"]
    if case["op"] == "attention":
        B, Tq, Tk, H, hd = (case[k] for k in ("B", "Tq", "Tk", "H", "hd"))
        w = 2 * H * hd
        s = dict(case=case, lam=(0.5 + 0.2 * normal(H)).requires_grad_(train), lengths=None)
        if Tq == Tk:    # one fused projection gives query | key | value
            s["qkv"] = normal(B, Tq, 3 * w, dtype=t).requires_grad_(train)
        else:
            s["q"] = normal(B, Tq, w, dtype=t).requires_grad_(train)
            s["k"], s["v"] = (normal(B, Tk, w, dtype=t).requires_grad_(train) for _ in range(2))
        if case["ragged"]:
            order = torch.randperm(B, generator=torch.Generator().manual_seed(seed))
            s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32)[order].to(DEVICE)
        if train:
            s["g"] = normal(B, Tq, w, dtype=t)
        return s
    rows, d, x = case["rows"], case["d"], TYPES[case["stream"]]
    s = dict(case=case, h=normal(rows, d, dtype=t).requires_grad_(train), resid=normal(rows, d, dtype=x, std=2.0).requires_grad_(train),
             rng=0x9E3779B97F4A7C15 ^ seed, offset=seed % 1000 + (1 << 33))
    if case["op"] != "dropout":
        s["w"] = (1.0 + normal(d, std=0.2)).requires_grad_(train)
    if train:
        s["gx"] = normal(rows, d, dtype=x)
        if case["op"] == "norm":
            s["gy"] = normal(rows, d, dtype=t)
    return s


# ---------------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    from gpt_amd import ops
    case = s["case"]
    train = case["train"]
    if case["op"] == "attention":
        if "qkv" in s:
            leaves = (s["qkv"], s["lam"])
            out = ops.diff_attention_qkv(s["qkv"], s["lam"], case["H"], lengths=s["lengths"])
        else:
            leaves = (s["q"], s["k"], s["v"], s["lam"])
            out = ops.diff_attention(s["q"], s["k"], s["v"], s["lam"], case["H"], lengths=s["lengths"])
        if not train:
            return {"out": out}
        return dict(zip(["out", "dlam", "dq", "dk", "dv"], _split(out, torch.autograd.grad(out, leaves, s["g"]))))
    if case["op"] == "dropout":
        x = ops.dropout_add(s["h"], s["resid"], case["p"], s["rng"], s["offset"])
        if not train:
            return {"x": x}
        dh, dr = torch.autograd.grad(x, (s["h"], s["resid"]), s["gx"])
        return {"x": x.detach(), "dh": dh, "dresid": dr}
    drop = dict(p=case["p"], seed=s["rng"], offset=s["offset"])
    if case["op"] == "norm8":
        q, scales, x = ops.add_rms_norm_mx8(s["h"], s["resid"], s["w"], **drop)
        return {"q": q, "scales": scales, "x": x}
    y, x = ops.add_rms_norm(s["h"], s["resid"], s["w"], **drop)
    if not train:
        return {"y": y, "x": x}
    dh, dr, dw = torch.autograd.grad((y, x), (s["h"], s["resid"], s["w"]), (s["gy"], s["gx"]))
    return {"y": y.detach(), "x": x.detach(), "dh": dh, "dresid": dr, "dw": dw}


def _split(out, grads):
    """(out, dlam, dq, dk, dv), the fused gradient cut into its three column ranges (views)."""
    dq, dk, dv = grads[0].chunk(3, -1) if len(grads) == 2 else grads[:3]
    return out.detach(), grads[-1], dq, dk, dv


# -------------------------------------------------------------------------------------------------------------- plain forms
def _keep_plain(rows, d, p, seed, offset):
    """Which elements stay, and the factor of those: Philox4x32-10 on 32-bit words held in int64, 8 elements a block."""
    n = rows * d
    blocks = torch.arange((n + 7) // 8, device=DEVICE)
    low = 0xFFFFFFFF
    c0, c1 = blocks & low, blocks >> 32
    c2, c3 = torch.full_like(c0, offset & low), torch.full_like(c0, offset >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):     # the generator's ten rounds
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], 1)
    halves = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n].view(rows, d)
    thr = round(65536 * p)
    return halves >= thr, 65536 / (65536 - thr)


def _drop_plain(v, s):
    case = s["case"]
    if round(65536 * case["p"]) == 0:
        return v
    if "keep" not in s:
        keep, factor = _keep_plain(case["rows"], case["d"], case["p"], s["rng"], s["offset"])
        s = dict(s, keep=keep, factor=factor)
    return torch.where(s["keep"], v * s["factor"], 0.0)


def _attention_plain(s):
    case = s["case"]
    B, Tq, Tk, H, hd = (case[k] for k in ("B", "Tq", "Tk", "H", "hd"))
    t, scale = TYPES[case["type"]], 1 / math.sqrt(hd)
    q, k, v = s["qkv"].chunk(3, -1) if "qkv" in s else (s["q"], s["k"], s["v"])
    q = q.float().view(B, Tq, H, 2, hd).permute(0, 2, 3, 1, 4).contiguous()     # [B, H, 2, T, hd]
    k = k.float().view(B, Tk, H, 2, hd).permute(0, 2, 3, 1, 4).contiguous()
    v = v.float().view(B, Tk, H, 2 * hd).permute(0, 2, 1, 3).contiguous()       # [B, H, T, 2 hd]
    sc = torch.matmul(q, k.transpose(-1, -2)) * scale
    if s["lengths"] is not None:
        valid = torch.arange(Tk, device=DEVICE) < s["lengths"].view(B, 1, 1, 1, 1)
        sc = torch.where(valid, sc, -math.inf)
        top = sc.amax(-1, keepdim=True)
        e = torch.where(valid, torch.exp(sc - top), 0.0)
        total = e.sum(-1, keepdim=True)
        P = e / torch.where(total > 0, total, 1.0)
    else:
        e = torch.exp(sc - sc.amax(-1, keepdim=True))
        P = e / e.sum(-1, keepdim=True)
    lam = s["lam"].view(1, H, 1, 1)
    A = P[:, :, 0] - lam * P[:, :, 1]
    rows = lambda x: x.permute(0, 2, 1, 3).reshape(B, x.shape[2], -1).to(t)                    # noqa: E731
    pairs = lambda x: x.permute(0, 3, 1, 2, 4).reshape(B, x.shape[3], -1).to(t)                # noqa: E731
    out = rows(torch.matmul(A, v))
    if not case["train"]:
        return {"out": out}
    g = s["g"].float().view(B, Tq, H, 2 * hd).permute(0, 2, 1, 3).contiguous()
    dv = torch.matmul(A.transpose(-1, -2), g)
    dP = torch.matmul(g, v.transpose(-1, -2)).unsqueeze(2)
    D = (P * dP).sum(-1, keepdim=True)
    sign = torch.cat([torch.ones_like(lam), -lam], 0).permute(1, 0, 2, 3).unsqueeze(0)         # [1, H, 2, 1, 1]
    dS = P * (dP - D) * (sign * scale)
    return {"out": out, "dlam": -D[:, :, 1].sum((0, 2, 3)), "dq": pairs(torch.matmul(dS, k)),
            "dk": pairs(torch.matmul(dS.transpose(-1, -2), q)), "dv": rows(dv)}


@torch.no_grad()
def _plain(s):
    case = s["case"]
    if case["op"] == "attention":
        return _attention_plain(s)
    t, xt, train = TYPES[case["type"]], TYPES[case["stream"]], case["train"]
    s = dict(s)
    if round(65536 * case["p"]):
        s["keep"], s["factor"] = _keep_plain(case["rows"], case["d"], case["p"], s["rng"], s["offset"])
    x = (s["resid"].float() + _drop_plain(s["h"].float(), s)).to(xt)
    if case["op"] == "dropout":
        if not train:
            return {"x": x}
        return {"x": x, "dh": _drop_plain(s["gx"].float(), s).to(t), "dresid": s["gx"]}
    f = x.float()
    rho = 1 / torch.sqrt((f * f).mean(-1, keepdim=True) + 1e-5)
    y = f * rho * s["w"]
    if case["op"] == "norm8":
        blocks = y.view(case["rows"], -1, 32)
        m, e = torch.frexp(blocks.abs().amax(-1, keepdim=True))
        e = torch.where(m > 0, e - 9 + (m > 0.875), -127).clamp(min=-127)       # the smallest e with amax <= 448 * 2^e
        q = torch.ldexp(blocks, -e).to(torch.float8_e4m3fn).view(case["rows"], -1)
        return {"q": q, "scales": (e + 127).to(torch.uint8).view(case["rows"], -1).view(torch.float8_e8m0fnu), "x": x}
    if not train:
        return {"y": y.to(t), "x": x}
    gy, gx = s["gy"].float(), s["gx"].float()
    wg = s["w"] * gy
    dx = gx + rho * wg - f * (rho ** 3 * (wg * f).mean(-1, keepdim=True))
    return {"y": y.to(t), "x": x, "dh": _drop_plain(dx, s).to(t), "dresid": dx.to(xt), "dw": (gy * f * rho).sum(0)}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------------ 64 bits
def _keep_exact(n, p, seed, offset):
    """Keep mask of n elements by the generator's definition, on the host in unsigned 64-bit words."""
    u = np.uint64
    lo, sh = u(0xFFFFFFFF), u(32)
    blk = np.arange((n + 7) // 8, dtype=u)
    ctr = [blk & lo, blk >> sh, np.full_like(blk, offset & 0xFFFFFFFF), np.full_like(blk, offset >> 32)]
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for r in range(10):
        p0, p1 = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
        ka, kb = u((key[0] + r * 0x9E3779B9) & 0xFFFFFFFF), u((key[1] + r * 0xBB67AE85) & 0xFFFFFFFF)
        ctr = [(p1 >> sh) ^ ctr[1] ^ ka, p1 & lo, (p0 >> sh) ^ ctr[3] ^ kb, p0 & lo]
    out = np.empty((len(blk), 8), dtype=np.uint16)
    for j in range(8):
        out[:, j] = ((ctr[j // 2] >> u(16 * (j % 2))) & u(0xFFFF)).astype(np.uint16)
    return out.reshape(-1)[:n] >= round(65536 * p)


def _attention_exact(s):
    case = s["case"]
    B, Tq, Tk, H, hd, train = (case[k] for k in ("B", "Tq", "Tk", "H", "hd", "train"))
    w = 2 * H * hd
    fused = [s["qkv"].detach()[..., i * w:(i + 1) * w] for i in range(3)] if "qkv" in s else [s[n].detach() for n in "qkv"]
    Q, K, V = (x.double().reshape(B, -1, H, 2 * hd) for x in fused)
    lam = s["lam"].detach().double()
    lens = [Tk] * B if s["lengths"] is None else s["lengths"].tolist()
    out = torch.zeros(B, Tq, H, 2 * hd, dtype=torch.float64, device=DEVICE)
    dq, dk, dv = (torch.zeros_like(x) for x in (Q, K, V)) if train else (None,) * 3
    dlam = torch.zeros(H, dtype=torch.float64, device=DEVICE)
    c = hd ** -0.5
    for b in range(B) if Tq * Tk > 1024 else []:
        for h in range(H):
            n = lens[b]
            if not n:
                continue
            q, k, v = Q[b, :, h], K[b, :n, h], V[b, :n, h]
            maps = [torch.softmax(c * (q[:, i * hd:(i + 1) * hd] @ k[:, i * hd:(i + 1) * hd].T), -1) for i in (0, 1)]
            diff = maps[0] - lam[h] * maps[1]
            out[b, :, h] = diff @ v
            if train:
                g = s["g"][b].double().view(Tq, H, 2 * hd)[:, h]
                dv[b, :n, h] = diff.T @ g
                gv = g @ v.T
                dlam[h] -= (maps[1] * gv).sum()
                for i, f in ((0, 1.0), (1, -lam[h])):
                    pg = maps[i] * gv
                    ds = f * c * (pg - maps[i] * pg.sum(-1, keepdim=True))
                    cols = slice(i * hd, (i + 1) * hd)
                    dq[b, :, h, cols] = ds @ k[:, cols]
                    dk[b, :n, h, cols] = ds.T @ q[:, cols]
    if Tq * Tk <= 1024:      # all samples at once
        alive = (torch.arange(Tk, device=DEVICE)[None] < torch.tensor(lens, device=DEVICE)[:, None])[:, None, None]
        halves = [slice(0, hd), slice(hd, 2 * hd)]
        maps = []
        for cols in halves:
            e = torch.einsum("bqhc,bkhc->bhqk", Q[..., cols], K[..., cols]) * c
            e = torch.exp(e - e.masked_fill(~alive, -1e300).amax(-1, keepdim=True)).masked_fill(~alive, 0.0)
            maps.append(e / e.sum(-1, keepdim=True).clamp(min=1e-300))
        diff = maps[0] - lam.view(1, H, 1, 1) * maps[1]
        out = torch.einsum("bhqk,bkhc->bqhc", diff, V)
        if train:
            g = s["g"].double().view(B, Tq, H, 2 * hd)
            dv = torch.einsum("bhqk,bqhc->bkhc", diff, g)
            gv = torch.einsum("bqhc,bkhc->bhqk", g, V)
            dlam = -(maps[1] * gv).sum((0, 2, 3))
            for m, cols, f in zip(maps, halves, (torch.ones_like(lam), -lam)):
                ds = m * (gv - (m * gv).sum(-1, keepdim=True)) * f.view(1, H, 1, 1) * c
                dq[..., cols] = torch.einsum("bhqk,bkhc->bqhc", ds, K[..., cols])
                dk[..., cols] = torch.einsum("bhqk,bqhc->bkhc", ds, Q[..., cols])
    if not train:
        return {"out": out.reshape(B, Tq, w)}
    return {"out": out.reshape(B, Tq, w), "dlam": dlam, "dq": dq.reshape(B, Tq, w), "dk": dk.reshape(B, Tk, w), "dv": dv.reshape(B, Tk, w)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        with torch.no_grad():
            return _attention_exact(s)
    rows, d = case["rows"], case["d"]
    thr = round(65536 * case["p"])
    factor = torch.ones(rows, d, dtype=torch.float64, device=DEVICE)
    if thr:
        keep = torch.from_numpy(_keep_exact(rows * d, case["p"], s["rng"], s["offset"])).view(rows, d).to(DEVICE)
        factor = keep.double() * (65536.0 / (65536 - thr))
    with torch.no_grad():
        stored = s["resid"].double() + factor * s["h"].double()
        gx = s["gx"].double() if case["train"] else None
        if case["op"] == "dropout":
            return {"x": stored, "dh": gx * factor, "dresid": gx} if case["train"] else {"x": stored}
        x = stored.to(torch.bfloat16).double() if case["stream"] == "bf16" else stored     # the norm reads the stream as it is stored
        norm = (x.pow(2).sum(-1, keepdim=True) / d + 1e-5).sqrt()
        w = s["w"].detach().double()
        y = x / norm * w
        if case["op"] == "norm8":
            # before its rounding to 8 bits, in units of the block's scale 2^e, e the smallest integer with amax <= 448 * 2^e
            blocks = y.view(rows, d // 32, 32)
            e = torch.ceil(torch.log2(blocks.abs().amax(-1).clamp(min=2.0 ** -160) / 448)).clamp(min=-127)
            return {"q": (blocks / torch.exp2(e)[..., None]).view(rows, d), "scales": torch.exp2(e), "x": stored}
        if not case["train"]:
            return {"y": y, "x": stored}
        gy = s["gy"].double()
        gn = gy * w                                            # d y / d (x / norm)
        dx = gx + (gn - (x / norm) * ((gn * x / norm).sum(-1, keepdim=True) / d)) / norm
        return {"y": y, "x": stored, "dh": dx * factor, "dresid": dx, "dw": (gy * x / norm).sum(0)}
