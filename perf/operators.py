"""Operators of a decoder's training step around its attention, each as one pass through its entry point.

Four kinds, in the order in which a training step meets them: the norms of queries and keys with the rotation of
positions (``pccl.ops.rotary``), attention (``pccl.ops.attention``), their backward passes, and the AdamW step over many
tensors (``pccl.ops.optim``).  The ranges are those of the GPT presets (4 to 32 heads of 64 or 128, sequences of up to
2048 tokens in a micro-batch of up to four, layers of 256 to 4096 columns), of packed documents of any length, and of
head sizes, shared key/value heads and 16-bit types beside them.

With ``own`` false the passes are the operators' plain forms in torch; with it true they are the library's calls.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BLOCK = 256                 # elements that share a scale in 8-bit optimizer states
_MASK32 = 0xFFFFFFFF


def listed():
    return [
        # the smallest preset's attention at its own sequence length: launches count
        {"name": "attn_fwd_small", "kind": "attn_fwd", "dtype": "bf16", "batch": 2, "q_len": 128, "k_len": 128, "heads": 4,
         "kv_heads": 4, "dim": 64, "causal": True, "lengths": ""},
        # a full micro-batch of the 1.3B preset
        {"name": "attn_fwd_large", "kind": "attn_fwd", "dtype": "bf16", "batch": 4, "q_len": 2048, "k_len": 2048, "heads": 16,
         "kv_heads": 16, "dim": 128, "causal": True, "lengths": ""},
        # a chunk of a sequence split over ranks against the keys gathered so far: odd lengths, shared key/value heads, fp16
        {"name": "attn_fwd_chunk", "kind": "attn_fwd", "dtype": "fp16", "batch": 1, "q_len": 1021, "k_len": 4093, "heads": 16,
         "kv_heads": 4, "dim": 80, "causal": True, "lengths": ""},
        # the backward pass of the 1.3B preset's micro-batch
        {"name": "attn_bwd_large", "kind": "attn_bwd", "dtype": "bf16", "batch": 4, "q_len": 2048, "k_len": 2048, "heads": 16,
         "kv_heads": 16, "dim": 128, "causal": True, "lengths": ""},
        # packed documents, from a single token to a long one, under a model with shared key/value heads; 5 rows of padding behind
        {"name": "attn_bwd_packed", "kind": "attn_bwd", "dtype": "bf16", "batch": 1, "q_len": 6144, "k_len": 6144, "heads": 16,
         "kv_heads": 8, "dim": 64, "causal": True, "lengths": "1,37,2048,512,1000,129,2412"},
        # queries and keys of the smallest preset, a quarter of each head left unrotated
        {"name": "qk_fwd_small", "kind": "qk_fwd", "dtype": "fp16", "batch": 2, "seq": 128, "heads": 4, "kv_heads": 4, "dim": 64,
         "rot": 48, "interleaved": True, "packed_positions": False, "weight": "fp16"},
        # queries and keys of the 1.3B preset, a full micro-batch, read out of the packed projection
        {"name": "qk_fwd_large", "kind": "qk_fwd", "dtype": "bf16", "batch": 4, "seq": 2048, "heads": 16, "kv_heads": 16, "dim": 128,
         "rot": 128, "interleaved": False, "packed_positions": False, "weight": "bf16"},
        # backward on an odd number of tokens whose positions start again with each document; shared key heads
        {"name": "qk_bwd_ragged", "kind": "qk_bwd", "dtype": "bf16", "batch": 1, "seq": 1501, "heads": 16, "kv_heads": 4, "dim": 64,
         "rot": 64, "interleaved": False, "packed_positions": True, "weight": "fp32"},
        # backward at the 7B preset's heads
        {"name": "qk_bwd_large", "kind": "qk_bwd", "dtype": "bf16", "batch": 4, "seq": 2048, "heads": 32, "kv_heads": 32, "dim": 128,
         "rot": 128, "interleaved": False, "packed_positions": False, "weight": "bf16"},
        # every tensor of a two-layer model of 256 columns, states in 32 bits: launches count
        {"name": "adamw32_small", "kind": "adamw", "bits": 32, "param": "bf16", "grad": "bf16", "layers": 2, "width": 256, "vocab": 1024,
         "ragged": "", "shift": 0},
        # four blocks of the 1.3B preset and its embedding, 308 million parameters, states in 8 bits
        {"name": "adamw8_large", "kind": "adamw", "bits": 8, "param": "bf16", "grad": "bf16", "layers": 4, "width": 2048, "vocab": 50304,
         "ragged": "", "shift": 0},
        # a list of odd sizes that do not start on vector boundaries, fp32 parameters without a second copy, states in 8 bits
        {"name": "adamw8_ragged", "kind": "adamw", "bits": 8, "param": "fp32", "grad": "fp32", "layers": 0, "width": 0, "vocab": 0,
         "ragged": "1,255,257,100003,31,4099,1500001,2047", "shift": 1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn_fwd", "attn_bwd", "qk_fwd", "qk_bwd", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    if kind in ("attn_fwd", "attn_bwd"):
        c = {"kind": kind, "dtype": dtype, "batch": 1, "q_len": 0, "k_len": 0, "heads": heads, "kv_heads": kv_heads,
             "dim": rng.choice([64, 128, 64, 128, 8 * rng.randint(2, 16)]), "causal": rng.random() < 0.75, "lengths": ""}
        packed, same = rng.random() < 0.4, rng.random() < 0.6
        most = next(x for x in listed() if x["name"] == kind + "_large")
        while True:
            if packed:
                c["q_len"] = c["k_len"] = left = _log(rng, 64, 6144)
                lengths = []
                while left > 0 and len(lengths) < 12:
                    lengths.append(min(left, _log(rng, 1, c["q_len"])))
                    left -= lengths[-1]
                c["lengths"] = ",".join(map(str, lengths))
            else:
                c["batch"], c["q_len"], c["k_len"] = _log(rng, 1, 8), _log(rng, 1, 4096), _log(rng, 1, 4096)
                if same:
                    c["k_len"] = c["q_len"]
            if work(c)["flops"] <= work(most)["flops"] and c["batch"] * heads * c["q_len"] * c["k_len"] <= 16 * 6144 * 6144:
                return c
    if kind in ("qk_fwd", "qk_bwd"):
        dim = rng.choice([64, 128, 64, 128, 8 * rng.randint(2, 16)])
        return {"kind": kind, "dtype": dtype, "batch": rng.randint(1, 4), "seq": _log(rng, 1, 2048), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "rot": dim if rng.random() < 0.6 else 8 * rng.randint(1, dim // 8),
                "interleaved": rng.random() < 0.3, "packed_positions": rng.random() < 0.3, "weight": rng.choice([dtype, "fp32"])}
    param = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    grad = "fp32" if rng.random() < 0.3 else param
    if rng.random() < 0.5:
        return {"kind": kind, "bits": rng.choice([8, 32]), "param": param, "grad": grad, "layers": rng.randint(1, 4),
                "width": rng.choice([256, 512, 1024, 2048]), "vocab": rng.choice([1024, 8192, 50304]), "ragged": "", "shift": 0}
    sizes = ",".join(str(_log(rng, 1, 4_000_000)) for _ in range(rng.randint(1, 40)))
    return {"kind": kind, "bits": rng.choice([8, 32]), "param": param, "grad": grad, "layers": 0, "width": 0, "vocab": 0,
            "ragged": sizes, "shift": rng.randint(0, 3)}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def _bounds(c):
    """Starts of the packed sequences and the end of the last one."""
    at = [0]
    for n in c["lengths"].split(","):
        at.append(at[-1] + int(n))
    return at


def _prepare_attention(c, g):
    dt, B, Sq, Sk, H, Hk, D = _DTYPES[c["dtype"]], c["batch"], c["q_len"], c["k_len"], c["heads"], c["kv_heads"], c["dim"]
    # the projections leave queries, keys and values side by side; a chunk against gathered keys has its queries apart
    if Sq == Sk:
        qkv = _randn(g, (B, Sq, H + 2 * Hk, D), dt)
        q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
    else:
        q, kv = _randn(g, (B, Sq, H, D), dt), _randn(g, (B, Sk, 2 * Hk, D), dt)
        k, v = kv[:, :, :Hk], kv[:, :, Hk:]
    s = {"causal": c["causal"], "scale": D ** -0.5, "cu": None}
    if c["lengths"]:
        q, k, v = q[0], k[0], v[0]
        s["cu"] = torch.tensor(_bounds(c), dtype=torch.int32, device=DEV)
    s.update(q=q, k=k, v=v)
    if c["kind"] == "attn_bwd":
        s["dout"] = _randn(g, q.shape, dt)
        s["out"], s["lse"] = _plain_attn_fwd(s)
    return s


def _prepare_qk(c, g):
    dt, B, S, H, Hk, D = _DTYPES[c["dtype"]], c["batch"], c["seq"], c["heads"], c["kv_heads"], c["dim"]
    qkv = _randn(g, (B, S, H + 2 * Hk, D), dt)
    wt = _DTYPES[c["weight"]]
    s = {"q": qkv[:, :, :H], "k": qkv[:, :, H:H + Hk], "interleaved": c["interleaved"], "eps": 1e-6,
         "qw": (1 + 0.2 * torch.randn(D, device=DEV, generator=g)).to(wt), "kw": (1 + 0.2 * torch.randn(D, device=DEV, generator=g)).to(wt)}
    half = c["rot"] // 2
    inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    angle = torch.arange(max(S, 16), dtype=torch.float64, device=DEV)[:, None] * inv
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    s["positions"] = None
    if c["packed_positions"]:       # documents of 7 to 300 tokens, one behind the other: positions start again at each
        n = int(torch.randint(7, 301, (1,), device=DEV, generator=g))
        s["positions"] = (torch.arange(S, device=DEV) % n).expand(B, S).contiguous()
    if c["kind"] == "qk_bwd":
        s["dq"], s["dk"] = _randn(g, (B, S, H, D), dt), _randn(g, (B, S, Hk, D), dt)
    return s


def _sizes(c):
    if c["ragged"]:
        return [int(n) for n in c["ragged"].split(",")]
    d = c["width"]
    block = [3 * d * d, 4 * d * d, d * d, 4 * d * d, 3 * d, 4 * d, d, d, d, d, d, d]
    return [c["vocab"] * d, 2048 * d, d, d] + block * c["layers"]


def _starts(sizes):
    """Where each tensor's part of the state begins: on a block of its own."""
    at = [0]
    for n in sizes:
        at.append(at[-1] + -(-n // _BLOCK) * _BLOCK)
    return at


def _prepare_adamw(c, g):
    sizes = _sizes(c)
    at = _starts(sizes)
    total, shift = at[-1], c["shift"]
    pt, gt = _DTYPES[c["param"]], _DTYPES[c["grad"]]

    def cut(flat):
        return [flat[shift + a:shift + a + n] for a, n in zip(at, sizes)]

    master = torch.randn(total + shift, device=DEV, generator=g) * 0.02
    grad = (torch.randn(total + shift, device=DEV, generator=g) * 1e-3).to(gt)
    param = master if pt == torch.float32 else master.to(pt)
    m = torch.randn(total, device=DEV, generator=g) * 3e-4
    v = (torch.randn(total, device=DEV, generator=g) * 1e-3).square_()
    inside = torch.zeros(total, dtype=torch.bool, device=DEV)
    for a, n in zip(at, sizes):
        inside[a:a + n] = True
    m, v = m * inside, v * inside
    s = {"at": at, "sizes": sizes, "bits": c["bits"], "param": param, "master": None if pt == torch.float32 else master,
         "params": cut(param), "grads": cut(grad), "masters": None if pt == torch.float32 else cut(master),
         # biases and gains are not decayed
         "decay": [0.1 if n > 50000 else 0.0 for n in sizes],
         # the squared norm that the step before it has formed, over all ranks
         "norm": (grad.double() ** 2).sum().float().view(1) * 1.7}
    if c["bits"] == 32:
        s.update(m=m, v=v)
    else:
        key = _key(0, 0)
        for name, x, signed in (("m", m, True), ("v", v, False)):
            s[name], s[name + "_scale"] = _quantize(x, torch.arange(total, device=DEV), key, signed)
    return s


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"].startswith("attn"):
        return {"kind": case["kind"], **_prepare_attention(case, g)}
    if case["kind"].startswith("qk"):
        return {"kind": case["kind"], **_prepare_qk(case, g)}
    return {"kind": case["kind"], **_prepare_adamw(case, g)}


# ---------------------------------------------------------------- attention, plain form
def _allowed(s):
    """Which key each query sees, [queries, keys]: those of its own sequence and, if causal, none behind it; the last
    query of a sequence stands at its last key."""
    Sq, Sk = s["q"].shape[-3], s["k"].shape[-3]
    i, j = torch.arange(Sq, device=DEV)[:, None], torch.arange(Sk, device=DEV)[None]
    if s["cu"] is None:
        return j <= i + (Sk - Sq) if s["causal"] else torch.ones(Sq, Sk, dtype=torch.bool, device=DEV)
    which = torch.bucketize(torch.arange(Sq, device=DEV), s["cu"][1:].long(), right=True)
    ok = (which[:, None] == which[None]) & (which < s["cu"].numel() - 1)[:, None]
    return ok & (j <= i) if s["causal"] else ok


def _heads(x, groups, n):
    """[B, S, H, D] or [S, H, D] to [B, key heads, heads that share one, S, D] in 32 bits."""
    x = x if x.dim() == 4 else x[None]
    B, S, H, D = x.shape
    return x.float().view(B, S, groups, n, D).permute(0, 2, 3, 1, 4)


def _back(x, like):
    """The way back, in the inputs' type."""
    B, g, n, S, D = x.shape
    return x.permute(0, 3, 1, 2, 4).reshape(like.shape).to(like.dtype)


def _scores(s):
    Hk, n = s["k"].shape[-2], s["q"].shape[-2] // s["k"].shape[-2]
    q, k, v = _heads(s["q"], Hk, n), _heads(s["k"], Hk, 1), _heads(s["v"], Hk, 1)
    x = (q @ k.transpose(-1, -2)) * s["scale"]
    return q, k, v, x.masked_fill_(~_allowed(s), -math.inf)


def _plain_attn_fwd(s):
    q, k, v, x = _scores(s)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = (x - m).exp()
    l = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(l == 0, 1.0, l)
    lse = (m + l.log()).flatten(1, 2).squeeze(-1)                   # [B, H, Sq]
    return _back(out, s["q"]), lse if s["q"].dim() == 4 else lse[0]


def _plain_attn_bwd(s):
    q, k, v, x = _scores(s)
    Hk, n = k.shape[1], q.shape[2]
    dout, out = _heads(s["dout"], Hk, n), _heads(s["out"], Hk, n)
    lse = s["lse"].view(q.shape[0], Hk, n, q.shape[3], 1)
    p = (x - torch.where(lse == -math.inf, 0.0, lse)).exp()
    dv = (p.transpose(-1, -2) @ dout).sum(2, keepdim=True)
    dp = dout @ v.transpose(-1, -2)
    ds = p * (dp - (dout * out).sum(-1, keepdim=True)) * s["scale"]
    dq = ds @ k
    dk = (ds.transpose(-1, -2) @ q).sum(2, keepdim=True)
    return _back(dq, s["q"]), _back(dk, s["k"]), _back(dv, s["v"])


# ---------------------------------------------------------------- norms of queries and keys, rotation: plain form
def _pairs(x, rot, interleaved):
    """The two halves of each rotated pair, and what is not rotated."""
    a, rest = x[..., :rot], x[..., rot:]
    return (a[..., 0::2], a[..., 1::2], rest) if interleaved else (a[..., :rot // 2], a[..., rot // 2:], rest)


def _join(a, b, rest, interleaved):
    both = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((both, rest), -1)


def _angles(s, x):
    cos, sin = (s["cos"][:x.shape[1]], s["sin"][:x.shape[1]]) if s["positions"] is None else (s["cos"][s["positions"]], s["sin"][s["positions"]])
    return cos.unsqueeze(-2), sin.unsqueeze(-2)


def _plain_qk(s, x, w):
    f = x.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + s["eps"]) * w.float()
    cos, sin = _angles(s, x)
    a, b, rest = _pairs(y, 2 * cos.shape[-1], s["interleaved"])
    return _join(a * cos - b * sin, b * cos + a * sin, rest, s["interleaved"]).to(x.dtype)


def _plain_qk_bwd(s, dy, x, w):
    f = x.float()
    r = torch.rsqrt(f.square().mean(-1, keepdim=True) + s["eps"])
    cos, sin = _angles(s, x)
    a, b, rest = _pairs(dy.float(), 2 * cos.shape[-1], s["interleaved"])
    dn = _join(a * cos + b * sin, b * cos - a * sin, rest, s["interleaved"])
    xh = f * r
    gx = dn * w.float()
    dx = r * (gx - xh * (gx * xh).mean(-1, keepdim=True))
    return dx.to(x.dtype), (dn * xh).flatten(0, -2).sum(0).to(w.dtype)


# ---------------------------------------------------------------- AdamW over many tensors, plain form
def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & _MASK32
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & _MASK32
    return x ^ (x >> 16)


def _key(seed, step):
    return _mix((_mix(seed & _MASK32) + step) & _MASK32)


def _noise(index, key):
    """A word of 32 bits for each element of the state, from its place, the step and the seed."""
    return _mix(((index & _MASK32) + (index >> 32) * 0x9E3779B1 + key) & _MASK32)


def _quantize(x, index, key, signed):
    """Codes and block maxima: x is about max * (code / 127)^2 with its sign, or max * (code / 255)^4 where there is none,
    rounded up or down by chance so that the mean is x."""
    top = 127 if signed else 255
    power = 2 if signed else 4
    b = x.view(-1, _BLOCK)
    size = b.abs()
    most = size.amax(-1, keepdim=True)
    most = torch.where(most < 2.0 ** -80, 0.0, torch.where(torch.isfinite(most), most, math.nan))
    inv = torch.where(most > 0, 1.0 / most, 0.0)
    y = (size * inv) * float(top ** power)
    c = y.double().pow(1.0 / power).floor().clamp(0, top)           # the largest c with c^power <= y, put right by one below

    def up(c):
        return (c * c).float() if signed else (c * c).float() * (c * c).float()

    c = torch.where(up(c + 1) <= y, c + 1, torch.where(up(c) > y, c - 1, c)).clamp(0, top)
    word = _noise(index.view(-1, _BLOCK), key)
    u = ((word >> 16) if signed else (word & 0xFFFF)).float() * 2.0 ** -16 + 2.0 ** -17
    c = (c + (u * (up(c + 1) - up(c)) < y - up(c))).clamp(max=top)
    if not signed:
        c = torch.where((size > 0) & (most > 0), c.clamp(min=1), c)
    c = torch.nan_to_num(c)
    code = (torch.where(b < 0, -c, c).to(torch.int8) if signed else c.to(torch.uint8)).view(-1)
    return code, most.view(-1)


def _dequantize(code, most, signed):
    c = code.view(-1, _BLOCK).float()
    unit = (most * np.float32(1 / 127 ** 2 if signed else 1 / 255 ** 4).item()).view(-1, 1)
    return (unit * (c.abs() * c if signed else (c * c) * (c * c))).view(-1)


_LR, _BETA1, _BETA2, _EPS, _STEP, _MAX_NORM, _SEED = 1e-4, 0.9, 0.95, 1e-8, 7, 1.0, 11


def _f32(x):
    return float(np.float32(x))


def _adamw_tensor(s, k, gs, key):
    p, grad, a, n = s["params"][k], s["grads"][k], s["at"][k], s["sizes"][k]
    w = p if s["masters"] is None else s["masters"][k]
    e = s["at"][k + 1]
    index = torch.arange(a, e, device=DEV)
    if s["bits"] == 8:
        blocks = slice(a // _BLOCK, e // _BLOCK)
        m = _dequantize(s["m"][a:e], s["m_scale"][blocks], True)
        v = _dequantize(s["v"][a:e], s["v_scale"][blocks], False)
    else:
        m, v = s["m"][a:e], s["v"][a:e]
    g = torch.nn.functional.pad(grad.float(), (0, e - a - n)) * gs
    m = m * _f32(_BETA1) + g * _f32(1 - _BETA1)
    v = v * _f32(_BETA2) + (g * g) * _f32(1 - _BETA2)
    mh, vh = m[:n] / (1 - _BETA1 ** _STEP), v[:n] / (1 - _BETA2 ** _STEP)
    w.copy_(w * (1 - _LR * s["decay"][k]) - _LR * (mh / (vh.sqrt() + _EPS)))
    if w is not p:
        p.copy_(w)
    if s["bits"] == 8:
        s["m"][a:e], s["m_scale"][blocks] = _quantize(m, index, key, True)
        s["v"][a:e], s["v_scale"][blocks] = _quantize(v, index, key, False)
    else:
        s["m"][a:e], s["v"][a:e] = m, v


def _plain_adamw(s):
    gs = torch.clamp(_MAX_NORM / (s["norm"].sqrt() + _f32(1e-6)), max=1.0)
    key = _key(_SEED, _STEP)
    [_adamw_tensor(s, k, gs, key) for k in range(len(s["sizes"]))]
    if s["bits"] == 8:
        return _adamw_outputs(s, _dequantize(s["m"], s["m_scale"], True), _dequantize(s["v"], s["v_scale"], False))
    return _adamw_outputs(s, s["m"], s["v"])


def _adamw_outputs(s, m, v):
    return {"param": s["param"], "master": s["master"], "exp_avg": m, "exp_avg_sq": v}


# ---------------------------------------------------------------- one pass
def run(state):
    s, kind = state, state["kind"]
    if kind == "attn_fwd":
        if own:
            from pccl.ops.attention import attention_forward

            return attention_forward(s["q"], s["k"], s["v"], causal=s["causal"], scale=s["scale"], cu_seqlens_q=s["cu"], cu_seqlens_k=s["cu"])
        return _plain_attn_fwd(s)
    if kind == "attn_bwd":
        if own:
            from pccl.ops.attention import attention_backward

            return attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], causal=s["causal"], scale=s["scale"],
                                      cu_seqlens_q=s["cu"], cu_seqlens_k=s["cu"])
        return _plain_attn_bwd(s)
    if kind == "qk_fwd":
        if own:
            from pccl.ops.rotary import qk_norm_rope_forward

            return qk_norm_rope_forward(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], positions=s["positions"], eps=s["eps"],
                                        interleaved=s["interleaved"])
        return _plain_qk(s, s["q"], s["qw"]), _plain_qk(s, s["k"], s["kw"])
    if kind == "qk_bwd":
        if own:
            from pccl.ops.rotary import qk_norm_rope_backward

            return qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"],
                                         positions=s["positions"], eps=s["eps"], interleaved=s["interleaved"])
        dq, dqw = _plain_qk_bwd(s, s["dq"], s["q"], s["qw"])
        dk, dkw = _plain_qk_bwd(s, s["dk"], s["k"], s["kw"])
        return dq, dk, dqw, dkw
    if own:
        from pccl.ops.optim import AdamWState, adamw_step

        st = AdamWState(s["m"], s["v"], s.get("m_scale"), s.get("v_scale"))
        adamw_step(s["params"], s["grads"], st, step=_STEP, lr=_LR, beta1=_BETA1, beta2=_BETA2, eps=_EPS, weight_decay=s["decay"],
                   masters=s["masters"], max_grad_norm=_MAX_NORM, total_sq_norm=s["norm"], seed=_SEED)
        return _adamw_outputs(s, *st.dequantize())
    return _plain_adamw(s)


# ---------------------------------------------------------------- what a pass cannot do without
def _spans(c):
    if c["lengths"]:
        return [(int(n), int(n)) for n in c["lengths"].split(",")]
    return [(c["q_len"], c["k_len"])] * c["batch"]


def _seen(c):
    """Pairs of a query and a key that it sees, over the batch, for one head."""
    n = 0
    for q, k in _spans(c):
        if not c["causal"]:
            n += q * k
        else:                               # query i sees i + (k - q) + 1 keys, none where that is not positive
            first = max(0, q - k)
            n += (q - first) * (2 * (first + k - q + 1) + (q - first - 1)) // 2
    return n


def work(case):
    c = case
    if c["kind"].startswith("attn"):
        q, k = c["batch"] * c["q_len"] * c["heads"], c["batch"] * c["k_len"] * c["kv_heads"]
        products = _seen(c) * c["heads"] * c["dim"] * 2
        if c["kind"] == "attn_fwd":
            return {"bytes": (2 * q + 2 * k) * c["dim"] * 2 + 4 * q, "flops": 2 * products}
        # reads dout, out, q, k, v and the row sums; writes dq, dk, dv: five products of the size of the scores
        return {"bytes": (4 * q + 4 * k) * c["dim"] * 2 + 4 * q, "flops": 5 * products}
    if c["kind"].startswith("qk"):
        rows, D = c["batch"] * c["seq"], c["dim"]
        n = rows * (c["heads"] + c["kv_heads"]) * D
        table = c["seq"] * c["rot"] * 4 + (8 * rows if c["packed_positions"] else 0)
        if c["kind"] == "qk_fwd":
            return {"bytes": 4 * n + table, "flops": 8 * n}
        return {"bytes": 6 * n + table, "flops": 16 * n}
    n = sum(_sizes(c))
    grad = 4 if c["grad"] == "fp32" else 2
    weight = 8 if c["param"] == "fp32" else 8 + 2                   # the 32-bit copy both ways, the 16-bit one out
    # 8 bits: codes both ways, and the values they stand for written out in 32 bits
    return {"bytes": n * (grad + weight + (4 + 8 if c["bits"] == 8 else 16)), "flops": 20 * n}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_attention(c, seed):
    s = prepare(c, seed)
    G = c["heads"] // c["kv_heads"]
    packed = s["q"].dim() == 3
    up = lambda x: (x[None] if packed else x).double().transpose(1, 2)                                   # noqa: E731
    q, k, v = up(s["q"]), up(s["k"]).repeat_interleave(G, 1), up(s["v"]).repeat_interleave(G, 1)
    B, H, Sq, D = q.shape
    Sk = k.shape[2]
    see = torch.zeros(Sq, Sk, dtype=torch.bool, device=DEV)
    at = _bounds(c) if c["lengths"] else None
    for a, b in ([(0, Sq)] if at is None else zip(at, at[1:])):
        ka, kb = (0, Sk) if at is None else (a, b)
        part = torch.ones(b - a, kb - ka, dtype=torch.bool, device=DEV)
        see[a:b, ka:kb] = part.tril((kb - ka) - (b - a)) if c["causal"] else part
    x = torch.einsum("bhid,bhjd->bhij", q, k) * s["scale"]
    x[:, :, ~see] = -math.inf
    down = lambda x: (x.transpose(1, 2)[0] if packed else x.transpose(1, 2)).contiguous()                # noqa: E731
    if c["kind"] == "attn_fwd":
        lse = torch.logsumexp(x, -1)
        p = torch.nan_to_num(torch.softmax(x, -1))
        return down(torch.einsum("bhij,bhjd->bhid", p, v)), lse[0] if packed else lse
    lse = (s["lse"][None] if packed else s["lse"]).double()
    p = torch.exp(x - lse.nan_to_num(neginf=0.0)[..., None])
    del x
    do, out = up(s["dout"]), up(s["out"])
    ds = torch.einsum("bhid,bhjd->bhij", do, v).sub_((do * out).sum(-1)[..., None]).mul_(p).mul_(s["scale"])
    share = lambda x: x.unflatten(1, (c["kv_heads"], G)).sum(2)                                          # noqa: E731
    return (down(torch.einsum("bhij,bhjd->bhid", ds, k)), down(share(torch.einsum("bhij,bhid->bhjd", ds, q))),
            down(share(torch.einsum("bhij,bhid->bhjd", p, do))))


def _exact_qk(c, seed):
    s = prepare(c, seed)
    D, rot = c["dim"], c["rot"]
    # the rotation as complex numbers: pair t of a head is the number first + i second
    first = torch.arange(0, rot, 2) if c["interleaved"] else torch.arange(rot // 2)
    second = first + 1 if c["interleaved"] else first + rot // 2
    pos = torch.arange(c["seq"], device=DEV).expand(c["batch"], -1) if s["positions"] is None else s["positions"]
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos].unsqueeze(2)

    def rotate(x, t):
        z = torch.complex(x[..., first], x[..., second]) * t
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    def both(f):
        return [f(s["q"].double(), s["qw"].double(), s.get("dq")), f(s["k"].double(), s["kw"].double(), s.get("dk"))]

    if c["kind"] == "qk_fwd":
        return tuple(both(lambda x, w, d: rotate(x / (x.pow(2).sum(-1, keepdim=True) / D + s["eps"]).sqrt() * w, turn)))

    def back(x, w, d):
        size = (x.pow(2).sum(-1, keepdim=True) / D + s["eps"]).sqrt()
        n = x / size
        t = rotate(d.double(), turn.conj())
        u = t * w
        return (u - n * (n * u).sum(-1, keepdim=True) / D) / size, torch.einsum("bshd,bshd->d", t, n)

    (dq, dqw), (dk, dkw) = both(back)
    return dq, dk, dqw, dkw


def _exact_adamw(c, seed):
    """Parameters and 32-bit states; the values of 8-bit states are chosen by rounding and have no other definition than the codes."""
    s = prepare(c, seed)
    at, sizes, shift = s["at"], s["sizes"], c["shift"]
    clip = min(1.0, _MAX_NORM / (math.sqrt(float(s["norm"])) + 1e-6))
    if s["bits"] == 8:
        m = s["m"].double()
        m = m * m.abs() / 127 ** 2 * s["m_scale"].double().repeat_interleave(_BLOCK)
        v = (s["v"].double() / 255) ** 4 * s["v_scale"].double().repeat_interleave(_BLOCK)
    else:
        m, v = s["m"].double(), s["v"].double()
    w = (s["param"] if s["master"] is None else s["master"]).double()
    for k, n in enumerate(sizes):
        here, there = slice(at[k], at[k] + n), slice(shift + at[k], shift + at[k] + n)
        g = s["grads"][k].double() * clip
        m[here] = _BETA1 * m[here] + (1 - _BETA1) * g
        v[here] = _BETA2 * v[here] + (1 - _BETA2) * g ** 2
        step = (m[here] / (1 - _BETA1 ** _STEP)) / ((v[here] / (1 - _BETA2 ** _STEP)).sqrt() + _EPS)
        w[there] -= _LR * (step + s["decay"][k] * w[there])
    state = (None, None) if s["bits"] == 8 else (m, v)
    return {"param": w, "master": None if s["master"] is None else w, "exp_avg": state[0], "exp_avg_sq": state[1]}


def exact(case, seed):
    if case["kind"].startswith("attn"):
        return _exact_attention(case, seed)
    return _exact_qk(case, seed) if case["kind"].startswith("qk") else _exact_adamw(case, seed)
