"""Attention, forward and backward, against the formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _visible(Sq, Sk, causal):
    see = torch.ones(Sq, Sk, dtype=torch.bool, device=DEV)
    return see.tril(Sk - Sq) if causal else see


def _oracle(q, k, v, see, scale, dout=None, out=None, lse=None):
    """One sequence, [rows, heads, dim]; returns values and how far each may be off.

    u: half a step of the 16-bit type.  Probabilities and score gradients are rounded to it before a product, results once at
    the end.  Everything else is 32-bit: a sum of D products is off by at most D + 2 roundings of the sum of their sizes."""
    u, f = torch.finfo(q.dtype).eps / 2, 2.0 ** -23
    G = q.shape[1] // k.shape[1]
    D = q.shape[2]
    up = lambda x: x.double().transpose(0, 1)                                    # noqa: E731
    Q, K, V = up(q), up(k).repeat_interleave(G, 0), up(v).repeat_interleave(G, 0)
    s = (Q @ K.transpose(1, 2)) * scale
    size = (Q.abs() @ K.abs().transpose(1, 2)) * scale if s.numel() else s.abs()
    s = s.masked_fill(~see, -math.inf)
    if dout is None:
        L = torch.logsumexp(s, -1) if s.shape[-1] else torch.full(s.shape[:2], -math.inf, dtype=s.dtype, device=DEV)
        p = torch.exp(s - L.nan_to_num(neginf=0.0)[..., None])
        o = p @ V
        e_s = (D + 4) * f * (size.amax() if size.numel() else 0.0) + 2.0 ** -20
        a = p @ V.abs()
        # a probability of a 16-bit type below its normal range is off by half of its smallest step; the running maximum
        # may be below the true one by 2^8, never above
        tiny = torch.finfo(q.dtype).tiny * u * V.abs().sum(1, keepdim=True)
        n = max(s.shape[-1], 1)
        return (o.transpose(0, 1), ((u + 2 * e_s + n * 2.0 ** -24) * a + u * o.abs() + tiny).transpose(0, 1) + torch.finfo(q.dtype).tiny * u,
                L, e_s + n * 2.0 ** -24 + f * L.nan_to_num(neginf=0.0).abs())
    L, dO, O = lse.double(), up(dout), up(out)
    p = torch.exp(s - L.nan_to_num(neginf=0.0)[..., None])
    dp, delta = dO @ V.transpose(1, 2), (dO * O).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_p = (D + 4) * f * (size.amax() if size.numel() else 0.0) + f * L.nan_to_num(neginf=0.0).abs().max() + 2.0 ** -20
    e_dp = (D + 4) * f * (dO.abs() @ V.abs().transpose(1, 2) + (dO * O).abs().sum(-1, keepdim=True))
    small = torch.finfo(q.dtype).tiny * u
    e_ds = (u + 2 * e_p) * ds.abs() + p * e_dp + small
    e_pr = (u + 2 * e_p) * p + small
    share = lambda x: x.unflatten(0, (k.shape[1], G)).sum(1)                      # noqa: E731
    n = G * max(s.shape[1], s.shape[2])
    dq, dk, dv = (ds @ K) * scale, share(ds.transpose(1, 2) @ Q) * scale, share(p.transpose(1, 2) @ dO)
    ads = e_ds + n * f * ds.abs()
    t_q = (ads @ K.abs()) * scale + u * dq.abs()
    t_k = share(ads.transpose(1, 2) @ Q.abs()) * scale + u * dk.abs()
    t_v = share((e_pr + n * f * p).transpose(1, 2) @ dO.abs()) + u * dv.abs()
    down = lambda x: x.transpose(0, 1)                                           # noqa: E731
    return [(down(x), down(t) + small) for x, t in ((dq, t_q), (dk, t_k), (dv, t_v))]


def _close(got, want, tol, what):
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got.double() - want).abs() - tol
    assert off.numel() == 0 or float(off.max()) <= 0, \
        f"{what}: {float(off.max()):.3e} over its bound, error {float((got.double() - want).abs().max()):.3e}"


def _check_forward(out, lse, q, k, v, causal, scale):
    for b in range(q.shape[0]):
        o, to, L, tl = _oracle(q[b], k[b], v[b], _visible(q.shape[1], k.shape[1], causal), scale)
        _close(out[b], o, to, "out")
        none = L == -math.inf
        assert torch.equal(lse[b] == -math.inf, none)
        _close(lse[b].masked_fill(none, 0), L.masked_fill(none, 0), tl, "lse")


def _given(q, k, v, causal, scale):
    """Output and row sums for a backward pass, from the oracle."""
    outs, lses = [], []
    for b in range(q.shape[0]):
        o, _t, L, _tl = _oracle(q[b], k[b], v[b], _visible(q.shape[1], k.shape[1], causal), scale)
        outs.append(o.to(q.dtype))
        lses.append(L.float())
    return torch.stack(outs), torch.stack(lses).contiguous()


def _inputs(B, Sq, Sk, H, Hk, D, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda *s: (torch.randn(*s, device=DEV, generator=g) * scale).to(dtype)  # noqa: E731
    if Sq == Sk:
        x = mk(B, Sq, H + 2 * Hk, D)
        return x[:, :, :H], x[:, :, H:H + Hk], x[:, :, H + Hk:], mk(B, Sq, H, D)
    kv = mk(B, Sk, 2 * Hk, D)
    return mk(B, Sq, H, D), kv[:, :, :Hk], kv[:, :, Hk:], mk(B, Sq, H, D)


BF, FP = torch.bfloat16, torch.float16
# batch, queries, keys, heads, key heads, dim, causal, type
CASES = [
    (1, 1, 1, 1, 1, 64, True, BF), (1, 1, 1, 1, 1, 128, False, FP), (2, 128, 128, 2, 2, 64, True, BF),
    (1, 127, 127, 2, 1, 128, True, BF), (1, 129, 129, 2, 2, 128, True, FP), (2, 256, 256, 2, 2, 128, False, BF),
    (1, 257, 257, 4, 2, 64, True, FP), (2, 300, 300, 4, 1, 128, True, BF), (1, 513, 513, 2, 2, 80, True, BF),
    (1, 640, 640, 2, 2, 8, False, BF), (1, 385, 385, 3, 3, 40, True, FP), (1, 200, 200, 2, 1, 72, False, FP),
    (1, 1, 700, 4, 2, 128, True, BF), (1, 130, 900, 4, 4, 64, True, FP), (2, 700, 100, 2, 2, 128, True, BF),
    (1, 900, 1, 2, 1, 64, True, BF), (1, 65, 1000, 2, 2, 128, False, BF), (3, 1000, 1000, 2, 1, 128, True, BF),
    (1, 2048, 2048, 2, 2, 128, True, FP), (1, 2047, 1025, 2, 2, 64, False, BF), (1, 1500, 1500, 2, 2, 96, True, BF),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_matches_formula(case):
    from pccl.ops.attention import attention_forward, check_errors

    B, Sq, Sk, H, Hk, D, causal, dtype = case
    q, k, v, _ = _inputs(B, Sq, Sk, H, Hk, D, dtype, 1)
    out, lse = attention_forward(q, k, v, causal=causal)
    check_errors()
    _check_forward(out, lse, q, k, v, causal, D ** -0.5)


@pytest.mark.parametrize("case", CASES, ids=str)
def test_backward_matches_formula(case):
    from pccl.ops.attention import attention_backward, check_errors

    B, Sq, Sk, H, Hk, D, causal, dtype = case
    q, k, v, dout = _inputs(B, Sq, Sk, H, Hk, D, dtype, 2)
    out, lse = _given(q, k, v, causal, D ** -0.5)
    got = attention_backward(dout, q, k, v, out, lse, causal=causal)
    check_errors()
    for b in range(B):
        want = _oracle(q[b], k[b], v[b], _visible(Sq, Sk, causal), D ** -0.5, dout[b], out[b], lse[b])
        for x, (w, t), what in zip(got, want, ("dq", "dk", "dv")):
            _close(x[b], w, t, what)
