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
    the end.  Everything else is 32-bit: a sum of D products is off by at most D + 2 roundings of the sum of their sizes.
    ``ftz``: the exponential and the tensor cores' sums flush what is below 2^-126 to zero, so a probability and each partial sum may
    be off by that much, whatever its size."""
    u, f, ftz = torch.finfo(q.dtype).eps / 2, 2.0 ** -23, 2.0 ** -126
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
        n = max(s.shape[-1], 1)
        tiny = (torch.finfo(q.dtype).tiny * u + ftz) * V.abs().sum(1, keepdim=True) + n * ftz
        return (o.transpose(0, 1), ((u + 2 * e_s + n * 2.0 ** -24) * a + u * o.abs() + tiny).transpose(0, 1) + torch.finfo(q.dtype).tiny * u,
                L, e_s + n * 2.0 ** -24 + f * L.nan_to_num(neginf=0.0).abs())
    L, dO, O = lse.double(), up(dout), up(out)
    p = torch.exp(s - L.nan_to_num(neginf=0.0)[..., None])
    dp, delta = dO @ V.transpose(1, 2), (dO * O).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_p = (D + 4) * f * (size.amax() if size.numel() else 0.0) + f * (L.nan_to_num(neginf=0.0).abs().max() if L.numel() else 0.0) + 2.0 ** -20
    e_dp = (D + 4) * f * (dO.abs() @ V.abs().transpose(1, 2) + (dO * O).abs().sum(-1, keepdim=True))
    small = torch.finfo(q.dtype).tiny * u
    e_ds = (u + 2 * e_p) * ds.abs() + p * e_dp + small + ftz * (1 + (dp - delta).abs())
    e_pr = (u + 2 * e_p) * p + small + ftz
    share = lambda x: x.unflatten(0, (k.shape[1], G)).sum(1)                      # noqa: E731
    n = G * max(s.shape[1], s.shape[2])
    dq, dk, dv = (ds @ K) * scale, share(ds.transpose(1, 2) @ Q) * scale, share(p.transpose(1, 2) @ dO)
    ads = e_ds + n * f * ds.abs()
    t_q = (ads @ K.abs()) * scale + u * dq.abs()
    t_k = share(ads.transpose(1, 2) @ Q.abs()) * scale + u * dk.abs()
    t_v = share((e_pr + n * f * p).transpose(1, 2) @ dO.abs()) + u * dv.abs()
    down = lambda x: x.transpose(0, 1)                                           # noqa: E731
    return [(down(x), down(t) + small + (n + 1) * ftz * max(scale, 1.0)) for x, t in ((dq, t_q), (dk, t_k), (dv, t_v))]


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
    (1, 1, 4000, 16, 2, 128, False, BF), (1, 256, 2500, 4, 1, 128, True, BF), (1, 800, 800, 16, 1, 64, True, FP), (2, 40, 3333, 3, 3, 80, True, FP),
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


# queries and keys of each packed sequence, rows behind the last one, heads, key heads, dim, causal
PACKED = [
    ([(1, 1)], 0, 1, 1, 64, True), ([(5, 5), (0, 0), (130, 130), (1, 1), (128, 128), (257, 257)], 7, 4, 2, 128, True),
    ([(300, 300), (0, 40), (40, 0), (77, 500), (129, 64)], 130, 2, 1, 64, True), ([(33, 33)] * 40, 3, 2, 2, 80, False),
    ([(0, 0), (0, 0)], 300, 2, 2, 128, True), ([(1 + i % 7, 1 + i % 7) for i in range(150)] + [(0, 0)] * 60 + [(400, 400)], 9, 2, 1, 64, True), ([(700, 300), (300, 700)], 1, 4, 4, 128, True), ([(7, 7), (2, 2)] * 37, 0, 3, 1, 40, True),
]


def _pack(lens, tail, H, Hk, D, dtype, seed, poison):
    """Packed inputs whose rows behind the last sequence are ``poison``."""
    q, _k, _v, dout = _inputs(1, sum(a for a, _ in lens) + tail, sum(b for _, b in lens) + tail + 1, H, Hk, D, dtype, seed)
    k, v = _k, _v
    q, k, v, dout = (x[0].clone() for x in (q, k, v, dout))
    cu = [torch.tensor([0] + [sum(x[i] for x in lens[:n + 1]) for n in range(len(lens))], dtype=torch.int32, device=DEV) for i in (0, 1)]
    for x, c in ((q, cu[0]), (dout, cu[0]), (k, cu[1]), (v, cu[1])):
        x[int(c[-1]):] = poison
    return q, k, v, dout, cu


@pytest.mark.parametrize("poison", [0.0, math.nan, math.inf])
@pytest.mark.parametrize("case", PACKED, ids=str)
def test_packed_sequences_stay_apart(case, poison):
    from pccl.ops.attention import attention_backward, attention_forward, check_errors

    lens, tail, H, Hk, D, causal = case
    q, k, v, dout, (cq, ck) = _pack(lens, tail, H, Hk, D, BF, 3, poison)
    out, lse = attention_forward(q, k, v, causal=causal, cu_seqlens_q=cq, cu_seqlens_k=ck)
    dq, dk, dv = attention_backward(dout, q, k, v, out, lse, causal=causal, cu_seqlens_q=cq, cu_seqlens_k=ck)
    check_errors()
    for i, (n, m) in enumerate(lens):
        a, b = int(cq[i]), int(ck[i])
        sq, sk, sv, sd = q[a:a + n], k[b:b + m], v[b:b + m], dout[a:a + n]
        see = _visible(n, m, causal)
        o, to, L, tl = _oracle(sq, sk, sv, see, D ** -0.5)
        _close(out[a:a + n], o, to, "out")
        got = lse[:, a:a + n]
        assert torch.equal(got == -math.inf, L == -math.inf)
        _close(got.masked_fill(L == -math.inf, 0), L.masked_fill(L == -math.inf, 0), tl, "lse")
        want = _oracle(sq, sk, sv, see, D ** -0.5, sd, out[a:a + n], got.contiguous())
        for x, (w, t), what in zip((dq[a:a + n], dk[b:b + m], dv[b:b + m]), want, ("dq", "dk", "dv")):
            _close(x, w, t, what)
    # what is allocated here holds zeros behind the last sequence
    for x, c in ((out, cq), (dq, cq), (dk, ck), (dv, ck)):
        assert torch.all(x[int(c[-1]):] == 0)
    assert torch.all(lse[:, int(cq[-1]):] == -math.inf)


def test_packed_outputs_of_the_caller_keep_the_rows_behind():
    from pccl.ops.attention import attention_backward, attention_forward

    q, k, v, dout, (cq, ck) = _pack([(50, 50), (90, 90)], 20, 2, 2, 64, BF, 4, 0.0)
    k, v = k[:160], v[:160]
    new = [torch.full_like(t, 7.0) for t in (q, q, k, v)]
    _out, lse = attention_forward(q, k, v, cu_seqlens_q=cq, out=new[0])
    attention_backward(dout, q, k, v, new[0], lse, cu_seqlens_q=cq, dq=new[1], dk=new[2], dv=new[3])
    ref, _ = attention_forward(q, k, v, cu_seqlens_q=cq)
    assert torch.equal(new[0][:140], ref[:140]) and torch.all(lse[:, 140:] == -math.inf)
    for x in new:
        assert torch.all(x[140:] == 7.0) and not torch.any(x[:140] == 7.0)


def test_neighbouring_sequences_may_hold_nan():
    from pccl.ops.attention import attention_backward, attention_forward

    lens = [(70, 70), (60, 60), (200, 200)]
    q, k, v, dout, (cq, ck) = _pack(lens, 0, 2, 1, 128, BF, 5, 0.0)
    k, v = k[:330], v[:330]
    good = attention_forward(q, k, v, cu_seqlens_q=cq)
    grads = attention_backward(dout, q, k, v, *good, cu_seqlens_q=cq)
    for x in (q, k, v, dout):
        x[70:130] = math.nan
    bad = attention_forward(q, k, v, cu_seqlens_q=cq)
    bgrads = attention_backward(dout, q, k, v, *bad, cu_seqlens_q=cq)
    for a, b in ((good[0], bad[0]), (good[1].t(), bad[1].t()), *zip(grads, bgrads)):
        assert torch.equal(a[:70], b[:70]) and torch.equal(a[130:], b[130:])
        assert torch.isnan(b[70:130]).all()


def test_large_scores_and_rising_maxima():
    """Scores of hundreds, rising along the keys, so that the running maximum is followed again and again."""
    from pccl.ops.attention import attention_backward, attention_forward, check_errors

    for dtype in (BF, FP):
        q, k, v, dout = _inputs(1, 600, 600, 2, 2, 64, dtype, 6)
        q, v = q * 4, v.contiguous()
        k = k * torch.linspace(0.1, 8, 600, device=DEV).view(1, -1, 1, 1).to(dtype)
        for causal in (True, False):
            out, lse = attention_forward(q, k, v, causal=causal)
            _check_forward(out, lse, q, k, v, causal, 64 ** -0.5)
            o, L = _given(q, k, v, causal, 64 ** -0.5)
            got = attention_backward(dout, q, k, v, o, L, causal=causal)
            check_errors()
            for x, (w, t), what in zip(got, _oracle(q[0], k[0], v[0], _visible(600, 600, causal), 64 ** -0.5, dout[0], o[0], L[0]),
                                       ("dq", "dk", "dv")):
                _close(x[0], w, t, what)


def test_other_scales_strides_and_outputs():
    from pccl.ops.attention import attention_backward, attention_forward

    g = torch.Generator(device=DEV).manual_seed(7)
    B, S, H, Hk, D = 2, 200, 4, 2, 64
    base = torch.randn(B, H, S, 72, device=DEV, generator=g).to(BF)              # heads before rows, gaps behind columns
    q = base[..., :D].transpose(1, 2)
    kv = torch.randn(S, B, 2 * Hk, D, device=DEV, generator=g).to(BF)            # rows before the batch
    k, v = kv[:, :, :Hk].transpose(0, 1), kv[:, :, Hk:].transpose(0, 1)
    out = torch.empty(B, S, 2 * H, D, device=DEV, dtype=BF)[:, :, ::2]
    got, lse = attention_forward(q, k, v, causal=True, scale=0.3, out=out)
    assert got.data_ptr() == out.data_ptr()
    _check_forward(out, lse, q, k, v, True, 0.3)
    dout = torch.randn(B, S, H, D, device=DEV, generator=g).to(BF)
    pack = torch.full((B, S, H + 2 * Hk, D), 9.0, device=DEV, dtype=BF)
    grads = (pack[:, :, :H], pack[:, :, H:H + Hk], pack[:, :, H + Hk:])
    attention_backward(dout, q, k, v, out, lse, causal=True, scale=0.3, dq=grads[0], dk=grads[1], dv=grads[2])
    plain = attention_backward(dout, q.contiguous(), k.contiguous(), v.contiguous(), out.contiguous(), lse, causal=True, scale=0.3)
    for a, b in zip(grads, plain):
        assert torch.equal(a, b)


def test_results_do_not_change_from_call_to_call():
    from pccl.ops.attention import attention_backward, attention_forward

    q, k, v, dout = _inputs(2, 500, 500, 8, 2, 64, BF, 8)
    first = attention_forward(q, k, v)
    grads = attention_backward(dout, q, k, v, *first)
    for _ in range(3):
        again = attention_forward(q, k, v)
        for a, b in zip((*first, *grads), (*again, *attention_backward(dout, q, k, v, *again))):
            assert torch.equal(a, b)


def test_captured_calls_and_other_streams():
    """Two captured graphs and eager calls on two streams at once: nothing is shared between them."""
    from pccl.ops.attention import attention_backward, attention_forward, check_errors

    data = [_inputs(1, 300, 300, 4, 4, 128, BF, s) for s in (20, 21, 22, 23)]
    run = lambda d: (lambda f: (*f, *attention_backward(d[3], *d[:3], *f)))(attention_forward(*d[:3]))      # noqa: E731
    want = [run(d) for d in data]
    graphs = []
    for d in data[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = run(d)
        graphs.append((g, res))
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(5):
        eager = []
        for s, (g, _r) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        for s, d in zip(streams[2:], data[2:]):
            with torch.cuda.stream(s):
                eager.append(run(d))
        torch.cuda.synchronize()
        for w, got in zip(want, [r for _g, r in graphs] + eager):
            for a, b in zip(w, got):
                assert torch.equal(a, b)
    check_errors()


def test_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from pccl.ops.attention import attention_backward, attention_forward, check_errors
from pccl.ops.rotary import qk_norm_rope_forward, rotary_table
from pccl.ops.optim import adamw_state, adamw_step
x = torch.randn(1, 300, 6, 64, device="cuda", dtype=torch.bfloat16)
w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
cos, sin = rotary_table(300, 64, device="cuda")
p = torch.ones(1000, device="cuda"); st = adamw_state([p], 8)
def run():
    q, k = qk_norm_rope_forward(x[:, :, :4], x[:, :, 4:5], w, w, cos, sin)
    out, lse = attention_forward(q, k, x[:, :, 5:6])
    g = attention_backward(out, q, k, x[:, :, 5:6], out, lse)
    return (q, k, out, lse, *g)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = run()
    adamw_step([p], [p * 0.5], st, step=1, lr=0.1)
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, run()))
assert float(p.max()) < 1.0
check_errors()
print("fine")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


def test_many_batch_entries_give_the_same_bits():
    from pccl.ops.attention import attention_backward

    q, k, v, dout = _inputs(1, 2049, 2049, 2, 2, 64, BF, 30)
    out, lse = _given(q, k, v, True, 0.125)
    want = _oracle(q[0], k[0], v[0], _visible(2049, 2049, True), 0.125, dout[0], out[0], lse[0])
    for n in (1, 150):
        got = attention_backward(*(t.expand(n, *t.shape[1:]).contiguous() for t in (dout, q, k, v, out)), lse.expand(n, 2, 2049).contiguous())
        for x, (w, t), what in zip(got, want, ("dq", "dk", "dv")):
            _close(x[0], w, t, what)
            assert torch.equal(x[0], x[n - 1])


@pytest.mark.parametrize("case", [(37, 37, 4, 2, 64, True, BF), (20, 150, 2, 2, 80, True, FP), (140, 30, 3, 1, 128, False, BF), (90, 33, 2, 1, 64, True, BF)], ids=str)
def test_gradient_against_differences(case):
    """The sum of out * dout, moved along a direction, against the gradients.  The formula in 64 bits is differenced; the kernel's
    gradient may be off by its roundings, the formula's by what the rounded output makes of the row sums."""
    from pccl.ops.attention import attention_backward

    Sq, Sk, H, Hk, D, causal, dtype = case
    q, k, v, dout = _inputs(1, Sq, Sk, H, Hk, D, dtype, 40)
    scale, see = D ** -0.5, _visible(Sq, Sk, causal)
    out, lse = _given(q, k, v, causal, scale)
    got = attention_backward(dout, q, k, v, out, lse, causal=causal)
    G, up = H // Hk, lambda x: x[0].double().transpose(0, 1)                     # noqa: E731

    def f(q, k, v):
        s = ((q @ k.repeat_interleave(G, 0).transpose(1, 2)) * scale).masked_fill(~see, -math.inf)
        return (s.softmax(-1).nan_to_num(0.0) @ v.repeat_interleave(G, 0))        # a query that sees nothing has an output of zero

    x, d = [up(q), up(k), up(v)], up(dout)
    exact = f(*x).transpose(0, 1)
    near = _oracle(q[0], k[0], v[0], see, scale, dout[0], out[0], lse[0])
    true = _oracle(q[0], k[0], v[0], see, scale, dout[0], exact, _oracle(q[0], k[0], v[0], see, scale)[2])
    gen = torch.Generator(device=DEV).manual_seed(41)
    for i, what in enumerate(("dq", "dk", "dv")):
        e = torch.randn(x[i].shape, dtype=torch.float64, device=DEV, generator=gen)
        h = 1e-5
        move = lambda t: [t * e + y if j == i else y for j, y in enumerate(x)]    # noqa: E731,B023
        want = float(((f(*move(h)) - f(*move(-h))) * d).sum() / (2 * h))
        along = lambda g: float((g.double().transpose(0, 1) * e).sum())           # noqa: E731,B023
        # central differences: h^2 times a third derivative, 2^-53 / h times the sum's size
        step = 1e-6 * (1 + float((f(*x).abs() * d.abs()).sum()))
        assert abs(along(true[i][0]) - want) <= step, f"{what}: the formula"
        off = float((near[i][1].transpose(0, 1) * e.abs()).sum()) + abs(along(near[i][0]) - along(true[i][0]))
        assert abs(along(got[i][0]) - want) <= off + step, what


def test_empty_calls():
    from pccl.ops.attention import attention_backward, attention_forward

    z = lambda *s: torch.zeros(*s, device=DEV, dtype=BF)                          # noqa: E731
    out, lse = attention_forward(z(1, 5, 2, 64) + 1, z(1, 0, 2, 64), z(1, 0, 2, 64))
    assert torch.all(out == 0) and torch.all(lse == -math.inf)
    dq, dk, dv = attention_backward(z(1, 5, 2, 64) + 1, z(1, 5, 2, 64) + 1, z(1, 0, 2, 64), z(1, 0, 2, 64), out, lse)
    assert torch.all(dq == 0) and dk.numel() == 0 and dv.numel() == 0
    out, lse = attention_forward(z(1, 0, 2, 64), z(1, 5, 2, 64), z(1, 5, 2, 64))
    assert out.numel() == 0 and lse.numel() == 0
    dq, dk, dv = attention_backward(z(1, 0, 2, 64), z(1, 0, 2, 64), z(1, 5, 2, 64), z(1, 5, 2, 64), out, lse)
    assert torch.all(dk == 0) and torch.all(dv == 0)
    assert attention_forward(z(0, 5, 2, 64), z(0, 5, 2, 64), z(0, 5, 2, 64))[0].shape == (0, 5, 2, 64)


def test_starts_out_of_order_or_range_touch_nothing_outside():
    """Broken starts give results that mean nothing, within the tensors: rows of guard around them keep their values."""
    from pccl.ops.attention import attention_backward, attention_forward, check_errors

    q, k, v, dout, _ = _pack([(300, 300)], 0, 2, 2, 64, BF, 9, 0.0)
    k, v = k[:300], v[:300]
    for starts in ([0, 1000], [-50, 200], [200, 100, 300], [300, 0], [2 ** 31 - 1, -2 ** 31, 5], [0, 300, 0, 300]):
        cu = torch.tensor(starts, dtype=torch.int32, device=DEV)
        guards = [torch.full((500, 2, 64), 3.0, device=DEV, dtype=BF) for _ in range(4)]
        outs = [g[100:400] for g in guards]
        _o, lse = attention_forward(q, k, v, cu_seqlens_q=cu, out=outs[0])
        attention_backward(dout, q, k, v, outs[0], lse.nan_to_num(0, 0, 0), cu_seqlens_q=cu, dq=outs[1], dk=outs[2], dv=outs[3])
        check_errors()
        for g in guards:
            assert torch.all(g[:100] == 3.0) and torch.all(g[400:] == 3.0)


def test_refusals():
    from pccl.ops.attention import attention_backward, attention_forward

    mk = lambda *s, dt=BF: torch.zeros(*s, device=DEV, dtype=dt)                  # noqa: E731
    q, k = mk(1, 8, 4, 64), mk(1, 8, 2, 64)
    cu = torch.tensor([0, 8], dtype=torch.int32, device=DEV)
    bad = [
        lambda: attention_forward(q.float(), k.float(), k.float()),
        lambda: attention_forward(q, k.half(), k),
        lambda: attention_forward(q, mk(1, 8, 3, 64), mk(1, 8, 3, 64)),            # 4 query heads on 3 key heads
        lambda: attention_forward(q, k, mk(1, 9, 2, 64)),
        lambda: attention_forward(mk(1, 8, 4, 136), mk(1, 8, 2, 136), mk(1, 8, 2, 136)),
        lambda: attention_forward(mk(1, 8, 4, 60), mk(1, 8, 2, 60), mk(1, 8, 2, 60)),
        lambda: attention_forward(q.cpu(), k, k),
        lambda: attention_forward(q, k.cpu(), k),
        lambda: attention_forward(q, mk(1, 8, 1, 64).expand(1, 8, 2, 64), k),      # expanded heads
        lambda: attention_forward(mk(1, 8, 4, 65)[..., 1:], k, k),                 # strides and start off the boundary
        lambda: attention_forward(mk(1, 8, 64, 4).transpose(2, 3), k, k),          # columns not contiguous
        lambda: attention_forward(q, k, k, scale=0.0),
        lambda: attention_forward(q, k, k, scale=-1.0),
        lambda: attention_forward(q, k, k, scale=math.nan),
        lambda: attention_forward(q, k, k, cu_seqlens_q=cu),                       # packed wants [rows, heads, dim]
        lambda: attention_forward(q[0], k[0], k[0]),                               # not packed wants a batch
        lambda: attention_forward(q[0], k[0], k[0], cu_seqlens_q=cu.long()),
        lambda: attention_forward(q[0], k[0], k[0], cu_seqlens_q=cu.cpu()),
        lambda: attention_forward(q[0], k[0], k[0], cu_seqlens_q=cu[:1]),
        lambda: attention_forward(q[0], mk(9, 2, 64), mk(9, 2, 64), cu_seqlens_q=cu),
        lambda: attention_forward(q[0], k[0], k[0], cu_seqlens_k=cu),
        lambda: attention_forward(q[0], k[0], k[0], cu_seqlens_q=cu, cu_seqlens_k=torch.zeros(3, dtype=torch.int32, device=DEV)),
        lambda: attention_forward(q, k, k, out=mk(1, 8, 4, 32)),
        lambda: attention_forward(q, k, k, out=q),
        lambda: attention_forward(q, k, k, out=mk(1, 8, 1, 64).expand(1, 8, 4, 64)),
    ]
    lse = torch.zeros(1, 4, 8, device=DEV)
    bad += [
        lambda: attention_backward(q, q, k, k, q, lse[:, :, :7]),
        lambda: attention_backward(q, q, k, k, q, lse.double()),
        lambda: attention_backward(q[:, :, :2], q, k, k, q, lse),
        lambda: attention_backward(q, q, k, k, q, lse, dq=torch.empty_like(q)),
        lambda: (lambda x: attention_backward(q, q, k, k, q, lse, dq=torch.empty_like(q), dk=x, dv=x))(torch.empty_like(k)),
        lambda: (lambda x: attention_backward(x, q, k, k, q, lse, dq=x, dk=torch.empty_like(k), dv=torch.empty_like(k)))(torch.empty_like(q)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was taken")


def test_outputs_between_the_inputs():
    """Views into one packed tensor: refused where an output touches an input, taken where it lies beside them."""
    from pccl.ops.attention import attention_backward, attention_forward

    x = torch.randn(2, 40, 8, 64, device=DEV).to(BF)                              # q 0-3, k 4, v 5, room 6 and 7
    q, k, v = x[:, :, :4], x[:, :, 4:5], x[:, :, 5:6]
    kept = x.clone()
    for h in (0, 1, 2, 3, 4):
        with pytest.raises(RuntimeError, match="overlap"):
            attention_forward(q, k, v, out=x[:, :, h:h + 4])
    with pytest.raises(RuntimeError, match="overlap"):
        attention_forward(q, k, v, out=x.view(-1)[:2 * 40 * 256].view(2, 40, 4, 64))
    with pytest.raises(RuntimeError, match="overlap"):
        attention_forward(q[:1], k[:1], v[:1], out=torch.as_strided(torch.zeros(1 << 14, device=DEV, dtype=BF), (1, 40, 4, 64), (0, 256, 8, 1)))
    out, lse = attention_forward(x[:, :, :2], k, v)
    o = x[:, :, 6:8]
    assert torch.equal(attention_forward(x[:, :, :2], k, v, out=o)[0], out) and torch.equal(x[:, :, :6], kept[:, :, :6])
    g = torch.zeros(2, 40, 4, 64, device=DEV, dtype=BF)
    want = attention_backward(out, x[:, :, :2], k, v, out, lse)
    got = attention_backward(out, x[:, :, :2], k, v, out, lse, dq=g[:, :, :2], dk=g[:, :, 2:3], dv=g[:, :, 3:])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="overlap"):
        attention_backward(out, x[:, :, :2], k, v, out, lse, dq=g[:, :, :2], dk=g[:, :, 1:2], dv=g[:, :, 3:])


def test_offsets_beyond_32_bits():
    """Rows four million elements apart: the last one's offset is above 2^31 elements.  The same bits as from contiguous tensors."""
    from pccl.ops.attention import attention_backward, attention_forward

    S, step = 600, 1 << 22
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB")
    far, grads = (torch.empty((S - 1) * step + 512, device=DEV, dtype=BF) for _ in range(2))
    cut = lambda x, at: torch.as_strided(x, (1, S, 1, 128), (S * step, step, 128, 1), at)    # noqa: E731
    q, k, v, dout = _inputs(1, S, S, 1, 1, 128, BF, 50)
    views = [cut(far, 128 * i) for i in range(4)]
    for x, y in zip(views, (q, k, v, dout)):
        x.copy_(y)
    out, lse = attention_forward(q, k, v)
    got, got_lse = attention_forward(*views[:3], out=cut(grads, 384))
    assert torch.equal(got, out) and torch.equal(got_lse, lse)
    want = attention_backward(dout, q, k, v, out, lse)
    near = attention_backward(views[3], *views[:3], got, lse, dq=cut(grads, 0), dk=cut(grads, 128), dv=cut(grads, 256))
    assert all(torch.equal(a, b) for a, b in zip(near, want))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("shape", [(1, 300, 2, 64), (1, 700, 16, 128)], ids=str)
def test_row_sums_of_the_call_in_front_are_not_read(shape, packed):
    """The kernel for dq begins before the one for dk and dv has ended.  Calls back to back, whose inputs, row sums and tile lists
    take the same memory and differ from call to call, give the bits of calls that stand alone."""
    from pccl.ops.attention import attention_backward, attention_forward, check_errors

    B, S, H, D = shape
    sets = []
    for seed in range(6):
        x = list(_inputs(B, S, S, H, H, D, BF, 60 + seed, 1.0 + seed))
        cu = None
        if packed:
            x = [t[0] for t in x]
            cu = torch.tensor([0, 30 * (seed + 1), 30 * (seed + 1), S - seed], dtype=torch.int32, device=DEV)
        out, lse = attention_forward(*x[:3], cu_seqlens_q=cu)
        sets.append((x[3].contiguous(), *(t.contiguous() for t in x[:3]), out, lse, cu))
    alone = []
    for s in sets:
        torch.cuda.synchronize()
        alone.append([t.clone() for t in attention_backward(*s[:6], cu_seqlens_q=s[6])])
        torch.cuda.synchronize()
    here = [None if t is None else t.clone() for t in sets[0]]
    for _ in range(20):
        got = []
        for s in sets:
            for a, b in zip(here, s):
                if a is not None:
                    a.copy_(b)
            got.append([t.clone() for t in attention_backward(*here[:6], cu_seqlens_q=here[6])])
        for a, b in zip(alone, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    check_errors()


def _kernel_nodes(run):
    """How many kernels a call launches: the kernel nodes of its captured graph."""
    from cuda.bindings import runtime as rt

    run()
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        run()
    raw = rt.cudaGraph_t(init_value=g.raw_cuda_graph())
    err, _nodes, n = rt.cudaGraphGetNodes(raw)
    assert err == rt.cudaError_t.cudaSuccess
    err, nodes, n = rt.cudaGraphGetNodes(raw, n)
    assert err == rt.cudaError_t.cudaSuccess
    kinds = [rt.cudaGraphNodeGetType(x) for x in nodes[:n]]
    assert all(e == rt.cudaError_t.cudaSuccess for e, _k in kinds)
    return sum(k == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for _e, k in kinds)


@pytest.mark.parametrize("shape,docs", [((1, 128, 2, 64), None), ((1, 1024, 4, 64), None), ((1, 2048, 2, 64), None), ((2, 160, 4, 64), [0, 1, 100, 320])],
                         ids=str)
def test_launches_are_counted(shape, docs):
    """What is reported as launched is what a captured call holds: whole, split (with sums or a join behind), packed."""
    from pccl import build_kernels
    from pccl.models import gpt
    from pccl.ops.attention import attention_backward, attention_forward

    C, (B, S, H, D) = build_kernels.load(), shape
    q, k, v, dout = _inputs(B, S, S, H, H, D, BF, 80)
    cu = None
    if docs:
        cu = torch.tensor(docs, dtype=torch.int32, device=DEV)
        q, k, v, dout = (t.reshape(B * S, H, D) for t in (q, k, v, dout))
    out, lse = attention_forward(q, k, v, cu_seqlens_q=cu)
    counts = []
    for run in (lambda: attention_forward(q, k, v, cu_seqlens_q=cu), lambda: attention_backward(dout, q, k, v, out, lse, cu_seqlens_q=cu)):
        before = C.attention_kernels_launched()
        run()
        counts.append(C.attention_kernels_launched() - before)
        assert counts[-1] == _kernel_nodes(run)
    assert tuple(counts) == {128: (1, 3), 1024: (2, 3), 2048: (2, 6), 160: (2, 4)}[S]
    # the same through a block: one more for the column sums of the projection's gradient, and with rotation one forward and two backward
    keep = gpt.native_attention
    try:
        gpt.native_attention = True
        for rope in (False, True):
            if docs and not rope:
                continue
            cfg = gpt.GPTConfig(1, H * D, H, 64, vocab=8, seq_len=S, qk_norm_rope=rope)
            pos = gpt.positions_of(cfg, B, S, DEV, None, cu) if rope else None
            w = {n: torch.ones(D, device=DEV, dtype=BF) for n in ("qn_w", "kn_w")}
            grads = {**{n: torch.empty_like(t) for n, t in w.items()}, "qkv_b": torch.empty(3 * H * D, device=DEV, dtype=BF)}
            qkv = torch.randn(B * S, 3 * H * D, device=DEV).to(BF)
            before = gpt.native_launches
            a, saved = gpt._attention(qkv, w, cfg, B, pos)
            assert gpt.native_launches - before == counts[0] + rope
            before = gpt.native_launches
            gpt._attention_backward(torch.randn_like(a), saved, w, grads, cfg, B, pos)
            assert gpt.native_launches - before == counts[1] + 2 * rope + 1
    finally:
        gpt.native_attention = keep


def test_outputs_apart_from_the_starts():
    """Every block reads the starts, so none may write them: such calls are refused."""
    from pccl.ops.attention import attention_backward, attention_forward

    q, k, v, dout = (t[0] for t in _inputs(1, 40, 40, 2, 2, 64, BF, 90))
    pool = torch.zeros(1 << 15, device=DEV, dtype=torch.uint8)
    new = pool[:40 * 2 * 64 * 2].view(BF).view(40, 2, 64)
    starts = pool[5120:5128].view(torch.int32)
    starts.copy_(torch.tensor([0, 40]))
    apart = starts.clone()
    out, lse = attention_forward(q, k, v, cu_seqlens_q=apart)
    for cu in (dict(cu_seqlens_q=starts), dict(cu_seqlens_q=apart, cu_seqlens_k=starts)):
        with pytest.raises(RuntimeError, match="overlap the starts"):
            attention_forward(q, k, v, out=new, **cu)
        for which in range(3):
            grads = [torch.empty_like(t) for t in (q, k, v)]
            grads[which] = new
            with pytest.raises(RuntimeError, match="overlap the starts"):
                attention_backward(dout, q, k, v, out, lse, dq=grads[0], dk=grads[1], dv=grads[2], **cu)
    assert torch.equal(attention_forward(q, k, v, cu_seqlens_q=apart, out=new)[0], out)


@pytest.mark.parametrize("poison", [0.0, math.nan])
@pytest.mark.parametrize("case", PACKED, ids=str)
def test_packed_sequences_in_fp16(case, poison, monkeypatch):
    import sys

    monkeypatch.setattr(sys.modules[__name__], "BF", FP)
    test_packed_sequences_stay_apart(case, poison)


@pytest.mark.parametrize("case", [([(2048, 2048)], 0, 16, 1, 64, True), ([(3, 2500), (129, 2200)], 5, 4, 1, 80, True), ([(1, 4000)], 0, 4, 2, 128, False)], ids=str)
def test_packed_calls_of_shapes_that_are_split_when_they_are_not(case):
    test_packed_sequences_stay_apart(case, 0.0)


@pytest.mark.parametrize("case", [(1, 1500, 1100, 4, 1, 64, True, BF), (1, 2500, 2100, 2, 1, 64, True, FP), (2, 1300, 1024, 2, 2, 128, True, BF)], ids=str)
def test_more_queries_than_keys_where_the_axes_are_split(case):
    """The first queries see nothing, in any part."""
    test_forward_matches_formula(case)
    test_backward_matches_formula(case)


def test_captured_packed_call_follows_the_starts():
    """The starts are read on the device: a replay takes those that are there then."""
    from pccl.ops.attention import attention_backward, attention_forward, check_errors

    q, k, v, dout = (t[0].contiguous() for t in _inputs(1, 500, 500, 4, 2, 64, BF, 70))
    cu = torch.tensor([0, 100, 300, 500], dtype=torch.int32, device=DEV)

    def run():
        out, lse = attention_forward(q, k, v, cu_seqlens_q=cu)
        return out, lse, *attention_backward(dout, q, k, v, out, lse, cu_seqlens_q=cu)

    run()
    graphs = []
    for _ in range(2):                  # two graphs that are replayed in turn share nothing
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = run()
        graphs.append((g, got))
    for starts in ([0, 100, 300, 500], [0, 1, 1, 490], [0, 500, 500, 500], [0, 0, 0, 0], [0, 257, 258, 499]):
        cu.copy_(torch.tensor(starts))
        want = run()
        for g, got in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, got in graphs:
            assert all(torch.equal(a, b) for a, b in zip(want, got)), starts
    check_errors()
