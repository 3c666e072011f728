"""Norms of queries and keys with the rotation of positions, against the formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float16


def _pairs(rot, interleaved):
    first = torch.arange(0, rot, 2, device=DEV) if interleaved else torch.arange(rot // 2, device=DEV)
    return first, first + (1 if interleaved else rot // 2)


def _turn(x, cos, sin, interleaved, back=False):
    """Rotated x, and the sum of the sizes of what was added up."""
    a, b = _pairs(2 * cos.shape[-1], interleaved)
    s = -sin if back else sin
    y, size = x.clone(), x.abs()
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * s, x[..., b] * cos + x[..., a] * s
    size[..., a] = (x[..., a] * cos).abs() + (x[..., b] * s).abs()
    size[..., b] = (x[..., b] * cos).abs() + (x[..., a] * s).abs()
    return y, size


def _oracle(x, w, cos, sin, interleaved, eps, dy=None):
    """Values and bounds.  u: half a step of the result's type, f: a step of 32 bits.  The norm's sum has D terms, its root
    halves their error; the hardware's reciprocal root and each product add a step."""
    D, f = x.shape[-1], 2.0 ** -23
    u, X, W = torch.finfo(x.dtype).eps / 2, x.double(), w.double()
    small = torch.finfo(x.dtype).tiny * u
    r = (X.square().mean(-1, keepdim=True) + eps).rsqrt()
    if dy is None:
        y, size = _turn(X * r * W, cos, sin, interleaved)
        return y, u * y.abs() + (D / 2 + 8) * f * size + small
    t, ts = _turn(dy.double(), cos, sin, interleaved, back=True)
    xh, g = X * r, t * W
    dot, dots = (g * xh).mean(-1, keepdim=True), (ts * (W * xh).abs()).mean(-1, keepdim=True)
    dx = r * (g - xh * dot)
    tol = u * dx.abs() + (2 * D + 16) * f * r * (ts * W.abs() + xh.abs() * dots) + small
    n = x.numel() // D
    dw = (t * xh).flatten(0, -2).sum(0)
    uw = torch.finfo(w.dtype).eps / 2
    return dx, tol, dw, uw * dw.abs() + (n + D) * f * (ts * xh.abs()).flatten(0, -2).sum(0) + torch.finfo(w.dtype).tiny * uw


def _close(got, want, tol, what):
    assert torch.isfinite(got).all(), what
    off = (got.double() - want).abs() - tol
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: {float(off.max()):.3e} over its bound"


# batch (0: none), rows, heads, key heads, dim, rotated, interleaved, type, type of the weights, positions
CASES = [
    (1, 1, 1, 1, 8, 8, False, BF, BF, None), (2, 128, 4, 4, 64, 64, False, BF, BF, None), (2, 37, 4, 2, 64, 48, True, FP, FP, None),
    (1, 300, 16, 4, 128, 128, False, BF, torch.float32, "int64"), (0, 129, 3, 1, 128, 64, False, FP, FP, "int32"),
    (1, 50, 9, 5, 72, 72, False, BF, BF, None), (2, 33, 2, 1, 40, 24, False, FP, torch.float32, None), (0, 1000, 8, 8, 96, 96, True, BF, BF, "int64"),
    (1, 65, 2, 2, 256, 256, False, BF, BF, None), (1, 64, 32, 32, 128, 128, False, BF, BF, None), (3, 700, 12, 3, 16, 8, True, BF, BF, "int32"),
    (1, 20, 2, 2, 200, 104, False, FP, FP, None), (0, 4000, 16, 16, 64, 64, False, BF, BF, None),
]


def _case(case, seed, scale=1.0):
    B, S, H, Hk, D, rot, inter, dt, wt, pos = case
    from pccl.ops.rotary import rotary_table

    g = torch.Generator(device=DEV).manual_seed(seed)
    lead = (S,) if B == 0 else (B, S)
    qkv = (torch.randn(*lead, H + 2 * Hk, D, device=DEV, generator=g) * scale).to(dt)
    q, k = qkv[..., :H, :], qkv[..., H:H + Hk, :]
    qw, kw = ((1 + 0.3 * torch.randn(D, device=DEV, generator=g)).to(wt) for _ in range(2))
    cos, sin = rotary_table(4096, rot, device=DEV)
    positions = None
    if pos:
        positions = torch.randint(0, 4096, lead, device=DEV, generator=g).to(getattr(torch, pos))
    at = torch.arange(S, device=DEV).expand(lead) if positions is None else positions.long()
    c, s = cos.double()[at].unsqueeze(-2), sin.double()[at].unsqueeze(-2)
    d = [torch.randn(*lead, n, D, device=DEV, generator=g).to(dt) for n in (H, Hk)]
    return q, k, qw, kw, cos, sin, positions, c, s, inter, d


@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_backward_match_formula(case):
    from pccl.ops.rotary import qk_norm_rope_backward, qk_norm_rope_forward

    q, k, qw, kw, cos, sin, positions, c, s, inter, (dq, dk) = _case(case, 1)
    qo, ko = qk_norm_rope_forward(q, k, qw, kw, cos, sin, positions, 1e-6, inter)
    got = qk_norm_rope_backward(dq, dk, q, k, qw, kw, cos, sin, positions, 1e-6, inter)
    for x, w, y, what in ((q, qw, qo, "q"), (k, kw, ko, "k")):
        _close(y, *_oracle(x, w, c, s, inter, 1e-6), what)
    for x, w, d, dx, dw, what in ((q, qw, dq, got[0], got[2], "q"), (k, kw, dk, got[1], got[3], "k")):
        wx, tx, ww, tw = _oracle(x, w, c, s, inter, 1e-6, d)
        _close(dx, wx, tx, "d" + what)
        _close(dw, ww, tw, f"d{what}_weight")
    again = qk_norm_rope_backward(dq, dk, q, k, qw, kw, cos, sin, positions, 1e-6, inter)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_gradient_against_differences():
    """The sum of y * dy, moved along a direction, against the gradient; the oracle's formula in 64 bits is differenced, the
    kernel's gradient compared with it within the bound of its own roundings."""
    from pccl.ops.rotary import qk_norm_rope_backward

    case = (1, 9, 2, 1, 64, 48, False, BF, torch.float32, None)
    q, k, qw, kw, cos, sin, positions, c, s, inter, (dq, dk) = _case(case, 2)
    gx, _gk, gw, _ = qk_norm_rope_backward(dq, dk, q, k, qw, kw, cos, sin, positions, 1e-6, inter)
    f = lambda x, w: (_turn(x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w, c, s, inter)[0] * dq.double()).sum()   # noqa: E731
    g = torch.Generator(device=DEV).manual_seed(3)
    for wrt, grad in (("x", gx), ("w", gw)):
        X, W = q.double(), qw.double()
        e = torch.randn((X if wrt == "x" else W).shape, dtype=torch.float64, device=DEV, generator=g)
        h = 1e-5
        up = f(X + h * e, W) - f(X - h * e, W) if wrt == "x" else f(X, W + h * e) - f(X, W - h * e)
        want, got = up / (2 * h), (grad.double() * e).sum()
        # each element of the gradient is off by half a step of its type at most, the differences by h^2 and 1e-16 / h
        u = torch.finfo(grad.dtype).eps / 2 + 300 * 2.0 ** -23
        assert abs(float(want - got)) <= float((grad.double().abs() * e.abs()).sum()) * u + 1e-6 * float(want.abs() + 1)


def test_in_place_and_into_a_packed_gradient():
    from pccl.ops.rotary import qk_norm_rope_backward, qk_norm_rope_forward

    case = (2, 77, 4, 2, 64, 64, False, BF, BF, None)
    q, k, qw, kw, cos, sin, positions, _c, _s, inter, (dq, dk) = _case(case, 4)
    want = qk_norm_rope_forward(q, k, qw, kw, cos, sin)
    grads = qk_norm_rope_backward(dq, dk, q, k, qw, kw, cos, sin)
    pack = torch.full((2, 77, 8, 64), 5.0, device=DEV, dtype=BF)
    pq, pk = pack[:, :, :4], pack[:, :, 4:6]
    pq.copy_(dq)
    pk.copy_(dk)
    gq, gk = torch.empty(64, device=DEV, dtype=BF), torch.empty(64, device=DEV, dtype=BF)
    qk_norm_rope_backward(pq, pk, q, k, qw, kw, cos, sin, dq_in=pq, dk_in=pk, dq_weight=gq, dk_weight=gk)
    for a, b in zip((pq, pk, gq, gk), grads):
        assert torch.equal(a, b)
    assert torch.all(pack[:, :, 6:] == 5.0)
    q1, k1 = qk_norm_rope_forward(q, k, qw, kw, cos, sin, q_out=q, k_out=k)
    assert q1.data_ptr() == q.data_ptr()
    assert torch.equal(q1, want[0]) and torch.equal(k1, want[1])


def test_rows_of_zeros_far_positions_and_unknown_ones():
    from pccl.ops.rotary import qk_norm_rope_backward, qk_norm_rope_forward, rotary_table

    x = torch.zeros(4, 2, 64, device=DEV, dtype=BF)
    x[2:] = 1.0
    w = torch.ones(64, device=DEV, dtype=BF)
    cos, sin = rotary_table(1 << 20, 64, device=DEV)
    p = torch.tensor([0, 7, (1 << 20) - 1, 1 << 20], device=DEV)
    y, z = qk_norm_rope_forward(x, x, w, w, cos, sin, positions=p)
    assert torch.all(y[:2] == 0) and torch.equal(y[:3], z[:3])
    assert torch.isnan(y[3]).all()
    ang = float((1 << 20) - 1) * 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    want = torch.cat((ang.cos() - ang.sin(), ang.cos() + ang.sin()))
    # the table is rounded to 32 bits, the result to 16: half a step of bf16 of values up to sqrt(2)
    assert float((y[2, 0].double().cpu() - want).abs().max()) <= 2.0 ** -8 * 1.4143 + 1e-6
    for bad in (-1, 1 << 40, -(1 << 62)):
        assert torch.isnan(qk_norm_rope_forward(x, x, w, w, cos, sin, positions=torch.full((4,), bad, device=DEV))[0]).all()
    d = qk_norm_rope_backward(x, x, x, x, w, w, cos, sin, positions=torch.zeros(4, device=DEV, dtype=torch.int32))
    assert all(torch.isfinite(t).all() for t in d)
    # a row that holds an infinity is NaN there and zero elsewhere; its neighbours are untouched
    x[2, 0, 5] = math.inf
    y = qk_norm_rope_forward(x, x, w, w, cos[:, :8].contiguous(), sin[:, :8].contiguous())[0]
    assert torch.isnan(y[2, 0, 5]) and torch.all(y[2, 0, 16:] == 0) and torch.isfinite(y[2, 1]).all()


def test_captured_call_and_empty_ones():
    from pccl.ops.rotary import qk_norm_rope_backward, qk_norm_rope_forward

    case = (1, 200, 4, 2, 64, 64, False, BF, BF, None)
    q, k, qw, kw, cos, sin, positions, _c, _s, inter, (dq, dk) = _case(case, 5)
    run = lambda: (*qk_norm_rope_forward(q, k, qw, kw, cos, sin), *qk_norm_rope_backward(dq, dk, q, k, qw, kw, cos, sin))   # noqa: E731
    want = run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    e = torch.zeros(0, 4, 64, device=DEV, dtype=BF)
    assert qk_norm_rope_forward(e, e, qw, kw, cos, sin)[0].numel() == 0
    assert torch.all(qk_norm_rope_backward(e, e, e, e, qw, kw, cos, sin)[2] == 0)


def test_refusals():
    from pccl.ops.rotary import qk_norm_rope_backward, qk_norm_rope_forward, rotary_table

    mk = lambda *s, dt=BF: torch.zeros(*s, device=DEV, dtype=dt)                  # noqa: E731
    q, w = mk(8, 2, 64), mk(64)
    cos, sin = rotary_table(16, 64, device=DEV)
    run = qk_norm_rope_forward
    bad = [
        lambda: run(q.float(), q.float(), w, w, cos, sin), lambda: run(q, q.half(), w, w, cos, sin), lambda: run(q.cpu(), q, w, w, cos, sin),
        lambda: run(q, mk(7, 2, 64), w, w, cos, sin), lambda: run(mk(8, 2, 60), mk(8, 2, 60), mk(60), mk(60), cos, sin),
        lambda: run(mk(8, 2, 264), mk(8, 2, 264), mk(264), mk(264), cos, sin), lambda: run(q, q, w[:63], w, cos, sin),
        lambda: run(q, q, w.half(), w.half(), cos, sin), lambda: run(q, q, w, w.float(), cos, sin), lambda: run(q, q, w, w, cos.double(), sin.double()),
        lambda: run(q, q, w, w, cos, sin[:, :28]), lambda: run(q, q, w, w, cos[:, :30].contiguous(), sin[:, :30].contiguous()),
        lambda: run(mk(8, 2, 32), mk(8, 2, 32), mk(32), mk(32), cos, sin), lambda: run(q, q, w, w, cos[:4], sin[:4]),
        lambda: run(q, q, w, w, cos, sin, positions=torch.zeros(7, device=DEV, dtype=torch.int64)),
        lambda: run(q, q, w, w, cos, sin, positions=torch.zeros(8, device=DEV)), lambda: run(q, q, w, w, cos, sin, eps=-1.0),
        lambda: run(q, q, w, w, cos, sin, eps=math.nan), lambda: run(mk(8, 2, 65)[..., 1:], q, w, w, cos, sin),
        lambda: run(mk(8, 64, 2).transpose(1, 2), q, w, w, cos, sin), lambda: run(q, q, w, w, cos, sin, q_out=mk(8, 2, 32)),
        lambda: run(q, q, w, w, cos, sin, q_out=mk(1, 2, 64).expand(8, 2, 64)),
        lambda: qk_norm_rope_backward(q, q, q, q, w, w, cos, sin, dq_weight=w, dk_weight=w),
        lambda: qk_norm_rope_backward(q, q, q, q, w, w, cos, sin, dq_weight=w.float()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was taken")


def test_outputs_between_the_inputs():
    from pccl.ops.rotary import qk_norm_rope_backward, qk_norm_rope_forward, rotary_table

    x = torch.randn(2, 20, 6, 64, device=DEV).to(BF)                              # q 0-1, k 2, room 3 to 5
    q, k = x[:, :, :2], x[:, :, 2:3]
    w = torch.ones(64, device=DEV, dtype=BF)
    tab = rotary_table(20, 64, device=DEV)
    want = qk_norm_rope_forward(q, k, w, w, *tab)
    for bad in (dict(q_out=x[:, :, 1:3]), dict(q_out=x[:, :, 2:4]), dict(k_out=x[:, :, 1:2]), dict(q_out=x[:, :, 3:5], k_out=x[:, :, 4:5])):
        with pytest.raises(RuntimeError, match="overlap"):
            qk_norm_rope_forward(q, k, w, w, *tab, **bad)
    with pytest.raises(RuntimeError, match="overlap"):
        qk_norm_rope_backward(*want, q, k, w, w, *tab, dq_in=x[:, :, 1:3])
    got = qk_norm_rope_forward(q, k, w, w, *tab, q_out=x[:, :, 3:5], k_out=x[:, :, 2:3])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_offsets_beyond_32_bits():
    from pccl.ops.rotary import qk_norm_rope_backward, qk_norm_rope_forward, rotary_table

    S, step = 600, 1 << 22
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GiB")
    far = torch.empty((S - 1) * step + 512, device=DEV, dtype=BF)
    cut = lambda at: torch.as_strided(far, (S, 1, 128), (step, 128, 1), at)                  # noqa: E731
    q, k, dq, dk = (torch.randn(S, 1, 128, device=DEV).to(BF) for _ in range(4))
    w, tab = torch.rand(128, device=DEV) + 0.5, rotary_table(S, 128, device=DEV)
    want = qk_norm_rope_forward(q, k, w, w, *tab)
    grad = qk_norm_rope_backward(dq, dk, q, k, w, w, *tab)
    for i, x in enumerate((q, k, dq, dk)):
        cut(128 * i).copy_(x)
    got = qk_norm_rope_backward(cut(256), cut(384), cut(0), cut(128), w, w, *tab, dq_in=cut(256), dk_in=cut(384))
    assert all(torch.equal(a, b) for a, b in zip(got, grad))
    got = qk_norm_rope_forward(cut(0), cut(128), w, w, *tab, q_out=cut(0), k_out=cut(128))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_outputs_apart_from_weights_tables_and_positions():
    """What every row reads must not be written by any: such calls are refused."""
    from pccl.ops.rotary import qk_norm_rope_backward, qk_norm_rope_forward, rotary_table

    S = 24
    pool = torch.zeros(1 << 16, device=DEV, dtype=torch.uint8)
    at = lambda i, n, dt: pool[i:i + n * dt.itemsize].view(dt)                              # noqa: E731
    q, k = (torch.randn(S, 2, 64, device=DEV).to(BF) for _ in range(2))
    w, (cos, sin) = torch.ones(64, device=DEV, dtype=BF), rotary_table(S, 64, device=DEV)
    out = at(0, S * 2 * 64, BF).view(S, 2, 64)                                              # the pool's first 6144 bytes
    pw, pc, pp = at(6016, 64, BF), at(3200, S * 32, torch.float32).view(S, 32), at(6080, S, torch.int64)
    pw.fill_(1.0)
    args = lambda **new: [{"qw": w, "kw": w, "cos": cos, "sin": sin, **new}[n] for n in ("qw", "kw", "cos", "sin")]  # noqa: E731
    for name in ("q", "k"):
        for new, pos in ((dict(qw=pw), None), (dict(kw=pw), None), (dict(cos=pc), None), (dict(sin=pc), None), ({}, pp)):
            with pytest.raises(RuntimeError, match="overlap the"):
                qk_norm_rope_forward(q, k, *args(**new), positions=pos, **{name + "_out": out})
            with pytest.raises(RuntimeError, match="overlap the"):
                qk_norm_rope_backward(q, k, q, k, *args(**new), positions=pos, **{f"d{name}_in": out})
        for weight in ("dq_weight", "dk_weight"):
            with pytest.raises(RuntimeError, match="overlap dq_in or dk_in"):
                qk_norm_rope_backward(q, k, q, k, *args(), **{f"d{name}_in": out, weight: pw})
    # beside the pool's first bytes all of that is taken, and a weight's gradient may take the weight's place
    far = at(8192, 64, BF)
    far.fill_(1.0)
    want = qk_norm_rope_backward(q, k, q, k, *args())
    got = qk_norm_rope_backward(q, k, q, k, *args(qw=far), dq_in=out, dq_weight=far)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
