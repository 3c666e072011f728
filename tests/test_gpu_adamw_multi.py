"""AdamW over lists of tensors, states in 32 and in 8 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8)


def _lists(sizes, pt, gt, seed, shift=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda n, s: (torch.randn(n + shift, device=DEV, generator=g) * s)[shift:]          # noqa: E731
    masters = [mk(n, 0.5) for n in sizes]
    grads = [torch.cat((torch.zeros(shift, device=DEV, dtype=gt), mk(n, 0.1).to(gt)))[shift:] for n in sizes]
    if pt == F32:
        return masters, grads, None
    params = [torch.cat((torch.zeros(shift, device=DEV, dtype=pt), m.to(pt)))[shift:] for m in masters]
    return params, grads, masters


def _formula(p, g, m, v, decay, step, clip, lr, beta1, beta2, eps):
    """The step in 64 bits."""
    g = g.double() * clip
    m, v = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
    upd = lr * (m / (1 - beta1 ** step)) / ((v / (1 - beta2 ** step)).sqrt() + eps)
    return p - lr * decay * p - upd, m, v, upd


def _cut(flat, sizes):
    at, out = 0, []
    for n in sizes:
        out.append(flat[at:at + n])
        at += (n + 255) // 256 * 256
    return out


SIZES = [[1], [256], [255, 257], [1, 2, 3, 100003, 5, 4096, 31], [7] * 900, [2048 * 300]]


@pytest.mark.parametrize("types", [(BF, BF), (FP, FP), (F32, F32), (BF, F32), (F32, BF), (FP, F32)], ids=str)
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("shift", [0, 1])
def test_states_in_32_bits_match_formula(types, sizes, shift):
    from pccl.ops.optim import adamw_state, adamw_step

    if len(sizes) > 100 and (types != (BF, BF) or shift):
        pytest.skip("the long list once")
    params, grads, masters = _lists(sizes, *types, 1, shift)
    decay = [0.1 * (i % 3) for i in range(len(sizes))]
    state = adamw_state(params, 32)
    norm = sum((g.double() ** 2).sum() for g in grads).float().view(1)
    clip = min(1.0, 0.7 / (math.sqrt(float(norm)) * 0.5 + 1e-6)) * 0.5
    f = 2.0 ** -24
    for step in (1, 2, 3):
        weights = masters if masters is not None else params
        before = [w.double() for w in weights]
        old = [[t.double().clone() for t in _cut(x, sizes)] for x in (state.exp_avg, state.exp_avg_sq)]
        adamw_step(params, grads, state, step=step, weight_decay=decay, masters=masters, grad_scale=0.5, max_grad_norm=0.7,
                   total_sq_norm=norm, **HYPER)
        for i, (p, w, g, b) in enumerate(zip(params, weights, grads, before)):
            want, m, v, upd = _formula(b, g, old[0][i], old[1][i], decay[i], step, clip, **HYPER)
            # a gradient is off by the roundings of the clip factor (its root, sum, quotient, product) and its own: six
            gm, gv = _cut(state.exp_avg, sizes)[i].double(), _cut(state.exp_avg_sq, sizes)[i].double()
            tiny = 1e-37
            assert torch.all((gm - m).abs() <= 10 * f * (old[0][i].abs() + (g.double() * clip).abs()) + tiny)
            assert torch.all((gv - v).abs() <= 16 * f * v + tiny)
            # the moments' errors move the update by as much of it, where they do not cancel
            slack = 0.01 * 10 * f * (old[0][i].abs() + (g.double() * clip).abs()) / (1 - 0.9 ** step) / ((v / (1 - 0.95 ** step)).sqrt() + 1e-8)
            assert torch.all((w.double() - want).abs() <= 4 * f * b.abs() + 24 * f * upd.abs() + slack + tiny)
            if w is not p:
                assert torch.equal(p, w.to(p.dtype))


def test_moments_are_rounded_product_by_product():
    """b1 m and (1 - b1) g are rounded to 32 bits before they are added, so that the codes of 8-bit states hang on the formula alone."""
    import numpy as np

    from pccl.ops.optim import adamw_state, adamw_step

    f = lambda x: float(np.float32(x))                                            # noqa: E731
    g = torch.Generator(device=DEV).manual_seed(8)
    n = 256 * 300
    for bits in (32, 8):
        grad = torch.randn(n, device=DEV, generator=g) * 1e-3
        state = adamw_state([grad], bits)
        for step in (1, 2):
            m, v = (x.clone() for x in state.dequantize())
            full = adamw_state([grad], 32)
            full.exp_avg.copy_(m)
            full.exp_avg_sq.copy_(v)
            p = torch.zeros(n, device=DEV)
            adamw_step([p], [grad], full, step=step, **HYPER)
            assert torch.equal(full.exp_avg, m * f(0.9) + grad * f(1 - 0.9))
            assert torch.equal(full.exp_avg_sq, v * f(0.95) + (grad * grad) * f(1 - 0.95))
            adamw_step([p], [grad], state, step=step, **HYPER)
            if bits == 8:
                assert torch.equal(state.exp_avg_scale, full.exp_avg.abs().view(-1, 256).amax(1))
                assert torch.equal(state.exp_avg_sq_scale, full.exp_avg_sq.view(-1, 256).amax(1))
            else:
                assert torch.equal(state.exp_avg, full.exp_avg)


@pytest.mark.parametrize("types", [(BF, BF), (F32, F32), (FP, F32)], ids=str)
@pytest.mark.parametrize("shift", [0, 1])
def test_8_bit_codes_are_the_neighbours_of_the_value(types, shift):
    from pccl.ops.optim import AdamWState, adamw_state, adamw_step

    sizes = [1, 300, 5000, 256, 70001]
    params, grads, masters = _lists(sizes, *types, 2, shift)
    state = adamw_state(params, 8)
    full = adamw_state(params, 32)
    for step in (1, 2, 3, 4):
        m0, v0 = state.dequantize()
        full.exp_avg.copy_(m0)
        full.exp_avg_sq.copy_(v0)
        copies = [[t.clone() for t in x] if x is not None else None for x in (params, masters)]
        adamw_step(copies[0], grads, full, step=step, masters=copies[1], **HYPER)
        adamw_step(params, grads, state, step=step, masters=masters, seed=3, **HYPER)
        # the parameters are stepped from the 32-bit moments: the same bits
        for a, b in zip(params, copies[0]):
            assert torch.equal(a, b)
        for x, code, scale, top, power in ((full.exp_avg, state.exp_avg, state.exp_avg_scale, 127, 2),
                                           (full.exp_avg_sq, state.exp_avg_sq, state.exp_avg_sq_scale, 255, 4)):
            x, c = x.view(-1, 256).double(), code.view(-1, 256).double()
            assert torch.equal(scale, x.abs().amax(1).float())
            y = x.abs() / scale.double()[:, None].clamp(min=1e-300) * top ** power
            # a code is the one below or above; 1e-5: the 32-bit roundings of y
            assert torch.all(c.abs() ** power <= ((y * (1 + 1e-5)) ** (1 / power) + 1) ** power)
            assert torch.all((c.abs() + 1) ** power >= y * (1 - 1e-5))
            assert torch.all((c == 0) | (torch.sign(c) == torch.sign(x)))
            if power == 4:
                assert torch.all((c > 0) == (x > 0))
        assert isinstance(state, AdamWState) and state.bits == 8


def test_8_bit_rounding_keeps_the_mean_and_the_seed():
    """Over many steps of the noise the mean of a rounded value is the value."""
    from pccl.ops.optim import adamw_state, adamw_step

    n, reps = 256, 600
    g = torch.Generator(device=DEV).manual_seed(5)
    p, grad = torch.zeros(n, device=DEV), torch.randn(n, device=DEV, generator=g)
    grad[0] = 8.0                       # the block's largest
    sums, first = None, None
    for seed in range(reps):
        state = adamw_state([p], 8)
        adamw_step([p.clone()], [grad], state, step=1, seed=seed, **HYPER)
        now = torch.stack(state.dequantize()).double()
        if seed == 0:
            first = now
            again = adamw_state([p], 8)
            adamw_step([p.clone()], [grad], again, step=1, seed=0, **HYPER)
            assert torch.equal(torch.stack(again.dequantize()).double(), first)
        sums = now if sums is None else sums + now
    assert not torch.equal(now, first)
    want = torch.stack(((1 - 0.9) * grad.double(), (1 - 0.95) * grad.double() ** 2))
    # a value lies between neighbours d apart: its deviation is at most d / 2, the mean's d / 2 / sqrt(reps); six of those
    for i, (top, power) in enumerate(((127, 2), (255, 4))):
        A = want[i].abs().max()
        c = (want[i].abs() / A * top ** power) ** (1 / power)
        d = ((c.floor() + 1) ** power - c.floor() ** power) / top ** power * A
        least = A / top ** power if power == 4 else 0.0          # a v below code 1 is held as code 1
        off = (sums[i] / reps - want[i]).abs()
        assert torch.all((off <= 3 * d / math.sqrt(reps) + 1e-6 * A) | (want[i].abs() < least))


def test_zeros_tiny_and_broken_blocks():
    from pccl.ops.optim import adamw_state, adamw_step

    n = 4 * 256
    p = torch.ones(n, device=DEV)
    grad = torch.zeros(n, device=DEV)
    grad[256:512] = 1e-25                # squares below 2^-80: held as zeros; first moments too
    grad[512 + 7] = math.nan
    grad[768:] = 1.0
    state = adamw_state([p], 8)
    adamw_step([p], [grad], state, step=1, weight_decay=0.0, **HYPER)
    m, v = (x.view(4, 256) for x in state.dequantize())
    assert torch.all(m[0] == 0) and torch.all(v[0] == 0) and torch.all(v[1] == 0) and torch.all(m[1] == 0)
    assert torch.isnan(m[2]).all() and torch.isnan(v[2]).all()
    assert torch.all(m[3] > 0) and torch.all(v[3] > 0)
    assert torch.all(p[:256] == 1) and torch.isnan(p[512 + 7]) and int(torch.isnan(p).sum()) == 1
    assert torch.all((p[768:] - 0.99).abs() < 1e-6)
    # many steps without a gradient: moments fade to zero and the parameter stays where it is
    q = torch.ones(300, device=DEV)
    st = adamw_state([q], 8)
    adamw_step([q], [torch.full((300,), 1e-3, device=DEV)], st, step=1, weight_decay=0.0, **HYPER)
    zero = torch.zeros(300, device=DEV)
    for step in range(2, 2200):
        adamw_step([q], [zero], st, step=step, weight_decay=0.0, **HYPER)
    assert torch.isfinite(q).all()
    last = q.clone()
    adamw_step([q], [zero], st, step=2200, weight_decay=0.0, **HYPER)
    assert torch.equal(q, last) and all(torch.all(x == 0) for x in st.dequantize())


def test_nan_norm_is_not_hidden_and_large_norm_clips():
    from pccl.ops.optim import adamw_state, adamw_step

    for norm, bad in ((math.nan, True), (1e30, False)):
        p = torch.ones(300, device=DEV)
        st = adamw_state([p], 32)
        adamw_step([p], [torch.ones(300, device=DEV)], st, step=1, max_grad_norm=1.0, total_sq_norm=torch.full((1,), norm, device=DEV), **HYPER)
        assert bool(torch.isnan(p).all()) == bad and bool(torch.isfinite(p).all()) != bad


def test_more_tensors_than_one_launch_takes_and_capture():
    from pccl.ops.optim import adamw_state, adamw_step

    sizes = [300 + i for i in range(1700)]
    for bits in (8, 32):
        runs = []
        for part in ("list", "flat", "graph"):
            params, grads, masters = _lists(sizes, BF, BF, 6)
            state = adamw_state(params, bits)
            if part == "list":
                adamw_step(params, grads, state, step=1, masters=masters, **HYPER)
            elif part == "graph":
                keep = [t.clone() for t in (state.exp_avg, state.exp_avg_sq)]
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    adamw_step(params, grads, state, step=1, masters=masters, **HYPER)
                assert torch.equal(state.exp_avg, keep[0]) and torch.equal(state.exp_avg_sq, keep[1])    # captured, not run
                g.replay()
            else:
                # every tensor by itself: its own state, the same blocks
                for i, (p, gr, w) in enumerate(zip(params, grads, masters)):
                    if bits == 32 and i % 100 == 0:
                        one = adamw_state([p], bits)
                        adamw_step([p], [gr], one, step=1, masters=[w], **HYPER)
                        assert torch.equal(one.exp_avg[:sizes[i]], _cut(runs[0][1].exp_avg, sizes)[i])
                        assert torch.equal(p, runs[0][0][i])
                continue
            torch.cuda.synchronize()
            runs.append((params, state))
        assert all(torch.equal(a, b) for a, b in zip(runs[0][0], runs[1][0]))
        assert torch.equal(runs[0][1].exp_avg, runs[1][1].exp_avg) and torch.equal(runs[0][1].exp_avg_sq, runs[1][1].exp_avg_sq)


def test_refusals():
    from pccl.ops.optim import AdamWState, adamw_state, adamw_step

    mk = lambda n=300, dt=F32: torch.zeros(n, device=DEV, dtype=dt)              # noqa: E731
    p, g = mk(), mk()
    st = adamw_state([p], 32)
    st8 = adamw_state([p], 8)
    both = mk(600)
    go = lambda params, grads, state=st, **kw: adamw_step(params, grads, state, **{"step": 1, **HYPER, **kw})     # noqa: E731
    bad = [
        lambda: go([p], []), lambda: go([p], [mk(299)]), lambda: go([p], [g], step=0), lambda: go([p], [g], beta1=1.0),
        lambda: go([p], [g], eps=-1.0), lambda: go([p], [g], lr=math.inf), lambda: go([p.cpu()], [g]), lambda: go([p], [g.cpu()]),
        lambda: go([p], [g], masters=[mk()]), lambda: go([p.to(BF)], [g]), lambda: go([p.to(BF)], [g], masters=[mk(dt=BF)]),
        lambda: go([p.double()], [g]), lambda: go([p], [g], weight_decay=[0.1, 0.2]), lambda: go([p, mk(dt=BF)], [g, g]),
        lambda: go([mk(900)], [mk(900)]),                                          # states of another list
        lambda: go([p, p], [g, mk()], state=adamw_state([p, p], 32)),              # the same tensor twice
        lambda: go([both[:300], both[299:599]], [g, mk()], state=adamw_state([p, p], 32)),
        lambda: go([p], [p]), lambda: go([p], [g], max_grad_norm=1.0),
        lambda: go([p], [g], max_grad_norm=1.0, total_sq_norm=torch.zeros(1)),
        lambda: go([torch.zeros(20, 15, device=DEV).t()], [g]),
        lambda: go([p], [g], state=AdamWState(st8.exp_avg, st8.exp_avg_sq)),
        lambda: go([p], [g], state=AdamWState(st8.exp_avg, st8.exp_avg_sq, st8.exp_avg_scale)),
        lambda: go([p], [g], state=AdamWState(st8.exp_avg, st8.exp_avg_sq, st8.exp_avg_scale[:1], st8.exp_avg_sq_scale)),
        lambda: go([p], [g], state=AdamWState(st.exp_avg, st.exp_avg_sq, st8.exp_avg_scale, st8.exp_avg_sq_scale)),
        lambda: go([p], [g], state=AdamWState(st.exp_avg, st.exp_avg)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(ValueError):
        adamw_state([p], 16)
    adamw_step([], [], st, step=1, **HYPER)
    adamw_step([mk(0), p], [mk(0), g], st, step=1, **HYPER)                        # an empty tensor has no part in the state


@pytest.mark.parametrize("bits", [8, 32])
def test_more_than_2_31_elements(bits):
    """The end of a long tensor, and the tensor behind it, change as they do alone (the first step reads no codes)."""
    from pccl.ops.optim import adamw_state, adamw_step

    n = (1 << 31) + 773
    if torch.cuda.mem_get_info()[0] < 44 << 30:
        pytest.skip("needs 44 GiB")
    p, g = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV, dtype=BF)
    q, h = torch.randn(1000, device=DEV), torch.randn(1000, device=DEV).to(BF)
    p[-773:].copy_(torch.randn(773, device=DEV))
    g[-773:].copy_(torch.randn(773, device=DEV))
    few, few_grads = [p[-773:].clone(), q.clone()], [g[-773:].clone(), h]
    state, own = adamw_state([p, q], bits), adamw_state(few, bits)
    adamw_step([p, q], [g, h], state, step=1, **HYPER)
    adamw_step(few, few_grads, own, step=1, **HYPER)
    assert torch.equal(p[-773:], few[0]) and torch.equal(q, few[1]) and float(p[:-773].abs().max()) == 0.0
    if bits == 8:
        assert torch.equal(state.exp_avg_scale[-8:], own.exp_avg_scale) and torch.equal(state.exp_avg_sq_scale[-8:], own.exp_avg_sq_scale)
        assert float(state.exp_avg_scale[:-8].abs().max()) == 0.0
    else:
        assert torch.equal(state.exp_avg[-2048:], own.exp_avg) and torch.equal(state.exp_avg_sq[-2048:], own.exp_avg_sq)


@pytest.mark.parametrize("beta2", [0.95, 0.999])
def test_second_moments_held_as_zeros_do_not_count(beta2):
    """Gradients around the size whose square is held as zero, then none, at the smallest eps that is taken.  A block's gradients
    are all alike, so its codes are its largest value and round nothing.  The root of v lacks at most eps / 32 (the kernel's head), so an
    update lies between that of the 32-bit states and 33/32 of it; beside that, ten roundings of 2^-24 in the moments and a dozen of 2^-23
    in the update (the hardware's root and reciprocal), and half a step of the parameter, which starts at zero."""
    from pccl.ops.optim import adamw_state, adamw_step, least_eps

    sizes = torch.logspace(-14, -8, 40, device=DEV)
    sizes[0] = 2e-12
    grad, none = sizes.repeat_interleave(256), torch.zeros(40 * 256, device=DEV)
    hyper = dict(lr=1.0, beta1=0.9, beta2=beta2, eps=least_eps(beta2), weight_decay=0.0)
    p8, p32 = none.clone(), none.clone()
    s8, s32 = adamw_state([p8], 8), adamw_state([p32], 32)
    for step in range(1, 250):
        g = grad if step < 50 else none
        for p, s in ((p8, s8), (p32, s32)):
            p.zero_()
            adamw_step([p], [g], s, step=step, **hyper)
        # what m keeps below 2^-80 is held as zero too: 2^-80 over eps of an update
        slack, least = 24 * 2.0 ** -23, 2.0 ** -80 / hyper["eps"] / (1 - 0.9) + 2.0 ** -126
        a, b = -p8.double(), -p32.double()
        assert torch.all(a >= b * (1 - slack * step) - least) and torch.all(a <= b * (33 / 32 + slack * step) + least), step
    assert torch.all(s8.dequantize()[1] <= s32.exp_avg_sq * (1 + 2.0 ** -10))


def test_a_norm_inside_what_the_step_writes_is_refused():
    from pccl.ops.optim import adamw_state, adamw_step

    p, g = torch.ones(300, device=DEV), torch.ones(300, device=DEV)
    for bits in (8, 32):
        st = adamw_state([p], bits)
        inside = [p[7:8], st.exp_avg_scale[:1] if bits == 8 else st.exp_avg[255:256], st.exp_avg_sq_scale[1:] if bits == 8 else st.exp_avg_sq[-1:]]
        for norm in inside:
            with pytest.raises(RuntimeError, match="overlaps another one"):
                adamw_step([p], [g], st, step=1, max_grad_norm=1.0, total_sq_norm=norm, **HYPER)
            assert torch.all(p == 1)
        adamw_step([p.clone()], [g], st, step=1, max_grad_norm=1.0, total_sq_norm=g[:1], **HYPER)       # a gradient is only read
        adamw_step([p.clone()], [g], st, step=1, total_sq_norm=p[:1], **HYPER)                         # not read without clipping


def test_all_64_bits_of_the_seed_count():
    from pccl.ops.optim import adamw_state, adamw_step

    grad = torch.randn(256 * 40, device=DEV, generator=torch.Generator(device=DEV).manual_seed(9))
    codes = []
    for seed in (3, 3 + (1 << 32), 3 + (5 << 40), (1 << 64) - 1, (1 << 32) - 1):
        state = adamw_state([grad], 8)
        adamw_step([torch.zeros_like(grad)], [grad], state, step=1, seed=seed, **HYPER)
        codes.append(torch.cat((state.exp_avg.int(), state.exp_avg_sq.int())))
    assert all(not torch.equal(a, b) for i, a in enumerate(codes) for b in codes[:i])


def test_8_bit_lists_of_several_launches_against_32_bits():
    """A list of more tensors than a launch takes, and one that needs the long table: scales are the block maxima of a 32-bit step from
    the moments that the codes stood for, codes the neighbours of its moments, parameters its bits; the second step reads codes."""
    from pccl.ops.optim import adamw_state, adamw_step

    for sizes in ([257 + 3 * i for i in range(1700)], [1 + 5 * i for i in range(200)]):
        params, grads, masters = _lists(sizes, BF, BF, 10)
        decay = [0.01 * (i % 7) for i in range(len(sizes))]
        state, full = adamw_state(params, 8), adamw_state(params, 32)
        for step in (1, 2, 3):
            for x, y in zip((full.exp_avg, full.exp_avg_sq), state.dequantize()):
                x.copy_(y)
            copies = [[t.clone() for t in x] for x in (params, masters)]
            adamw_step(copies[0], grads, full, step=step, masters=copies[1], weight_decay=decay, **HYPER)
            adamw_step(params, grads, state, step=step, masters=masters, weight_decay=decay, seed=step, **HYPER)
            assert all(torch.equal(a, b) for x, y in zip((params, masters), copies) for a, b in zip(x, y))
            for x, code, scale, top, power in ((full.exp_avg, state.exp_avg, state.exp_avg_scale, 127, 2),
                                               (full.exp_avg_sq, state.exp_avg_sq, state.exp_avg_sq_scale, 255, 4)):
                x, c = x.view(-1, 256).double(), code.view(-1, 256).double()
                assert torch.equal(scale, x.abs().amax(1).float())
                y = x.abs() / scale.double()[:, None].clamp(min=1e-300) * top ** power
                # 1e-5: the 32-bit roundings of y
                assert torch.all(c.abs() ** power <= ((y * (1 + 1e-5)) ** (1 / power) + 1) ** power)
                assert torch.all((c.abs() + 1) ** power >= y * (1 - 1e-5))
                assert torch.all((c == 0) | (torch.sign(c) == torch.sign(x)))
