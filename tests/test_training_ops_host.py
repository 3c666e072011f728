"""What the training operators do on the host: layouts, tables, positions, parameters, refusals."""
import dataclasses
import math
import warnings

import pytest
import torch

from pccl.models import gpt
from pccl.models.gpt import GPTConfig, positions_of, unit_specs
from pccl.ops.attention import attention_backward, attention_forward
from pccl.ops.optim import BLOCK, adamw_state, adamw_step, state_offsets
from pccl.ops.rotary import qk_norm_rope_backward, qk_norm_rope_forward, rotary_table

CFG = GPTConfig(2, 64, 4, 256, vocab=96, seq_len=16, name="host-test")
ROPE = dataclasses.replace(CFG, qk_norm_rope=True)


def test_tensors_of_the_host_are_refused():
    q, w = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    cos, sin = rotary_table(16, 64)
    p = [torch.zeros(300)]
    for call in (lambda: attention_forward(q, q, q), lambda: attention_backward(q, q, q, q, q, torch.zeros(1, 2, 4)),
                 lambda: qk_norm_rope_forward(q, q, w, w, cos, sin), lambda: qk_norm_rope_backward(q, q, q, q, w, w, cos, sin),
                 lambda: adamw_step(p, [torch.zeros(300)], adamw_state(p), step=1, lr=1e-3),
                 lambda: adamw_state(p, bits=8).dequantize()):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_states_begin_on_whole_blocks():
    sizes = [1, 0, 256, 257, 1000]
    params = [torch.zeros(n) for n in sizes]
    at = state_offsets(params)
    assert at == [0, 256, 256, 512, 1024, 2048] and all(a % BLOCK == 0 for a in at)
    wide, narrow = adamw_state(params), adamw_state(params, bits=8)
    assert wide.bits == 32 and narrow.bits == 8 and wide.dequantize()[0] is wide.exp_avg
    assert wide.exp_avg.numel() == narrow.exp_avg.numel() == at[-1] and narrow.exp_avg_scale.numel() == at[-1] // BLOCK
    assert narrow.exp_avg.dtype == torch.int8 and narrow.exp_avg_sq.dtype == torch.uint8
    with pytest.raises(ValueError, match="bits"):
        adamw_state(params, bits=16)
    with pytest.raises(ValueError, match="at least one"):
        adamw_state([])


def test_far_positions_keep_their_digits():
    cos, sin = rotary_table(70000, 16, theta=500000.0)
    for pos in (0, 1, 65535, 69999):
        for i in range(8):
            angle = math.fmod(pos * 500000.0 ** (-2 * i / 16), 2 * math.pi)
            # fmod's argument is off by 2^-53 of itself and by the power's own rounding, results by half a step of fp32
            assert abs(float(cos[pos, i]) - math.cos(angle)) <= 2.0 ** -24 + pos * 2.0 ** -51
            assert abs(float(sin[pos, i]) - math.sin(angle)) <= 2.0 ** -24 + pos * 2.0 ** -51
    for rot in (0, 4, 12):
        with pytest.raises(ValueError, match="multiple of 8"):
            rotary_table(4, rot)


def test_parameters_of_a_configuration_with_rotation():
    names = [[p.name for p in u.params] for u in unit_specs(CFG)]
    assert "wpe" in names[0] and "qn_w" not in names[1]
    units = unit_specs(ROPE)
    names = [[p.name for p in u.params] for u in units]
    assert "wpe" not in names[0] and names[1][-2:] == ["qn_w", "kn_w"]
    flat = torch.empty(units[1].numel)
    gpt.init_unit(units[1], flat, ROPE, seed=1)
    views = gpt.views(units[1], flat)
    assert views["qn_w"].shape == (16,) and torch.all(views["qn_w"] == 1) and torch.all(views["kn_w"] == 1)
    used = lambda cfg: sum(math.prod(p.shape) for u in unit_specs(cfg) for p in u.params)          # noqa: E731
    assert used(CFG) - used(ROPE) == 16 * 64 - 2 * 2 * 16


def test_positions_of_packed_documents():
    pos = positions_of(ROPE, 2, 16, "cpu")
    assert pos.place is None and pos.cos.shape == (16, 8)
    cu = torch.tensor([0, 3, 3, 10, 29], dtype=torch.int32)
    packed = positions_of(ROPE, 2, 16, "cpu", (pos.cos, pos.sin), cu)
    want = list(range(3)) + list(range(7)) + [i % 16 for i in range(19)] + list(range(3))
    assert packed.cos is pos.cos and packed.place.tolist() == want
    with pytest.raises(ValueError, match="does not hold"):
        positions_of(ROPE, 1, 17, "cpu")


def test_what_the_attention_kernels_take():
    takes = lambda d: gpt.native_attention_takes(GPTConfig(1, 4 * d, 4, 64, vocab=8, seq_len=8))      # noqa: E731
    assert takes(8) and takes(64) and takes(80) and takes(128) and not takes(136) and not takes(12)


def test_8_bit_states_refuse_a_small_eps():
    from pccl.ops.optim import least_eps
    from pccl.parallel.zero3 import OptimConfig, Zero3Engine

    p, g = [torch.zeros(300)], [torch.zeros(300)]
    for beta2 in (0.0, 0.95, 0.999, 0.99999):
        least = 2.0 ** -35 / math.sqrt(1 - beta2)
        assert abs(least_eps(beta2) / least - 1) < 1e-12
        go = lambda eps, bits: adamw_step(p, g, adamw_state(p, bits), step=1, lr=1e-3, beta2=beta2, eps=eps)      # noqa: E731,B023
        for eps in (0.0, 1e-15, least * 0.999):
            with pytest.raises(RuntimeError, match="eps of at least"):
                go(eps, 8)
        for eps, bits in ((least * 1.001, 8), (1e-8, 8), (0.0, 32)):
            with pytest.raises(RuntimeError, match="CUDA"):                        # taken, but for where the tensors lie
                go(eps, bits)
    with pytest.raises(ValueError, match="eps of at least"):
        Zero3Engine(CFG, optim=OptimConfig(eps=1e-12), device=torch.device("cpu"), optim_bits=8)


def test_engine_refuses_head_sizes_that_the_rotation_does_not_take():
    from pccl.parallel.zero3 import Zero3Engine

    for d_model in (4 * 12, 4 * 264, 4 * 512):
        cfg = GPTConfig(1, d_model, 4, 64, vocab=8, seq_len=8, qk_norm_rope=True)
        with pytest.raises(ValueError, match="multiple of 8 up to 256"):
            Zero3Engine(cfg, device=torch.device("cpu"))


def test_engine_refuses_long_sequences_before_the_step_begins():
    """With nothing of the step begun: the engine here has no more than its configuration."""
    from pccl.parallel.zero3 import Zero3Engine

    eng = Zero3Engine.__new__(Zero3Engine)
    eng.cfg, eng.C, eng.native_attention, eng.device = ROPE, None, True, torch.device("cpu")
    tokens = torch.zeros(2, 17, dtype=torch.int64)
    with pytest.raises(ValueError, match="17 tokens have positions"):
        eng.train_step(tokens, tokens)


def test_engine_says_where_native_attention_does_not_take_a_head_size():
    from pccl.parallel.zero3 import Zero3Engine

    def build(d):
        try:
            Zero3Engine(GPTConfig(1, 4 * d, 4, 64, vocab=8, seq_len=8), device=torch.device("cpu"), native_attention=True)
        except Exception:           # noqa: BLE001  (the engine wants a GPU, later on)
            pass

    for d in (12, 136):
        with pytest.warns(UserWarning, match=f"heads of {d} columns"):
            build(d)
    with warnings.catch_warnings(record=True) as said:
        warnings.simplefilter("always")
        build(64)
    assert not [w for w in said if "native_attention" in str(w.message)]


def test_a_largest_norm_that_is_nan_is_refused():
    p = [torch.zeros(300)]
    go = lambda most: adamw_step(p, p, adamw_state(p), step=1, lr=1e-3, max_grad_norm=most, total_sq_norm=torch.zeros(1))      # noqa: E731
    with pytest.raises(RuntimeError, match="max_grad_norm must be a number"):
        go(math.nan)
    for most in (-1.0, 0.0, 1.0, math.inf):
        with pytest.raises(RuntimeError, match="CUDA"):                            # taken, but for where the tensors lie
            go(most)
