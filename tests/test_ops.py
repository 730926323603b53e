"""Refusals of the operators (svl.ops): every check runs on the host before
any device is touched, so these need no GPU.  The addresses passed here are
never read."""

import ctypes

import numpy as np
import pytest

from svl import errors
from svl._abi import ErrBuf, SvlAttentionConfig, SvlRopeConfig, load_library
from svl.ops import AttentionPlan, AxisRope, Q4Weight

FAKE = 1 << 20  # 16-byte aligned, never dereferenced


@pytest.mark.parametrize("kwargs", [
    dict(head_dim=1, pairs=[1]),
    dict(head_dim=514, pairs=[1]),
    dict(head_dim=64, pairs=[]),
    dict(head_dim=64, pairs=[1] * 5),
    dict(head_dim=64, pairs=[16, 0]),
    dict(head_dim=64, pairs=[16, 17]),
    dict(head_dim=64, pairs=[(1 << 32) - 1, 2]),
    dict(head_dim=64, pairs=[1 << 32]),
    dict(head_dim=64, pairs=[8, -1]),
    dict(head_dim=64, pairs=[1.5]),
    dict(head_dim=64, pairs=[32], theta=0.0),
    dict(head_dim=64, pairs=[32], theta=float("inf")),
    dict(head_dim=64, pairs=[16, 16], theta=[1e4, -1.0]),
    dict(head_dim=64, pairs=[16, 16], theta=[1e4]),
    dict(head_dim=64, pairs=[16, 16], theta=[1e4, 1e4, 1e4]),
    dict(head_dim=64, pairs=[32], arrangement="halves"),
])
def test_rope_configuration_refusals(kwargs):
    with pytest.raises(errors.UsageError):
        AxisRope(**kwargs)


@pytest.mark.parametrize("theta", [1e-3, 1.0 / 129, 5e-324])
def test_rope_refuses_bases_whose_angles_are_lost(theta):
    """Frequencies of many turns a position leave too few bits of the angle at far positions; 1/128 is the least base."""
    with pytest.raises(errors.UsageError):
        AxisRope(64, [32], theta)
    with pytest.raises(errors.UsageError):
        AxisRope(64, [16, 16], [1e4, theta])
    AxisRope(64, [32], 1.0 / 128).close()


def test_rope_c_configuration_refusals():
    lib = load_library()
    for change in (dict(arrangement=3), dict(reserved=1), dict(n_axes=0), dict(n_axes=5)):
        c = SvlRopeConfig(head_dim=64, n_axes=1)
        c.pairs[0], c.theta[0] = 8, 1e4
        for k, v in change.items():
            setattr(c, k, v)
        out, eb = ctypes.c_void_p(), ErrBuf()
        assert lib.svl_rope_create(ctypes.byref(c), ctypes.byref(out), *eb.args) == errors.USAGE
        assert not out.value and eb.buf.value


@pytest.mark.parametrize("change", [
    dict(dtype="f64"), dict(n_tokens=1 << 31), dict(positions=0), dict(q=0), dict(q_out=0), dict(k_out=0),
    dict(ld_q=127), dict(ld_k_out=63), dict(q=FAKE + 1), dict(k_out=FAKE + 2), dict(q_out=FAKE, ld_q_out=160),
    dict(q_heads=65536, ld_q=1 << 30, ld_q_out=1 << 30),
])
def test_rope_call_refusals(change):
    rope = AxisRope(64, [32])
    call = dict(dtype="f32", positions=FAKE, n_tokens=4, q=FAKE, ld_q=128, q_heads=2, q_out=2 * FAKE, ld_q_out=128,
                k=FAKE, ld_k=64, k_heads=1, k_out=2 * FAKE, ld_k_out=64)
    with pytest.raises(errors.UsageError):
        rope.apply_device(**{**call, **change})


@pytest.mark.parametrize("change", [dict(ld_q=1 << 36), dict(ld_q=-128), dict(ld_q_out=-128), dict(ld_k=1 << 36),
                                    dict(ld_k_out=-64)])
def test_rope_refuses_strides_that_wrap(change):
    call = dict(dtype="f32", positions=FAKE, n_tokens=3, q=FAKE, ld_q=128, q_heads=2, q_out=2 * FAKE, ld_q_out=128,
                k=FAKE, ld_k=64, k_heads=1, k_out=2 * FAKE, ld_k_out=64)
    with pytest.raises(errors.UsageError):
        AxisRope(64, [32]).apply_device(**{**call, **change})


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_rope_refuses_misaligned_positions(offset):
    call = dict(dtype="bf16", positions=FAKE + offset, n_tokens=4, q=FAKE, ld_q=128, q_heads=2, q_out=2 * FAKE,
                ld_q_out=128)
    with pytest.raises(errors.UsageError):
        AxisRope(64, [32]).apply_device(**call)


@pytest.mark.parametrize("change", [dict(q_heads=(1 << 32) + 2), dict(k_heads=(1 << 32) + 1), dict(q_heads=-2)])
def test_rope_refuses_head_counts_that_would_be_cut(change):
    call = dict(dtype="f32", positions=FAKE, n_tokens=0, q=FAKE, ld_q=128, q_heads=2, q_out=2 * FAKE, ld_q_out=128,
                k=FAKE, ld_k=64, k_heads=1, k_out=2 * FAKE, ld_k_out=64)
    with pytest.raises(errors.UsageError):
        AxisRope(64, [32]).apply_device(**{**call, **change})


def test_rope_of_nothing_needs_no_device():
    AxisRope(64, [32]).apply_device("f32", 0, 0, 0, 0, 2, 0, 0)
    AxisRope(64, [32]).apply_device("f32", 0, 9, 0, 0, 0, 0, 0)


PLAN = dict(q_heads=4, kv_heads=2, head_dim=64, cu_q=[0, 3, 8])


@pytest.mark.parametrize("change", [
    dict(dtype="f64"), dict(kv_heads=0), dict(kv_heads=3), dict(q_heads=0), dict(q_heads=1 << 32), dict(head_dim=0),
    dict(head_dim=513), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf")), dict(cap=1e-31), dict(cap=2e30), dict(scale=1e-31),
    dict(scale=2e30), dict(scale=1e3, cap=1e-28), dict(slopes=[1.0, 1.0, 2e20, 1.0]), dict(window=-2), dict(window=1 << 31),
    dict(cu_q=[1, 3, 8]), dict(cu_q=[0, 5, 3]), dict(cu_q=[]), dict(cu_q=[0.0, 1.5, 3.0]), dict(cu_q=[0, -1, 3]),
    dict(cu_k=[0, 3]), dict(cu_k=[0, 9, 8]), dict(prefix=[1]), dict(prefix=[1, -1]), dict(doc_q=[0] * 7),
    dict(doc_k=[0] * 8), dict(doc_q=[0] * 8, cu_k=[0, 1, 2]), dict(doc_q=[1 << 31] * 8), dict(slopes=[1.0] * 3),
    dict(slopes=[1.0, 1.0, float("nan"), 1.0]), dict(slopes=[1.0, 1.0, float("inf"), 1.0]),
])
def test_attention_plan_refusals(change):
    with pytest.raises(errors.UsageError):
        AttentionPlan(**{**PLAN, **change})


@pytest.mark.parametrize("change", [
    dict(cu_k=[0, 1 << 31, 1 << 31]), dict(cu_q=[0, 1 << 30, 1 << 30]), dict(cu_k=[0, 1 << 41, 1 << 41]),
])
def test_attention_plan_limits(change):
    with pytest.raises(errors.LimitExceededError):
        AttentionPlan(**{**PLAN, **change})


@pytest.mark.parametrize("cap", [1e-46, 1e-300, -1e-46])
def test_attention_refuses_caps_that_round_to_none(cap):
    """A cap too small for the C float would arrive as 0, which is no cap."""
    with pytest.raises(errors.UsageError):
        AttentionPlan(**PLAN, cap=cap)


@pytest.mark.parametrize("build", [
    lambda x: AxisRope(64, [x]), lambda x: AxisRope(x, [8]), lambda x: AttentionPlan(**{**PLAN, "q_heads": x}),
    lambda x: AttentionPlan(**PLAN, window=x), lambda x: Q4Weight.from_codes(FAKE, FAKE, x, 64, 32),
])
@pytest.mark.parametrize("x", [float("nan"), float("inf"), 2.5])
def test_counts_that_are_no_whole_numbers(build, x):
    with pytest.raises(errors.UsageError):
        build(x)


def test_attention_c_configuration_refusals():
    lib = load_library()
    cu = np.array([0, 4], np.uint64)
    for change in (dict(causal=2), dict(reserved=(ctypes.c_uint32 * 4)(0, 0, 0, 1)), dict(dtype=3),
                   dict(q_heads=65536, kv_heads=1), dict(kv_heads=65536, q_heads=65536)):
        c = SvlAttentionConfig(dtype=0, q_heads=2, kv_heads=1, head_dim=64, scale=1.0, window=-1)
        for k, v in change.items():
            setattr(c, k, v)
        out, eb = ctypes.c_void_p(), ErrBuf()
        rc = lib.svl_attention_plan_create(0, ctypes.byref(c), cu.ctypes.data, None, 1, None, None, None, None,
                                           ctypes.byref(out), *eb.args)
        assert rc == errors.USAGE and not out.value and eb.buf.value
    for call in ((None, cu.ctypes.data), (ctypes.byref(SvlAttentionConfig()), None)):
        out, eb = ctypes.c_void_p(), ErrBuf()
        assert lib.svl_attention_plan_create(0, *call, None, 1, None, None, None, None, ctypes.byref(out),
                                             *eb.args) == errors.USAGE
    assert lib.svl_attention_plan_workspace(None, None) == errors.USAGE
    eb = ErrBuf()
    assert lib.svl_attention_device(None, *[0] * 12, *eb.args) == errors.USAGE
    assert lib.svl_attention_check(None, *eb.args) == errors.USAGE


@pytest.mark.parametrize("change", [
    dict(group=16), dict(group=256), dict(k=96, group=64), dict(n=0), dict(k=0), dict(n=1 << 31), dict(k=1 << 31),
    dict(scale_dtype="f32"), dict(codes=0), dict(scales=0),
])
def test_q4_create_refusals(change):
    # without a GPU the sizes are refused before the device is asked for; with one, the same
    call = dict(codes=FAKE, scales=FAKE, n=8, k=64, group=32)
    with pytest.raises(errors.UsageError):
        Q4Weight.from_codes(**{**call, **change})


@pytest.mark.parametrize("weight,kwargs", [
    (np.zeros((4, 4, 64), np.float32), {}),
    (np.zeros(64, np.float32), {}),
    (np.zeros((4, 96), np.float32), dict(group=64)),
    (np.zeros((4, 64), np.float32), dict(group=48)),
    (np.zeros((0, 64), np.float32), {}),
])
def test_q4_quantize_refusals(weight, kwargs):
    with pytest.raises(errors.UsageError):
        Q4Weight.quantize(weight, **kwargs)


def test_q4_null_handle():
    lib, eb = load_library(), ErrBuf()
    assert lib.svl_q4_linear_device(None, 0, FAKE, 64, 1, FAKE, 64, None, *eb.args) == errors.USAGE
    assert lib.svl_q4_read(None, *[None] * 7, *eb.args) == errors.USAGE
    lib.svl_q4_destroy(None)
    lib.svl_rope_destroy(None)
    lib.svl_attention_plan_destroy(None)
