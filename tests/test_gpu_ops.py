"""svl.ops on the GPU against their definitions in 64 bits.

Tolerances count roundings.  A rounding to a type t is off by at most
eps(t) / 2 of the value; FP32 sums of n products by at most n 2^-23 of the sum
of the magnitudes (2^-23, a whole unit in the last place, because a tensor core
may cut where an adder rounds).  Each test writes its own sum below.
"""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from svl import errors  # noqa: E402
from svl.ops import AttentionPlan, AxisRope, Q4Weight  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ULP = 2.0 ** -23


def half_step(dtype):
    return torch.finfo(TYPES[dtype]).eps / 2


def least_half_step(dtype):
    """Half the spacing of the type's smallest values (FP16: 2^-24 below 2^-14), where half_step is no longer relative."""
    info = torch.finfo(TYPES[dtype])
    return info.eps * info.tiny / 2


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------- rope --


def rope_pairs(pairs, theta, arrangement):
    """(axis, first, second, frequency) by the definition."""
    out, total = [], sum(pairs)
    if arrangement == "split":
        start = 0
        for a, n in enumerate(pairs):
            out += [(a, start + i, start + n + i, theta[a] ** (-i / n)) for i in range(n)]
            start += 2 * n
        return out
    if arrangement == "sections":
        axes = [a for a, n in enumerate(pairs) for _ in range(n)]
    else:
        axes = [a for r in range(max(pairs)) for a, n in enumerate(pairs) if r < n]
    return [(a, p, p + total, theta[0] ** (-p / total)) for p, a in enumerate(axes)]


def rope_reference(x, positions, pairs, theta, arrangement):
    """x [T, heads, hd] float64 on the CPU; (result, |x| + |y| of each result's pair)."""
    y, size = x.clone(), torch.zeros_like(x)
    for a, d, e, f in rope_pairs(pairs, theta, arrangement):
        # the angle modulo a turn, in integers: position * f / 2 pi has 2^31 * 2^-53 left to lose in 64 bits
        angle = (positions[a].double() * f)[:, None]
        c, s = angle.cos(), angle.sin()
        y[..., d] = x[..., d] * c - x[..., e] * s
        y[..., e] = x[..., e] * c + x[..., d] * s
        size[..., d] = size[..., e] = x[..., d].abs() + x[..., e].abs()
    return y, size


def rope_tolerance(dtype, y, size, far):
    # the angle in half turns is rounded to FP32 (2^-25 of a half turn: 3.2 2^-25 rad, under 2 2^-24), sine and
    # cosine are within 2 units, two products and a sum round: 6 2^-24 of |x| + |y| in all; the 64-bit reference's own
    # angle is off by far * 2^-53 (its product's rounding) and as much for its frequency
    return size * (6 * 2.0 ** -24 + far * 2.0 ** -52) + half_step(dtype) * y.abs() + least_half_step(dtype)


def run_rope(dtype, tokens, qh, kh, hd, pairs, arrangement, far=0, pad=0, offset=0, in_place=False, seed=0, theta=None):
    g, t = gen(seed), TYPES[dtype]
    theta = theta or [10000.0, 500.0, 100.0, 7.0][: len(pairs)]
    ld = (qh + kh) * hd + pad
    store = torch.randn(tokens * ld + offset, device="cuda", generator=g).to(t)
    x = store[offset:].view(tokens, ld)
    pos = (torch.randint(-40, 400, (len(pairs), tokens), device="cuda", generator=g) + far).to(torch.int32)
    out_store = store.clone() if in_place else torch.full_like(store, 5.0)
    out = out_store[offset:].view(tokens, ld)
    src = out if in_place else x
    rope = AxisRope(hd, pairs, theta, arrangement)
    ahead = qh * hd * x.element_size()
    rope.apply_device(dtype, pos.data_ptr(), tokens, src.data_ptr(), ld, qh, out.data_ptr(), ld,
                      src.data_ptr() + ahead, ld, kh, out.data_ptr() + ahead, ld, stream=stream())
    torch.cuda.synchronize()
    got = out.cpu().double()
    n = (qh + kh) * hd
    y, size = rope_reference(x.cpu().double()[:, :n].reshape(tokens, qh + kh, hd), pos.cpu(), pairs, theta, arrangement)
    err = (got[:, :n].reshape(y.shape) - y).abs()
    assert (err <= rope_tolerance(dtype, y, size, abs(far) + 400)).all(), (err.max(), err.argmax())
    # columns behind the heads and values before the first row stay as they were
    want = x.cpu().double() if in_place else torch.full_like(got, 5.0)
    assert torch.equal(got[:, n:], want[:, n:])
    assert torch.equal(out_store[:offset], store[:offset] if in_place else torch.full_like(store[:offset], 5.0))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("arrangement", ["split", "sections", "interleaved"])
@pytest.mark.parametrize("tokens,qh,kh,hd,pairs", [
    (1, 1, 1, 2, [1]), (33, 4, 2, 256, [128]), (17, 16, 16, 72, [18, 18]), (130, 16, 4, 128, [24, 20, 20]),
    (5, 3, 1, 66, [3, 7, 2, 5]), (9, 2, 2, 67, [11, 5]), (3, 1, 1, 512, [100, 156]), (64, 5, 0, 80, [16, 24]),
    (70, 0, 7, 96, [40]), (4, 1, 2, 512, [1]), (700, 2, 1, 128, [20, 44]),
])
def test_rope(dtype, arrangement, tokens, qh, kh, hd, pairs):
    run_rope(dtype, tokens, qh, kh, hd, pairs, arrangement)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("far", [1 << 20, 2147483247, -2147483000])
def test_rope_far_positions(dtype, far):
    run_rope(dtype, 40, 4, 2, 128, [24, 20, 20], "interleaved", far=far)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 0), (3, 0), (0, 1), (5, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rope_strides_and_alignment(dtype, pad, offset, in_place):
    run_rope(dtype, 21, 4, 2, 72, [18, 10], "split", pad=pad, offset=offset, in_place=in_place)


def test_rope_small_base():
    run_rope("f32", 31, 2, 1, 64, [16, 16], "split", theta=[0.5, 0.01])


@pytest.mark.parametrize("theta", [1.0 / 128, 0.01, 0.5, 1.0, 3.0])
@pytest.mark.parametrize("far", [0, 1 << 20, 2147483000, -2147483648])
def test_rope_small_bases_far_out(theta, far):
    """Frequencies of up to 20 turns a position, against angles of 60 digits."""
    from decimal import Decimal, getcontext

    getcontext().prec = 60
    turn = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494")
    n, tokens = 16, 40
    pos = torch.arange(tokens, dtype=torch.int64) + far
    x = torch.randn(tokens, 2 * n, device="cuda", generator=gen(2))
    y = torch.empty_like(x)
    p32 = pos.to(torch.int32).cuda()
    AxisRope(2 * n, [n], theta).apply_device("f32", p32.data_ptr(), tokens, x.data_ptr(), 2 * n, 1, y.data_ptr(), 2 * n,
                                             stream=stream())
    torch.cuda.synchronize()
    base = Decimal(theta).ln()
    f = [(-base * i / n).exp() for i in range(n)]
    angle = np.array([[float((int(p) * w) % turn) for w in f] for p in pos])
    c, s = np.cos(angle), np.sin(angle)
    xs, got = x.cpu().double().numpy(), y.cpu().double().numpy()
    a, b = xs[:, :n], xs[:, n:]
    size = np.abs(a) + np.abs(b)
    # the angle within 2^-25 of a turn (6.3 2^-25 rad), sine and cosine within 2 units, two products and a sum rounded
    tol = size * (6.3 * 2.0 ** -25 + 4 * 2.0 ** -24) + least_half_step("f32")
    assert (np.abs(got[:, :n] - (a * c - b * s)) <= tol).all()
    assert (np.abs(got[:, n:] - (b * c + a * s)) <= tol).all()


# ----------------------------------------------------------------- linear --


def dequantised(codes, scales, zeros, group):
    codes = codes.astype(np.int64)
    w = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1).astype(np.float64)
    z = np.full(scales.shape, 8.0) if zeros is None else zeros.astype(np.float64)
    return (w - np.repeat(z, group, 1)) * np.repeat(scales, group, 1)


def run_linear(dtype, rows, n, k, group, zeros, scale_dtype="bf16", pad=0, offset=0, seed=0, host=False, spoil=None):
    g, t = gen(seed), TYPES[dtype]
    codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = ((torch.rand(n, k // group, device="cuda", generator=g) + 0.1) * 0.02).to(TYPES[scale_dtype])
    z = torch.randint(0, 16, scales.shape, device="cuda", generator=g, dtype=torch.uint8) if zeros else None
    store = torch.randn(rows * (k + pad) + offset, device="cuda", generator=g).to(t)
    x = store[offset:].view(rows, k + pad)
    if spoil is not None:
        x[spoil[0], spoil[1]] = spoil[2]
    y_store = torch.full((rows * (n + pad) + offset + 7,), 5.0, device="cuda", dtype=t)
    y = y_store[offset:offset + rows * (n + pad)].view(rows, n + pad)
    torch.cuda.synchronize()
    if host:
        kept = [codes.cpu(), scales.cpu(), None if z is None else z.cpu()]
    else:
        kept = [codes, scales, z]
    w = Q4Weight.from_codes(kept[0].data_ptr(), kept[1].data_ptr(), n, k, group,
                            zeros=kept[2].data_ptr() if zeros else 0, scale_dtype=scale_dtype)
    w.linear_device(dtype, x.data_ptr(), k + pad, rows, y.data_ptr(), n + pad, stream=stream())
    torch.cuda.synchronize()
    full = dequantised(codes.cpu().numpy(), scales.cpu().double().numpy(), None if z is None else z.cpu().numpy(), group)
    xs = x[:, :k].cpu().double().numpy()
    got = y.cpu().double().numpy()
    with np.errstate(invalid="ignore"):
        want, size = xs @ full.T, np.abs(xs) @ np.abs(full).T
        # k products summed, the group's sum scaled (one more rounding each), and y rounded
        bound = (k + k // group + 2) * ULP * size + half_step(dtype) * np.abs(want) + least_half_step(dtype)
        good = np.ones(rows, bool)
        if spoil is not None:
            good[spoil[0]] = False
            assert not np.isfinite(got[spoil[0], :n]).any()
        assert (np.abs(got[good, :n] - want[good]) <= bound[good]).all()
    assert (got[:, n:] == 5.0).all() and (y_store[:offset] == 5.0).all() and (y_store[-7:] == 5.0).all()
    return w, codes, scales, z


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("group,zeros,scale_dtype", [(32, False, "bf16"), (64, True, "f16"), (128, True, "bf16")])
@pytest.mark.parametrize("rows,n,k", [(1, 512, 512), (1, 1, 128), (2, 17, 384), (3, 100, 640), (7, 130, 256), (8, 33, 1152),
                                      (9, 64, 128), (17, 200, 512), (33, 65, 256), (64, 96, 384), (71, 48, 2048),
                                      (200, 31, 256)])
def test_linear(dtype, group, zeros, scale_dtype, rows, n, k):
    run_linear(dtype, rows, n, k, group, zeros, scale_dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("k", [32, 96, 160, 2080])
def test_linear_odd_depth(dtype, k):
    run_linear(dtype, 5, 77, k, 32, True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 2, 5, 11, 17, 33, 70, 130])
@pytest.mark.parametrize("k,group", [(96, 32), (160, 32), (1056, 32), (2080, 32), (192, 64), (1088, 64), (2112, 64)])
def test_linear_last_span_in_part(dtype, rows, k, group):
    """Depths that end inside a span of 128 columns, in every kernel and with the span run of every rank of a cluster."""
    run_linear(dtype, rows, 77, k, group, True)
    run_linear(dtype, rows, 300, k, group, False, scale_dtype="f16")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_linear_padding_behind_a_row_is_not_read_into_it(dtype, rows):
    """Columns of x behind k, inside the last span or not, may hold anything."""
    for k, group in ((96, 32), (160, 32), (2112, 64)):
        g, t, n, ld = gen(k), TYPES[dtype], 50, k + 64
        codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.uint8)
        scales = torch.ones(n, k // group, device="cuda", dtype=torch.bfloat16)
        x = torch.randn(rows, ld, device="cuda", generator=g).to(t)
        w = Q4Weight.from_codes(codes.data_ptr(), scales.data_ptr(), n, k, group)
        ys = []
        for fill in (0.0, float("nan"), float("inf")):
            x[:, k:] = fill
            ys.append(torch.empty(rows, n, device="cuda", dtype=t))
            w.linear_device(dtype, x.data_ptr(), ld, rows, ys[-1].data_ptr(), n, stream=stream())
        torch.cuda.synchronize()
        assert torch.isfinite(ys[0].float()).all() and torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (0, 1), (5, 3)])
def test_linear_strides_and_alignment(dtype, pad, offset):
    run_linear(dtype, 6, 50, 192, 64, False, pad=pad, offset=offset, host=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_linear_non_finite_row(dtype, value):
    # every weight of the spoiled column is non-zero or meets the NaN of inf * 0: no finite result in that row
    run_linear(dtype, 4, 40, 128, 32, False, spoil=(2, 50, value))


def test_linear_large_values_f32():
    """24-bit activations of very different sizes keep their precision."""
    g = gen(3)
    k, n = 256, 40
    codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = torch.ones(n, k // 32, device="cuda", dtype=torch.bfloat16)
    for power in (-60, 0, 60):
        x = torch.randn(3, k, device="cuda", generator=g) * 2.0 ** power
        y = torch.empty(3, n, device="cuda")
        w = Q4Weight.from_codes(codes.data_ptr(), scales.data_ptr(), n, k, 32)
        w.linear_device("f32", x.data_ptr(), k, 3, y.data_ptr(), n, stream=stream())
        full = dequantised(codes.cpu().numpy(), np.ones((n, k // 32)), None, 32)
        xs = x.cpu().double().numpy()
        assert (np.abs(y.cpu().double().numpy() - xs @ full.T) <= (k + 10) * ULP * (np.abs(xs) @ np.abs(full).T)).all()


@pytest.mark.parametrize("rows", [1, 3, 14, 40])
@pytest.mark.parametrize("power", [-100, -109, -116, -124, -132, -140])
def test_linear_tiny_values_f32(rows, power):
    """FP32 values keep their 24 bits down to 2^-110; below, what lies under 2^-133 is cut off."""
    g, k, n = gen(4), 256, 40
    codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = torch.full((n, k // 32), 2.0 ** 60, device="cuda", dtype=torch.bfloat16)
    x = (torch.rand(rows, k, device="cuda", generator=g) + 1.0).double().mul(2.0 ** power).float()
    x *= torch.randint(0, 2, x.shape, device="cuda", generator=g) * 2 - 1
    y = torch.empty(rows, n, device="cuda")
    w = Q4Weight.from_codes(codes.data_ptr(), scales.data_ptr(), n, k, 32)
    w.linear_device("f32", x.data_ptr(), k, rows, y.data_ptr(), n, stream=stream())
    full = dequantised(codes.cpu().numpy(), np.full((n, k // 32), 2.0 ** 60), None, 32)
    xs = x.cpu().double().numpy()
    cut = 2.0 ** -133 * np.abs(full).sum(1) if power < -110 else 0.0
    bound = (k + 10) * ULP * (np.abs(xs) @ np.abs(full).T) + cut
    assert (np.abs(y.cpu().double().numpy() - xs @ full.T) <= bound).all()


def test_q4_read_returns_what_was_given():
    for zeros in (False, True):
        w, codes, scales, z = run_linear("f32", 1, 37, 160, 32, zeros)
        c, s, zz = w.read()
        assert np.array_equal(c, codes.cpu().numpy())
        assert np.array_equal(s, scales.view(torch.int16).cpu().numpy().view(np.uint16))
        assert np.array_equal(zz, z.cpu().numpy() if zeros else np.full_like(zz, 8))


def test_q4_create_misaligned_scales():
    """Scales at an odd address: refused in device memory, which is read in place; copied from host memory."""
    n, k, group = 24, 128, 32
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, generator=torch.Generator().manual_seed(0))
    scales = (torch.rand(n, k // group, generator=torch.Generator().manual_seed(1)) + 0.5).to(torch.float16)
    odd = torch.zeros(2 * scales.numel() + 1, dtype=torch.uint8)
    odd[1:] = scales.reshape(-1).view(torch.uint8)
    assert odd.data_ptr() % 2 == 0
    on_gpu, c = odd.cuda(), codes.cuda()
    with pytest.raises(errors.UsageError):
        Q4Weight.from_codes(c.data_ptr(), on_gpu.data_ptr() + 1, n, k, group, scale_dtype="f16")
    w = Q4Weight.from_codes(c.data_ptr(), odd.data_ptr() + 1, n, k, group, scale_dtype="f16")
    assert np.array_equal(w.read()[1], scales.view(torch.int16).numpy().view(np.uint16))
    # the same bytes, aligned
    w = Q4Weight.from_codes(c.data_ptr(), on_gpu[1:].clone().data_ptr(), n, k, group, scale_dtype="f16")
    assert np.array_equal(w.read()[1], scales.view(torch.int16).numpy().view(np.uint16))


def as_bf16(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


@pytest.mark.parametrize("asymmetric", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_q4_quantize_is_nearest(asymmetric, group):
    r = np.random.default_rng(group)
    w = r.standard_normal((19, 256), dtype=np.float32) * 0.02
    w[3, :group] = 0.0            # a group of zeros stays zero
    w[4, :group] = np.abs(w[4, :group])  # one-sided groups
    w[5, :group] *= 1e30
    q = Q4Weight.quantize(w, group, asymmetric)
    codes, bits, zeros = q.read()
    scales = as_bf16(bits)
    got = dequantised(codes, scales, zeros, group)
    step = np.repeat(scales, group, 1)
    # the nearest code is within half a step; the scale's rounding to 8 bits moves the ends of the range by 15 * 2^-8
    # of a step (8 steps * 2^-9 symmetric), and a rounded zero by half a step more where the range is cut
    slack = 0.5 + 15 * 2.0 ** -8 + (0.5 if asymmetric else 0.0)
    assert (np.abs(got - w) <= slack * step).all()
    assert (got[3, :group] == 0).all()
    c = np.stack([codes & 15, codes >> 4], -1).reshape(w.shape)
    if not asymmetric:
        assert (zeros == 8).all() and c.min() >= 1
        lo, hi = 1, 15
    else:
        lo, hi = 0, 15
    z = np.repeat(zeros, group, 1).astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        exact = np.where(step > 0, w / step + z, z)
    # nearest: no other code is closer by more than the FP32 quotient's rounding
    best = np.clip(np.rint(exact), lo, hi)
    near = np.abs(c - exact) <= np.abs(best - exact) + 16 * 2.0 ** -22
    assert near.all()


def test_q4_quantize_bf16_and_corrupt():
    from svl.safetensors import TensorEntry

    r = np.random.default_rng(1)
    w = r.standard_normal((8, 64), dtype=np.float32)
    bits = (w.view(np.uint32) >> 16).astype(np.uint16)
    entry = TensorEntry.__new__(TensorEntry)
    entry.raw, entry.dtype, entry.shape = bits, "BF16", (8, 64)
    a = Q4Weight.quantize(entry, 32).read()
    b = Q4Weight.quantize((bits.astype(np.uint32) << 16).view(np.float32), 32).read()
    assert all(np.array_equal(x, y) for x, y in zip(a, b))
    for bad in (np.nan, np.inf):
        w[7, 63] = bad
        with pytest.raises(errors.CorruptError):
            Q4Weight.quantize(w, 32)


def test_linear_refusals():
    codes = torch.zeros(8, 32, dtype=torch.uint8, device="cuda")
    scales = torch.ones(8, 2, dtype=torch.bfloat16, device="cuda")
    w = Q4Weight.from_codes(codes.data_ptr(), scales.data_ptr(), 8, 64, 32)
    x, y = torch.zeros(2, 64, device="cuda"), torch.full((2, 8), 5.0, device="cuda")
    for call in (("f64", x.data_ptr(), 64, 2, y.data_ptr(), 8), ("f32", 0, 64, 2, y.data_ptr(), 8),
                 ("f32", x.data_ptr(), 64, 2, 0, 8), ("f32", x.data_ptr(), 63, 2, y.data_ptr(), 8),
                 ("f32", x.data_ptr(), 64, 2, y.data_ptr(), 7), ("f32", x.data_ptr() + 2, 64, 1, y.data_ptr(), 8),
                 ("f32", x.data_ptr(), 64, 1 << 31, y.data_ptr(), 8)):
        with pytest.raises(errors.UsageError):
            w.linear_device(*call)
    w.linear_device("f32", 0, 64, 0, 0, 8)  # no rows
    torch.cuda.synchronize()
    assert (y == 5.0).all()


@pytest.mark.parametrize("change", [dict(ld_x=-64), dict(ld_x=1 << 36), dict(ld_y=-8), dict(ld_y=1 << 36)])
def test_linear_refuses_strides_that_wrap(change):
    codes = torch.zeros(8, 32, dtype=torch.uint8, device="cuda")
    scales = torch.ones(8, 2, dtype=torch.bfloat16, device="cuda")
    w = Q4Weight.from_codes(codes.data_ptr(), scales.data_ptr(), 8, 64, 32)
    x, y = torch.zeros(2, 64, device="cuda"), torch.full((2, 8), 5.0, device="cuda")
    call = dict(dtype="f32", x=x.data_ptr(), ld_x=64, rows=2, y=y.data_ptr(), ld_y=8)
    with pytest.raises(errors.UsageError):
        w.linear_device(**{**call, **change})
    torch.cuda.synchronize()
    assert (y == 5.0).all()


# -------------------------------------------------------------- attention --


def visible(c, n_q, n_k, prefix, dq, dk):
    p = np.arange(n_q)[:, None] + n_k - n_q
    j = np.arange(n_k)[None]
    near = np.ones((n_q, n_k), bool)
    if c["causal"]:
        near &= j <= p
    if c["window"] is not None:
        near &= np.abs(p - j) <= c["window"]
    if dq is not None:
        near &= dq[:, None] == dk[None]
    seen = near | (j < prefix)
    if dq is not None:
        seen &= (dq >= 0)[:, None] & (dk >= 0)[None]
    return seen, np.abs(p - j)


def attention_reference(c, q, k, v, seen, gap, slope):
    """One head in float64: (out, lse, tolerance of out, tolerance of lse).  Values of masked keys are not looked at."""
    used = seen.any(0)
    k, v = np.where(used[:, None], k, 0.0), np.where(used[:, None], v, 0.0)
    t = c["scale"] * (q @ k.T)
    size = c["scale"] * (np.abs(q) @ np.abs(k).T)
    if c["cap"]:
        t = c["cap"] * np.tanh(t / c["cap"])
    t = np.where(seen, t - slope * gap, -np.inf)
    m = t.max(1, initial=-np.inf)
    base = np.where(np.isfinite(m), m, 0.0)
    e = np.exp(t - base[:, None])
    total = e.sum(1)
    w = e / np.where(total == 0, 1.0, total)[:, None]
    with np.errstate(divide="ignore"):
        lse = base + np.log(total)
    out, mass = w @ v, w @ np.abs(v)
    # a score: hd products and a scale; the cap's tanh to 8 units of the cap; the bias a product and a difference
    hd = q.shape[1]
    bias = np.where(seen, np.abs(slope) * gap, 0.0).max(1, initial=0.0)
    span = np.where(seen, size, 0.0).max(1, initial=0.0)
    score = (hd + 4) * ULP * span + 8 * ULP * c["cap"] + 4 * ULP * (bias + np.abs(base) + c["cap"])
    # a weight: e^score, the exponential's own error, and n additions of the row's sum
    weight = 2 * score + (seen.shape[1] + 16) * ULP
    half = half_step(c["dtype"])
    # 16-bit weights are rounded before they multiply v; FP32 ones are not
    rounded = half if c["dtype"] != "f32" else 0.0
    tol = (2 * weight + rounded)[:, None] * mass + half * np.abs(out) + np.finfo(np.float32).tiny
    if c["dtype"] == "f16":
        # results and weights (of 1 at the row's maximum) below the normal range are off by half of 2^-24
        tol = tol + 2.0 ** -25 * (1 + seen.shape[1] * np.abs(v).max(initial=0.0))
    return out, lse, tol, score + (seen.shape[1] + 16) * ULP + ULP * np.abs(np.where(np.isfinite(lse), lse, 0.0))


def run_attention(dtype, hq, hk, hd, lens, *, scale=None, cap=0.0, causal=False, window=None, prefix=None, docs=None,
                  slopes=False, seed=0, spoil=None, pad=8, fused=True, lse=True, by=1.0, graph=False, offset=0):
    """lens: (queries, keys) of each sequence; docs(n) -> documents of n keys.  spoil: a value put into every key
    and value row that no query of its sequence sees."""
    rng = np.random.default_rng(seed)
    c = dict(dtype=dtype, scale=scale or hd ** -0.5, cap=cap, causal=causal, window=window)
    t = TYPES[dtype]
    cu_q = np.concatenate([[0], np.cumsum([a for a, _ in lens])]).astype(np.int64)
    cu_k = np.concatenate([[0], np.cumsum([b for _, b in lens])]).astype(np.int64)
    tq, tk = int(cu_q[-1]), int(cu_k[-1])
    dk = np.concatenate([docs(b) for _, b in lens] or [[]]).astype(np.int32) if docs else None
    dq = np.concatenate([dk[cu_k[i + 1] - min(a, b):cu_k[i + 1]] if a <= b else
                         np.concatenate([np.zeros(a - b), dk[cu_k[i]:cu_k[i + 1]]]) for i, (a, b) in enumerate(lens)] or
                        [[]]).astype(np.int32) if docs else None
    sl = [0.5 * 2.0 ** (-8.0 * (h + 1) / hq) * (-1 if h % 5 == 4 else 1) for h in range(hq)] if slopes else None

    def rows(n, width):
        store = torch.from_numpy(rng.standard_normal((n, width + pad)) * by).to(t).cuda().reshape(-1)
        if offset:
            store = torch.cat([torch.zeros(offset, device="cuda", dtype=t), store])[offset:]
        return store.view(n, width + pad)

    self_attention = fused and tq == tk
    if self_attention:
        x = rows(tq, (hq + 2 * hk) * hd)
        q, k, v = x[:, :hq * hd], x[:, hq * hd:(hq + hk) * hd], x[:, (hq + hk) * hd:]
    else:
        q, k, v = rows(tq, hq * hd), rows(tk, hk * hd), rows(tk, hk * hd)
    masks = []
    for i, (a, b) in enumerate(lens):
        masks.append(visible(c, a, b, prefix[i] if prefix else 0, dq[cu_q[i]:cu_q[i + 1]] if docs else None,
                             dk[cu_k[i]:cu_k[i + 1]] if docs else None))
        if spoil is not None:
            hidden = torch.from_numpy(np.flatnonzero(~masks[-1][0].any(0)) + cu_k[i]).cuda()
            k[hidden, :hk * hd] = spoil
            v[hidden, :hk * hd] = spoil
    out_store = torch.full((tq + 2, hq * hd + pad), 5.0, device="cuda", dtype=t)
    out = out_store[1:tq + 1]
    lse_store = torch.full((tq + 2, hq), 5.0, device="cuda")
    plan = AttentionPlan(hq, hk, hd, cu_q, cu_k, dtype=dtype, scale=c["scale"], cap=cap, causal=causal, window=window,
                         prefix=prefix, doc_q=dq, doc_k=dk, slopes=sl)
    ws = torch.full((plan.workspace_bytes + 64,), 255, dtype=torch.uint8, device="cuda")  # NaN patterns: nothing is assumed

    def call():
        plan.run_device(q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), out.data_ptr(),
                        out.stride(0), lse=lse_store[1:].data_ptr() if lse else 0, workspace=ws.data_ptr(),
                        workspace_bytes=plan.workspace_bytes, stream=stream())

    if graph:
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        out_store.fill_(5.0)
        lse_store.fill_(5.0)
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            call()
        assert (out_store == 5.0).all()
        for _ in range(graph):
            captured.replay()
    else:
        call()
    plan.check()
    got, got_lse = out.float().cpu().double().numpy(), lse_store[1:tq + 1].cpu().double().numpy()
    qs, ks, vs = (y.float().cpu().double().numpy() for y in (q, k, v))
    for i, (a, b) in enumerate(lens):
        seen, gap = masks[i]
        for h in range(hq):
            at, kv = slice(h * hd, (h + 1) * hd), slice(h // (hq // hk) * hd, (h // (hq // hk) + 1) * hd)
            want, want_lse, tol, tol_lse = attention_reference(
                c, qs[cu_q[i]:cu_q[i + 1], at], ks[cu_k[i]:cu_k[i + 1], kv], vs[cu_k[i]:cu_k[i + 1], kv], seen, gap,
                sl[h] if sl else 0.0)
            err = np.abs(got[cu_q[i]:cu_q[i + 1], at] - want)
            assert (err <= tol).all(), (i, h, float(np.nanmax(err - tol)), np.argwhere(~(err <= tol))[:4].tolist())
            if lse:
                mine = got_lse[cu_q[i]:cu_q[i + 1], h]
                empty = ~seen.any(1)
                assert (mine[empty] == -np.inf).all()
                assert (np.abs(mine[~empty] - want_lse[~empty]) <= tol_lse[~empty]).all(), (i, h)
    assert (out_store[0] == 5.0).all() and (out_store[-1] == 5.0).all() and (out_store[:, hq * hd:] == 5.0).all()
    assert (lse_store[0] == 5.0).all() and (lse_store[-1] == 5.0).all()
    assert (ws[plan.workspace_bytes:] == 255).all()
    return plan


def runs_of(size, padding=0):
    """Documents as runs of about `size` keys, the last `padding` keys padding."""

    def docs(n):
        d = np.arange(n) // max(1, size)
        d[n - min(padding, n):] = -1
        return d

    return docs


def shuffled(n):
    """Documents that alternate, with padding between."""
    d = (np.arange(n) * 7 + 3) % 5
    return np.where(d == 4, -1, d)


ODD = [(1, 1), (5, 5), (127, 127), (128, 128), (129, 129), (300, 300)]
HEADS = [(4, 2, 64), (4, 1, 128), (2, 2, 256), (3, 1, 72), (6, 2, 80), (5, 1, 192), (16, 2, 128)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hq,hk,hd", HEADS + [(2, 1, 512), (2, 2, 36), (3, 3, 1), (1, 1, 67), (64, 1, 16)])
def test_attention_heads(dtype, hq, hk, hd):
    run_attention(dtype, hq, hk, hd, [(1, 1), (130, 130), (45, 45)])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [8, 16, 24, 40, 48, 56, 88, 104, 112, 120, 136, 160, 168, 200, 216, 240, 248])
@pytest.mark.parametrize("kwargs", [dict(cap=4.0, causal=True), dict(slopes=True), dict(docs=shuffled, prefix=[3, 40])],
                         ids=lambda d: ",".join(d))
def test_attention_every_head_size(dtype, hd, kwargs):
    """Heads that end inside a slab of 64 columns or a step of 16, for the tiles and for few rows."""
    run_attention(dtype, 3, 1, hd, [(130, 130), (301, 301)], **kwargs)
    run_attention(dtype, 3, 1, hd, [(2, 400), (1, 129)], **kwargs)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group", [3, 7, 12, 33, 60, 65, 100, 127, 128])
@pytest.mark.parametrize("hd", [64, 136])
def test_attention_every_group(dtype, group, hd):
    """Row tiles of whole queries that leave rows of the tile empty."""
    run_attention(dtype, group, 1, hd, [(9, 9), (70, 200)], cap=4.0, causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kwargs", [
    {}, dict(causal=True), dict(window=0), dict(window=40), dict(causal=True, window=130), dict(cap=5.0),
    dict(slopes=True), dict(cap=3.0, slopes=True, causal=True), dict(causal=True, prefix=[0, 5, 300, 64, 1, 128]),
    dict(window=10, prefix=[1, 0, 3, 128, 129, 200]), dict(docs=runs_of(50)), dict(docs=runs_of(64, 3), prefix=[9] * 6),
    dict(docs=shuffled), dict(docs=shuffled, causal=True, prefix=[2] * 6, cap=2.0, slopes=True, window=90),
    dict(docs=lambda n: np.full(n, -1)), dict(docs=lambda n: np.full(n, 2147483647)),
], ids=lambda d: ",".join(d) or "plain")
@pytest.mark.parametrize("hq,hk,hd", [(4, 2, 64), (2, 1, 256), (6, 2, 72)])
def test_attention_masks(dtype, kwargs, hq, hk, hd):
    run_attention(dtype, hq, hk, hd, ODD, **kwargs)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens", [
    [(1, 700)], [(0, 5), (1, 1), (0, 0), (3, 0), (2, 129)], [(1, 5000), (1, 3), (4, 260)], [(7, 2)], [(200, 50), (50, 200)],
    [(0, 0)], [(1, 127), (1, 128), (1, 129), (1, 255), (1, 256), (1, 257)],
], ids=str)
@pytest.mark.parametrize("kwargs", [{}, dict(causal=True, cap=20.0), dict(window=33, slopes=True)],
                         ids=lambda d: ",".join(d) or "plain")
def test_attention_fewer_queries_than_keys(dtype, lens, kwargs):
    run_attention(dtype, 8, 2, 128, lens, **kwargs)


@pytest.mark.parametrize("dtype,hd", [("f32", 64), ("bf16", 128), ("f16", 64), ("bf16", 256)])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_attention_cut_axis(dtype, hd, rows):
    """A long axis and few rows: the plan cuts it and joins the parts."""
    plan = run_attention(dtype, 4, 1, hd, [(rows, 9001), (rows, 2000)], cap=30.0, docs=runs_of(7000, 2), prefix=[50, 50])
    # the last two queries are padding and see nothing: with fewer than three there is no axis to cut
    assert (plan.workspace_bytes > 0) == (rows > 2)
    plan = run_attention(dtype, 4, 1, hd, [(rows, 9001), (rows, 2000)], cap=30.0, docs=runs_of(7000), prefix=[50, 50])
    assert plan.workspace_bytes > 0


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("spoil", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("kwargs", [
    dict(docs=runs_of(1000, 20)), dict(causal=True, window=3, docs=runs_of(90, 7)), dict(docs=runs_of(10 ** 6, 150)),
], ids=lambda d: ",".join(d))
def test_attention_hidden_values(dtype, spoil, kwargs):
    """NaN and infinities in keys that nobody sees reach nobody, in their own tile or the next sequence's."""
    run_attention(dtype, 4, 2, 64, [(200, 200), (131, 131), (64, 64), (2, 500)], spoil=spoil, fused=False, **kwargs)
    run_attention(dtype, 2, 2, 256, [(200, 200), (131, 131), (2, 500)], spoil=spoil, fused=False, **kwargs)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("spoil", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("hq,hk,hd", [(4, 2, 64), (8, 1, 128), (2, 2, 256), (3, 1, 72)])
def test_attention_few_rows_hidden_values(dtype, spoil, hq, hk, hd):
    run_attention(dtype, hq, hk, hd, [(2, 500), (1, 131), (3, 64), (4, 1290)], spoil=spoil, docs=runs_of(90, 1), window=40)
    run_attention(dtype, hq, hk, hd, [(2, 500), (1, 131), (3, 64), (1, 129)], spoil=spoil, causal=True, window=3,
                  docs=runs_of(10 ** 6, 0))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hq,hk,hd", HEADS + [(2, 1, 512), (1, 1, 8), (32, 1, 64), (16, 1, 256), (12, 1, 128)])
@pytest.mark.parametrize("kwargs", [{}, dict(cap=4.0, slopes=True), dict(causal=True, window=200, docs=runs_of(300, 1)),
                                    dict(docs=shuffled, prefix=[3, 0, 130])], ids=lambda d: ",".join(d) or "plain")
def test_attention_few_rows(dtype, hq, hk, hd, kwargs):
    run_attention(dtype, hq, hk, hd, [(1, 700), (2, 129), (1, 1)], **kwargs)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_attention_value_seen_by_some(dtype, hd, bad):
    """A non-finite value reaches exactly the rows that see it, in its own column."""
    n, at, col = 300, 200, 5
    t = TYPES[dtype]
    x = torch.randn(n, 3 * hd, device="cuda", generator=gen(hd)).to(t)
    q, k, v = x[:, :hd], x[:, hd:2 * hd], x[:, 2 * hd:]
    v[at, col] = bad
    for causal, window in ((True, None), (False, 20), (False, None)):
        plan = AttentionPlan(1, 1, hd, [0, n], dtype=dtype, causal=causal, window=window)
        ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device="cuda")
        out = torch.empty(n, hd, device="cuda", dtype=t)
        plan.run_device(q.data_ptr(), 3 * hd, k.data_ptr(), 3 * hd, v.data_ptr(), 3 * hd, out.data_ptr(), hd,
                        workspace=ws.data_ptr(), workspace_bytes=plan.workspace_bytes, stream=stream())
        plan.check()
        p = torch.arange(n, device="cuda")
        sees = (p >= at) if causal else ((p - at).abs() <= window) if window else torch.ones_like(p, dtype=torch.bool)
        want = torch.zeros(n, hd, dtype=torch.bool, device="cuda")
        # the last eight rows alone: the kernel for few rows
        few = AttentionPlan(1, 1, hd, [0, 8], [0, n], dtype=dtype, causal=causal, window=window and 97)
        part = torch.empty(8, hd, device="cuda", dtype=t)
        ws = torch.empty(few.workspace_bytes, dtype=torch.uint8, device="cuda")
        few.run_device(q[-8:].data_ptr(), 3 * hd, k.data_ptr(), 3 * hd, v.data_ptr(), 3 * hd, part.data_ptr(), hd,
                       workspace=ws.data_ptr(), workspace_bytes=few.workspace_bytes, stream=stream())
        few.check()
        near = (p[-8:] - at <= 97) if window else torch.ones_like(p[-8:], dtype=torch.bool)
        seen = torch.zeros(8, hd, dtype=torch.bool, device="cuda")
        seen[near, col] = True
        assert torch.equal(~torch.isfinite(part.float()), seen)
        if not math.isnan(bad):
            assert (part[near, col].float() == bad).all()
        want[sees, col] = True
        assert torch.equal(~torch.isfinite(out.float()), want)
        if not math.isnan(bad):
            assert (out[sees, col].float() == bad).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_value_seen_with_a_vanishing_weight(dtype, rows):
    """An infinite value reaches the rows that see it although their weight for it is below FP32's range, in the part
    of a cut axis that holds the largest scores as in any other."""
    n, hd, col = 9001, 64, 5
    t = TYPES[dtype]
    q = torch.full((rows, hd), 8.0, device="cuda", dtype=t)
    k = torch.zeros(n, hd, device="cuda", dtype=t)
    k[-1] = 8.0  # a score of 64 * 64 / 8 = 512 against 0
    v = torch.ones(n, hd, device="cuda", dtype=t)
    v[3, col] = float("inf")
    plan = AttentionPlan(1, 1, hd, [0, rows], [0, n], dtype=dtype)
    assert plan.workspace_bytes > 0
    ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device="cuda")
    out = torch.empty(rows, hd, device="cuda", dtype=t)
    plan.run_device(q.data_ptr(), hd, k.data_ptr(), hd, v.data_ptr(), hd, out.data_ptr(), hd, workspace=ws.data_ptr(),
                    workspace_bytes=plan.workspace_bytes, stream=stream())
    plan.check()
    want = torch.zeros(rows, hd, dtype=torch.bool, device="cuda")
    want[:, col] = True
    assert torch.equal(~torch.isfinite(out.float()), want)
    assert (out[~want] == 1.0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_attention_non_finite_query_and_key(dtype):
    """A NaN query spoils its own row, a NaN key the rows that see it; nothing else."""
    n, hd = 260, 64
    x = torch.randn(n, 3 * hd, device="cuda", generator=gen(1)).to(TYPES[dtype])
    x[37, 3] = float("nan")
    x[180, hd + 9] = float("nan")
    plan = AttentionPlan(1, 1, hd, [0, n], dtype=dtype, causal=True)
    ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device="cuda")
    out, lse = torch.empty(n, hd, device="cuda", dtype=TYPES[dtype]), torch.empty(n, 1, device="cuda")
    size = x.element_size()
    plan.run_device(x.data_ptr(), 3 * hd, x.data_ptr() + hd * size, 3 * hd, x.data_ptr() + 2 * hd * size, 3 * hd,
                    out.data_ptr(), hd, lse=lse.data_ptr(), workspace=ws.data_ptr(),
                    workspace_bytes=plan.workspace_bytes, stream=stream())
    plan.check()
    p = torch.arange(n, device="cuda")
    bad = (p == 37) | (p >= 180)
    assert torch.equal(torch.isnan(out.float()).all(1), bad) and torch.equal(torch.isnan(out.float()).any(1), bad)
    assert torch.equal(torch.isnan(lse[:, 0]), bad)


@pytest.mark.parametrize("dtype,hd,pad,offset", [("f32", 64, 1, 1), ("bf16", 36, 3, 1), ("f16", 67, 5, 3), ("bf16", 64, 8, 8)])
def test_attention_strides_and_alignment(dtype, hd, pad, offset):
    run_attention(dtype, 4, 2, hd, [(33, 33), (130, 130)], pad=pad, offset=offset, fused=False)
    run_attention(dtype, 4, 2, hd, [(33, 33), (130, 130)], pad=pad, offset=offset, lse=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("by", [1e-3, 12.0])
def test_attention_flat_and_sharp_scores(dtype, by):
    run_attention(dtype, 2, 1, 128, [(150, 150)], by=by)
    run_attention(dtype, 2, 1, 128, [(150, 150)], by=by, cap=50.0, slopes=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_attention_small_caps_and_scales(dtype):
    """Caps far below and far above the scores, for both kernels of the 16-bit types."""
    for lens in ([(130, 130)], [(2, 300)]):
        for cap in (1e-6, 1e-3, 0.3, 1e6, 1e20):
            run_attention(dtype, 2, 1, 64, lens, cap=cap)
        run_attention(dtype, 2, 1, 64, lens, scale=1e-20, cap=1e-25)
        run_attention(dtype, 2, 1, 64, lens, scale=1e-6)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_attention_zero_scores_under_a_tiny_cap(dtype):
    """Zero queries: every visible key weighs the same, whatever the cap."""
    t = TYPES[dtype]
    for n_q in (3, 200):
        q, k = torch.zeros(n_q, 64, device="cuda", dtype=t), torch.randn(256, 64, device="cuda", generator=gen(2)).to(t)
        out, lse = torch.empty(n_q, 64, device="cuda", dtype=t), torch.empty(n_q, 1, device="cuda")
        plan = AttentionPlan(1, 1, 64, [0, n_q], [0, 256], dtype=dtype, scale=1.0, cap=1e-30)
        ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device="cuda")
        plan.run_device(q.data_ptr(), 64, k.data_ptr(), 64, k.data_ptr(), 64, out.data_ptr(), 64, lse=lse.data_ptr(),
                        workspace=ws.data_ptr(), workspace_bytes=plan.workspace_bytes, stream=stream())
        plan.check()
        # 256 weights of 1 (exact in every type), a sum of 256 products and a division
        want = k.double().mean(0)
        assert ((out.double() - want).abs() <= 260 * ULP * k.double().abs().mean(0) + half_step(dtype) * want.abs() +
                least_half_step(dtype)).all()
        assert ((lse.double() - math.log(256)).abs() <= 16 * ULP * math.log(256)).all()


def test_attention_group_above_a_tile():
    """130 query heads on one key head: more rows than a tensor-core tile for a single query."""
    run_attention("bf16", 130, 1, 16, [(1, 40), (3, 200)])


def attend(plan, q, k, v, hq, hd):
    out = torch.full((q.shape[0], hq * hd), 5.0, device="cuda", dtype=q.dtype)
    lse = torch.full((q.shape[0], hq), 5.0, device="cuda")
    ws = torch.full((plan.workspace_bytes,), 255, dtype=torch.uint8, device="cuda")
    plan.run_device(q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), out.data_ptr(),
                    hq * hd, lse=lse.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=plan.workspace_bytes,
                    stream=stream())
    plan.check()
    return out, lse


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hq,hk,hd", [(3, 1, 64), (5, 1, 128), (12, 1, 256), (6, 2, 72)])
@pytest.mark.parametrize("n_q,n_k", [(2, 300), (200, 200)])
@pytest.mark.parametrize("kwargs", [{}, dict(causal=True), dict(slopes=True)], ids=lambda d: ",".join(d) or "plain")
def test_capped_rows_do_not_depend_on_strangers(dtype, hq, hk, hd, n_q, n_k, kwargs):
    """The same bits whatever masked keys, the next sequence, other queries of the sequence and an earlier call hold:
    scores of their own size (about 1, far inside the cap) and of thirty times that and more (far outside)."""
    g, t = gen(11), TYPES[dtype]
    pad = 5
    q = torch.randn(2 * n_q, hq * hd, device="cuda", generator=g).to(t)
    k = torch.randn(2 * n_k, hk * hd, device="cuda", generator=g).to(t)
    v = torch.randn(2 * n_k, hk * hd, device="cuda", generator=g).to(t)
    docs = ([0] * (n_k - pad) + [-1] * pad) * 2
    slopes = [0.5 ** (h + 1) for h in range(hq)] if kwargs.get("slopes") else None
    plan = AttentionPlan(hq, hk, hd, [0, n_q, 2 * n_q], [0, n_k, 2 * n_k], dtype=dtype, cap=50.0,
                         causal=kwargs.get("causal", False), doc_q=[0] * 2 * n_q, doc_k=docs, slopes=slopes)
    before = AttentionPlan(4, 1, hd, [0, 9600], [0, 128], dtype=dtype)  # whole tiles of rows on every SM
    fill_q = torch.ones(9600, 4 * hd, device="cuda", dtype=t)
    fill_k = torch.ones(128, hd, device="cuda", dtype=t)

    def first(rows=n_q, past=0.0, **change):
        a, b, c = q.clone(), k.clone(), v.clone()
        hidden = slice(n_k - pad, n_k)
        if "hidden" in change:
            for x in (b, c):
                x[hidden] = x[hidden] * change["hidden"] if math.isfinite(change["hidden"]) else change["hidden"]
        if "next" in change:
            for x, n in ((a, n_q), (b, n_k), (c, n_k)):
                x[n:] *= change["next"]
        if "last" in change:
            a[n_q - 1] *= change["last"]
        attend(before, fill_q * past, fill_k, fill_k, 4, hd)
        out, lse = attend(plan, a, b, c, hq, hd)
        return out[:rows].clone(), lse[:rows].clone()

    for rows, change in ((n_q, dict(hidden=30.0)), (n_q, dict(hidden=float("nan"))), (n_q, dict(hidden=float("inf"))),
                         (n_q, dict(next=30.0)), (n_q, dict(past=100.0)), (n_q - 1, dict(last=30.0))):
        want, got = first(rows), first(rows, **change)
        assert torch.isfinite(want[0].float()).all()
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1]), change


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("causal,window", [(True, None), (True, 30), (False, 30), (False, None)])
def test_attention_values_seen_across_many_segments(dtype, hd, causal, window):
    """Infinite values in several sequences reach exactly the rows that see them where a block walks many segments, of one
    and of two row tiles in turn, with and without such values."""
    lens = [300, 40, 150, 7, 260, 129, 64, 20] * 75
    cu = np.concatenate([[0], np.cumsum(lens)])
    g, t = gen(hd), TYPES[dtype]
    x = torch.randn(cu[-1], 4 * hd, device="cuda", generator=g).to(t)
    q, k, v = x[:, :2 * hd], x[:, 2 * hd:3 * hd], x[:, 3 * hd:]
    rng = np.random.default_rng(hd)
    want = np.zeros((cu[-1], 2 * hd), bool)
    for s, n in enumerate(lens):
        p = np.arange(n)
        for _ in range(rng.integers(0, 4)):
            at, col = int(rng.integers(n)), int(rng.integers(hd))
            v[int(cu[s]) + at, col] = float("inf")
            sees = (p >= at) if causal else np.ones(n, bool)
            if window is not None:
                sees &= np.abs(p - at) <= window
            for h in range(2):
                want[cu[s]:cu[s + 1], h * hd + col] |= sees
    plan = AttentionPlan(2, 1, hd, cu, dtype=dtype, causal=causal, window=window)
    for _ in range(3):
        out, _ = attend(plan, q, k, v, 2, hd)
        assert torch.equal(torch.isinf(out.float()), torch.from_numpy(want).cuda())
        assert not torch.isnan(out.float()).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cap", [1e5, 1e7, 1e8, 1e9, 1e10, 1e12])
@pytest.mark.parametrize("n_q,n_k,hd", [(256, 256, 64), (256, 512, 128), (130, 256, 256), (2, 512, 128)])
def test_attention_caps_far_above_the_scores(dtype, cap, n_q, n_k, hd):
    """A cap far above every score changes nothing: cap tanh(t / cap) = t (1 - (t / cap)^2 / 3), scores here lie below
    200, and (200 / 1e5)^2 / 3 is 1.4e-6 of t, at most 2.7e-4 in a score."""
    g, t = gen(7), TYPES[dtype]
    q = (torch.randn(n_q, hd, device="cuda", generator=g) * 6).to(t)
    k = (torch.randn(n_k, hd, device="cuda", generator=g) * 6).to(t)
    v = torch.randn(n_k, hd, device="cuda", generator=g).to(t)
    out, lse = attend(AttentionPlan(1, 1, hd, [0, n_q], [0, n_k], dtype=dtype, cap=cap), q, k, v, 1, hd)
    c = dict(dtype=dtype, scale=hd ** -0.5, cap=0.0)
    qs, ks, vs = (x.cpu().double().numpy() for x in (q, k, v))
    seen, gap = visible(dict(causal=False, window=None), n_q, n_k, 0, None, None)
    want, want_lse, tol, tol_lse = attention_reference(c, qs, ks, vs, seen, gap, 0.0)
    most = np.abs(c["scale"] * qs @ ks.T).max()
    assert most < 200
    moved = most ** 3 / (3 * cap ** 2)  # of a score; a weight by twice that, out by twice that of the magnitudes
    # FP32's own score under a cap: 8 units of the score for tanh, where the general kernel's quotient t / cap rounds
    score = moved + 8 * ULP * most
    assert (np.abs(out.cpu().double().numpy() - want) <= tol + 4 * score * np.abs(vs).max()).all()
    assert (np.abs(lse[:, 0].cpu().double().numpy() - want_lse) <= tol_lse + score).all()


@pytest.mark.parametrize("dtype,by", [("f32", 3e4), ("bf16", 3e4), ("f16", 200.0)])
@pytest.mark.parametrize("n_q,n_k,hd", [(256, 256, 64), (256, 512, 128), (130, 256, 256), (2, 512, 128)])
@pytest.mark.parametrize("of_scores", [1e-3, 0.1, 1.0, 10.0])
def test_attention_large_caps_reached(dtype, by, n_q, n_k, hd, of_scores):
    """Scores of 2e6 to 1e10 and caps of that size: a weighted mean of ones is one."""
    g, t = gen(9), TYPES[dtype]
    q = (torch.randn(n_q, hd, device="cuda", generator=g) * by).to(t)
    k = (torch.randn(n_k, hd, device="cuda", generator=g) * by).to(t)
    v = torch.ones(n_k, hd, device="cuda", dtype=t)
    plan = AttentionPlan(1, 1, hd, [0, n_q], [0, n_k], dtype=dtype, scale=1.0, cap=of_scores * by * by * hd ** 0.5)
    out, lse = attend(plan, q, k, v, 1, hd)
    # weights rounded to the type before and not in their sum, n additions each, the result rounded
    tol = 2 * half_step(dtype) + 2 * (n_k + 4) * ULP
    assert ((out.double() - 1).abs() <= tol).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n_q,n_k,hd", [(256, 256, 64), (256, 512, 128), (130, 256, 256), (2, 512, 128)])
@pytest.mark.parametrize("by", [300.0, 3e3, 1.2e4])
def test_attention_scores_far_above_one(dtype, by, n_q, n_k, hd):
    """Scores of 1e6 to 1e10, where FP32 steps over whole units: a weighted mean of ones is one, and the log sum is the
    largest score."""
    g, t = gen(9), TYPES[dtype]
    q = (torch.randn(n_q, hd, device="cuda", generator=g) * by).to(t)
    k = (torch.randn(n_k, hd, device="cuda", generator=g) * by).to(t)
    v = torch.ones(n_k, hd, device="cuda", dtype=t)
    out, lse = attend(AttentionPlan(1, 1, hd, [0, n_q], [0, n_k], dtype=dtype, scale=1.0), q, k, v, 1, hd)
    tol = 2 * half_step(dtype) + 2 * (n_k + 4) * ULP
    assert ((out.double() - 1).abs() <= tol).all()
    top, size = (q.double() @ k.double().T).amax(1), (q.double().abs() @ k.double().abs().T).amax(1)
    # hd products, a scale in log2 units and back; at most n_k scores as large as the largest
    assert ((lse[:, 0].double() - top).abs() <= (hd + 8) * ULP * size + math.log(n_k)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("slope", [1e3, -1e3, 1e5, -1e5, 1e12, -1e12, 1e20, -1e20])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [2, 300])
def test_attention_steep_slopes(dtype, slope, hd, rows):
    """Slopes of any allowed size, keys near and far preferred: the mean of ones is one, the values are the preferred
    keys', and the log sum is their score and bias."""
    n_k, t = 900, TYPES[dtype]
    for docs in (None, [0] * 400 + [1] * 500):
        q = torch.randn(rows, 2 * hd, device="cuda", generator=gen(1)).to(t)
        k = torch.randn(n_k, hd, device="cuda", generator=gen(2)).to(t)
        v = torch.ones(n_k, hd, device="cuda", dtype=t)
        where = torch.arange(n_k, device="cuda") % 64  # exact in every type
        v[:, 1] = where.to(t)
        # with documents the rows are the first one's: every key that they see is far away
        plan = AttentionPlan(2, 1, hd, [0, rows], [0, n_k], dtype=dtype, slopes=[slope, slope / 4],
                             doc_q=None if docs is None else [0] * rows, doc_k=docs)
        out, lse = attend(plan, q, k, v, 2, hd)
        out = out.view(rows, 2, hd)
        tol = 2 * half_step(dtype) + 2 * (n_k + 4) * ULP
        assert ((out[..., 2:].double() - 1).abs() <= tol).all()
        p = torch.arange(n_k - rows, n_k, device="cuda")
        seen = 400 if docs else n_k
        at = p.clamp(max=seen - 1) if slope > 0 else torch.zeros_like(p)  # nearest or farthest, unless two are as far
        for h, s in enumerate((slope, slope / 4)):
            gap = (p - at).abs().double()
            score = (q.view(rows, 2, hd)[:, h].double() * k[at].double()).sum(1) * hd ** -0.5 - s * gap
            far = (gap > 0) | (slope > 0)
            err = (lse[:, h].double() - score).abs()
            assert (err[far] <= 1e-3 + 8 * ULP * abs(s) * (gap[far] + 64)).all()
            if abs(s) * (gap.max() + 64) * 16 * ULP < 1:  # FP32 tells neighbours apart: one key has all the weight
                assert (out[:, h, 1].double() - where[at].double()).abs().max() <= 64 * tol


@pytest.mark.parametrize("dtype,by", [("f32", 1.0), ("f32", 3e4), ("f32", 3e8), ("bf16", 1.0), ("bf16", 60.0), ("bf16", 3e4),
                                      ("bf16", 3e8), ("f16", 1.0), ("f16", 60.0), ("f16", 1e3)])
@pytest.mark.parametrize("n_q,n_k", [(256, 256), (2, 512)])
@pytest.mark.parametrize("of_cap", [1e-4, 1e-3, 0.01, 0.05, 0.2, 0.3, 0.34, 1.0])
def test_attention_scores_near_a_large_cap(dtype, by, n_q, n_k, of_cap):
    """Caps of any size whose scores reach a given part of them: the log sum, which is the largest score's, is off by units
    of the cap at most."""
    g, t, hd = gen(9), TYPES[dtype], 64
    q = (torch.randn(n_q, hd, device="cuda", generator=g) * by).to(t)
    k = (torch.randn(n_k, hd, device="cuda", generator=g) * by).to(t)
    s = q.double() @ k.double().T
    cap = float(np.float32(s.abs().max().item() / of_cap))
    out, lse = attend(AttentionPlan(1, 1, hd, [0, n_q], [0, n_k], dtype=dtype, scale=1.0, cap=cap), q, k, torch.ones_like(k), 1, hd)
    want = torch.logsumexp(cap * torch.tanh(s / cap), 1)
    size = (q.double().abs() @ k.double().abs().T).amax(1)
    # as in attention_reference: hd products and a scale; 8 units of the cap for tanh; 4 of the cap and of the result
    tol = (hd + 4) * ULP * size + 12 * ULP * cap + (n_k + 16) * ULP + 5 * ULP * want.abs()
    err = (lse[:, 0].double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
    assert ((out.double() - 1).abs() <= 2 * half_step(dtype) + 2 * (n_k + 4) * ULP).all()


@pytest.mark.parametrize("hd", [64, 128, 200, 256, 512])
@pytest.mark.parametrize("n_q", [1, 3, 200])
def test_attention_f32_scores_are_summed_in_parts(hd, n_q):
    """The log sum over one key is its score.  Values just above 1, whose excess a running sum near the head's size would
    lose in every step: sums of 16 products, two additions, one for each 64 dimensions and the scale's rounding."""
    value = 1.0 + 0.49 * 2.0 ** -24 * hd
    q = torch.full((n_q, hd), value, device="cuda")
    k = torch.ones(n_q, hd, device="cuda")
    cu = list(range(n_q + 1))
    out, lse = attend(AttentionPlan(1, 1, hd, cu, cu, dtype="f32", scale=1.0), q, k, k, 1, hd)
    want = hd * float(np.float32(value))
    assert ((lse.double() - want).abs() <= (16 + 2 + hd / 64 + 1) * 2.0 ** -24 * want).all()
    assert (out == 1.0).all()


FIRST_CALLS = """
import sys
sys.path.insert(0, {pkg!r})
import torch
from svl.ops import AttentionPlan, AxisRope, Q4Weight
torch.manual_seed(0)
n, hd = 200, 64
qkv = torch.randn(n, 4 * hd, device="cuda").half()
pos = torch.arange(n, device="cuda", dtype=torch.int32)
rope, plan = AxisRope(hd, [32]), AttentionPlan(2, 1, hd, [0, n], dtype="f16")
few = AttentionPlan(2, 1, hd, [0, 1], [0, n], dtype="f16")
w = Q4Weight.quantize(torch.randn(96, 2 * hd).numpy(), 32)
ws = torch.empty(max(plan.workspace_bytes, few.workspace_bytes) + 16, dtype=torch.uint8, device="cuda")
turned, out, last, y = qkv.clone(), qkv.new_empty(n, 2 * hd), qkv.new_empty(1, 2 * hd), qkv.new_empty(n, 96)

def block():
    s = torch.cuda.current_stream().cuda_stream
    a, t = qkv.data_ptr(), turned.data_ptr()
    rope.apply_device("f16", pos.data_ptr(), n, a, 4 * hd, 2, t, 4 * hd, a + 4 * hd, 4 * hd, 1, t + 4 * hd, 4 * hd, stream=s)
    plan.run_device(t, 4 * hd, t + 4 * hd, 4 * hd, t + 6 * hd, 4 * hd, out.data_ptr(), 2 * hd, workspace=ws.data_ptr(),
                    workspace_bytes=plan.workspace_bytes, stream=s)
    few.run_device(t, 4 * hd, t + 4 * hd, 4 * hd, t + 6 * hd, 4 * hd, last.data_ptr(), 2 * hd, workspace=ws.data_ptr(),
                   workspace_bytes=few.workspace_bytes, stream=s)
    w.linear_device("f16", out.data_ptr(), 2 * hd, n, y.data_ptr(), 96, stream=s)

torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):  # the process's first calls
    block()
g.replay()
torch.cuda.synchronize()
got = [x.clone() for x in (turned, out, last, y)]
block()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, (turned, out, last, y))) and bool(torch.isfinite(y).all())
print("same")
"""


def test_first_calls_inside_a_capture():
    import subprocess
    import sys
    from pathlib import Path

    pkg = str(Path(__file__).resolve().parent.parent / "seldon-vault-lite-rust_b200")
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(pkg=pkg)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_graph(dtype):
    run_attention(dtype, 4, 2, 128, [(60, 60), (1, 900)], fused=False, causal=True, graph=3)
    run_attention(dtype, 4, 1, 128, [(2, 9000)], fused=False, graph=2)


def test_attention_repeats_bit_for_bit():
    x = torch.randn(700, 4 * 128, device="cuda", generator=gen(4)).to(torch.bfloat16)
    plan = AttentionPlan(2, 1, 128, [0, 300, 700], dtype="bf16", cap=30.0)
    outs = []
    for _ in range(4):
        out = torch.empty(700, 256, device="cuda", dtype=torch.bfloat16)
        ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device="cuda")
        plan.run_device(x.data_ptr(), 512, x.data_ptr() + 512, 512, x.data_ptr() + 768, 512, out.data_ptr(), 256,
                        workspace=ws.data_ptr(), workspace_bytes=plan.workspace_bytes, stream=stream())
        outs.append(out)
    plan.check()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_attention_two_streams_and_threads():
    """One plan, two streams from two threads, each with its own workspace."""
    import threading

    plan = AttentionPlan(4, 1, 128, [0, 2], [0, 9000], dtype="f16")
    g = gen(5)
    data = [[torch.randn(n, w, device="cuda", generator=g).half() for n, w in ((2, 512), (9000, 128), (9000, 128))]
            for _ in range(2)]

    def attend(d, s):
        out = torch.empty(2, 512, device="cuda", dtype=torch.float16)
        ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device="cuda")
        for _ in range(20):
            plan.run_device(d[0].data_ptr(), 512, d[1].data_ptr(), 128, d[2].data_ptr(), 128, out.data_ptr(), 512,
                            workspace=ws.data_ptr(), workspace_bytes=plan.workspace_bytes, stream=s)
        return out, ws

    alone = [attend(d, stream())[0] for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = [None, None]

    def work(i):
        with torch.cuda.stream(streams[i]):
            got[i] = attend(data[i], streams[i].cuda_stream)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    plan.check()
    assert all(torch.equal(a, b[0]) for a, b in zip(alone, got))


def test_attention_call_refusals():
    x = torch.zeros(16, 256, device="cuda", dtype=torch.bfloat16)
    out = torch.full((16, 64), 5.0, device="cuda", dtype=torch.bfloat16)
    plan = AttentionPlan(1, 1, 64, [0, 16], dtype="bf16")
    p = x.data_ptr()
    good = dict(q=p, ld_q=256, k=p + 128, ld_k=256, v=p + 256, ld_v=256, out=out.data_ptr(), ld_out=64)
    for change in (dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(ld_q=63), dict(ld_k=8), dict(ld_v=0), dict(ld_out=32),
                   dict(q=p + 2), dict(k=p + 8), dict(ld_v=260), dict(out=out.data_ptr() + 4), dict(ld_q=1 << 36),
                   dict(lse=out.data_ptr() + 2)):
        with pytest.raises(errors.UsageError):
            plan.run_device(**{**good, **change})
    long = AttentionPlan(1, 1, 64, [0, 1], [0, 100000], dtype="bf16")
    assert long.workspace_bytes > 0
    for change in (dict(), dict(workspace=p), dict(workspace=p + 4, workspace_bytes=long.workspace_bytes),
                   dict(workspace=p, workspace_bytes=long.workspace_bytes - 1)):
        with pytest.raises(errors.UsageError):
            long.run_device(**{**good, **change})
    torch.cuda.synchronize()
    assert (out == 5.0).all()


@pytest.mark.parametrize("mode", ["global", "thread_local", "relaxed"])
@pytest.mark.parametrize("other_thread", [False, True])
def test_handles_freed_inside_a_capture(mode, other_thread):
    """The last reference to a handle may go while an unrelated graph is captured: the capture goes on."""
    import threading

    handles = [AttentionPlan(1, 1, 64, [0, 16], dtype="bf16"),
               Q4Weight.quantize(np.ones((64, 64), np.float32), 32), AxisRope(64, [32])]
    x = torch.ones(1000, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode=mode):
        y = x * 2
        if other_thread:
            t = threading.Thread(target=handles.clear)
            t.start()
            t.join()
        else:
            handles.clear()
        z = y + 1
    assert not handles
    graph.replay()
    torch.cuda.synchronize()
    assert (z == 3).all()


# --------------------------------------------------------------- together --


def test_tower_block_feeds_the_text_model(tiny_config, tiny_tensors):
    """An image's patches through 4-bit projections, two-axis rotary positions and masked attention, and the result as
    the soft tokens of a text forward: each step against 64 bits, the embedding against the same features."""
    from svl.text import TextModel

    r = np.random.default_rng(8)
    hidden, hq, hk, hd, patches = tiny_config.hidden_size, 4, 2, 32, 30
    width = 64
    w_qkv = Q4Weight.quantize(r.standard_normal(((hq + 2 * hk) * hd, width), dtype=np.float32) * 0.2, 32)
    w_o = Q4Weight.quantize(r.standard_normal((hidden, hq * hd), dtype=np.float32) * 0.2, 32, asymmetric=True)
    x = torch.from_numpy(r.standard_normal((patches, width), dtype=np.float32)).cuda()
    pos = torch.stack([torch.arange(patches) // 6, torch.arange(patches) % 6]).int().cuda()
    qkv = torch.empty(patches, (hq + 2 * hk) * hd, device="cuda")
    att = torch.empty(patches, hq * hd, device="cuda")
    feats = torch.empty(patches, hidden, device="cuda")
    rope = AxisRope(hd, [8, 8], [100.0, 100.0])
    docs = [0] * 20 + [1] * 8 + [-1] * 2  # two images and padding
    plan = AttentionPlan(hq, hk, hd, [0, patches], dtype="f32", cap=50.0, doc_q=docs)
    ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device="cuda")
    s, ld, f4 = stream(), qkv.shape[1], 4

    def block():
        w_qkv.linear_device("f32", x.data_ptr(), width, patches, qkv.data_ptr(), ld, stream=s)
        q, k, v = qkv.data_ptr(), qkv.data_ptr() + hq * hd * f4, qkv.data_ptr() + (hq + hk) * hd * f4
        rope.apply_device("f32", pos.data_ptr(), patches, q, ld, hq, q, ld, k, ld, hk, k, ld, stream=s)
        plan.run_device(q, ld, k, ld, v, ld, att.data_ptr(), hq * hd, workspace=ws.data_ptr(),
                        workspace_bytes=plan.workspace_bytes, stream=s)
        w_o.linear_device("f32", att.data_ptr(), hq * hd, patches, feats.data_ptr(), hidden, stream=s)

    block()
    plan.check()
    full = [dequantised(c, as_bf16(b), z, 32) for c, b, z in (w_qkv.read(), w_o.read())]
    want = x.cpu().double().numpy() @ full[0].T
    turned, _ = rope_reference(torch.from_numpy(want[:, :(hq + hk) * hd]).view(patches, -1, hd), pos.cpu(), [8, 8],
                               [100.0, 100.0], "split")
    turned = turned.reshape(patches, -1).numpy()
    c = dict(dtype="f32", scale=hd ** -0.5, cap=50.0, causal=False, window=None)
    d = np.array(docs)
    seen, gap = visible(c, patches, patches, 0, d, d)
    o = np.zeros((patches, hq * hd))
    for h in range(hq):
        kv = h // (hq // hk)
        o[:, h * hd:(h + 1) * hd] = attention_reference(
            c, turned[:, h * hd:(h + 1) * hd], turned[:, (hq + kv) * hd:(hq + kv + 1) * hd],
            want[:, (hq + hk + kv) * hd:(hq + hk + kv + 1) * hd], seen, gap, 0.0)[0]
    final = o @ full[1].T
    # FP32 throughout: scores of about 10 with 64 + 32 roundings each, then two sums of 64 and 128 terms
    scale = np.abs(o).max() * np.abs(full[1]).sum(1).max()
    assert np.abs(feats.cpu().double().numpy() - final).max() <= 2000 * ULP * scale
    assert (att[28:] == 0).all()
    # the same block captured: q and k are rotated in place, so the capture starts from the projection again
    eager = feats.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        s = stream()
        block()
    feats.fill_(7.0)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(feats, eager)
    model = TextModel(tiny_config, tiny_tensors)
    ids = [2] + [tiny_config.pad_token_id or 0] * 28 + [1]
    a = model.forward_with_features(ids, feats[:28].cpu().numpy(), 1, 28).normalized()
    b = model.forward_with_features(ids, final[:28].astype(np.float32), 1, 28).normalized()
    assert np.isfinite(a).all() and float(a.astype(np.float64) @ b) >= 0.9999
