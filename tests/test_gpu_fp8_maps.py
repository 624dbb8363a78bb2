"""The 8-bit maps on matrices large enough for four blocks a thread, and what a row's codes depend on.

A map works on each row's block of 128 by itself, so a large matrix gives bit for bit what
its strips of rows give one by one (which take one block a thread), and sampled rows are
held against the restatement in 64 bits as the small sizes are: codes and scales of an input
bit for bit, an activation's up to ties, a derivative within 1e-5 |g| (2^-8 more in bf16)."""
from __future__ import annotations

import numpy as np
import pytest

import fp8_reference as ref
from test_gpu_fp8 import ACT, CLIP, SLOPE, assert_codes_of, held, matrix, rng_of, upload_held, values

pytestmark = pytest.mark.gpu

# Four blocks a thread from 4 x 256 workgroups of 16 rows x 4 blocks on: whole 128-byte lines
# (streamed past the caches), lines of odd lengths, a part group of blocks, a ragged last strip.
SHAPES = [(16400, 512), (16399, 500), (8200, 640), (2051, 4100)]
STRIP = 1024


def strips(rows):
    return [(r, min(rows, r + STRIP)) for r in range(0, rows, STRIP)]


def sample(rng, rows):
    return np.unique(np.concatenate([np.arange(24), np.arange(rows - 24, rows), rng.integers(0, rows, 200)]))


def rows_of(t, r0, r1):
    """Rows r0 .. r1 of a device matrix, in place."""
    return t.sub(r0 * t.shape[1], (r1 - r0, t.shape[1]))


def codes_of(ca, t):
    return t.codes.numpy(), t.scales.numpy()


def joined(parts, rows):
    """The codes and scales of a matrix from those of its strips (1024 rows: whole groups of 16 scales)."""
    return np.concatenate([c for c, _ in parts]), np.concatenate([s for _, s in parts], axis=1)


def assert_same(t, parts, what):
    codes, scales = joined(parts, t.shape[0])
    assert np.array_equal(t.codes.numpy(), codes), what
    assert np.array_equal(t.scales.numpy(), scales), what


def pick(t, rows):
    """(codes, scales) of some rows, as a small matrix holds them."""
    codes, scales = t.codes.numpy()[rows], t.scales.numpy()[:, rows]
    full = np.full((scales.shape[0], ref.up(len(rows), 16)), 127, np.uint8)
    full[:, : len(rows)] = scales
    return codes, full


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_and_back(hip, rows, cols, dtype):
    rng = rng_of("large quantise", rows, cols, dtype)
    x, x64 = matrix(rng, rows, cols, dtype)
    t = hip.quantize_fp8(x)
    assert_same(t, [codes_of(hip, hip.quantize_fp8(rows_of(x, *r))) for r in strips(rows)], "strips")
    at = sample(rng, rows)
    codes, scales = ref.quantize(x64[at])
    assert all(np.array_equal(a, b) for a, b in zip(pick(t, at), (codes, scales)))
    assert (t.scales.numpy()[:, rows:] == 127).all()  # the padded rows' scale is 1
    for out in ("f32", "bf16"):
        back = values(hip.dequantize_fp8(t, out))
        assert np.array_equal(back, held(t)), out


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["relu", "sigmoid", "tanh"])
def test_activation(hip, rows, cols, dtype, act):
    rng = rng_of("large act", rows, cols, act)
    z, z64 = matrix(rng, rows, cols, dtype, 2.0)
    at = sample(rng, rows)
    fn = {"relu": hip.relu_fp8, "sigmoid": hip.sigmoid_fp8, "tanh": hip.tanh_fp8}[act]
    small = [fn(rows_of(z, *r)) for r in strips(rows)]
    if act == "relu":
        h8 = fn(z)
        assert_same(h8, [codes_of(hip, s) for s in small], "strips")
        assert all(np.array_equal(a, b) for a, b in zip(pick(h8, at), ref.quantize(ACT[act](z64[at]), keep_positive=True)))
        return
    h8, z8 = fn(z)
    alone, none = fn(z, save=False)
    assert none is None and np.array_equal(alone.codes.numpy(), h8.codes.numpy())
    assert np.array_equal(alone.scales.numpy(), h8.scales.numpy())
    assert_same(h8, [codes_of(hip, s[0]) for s in small], "h, strips")
    assert_same(z8, [codes_of(hip, s[1]) for s in small], "z, strips")
    part = hip.empty_fp8((len(at), cols))
    for a, b in zip((part.codes, part.scales), pick(h8, at)):
        a.upload(b)
    assert_codes_of(part, ACT[act](z64[at]).astype(np.float32).astype(np.float64), f"{act} h")
    assert all(np.array_equal(a, b) for a, b in zip(pick(z8, at), ref.quantize(np.clip(z64[at], -CLIP[act], CLIP[act]))))
    for t in (h8, z8):
        assert (t.codes.numpy()[:, cols:] == 0).all() and (t.scales.numpy()[:, rows:] == 127).all()


def assert_derivative_codes(dz8, dz, want, tol, what):
    """dz8 (codes, scales) holds want to tol: its scales are the least that hold the largest value, one binade
    off only where that value is within tol of the edge between two; its codes the nearest to a value within
    tol of want; its padding 0.  Of an f32 dz it holds just that dz."""
    codes, scales = dz8
    rows, cols = want.shape
    pitch = codes.shape[1]
    assert (codes[:, cols:] == 0).all() and (scales[:, rows:] == 127).all(), what
    if dz is not None:
        rc, rs = ref.quantize(dz)
        assert np.array_equal(scales, rs) and np.array_equal(codes, rc), what
        return
    def tops(v):
        full = np.zeros((rows, pitch))
        full[:, :cols] = v
        return full.reshape(rows, pitch // 128, 128).max(axis=2).T
    low, high = tops(np.maximum(np.abs(want) - tol, 0)), tops(np.abs(want) + tol)
    got = scales[:, :rows].astype(int) - 127
    zero = high == 0  # a block of zeros has the scale 1; one that may be zero, any up to its largest's
    least = np.where(low > 0, ref.exponents(low), -126)
    assert np.where(zero, got == 0, (least <= got) & (got <= ref.exponents(high)) | (low == 0) & (got == 0)).all(), what
    s = np.repeat(2.0 ** got.T, 128, axis=1)[:, :cols]
    q, step = ref.VALUES[codes[:, :cols]], np.maximum(np.abs(want) / s, 2.0**-6)
    half = 2.0 ** (np.floor(np.log2(step)) - 4)  # half the distance between codes there
    assert (np.abs(q * s - want) <= half * s * (1 + 1e-6) + tol).all(), what


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["relu", "sigmoid", "tanh"])
def test_derivative(hip, rows, cols, dtype, act):
    rng = rng_of("large bwd", rows, cols, act)
    z = matrix(rng, rows, cols, std=3.0)[0]
    save = {"relu": lambda v: hip.relu_fp8(v), "sigmoid": lambda v: hip.sigmoid_fp8(v)[1],
            "tanh": lambda v: hip.tanh_fp8(v)[1]}[act]
    fn = {"relu": hip.relu_bwd_fp8, "sigmoid": hip.sigmoid_bwd_fp8, "tanh": hip.tanh_bwd_fp8}[act]
    z8 = save(z)
    g, g64 = matrix(rng, rows, cols, dtype, 0.01)
    dz, dz8 = fn(z8, g)
    small = [fn(save(rows_of(z, *r)), rows_of(g, *r)) for r in strips(rows)]
    assert np.array_equal(dz.numpy(), np.concatenate([d.numpy() for d, _ in small]))
    assert_same(dz8, [codes_of(hip, d) for _, d in small], "strips")
    at = sample(rng, rows)
    z64 = ref.dequantize(*pick(z8, at), cols)
    want = g64[at] * SLOPE[act](z64)
    tol = 1e-5 * np.abs(g64[at])
    got = values(dz)[at]
    assert (np.abs(got - want) <= tol + (2.0**-8 * np.abs(want) if dtype == "bf16" else 0.0)).all()
    assert_derivative_codes(pick(dz8, at), got if dtype == "f32" else None, want, tol, act)
    alone, none = fn(z8, g, codes=False)
    assert none is None and np.array_equal(alone.numpy(), dz.numpy())
    fn(z8, g, out=g)  # in place
    assert np.array_equal(g.numpy(), dz.numpy())


@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 127), (3, 129), (17, 300), (130, 1000)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["relu", "sigmoid", "tanh"])
def test_derivative_scales_and_padding(hip, rows, cols, dtype, act):
    rng = rng_of("bwd scales", rows, cols, act)
    z64 = matrix(rng, rows, cols, std=3.0)[1]
    z64 = np.maximum(z64, 0) if act == "relu" else np.clip(z64, -CLIP[act], CLIP[act])
    z8, z64 = upload_held(hip, z64)
    g, g64 = matrix(rng, rows, cols, dtype, 0.01)
    dz, dz8 = {"relu": hip.relu_bwd_fp8, "sigmoid": hip.sigmoid_bwd_fp8, "tanh": hip.tanh_bwd_fp8}[act](z8, g)
    assert_derivative_codes(codes_of(hip, dz8), values(dz) if dtype == "f32" else None, g64 * SLOPE[act](z64),
                            1e-5 * np.abs(g64), act)


@pytest.mark.parametrize("act", ["sigmoid", "tanh"])
@pytest.mark.parametrize("other", [100.0, -100.0, np.inf, -np.inf, np.nan])
def test_a_row_does_not_depend_on_the_others(hip, act, other):
    # 2^25 values of every magnitude, each fourth row's neighbours put past the clip: any dependence on the way
    # that the others take (an ulp apart in f32) would flip the code of some value near a tie
    rows, cols = 1 << 16, 512
    rng = rng_of("neighbours", act)
    z = (rng.uniform(-20, 20, (rows, 1)) + rng.uniform(-1, 1, (rows, cols))).astype(np.float32)
    fn = {"sigmoid": hip.sigmoid_fp8, "tanh": hip.tanh_fp8}[act]
    before = fn(hip.from_numpy(z))
    z[3::4, 5] = other
    after = fn(hip.from_numpy(z))
    keep = np.arange(rows) % 4 != 3
    for a, b in zip(before, after):
        assert np.array_equal(a.codes.numpy()[keep], b.codes.numpy()[keep])
        assert np.array_equal(a.scales.numpy()[:, keep], b.scales.numpy()[:, keep])


def test_sigmoid_of_large_negative_arguments(hip):
    # blocks of e^z down to f32's subnormals, at their own scales (2^-126 at the least)
    z = np.repeat(np.linspace(-60.0, -115.0, 56), 128).reshape(56, 128).astype(np.float32)
    z += np.linspace(0, 0.5, 128, dtype=np.float32)
    h8 = hip.sigmoid_fp8(hip.from_numpy(z), save=False)[0]
    z64 = z.astype(np.float64)
    want = np.exp(z64) / (1 + np.exp(z64))
    scales = h8.scales.numpy()[:, :56]
    s = 2.0 ** (scales.T.astype(np.float64) - 127)
    # of the exponent -z log2(e), up to 166: its rounding and the constant's, 2^-17 and 166 2^-25, and an ulp of
    # exp2 and of the reciprocal: 1.5e-5 of the value, and the steps of the subnormals; then half a code's step
    tol = 1.5e-5 * want + 2.0**-149
    low, high = (want - tol).max(axis=1), (want + tol).max(axis=1)
    got = scales[0].astype(int) - 127  # a block of zeros, as e^z below 2^-149 may give, has the scale 1
    least = np.where(low > 0, ref.exponents(low), -126)
    assert ((least <= got) & (got <= ref.exponents(high)) | (low <= 0) & (got == 0)).all()
    step = np.maximum(2.0 ** (np.floor(np.log2(np.maximum(want / s, 2.0**-6))) - 3), 2.0**-9)
    assert (np.abs(held(h8) - want) <= step * s / 2 * (1 + 1e-6) + tol).all()


@pytest.mark.parametrize("act,top", [("sigmoid", 0.25), ("tanh", 1.0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_derivative_is_at_most_its_largest(hip, act, top, dtype):
    # z near 0, where the slope is its largest but for less than f32 holds: every code at scales down to 2^-40.
    # g = 1.75 puts the largest dz of each block (z = 0) on the edge between two scales: an ulp more doubles it.
    codes = np.zeros((40, 256), np.uint8)
    codes[:, :127], codes[:, 128:255] = np.arange(127), 128 + np.arange(127)
    scales = np.full((2, 48), 127, np.uint8)
    scales[:, :40] = 127 - 8 - np.arange(40)  # |z| up to 1.75 2^0, 2^-1, ...
    z8 = hip.empty_fp8((40, 256))
    z8.codes.upload(codes)
    z8.scales.upload(scales)
    g = np.full((40, 256), 1.75, np.float32)
    dz, dz8 = {"sigmoid": hip.sigmoid_bwd_fp8, "tanh": hip.tanh_bwd_fp8}[act](
        z8, hip.from_numpy(g if dtype == "f32" else ref.to_bf16(g), dtype))
    assert (values(dz) <= 1.75 * top).all()
    assert (dz8.scales.numpy()[:, :40].astype(int) - 127 == ref.exponents(np.array(1.75 * top))).all()
    z64 = held(z8)
    assert (np.abs(held(dz8) - 1.75 * SLOPE[act](z64)) <= 1.75 * top / 16 + 1e-5).all()
