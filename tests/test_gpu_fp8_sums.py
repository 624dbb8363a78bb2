"""What the 8-bit products round on the way to their sums, as the header states it.

  f32 results, bf16 ones of up to 32 rows   f32 sums of the exact products: small products
                                            survive beside large ones that cancel
  bf16 results of more than 32 rows         of each 8 consecutive k, every product is cut off
                                            below 2^-13 of the largest (a code below 2^-6
                                            counts as 2^-6), at most 7 of them; sums rounded
                                            down, one f32 step (2^-23 of at most sum |a||b|)
                                            for each 8 and for each joined slice; the result is
                                            the nearest bf16 to a value within that of a b

and, exactly, on small integers: with products up to 64 of at least 1 nothing is cut off and
every partial sum is a whole number below 2^24, so each k, lane, tile and ragged edge has to
be in its place once."""
from __future__ import annotations

import numpy as np
import pytest

import fp8_reference as ref
from test_gpu_fp8 import rng_of, upload_held, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("trans_b", [False, True])
@pytest.mark.parametrize("M,dtype", [(1, "bf16"), (4, "bf16"), (16, "bf16"), (17, "bf16"), (32, "bf16"),
                                     (3, "f32"), (48, "f32"), (1500, "f32")])
def test_full_sums_keep_small_products_beside_cancelling_ones(hip, M, dtype, trans_b):
    K, N = 300, 200 if M < 1500 else 1400
    a, b = np.zeros((M, K)), np.zeros((K, N))
    a[:, 0] = a[:, 1] = 256.0
    b[0], b[1] = 256.0, -256.0  # 2^16 - 2^16, at a scale of 1
    a[:, 2:8] = 2.0 ** -(np.arange(M)[:, None] % 5)
    b[2:8] = 0.25  # six products from 2^-2 down to 2^-6: 2^-18 to 2^-22 of the large ones
    qa, a64 = upload_held(hip, a)
    qb, b64 = upload_held(hip, np.ascontiguousarray(b.T) if trans_b else b, 128)
    assert np.array_equal(a64, a) and np.array_equal(b64.T if trans_b else b64, b)
    assert np.array_equal(values(hip.matmul_fp8(qa, qb, trans_b=trans_b, dtype=dtype)), a @ b)


def cut_off(a8, b8, K):
    """The least and the largest bf16 that every element of a8 b8 may be (M x K, K x N: (codes' values, scales))."""
    (ac, ae), (bc, be) = a8, b8
    a, b = ac * ae, bc * be
    want, den = a @ b, np.abs(a) @ np.abs(b)
    big_a, big_b = np.maximum(np.abs(ac), 2.0**-6) * ae, np.maximum(np.abs(bc), 2.0**-6) * be
    lost = np.zeros(want.shape)
    for k in range(0, K, 8):  # no 8 lie across two blocks
        top = np.zeros(want.shape)
        for i in range(k, min(k + 8, K)):
            np.maximum(top, big_a[:, i, None] * big_b[i], out=top)
        lost += top
    err = 7 * 2.0**-13 * lost + (K / 8 + 32) * 2.0**-23 * den
    # rounding keeps the order: the ends of the range, outwards to f32, rounded as the result is
    low = np.nextafter((want - err).astype(np.float32), np.float32(-np.inf))
    high = np.nextafter((want + err).astype(np.float32), np.float32(np.inf))
    return ref.from_bf16(ref.to_bf16(low)), ref.from_bf16(ref.to_bf16(high))


def parts(x, block_rows=1):
    """(the codes' values, their scales) of x in 8 bits, each of x's shape."""
    codes, scales = ref.quantize(x, block_rows)
    s = 2.0 ** (scales[:, : x.shape[0]].T.astype(np.float64) - 127)
    return ref.VALUES[codes][:, : x.shape[1]], np.repeat(s, 128, axis=1)[:, : x.shape[1]]


# one for each way of a bf16 result past 32 rows: 64 x 64 tiles, K in slices, 128 x 128, 256 x 256 in one round and in two
@pytest.mark.parametrize("M,N,K", [(33, 70, 300), (64, 64, 4100), (1500, 1400, 203), (2900, 2817, 130), (4500, 4700, 130)])
@pytest.mark.parametrize("trans_b", [False, True])
def test_bf16_sums_lose_no_more_than_stated(hip, M, N, K, trans_b):
    # magnitudes over many binades, and columns of a that cancel against each other
    rng = rng_of("cut", M, N, K, trans_b)
    a = rng.standard_normal((M, K)) * np.exp(rng.uniform(-6, 2, (1, K)))
    b = rng.standard_normal((K, N)) * np.exp(rng.uniform(-3, 3, (K, 1)))
    a[:, 8:K - 8:16] = a[:, 9:K - 7:16]
    b[8:K - 8:16] = -b[9:K - 7:16] * (1 + 2.0**-3 * rng.integers(0, 2, (len(range(8, K - 8, 16)), 1)))
    b = np.ascontiguousarray(b.T) if trans_b else b
    a8, b8 = upload_held(hip, a)[0], upload_held(hip, b, 128)[0]
    got = values(hip.matmul_fp8(a8, b8, trans_b=trans_b, dtype="bf16"))
    pa, pb = parts(a), parts(b, 128)
    if trans_b:
        pb = tuple(p.T for p in pb)
    rows = np.unique(np.concatenate([np.arange(min(M, 20)), np.arange(M - 20, M), rng.integers(0, M, 20)]))
    cols = np.unique(np.concatenate([np.arange(min(N, 20)), np.arange(N - 20, N), rng.integers(0, N, 20)]))
    for r, c in ((rows, np.arange(N)), (np.arange(M), cols)):
        low, high = cut_off(tuple(p[r] for p in pa), tuple(p[:, c] for p in pb), K)
        some = got[np.ix_(r, c)]
        assert ((low <= some) & (some <= high)).all()


INTEGERS = [(33, 70, 300), (100, 130, 129), (64, 64, 8192), (100, 200, 2100), (1000, 33, 2049),  # 64 x 64, whole and in slices
            (1500, 1400, 700), (1409, 1537, 200),                                               # 128 x 128
            (2817, 3001, 300), (2900, 2817, 8300),               # 256 x 256, a tile a workgroup; past 64 k-blocks
            (4500, 4700, 300), (4353, 4097, 129), (4200, 4300, 8333),   # several tiles a workgroup, edges after whole ones
            (8192, 8192, 256), (12288, 5632, 384)]               # ... and C of 128 MiB and more, in whole lines


@pytest.mark.parametrize("M,N,K", INTEGERS)
@pytest.mark.parametrize("trans_b", [False, True])
def test_bf16_results_of_integers_are_exact(hip, M, N, K, trans_b):
    rng = rng_of("bf16 integers", M, N, K, trans_b)
    a = rng.integers(-8, 9, (M, K)).astype(np.float32)
    b = rng.integers(-8, 9, (K, N)).astype(np.float32)
    a8 = hip.quantize_fp8(hip.from_numpy(a))
    b8 = hip.quantize_fp8(hip.from_numpy(np.ascontiguousarray(b.T) if trans_b else b), 128)
    first = hip.matmul_fp8(a8, b8, trans_b=trans_b, dtype="bf16").numpy()
    assert np.array_equal(first, ref.to_bf16(a @ b))  # an f32 product of whole numbers below 2^24: exact in any order
    assert np.array_equal(first, hip.matmul_fp8(a8, b8, trans_b=trans_b, dtype="bf16").numpy())


@pytest.mark.parametrize("M,N,K", [(140, 260, 300), (1500, 1400, 130), (2900, 2817, 300), (4500, 4700, 200)])
@pytest.mark.parametrize("trans_b", [False, True])
def test_bf16_nan_stays_in_its_row_and_column(hip, M, N, K, trans_b):
    rng = rng_of("bf16 nan", M, N, K)
    a = rng.standard_normal((M, K), np.float32)
    b = rng.standard_normal((K, N), np.float32)
    a[3, K - 1] = a[M - 1, 0] = np.nan
    b[K - 1, N - 1] = b[0, 5] = np.nan
    a8 = hip.quantize_fp8(hip.from_numpy(a))
    b8 = hip.quantize_fp8(hip.from_numpy(np.ascontiguousarray(b.T) if trans_b else b), 128)
    c = values(hip.matmul_fp8(a8, b8, trans_b=trans_b, dtype="bf16"))
    want = np.zeros((M, N), bool)
    want[[3, M - 1]] = True
    want[:, [5, N - 1]] = True
    assert np.array_equal(np.isnan(c), want)


@pytest.mark.parametrize("trans_b", [False, True])
def test_several_tiles_a_workgroup_into_offset_memory(hip, trans_b):
    # C on no 16-byte boundary and of whole 128-byte lines' length: its neighbours stay, and it is not streamed
    M, N, K = 8192, 8192, 128
    rng = rng_of("offset walk", trans_b)
    a = rng.integers(-8, 9, (M, K)).astype(np.float32)
    b = rng.integers(-8, 9, (K, N)).astype(np.float32)
    a8 = hip.quantize_fp8(hip.from_numpy(a))
    b8 = hip.quantize_fp8(hip.from_numpy(np.ascontiguousarray(b.T) if trans_b else b), 128)
    raw = hip.from_numpy(np.full(M * N + 2, 0x40E0, np.uint16), "bf16")
    hip.matmul_fp8(a8, b8, trans_b=trans_b, out=raw.sub(1, (M, N)))
    got = raw.numpy()
    assert got[0] == 0x40E0 and got[-1] == 0x40E0
    assert np.array_equal(got[1:-1].reshape(M, N), ref.to_bf16(a @ b))
