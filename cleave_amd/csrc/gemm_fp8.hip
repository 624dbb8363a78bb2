// gemm_fp8.hip -- entry points of the 8-bit products: matmul_fp8, linear_fp8
// (quantise, then the product) and weight_grad_fp8 (the product that reads a
// layer's saved input), and which kernel takes a product.
#include <algorithm>

#include "gemm_fp8_grad.hpp"
#include "gemm_fp8_pingpong.hpp"
#include "gemm_fp8_rows.hpp"
#include "gemm_fp8_tiled.hpp"

namespace ch {
// c[i] = part[i] + part[stride + i] + ..., S slices in order (gemm_f32.hip).
int32_t sum_slices_f32(const float* part, float* c, int64_t n, int S, int64_t stride);
}  // namespace ch

#define CH_OK(expr)                           \
    do {                                      \
        int32_t _st = (expr);                 \
        if (_st != CLEAVE_HIP_OK) return _st; \
    } while (0)

namespace {

using namespace ch::fp8;

constexpr int kMaxPitch = 1 << 23;
constexpr int kHeldSlot = 13;  // scratch: an input quantised on the way, or dequantised
constexpr int kPartSlot = 14;  // scratch: sums of slices of K

// A C of whole 128-byte lines and at least this size is stored non-temporally:
// alone, 65536 x 4096 x 1024 (512 MiB) 282 -> 266 us and 8192^3 (128 MiB) 377 ->
// 367; in a loop, where power bounds both, level.
constexpr int64_t kNtStoreBytes = 128ll << 20;

// At least half a round of 256 x 256 tiles: the ping-pong kernel.
template <bool NT>
bool launch_pingpong(const Operands& o, uint16_t* c) {
    const int tiles_m = ch::tiles_of(o.M, 256), tiles_n = ch::tiles_of(o.N, 256);
    const int64_t tiles = (int64_t)tiles_m * tiles_n;
    if (tiles * 2 < ch::num_cus() || tiles > INT32_MAX / 2) return false;
    // one workgroup per CU (its LDS); a multiple of 8 keeps a workgroup's tiles on one XCD
    const int64_t resident = ch::num_cus() / 8 * 8;
    const int nt_c = (int64_t)o.M * o.N * 2 >= kNtStoreBytes && o.N % 64 == 0 && ((uintptr_t)c & 127) == 0;
    const unsigned grid = (unsigned)(tiles < resident ? tiles : resident);
    if constexpr (!NT) {
        if (o.K % PingPong::BK) {
            gemm_fp8_pingpong_kernel<false, true><<<grid, 512, 0, ch::stream()>>>(o, c, tiles_m, tiles_n, nt_c);
            return true;
        }
    }
    gemm_fp8_pingpong_kernel<NT, false><<<grid, 512, 0, ch::stream()>>>(o, c, tiles_m, tiles_n, nt_c);
    return true;
}

template <bool NT, bool WIDE, class T, int BM, int BN, int TM, int S>
int32_t launch_tiled(const char* fn, const Operands& o, T* c, int slices = 1, int64_t part = 0) {
    using P = Tiled<BM, BN, TM, S>;
    const int tiles_m = ch::tiles_of(o.M, BM), tiles_n = ch::tiles_of(o.N, BN);
    const int64_t blocks = (int64_t)tiles_m * tiles_n * slices;
    static_assert(P::THREADS <= 256, "what kMaxBlocks counts");
    CH_REQUIRE(blocks <= ch::kMaxBlocks, "%s: %d x %d is more than one launch covers", fn, o.M, o.N);
    const unsigned grid = (unsigned)blocks;
    if constexpr (!NT) {
        if (o.K % P::BK) {
            gemm_fp8_tiled_kernel<false, true, WIDE, T, BM, BN, TM, S>
                <<<grid, P::THREADS, 0, ch::stream()>>>(o, c, tiles_m, tiles_n, slices, part);
            CH_LAUNCHED(fn);
            return CLEAVE_HIP_OK;
        }
    }
    gemm_fp8_tiled_kernel<NT, false, WIDE, T, BM, BN, TM, S>
        <<<grid, P::THREADS, 0, ch::stream()>>>(o, c, tiles_m, tiles_n, slices, part);
    CH_LAUNCHED(fn);
    return CLEAVE_HIP_OK;
}

// c[i] = the slices' f32 sums of element i, added in order.
template <class T>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* __restrict__ part, T* __restrict__ c, int64_t n,
                                                        int slices, int64_t stride) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float y = part[i];
        for (int s = 1; s < slices; ++s) y += part[s * stride + i];
        store_c(c, i, y);
    }
}

template <bool NT, class T>
int32_t launch_layout(const char* fn, const Operands& o, T* c) {
    if constexpr (sizeof(T) == 2) {
        if (launch_pingpong<NT>(o, c)) {
            CH_LAUNCHED(fn);
            return CLEAVE_HIP_OK;
        }
    }
    constexpr bool WIDE = sizeof(T) == 4;
    auto tiles = [&](int bm, int bn) { return (int64_t)ch::tiles_of(o.M, bm) * ch::tiles_of(o.N, bn); };
    const int64_t cus = ch::num_cus();
    // Two rounds of 256 x 128 tiles, f32 results (so many of bf16 are the ping-pong
    // kernel's): they read half the operand bytes of 128 x 128 (us: 4096^3 120 against
    // 128, 8192^2 x 1024 151 and 163); below, the smaller tiles lose less to a
    // part-filled round (3000 x 4000 x 2000 56 against 53, 2900^2 x 1000 34 and 32).
    if constexpr (WIDE) {
        if (tiles(256, 128) >= 2 * cus) return launch_tiled<NT, WIDE, T, 256, 128, 128, 3>(fn, o, c);
    }
    // Half a round of 128 x 128 tiles, or 64 x 64 (128 against 64, us: 2048^3 f32 24
    // and 31, 1500^3 bf16 15 and 17; below, 512^2 x 4096 21 and 14, 64 x 4096^2 20
    // and 12, 1000^3 11.4 and 9.8).
    if (tiles(128, 128) * 2 >= cus) return launch_tiled<NT, WIDE, T, 128, 128, 64, 4>(fn, o, c);
    // Tiles that leave CUs without one: K in slices of at least 8 blocks, less than
    // which the second launch outweighs (whole against sliced, us: 300 x 500 x 16384
    // 36 and 17, 128^2 x 16384 f32 67 and 15, 33 x 4096^2 f32 21 and 13, 512^2 x 4096
    // 13.6 and 12; two slices of 4 blocks, 1000^3: 9.8 and 14).
    const int64_t count = tiles(64, 64), nkb = pitch_of(o.K) / kBlock;
    const int64_t slices = std::min(cus / count, nkb / 8);
    if (slices <= 1) return launch_tiled<NT, WIDE, T, 64, 64, 32, 6>(fn, o, c);
    const int64_t n = (int64_t)o.M * o.N;
    float* const part = (float*)ch::scratch(kPartSlot, sizeof(float) * (size_t)(n * slices));
    if (!part) return CLEAVE_HIP_ERR_OOM;
    CH_OK((launch_tiled<NT, WIDE, float, 64, 64, 32, 6>(fn, o, part, (int)slices, n)));
    sum_parts_kernel<T><<<(unsigned)std::min<int64_t>((n + 255) / 256, 16 * cus), 256, 0, ch::stream()>>>(
        part, c, n, (int)slices, n);
    CH_LAUNCHED(fn);
    return CLEAVE_HIP_OK;
}

// Products of up to kFewRows rows.
constexpr int kFewRows = 32;
template <bool NT, class X, class T>
int32_t launch_rows(const char* fn, const RowsIn<X>& in, const Operands& o, T* c) {
    using P = Rows<NT>;
    // Fewer column groups than CUs: K cut into slices that fill them, each with a
    // k-block for every wave.
    const int64_t groups = ((int64_t)o.N + P::COLS - 1) / P::COLS, cus = ch::num_cus();
    const int64_t nkb = pitch_of(o.K) / kBlock;
    int64_t slices = 1;
    if (groups <= kMaxSliced) slices = std::min<int64_t>(cus / groups, nkb / P::NW);
    const int fr = o.M <= 16 ? 1 : 2;
    float* part = nullptr;
    if (slices > 1) {
        part = (float*)ch::scratch(kPartSlot, sizeof(float) * (size_t)(groups * slices * fr * 16 * P::COLS));
        if (!part) return CLEAVE_HIP_ERR_OOM;
    } else {
        slices = 1;
    }
    const dim3 grid((unsigned)groups, (unsigned)slices);
    if constexpr (sizeof(X) != 1) {
        if (o.M <= kSegRows) {
            gemm_fp8_rows_kernel<NT, 0, X, T><<<grid, P::THREADS, 0, ch::stream()>>>(in, o, c, part);
            CH_LAUNCHED(fn);
            return CLEAVE_HIP_OK;
        }
    }
    if (fr == 1) gemm_fp8_rows_kernel<NT, 1, X, T><<<grid, P::THREADS, 0, ch::stream()>>>(in, o, c, part);
    else gemm_fp8_rows_kernel<NT, 2, X, T><<<grid, P::THREADS, 0, ch::stream()>>>(in, o, c, part);
    CH_LAUNCHED(fn);
    return CLEAVE_HIP_OK;
}

template <class T>
int32_t launch(const char* fn, const Operands& o, T* c, bool nt) {
    if (o.M <= kFewRows) {
        const RowsIn<uint8_t> in{nullptr, nullptr, nullptr};
        return nt ? launch_rows<true>(fn, in, o, c) : launch_rows<false>(fn, in, o, c);
    }
    return nt ? launch_layout<true, T>(fn, o, c) : launch_layout<false, T>(fn, o, c);
}

Operands operands(const uint8_t* a, const uint8_t* as, const uint8_t* b, const uint8_t* bs, int M, int N, int K,
                  bool nt) {
    return {a, as, b, bs, M, N, K, pitch_of(K), pitch_of(nt ? K : N), scale_pitch(M), scale_pitch(nt ? N : K)};
}

int32_t check_dims(const char* fn, int M, int N, int K, int trans_b) {
    CH_REQUIRE(M > 0 && N > 0 && K > 0, "%s: M, N and K must be positive (%d, %d, %d)", fn, M, N, K);
    CH_REQUIRE(trans_b == 0 || trans_b == 1, "%s: trans_b must be 0 or 1 (got %d)", fn, trans_b);
    // a tile's 256 rows lie within the 32-bit offsets of its copies
    CH_REQUIRE(K <= kMaxPitch && N <= kMaxPitch, "%s: rows of more than %d codes (%d, %d)", fn, kMaxPitch, N, K);
    return CLEAVE_HIP_OK;
}
// Codes and scales are copied 16 bytes at a time.
#define CH_TILES(fn, q, qlen)                                                           \
    do {                                                                                \
        CH_REQUIRE(((uintptr_t)(q) & 15) == 0, "%s: " #q " is not 16-byte aligned", fn); \
        CH_DEVICE((fn), (q), (qlen));                                                   \
    } while (0)

template <class T>
int32_t run_matmul(const char* fn, const uint8_t* a, int64_t alen, const uint8_t* as, int64_t aslen, const uint8_t* b,
                   int64_t blen, const uint8_t* bs, int64_t bslen, T* c, int64_t clen, int M, int N, int K,
                   int trans_b) {
    CH_OK(check_dims(fn, M, N, K, trans_b));
    CH_HELD(fn, a, alen, as, aslen, M, K);
    CH_HELD(fn, b, blen, bs, bslen, trans_b ? N : K, trans_b ? K : N);
    CH_REQUIRE(clen == (int64_t)M * N, "%s: clen %lld != M*N (%d x %d)", fn, (long long)clen, M, N);
    CH_REQUIRE(a && as && b && bs && c, "%s: null buffer", fn);
    CH_INIT_OR_RETURN();
    CH_TILES(fn, a, alen);
    CH_TILES(fn, as, aslen);
    CH_TILES(fn, b, blen);
    CH_TILES(fn, bs, bslen);
    CH_REQUIRE(((uintptr_t)c & (sizeof(T) - 1)) == 0, "%s: c is not element-aligned", fn);
    CH_DEVICE(fn, c, clen * (int64_t)sizeof(T));
    return launch<T>(fn, operands(a, as, b, bs, M, N, K, trans_b != 0), c, trans_b != 0);
}

template <class X, class T>
int32_t run_linear(const char* fn, const X* x, int64_t xlen, const uint8_t* w, int64_t wlen, const uint8_t* ws,
                   int64_t wslen, T* y, int64_t ylen, uint8_t* xq, int64_t xqlen, uint8_t* xs, int64_t xslen, int M,
                   int N, int K, int trans_b) {
    CH_OK(check_dims(fn, M, N, K, trans_b));
    CH_REQUIRE(xlen == (int64_t)M * K, "%s: xlen %lld != M*K (%d x %d)", fn, (long long)xlen, M, K);
    CH_HELD(fn, w, wlen, ws, wslen, trans_b ? N : K, trans_b ? K : N);
    CH_REQUIRE(ylen == (int64_t)M * N, "%s: ylen %lld != M*N (%d x %d)", fn, (long long)ylen, M, N);
    const bool keep = xq != nullptr || xs != nullptr;
    if (keep) CH_HELD(fn, xq, xqlen, xs, xslen, M, K);
    CH_REQUIRE(x && w && ws && y && (!keep || (xq && xs)), "%s: null buffer", fn);
    CH_INIT_OR_RETURN();
    CH_REQUIRE(((uintptr_t)x & (sizeof(X) - 1)) == 0, "%s: x is not element-aligned", fn);
    CH_DEVICE(fn, x, xlen * (int64_t)sizeof(X));
    CH_TILES(fn, w, wlen);
    CH_TILES(fn, ws, wslen);
    CH_REQUIRE(((uintptr_t)y & (sizeof(T) - 1)) == 0, "%s: y is not element-aligned", fn);
    CH_DEVICE(fn, y, ylen * (int64_t)sizeof(T));
    if (keep) {
        CH_TILES(fn, xq, xqlen);
        CH_TILES(fn, xs, xslen);
    }
    // A few rows are quantised by each workgroup of the product, unless that is more
    // work than a launch of its own (one launch against two, us, N x K weights, bf16
    // x: 16 x 4096^2 9.3 and 8.9, 16 x 8192^2 29 and 20; f32 x: 32 x 2048^2 8.7 and
    // 8.6, 16 x 4096^2 12.1 and 9.1).  Up to kSegRows rows it is always less.
    const int64_t groups = ((int64_t)N + (trans_b ? Rows<true>::COLS : Rows<false>::COLS) - 1) /
                           (trans_b ? Rows<true>::COLS : Rows<false>::COLS);
    if (M <= kSegRows || (M <= kFewRows && (int64_t)sizeof(X) * M * K * groups < 1 << 26)) {
        const RowsIn<X> in{x, xq, xs};
        const Operands o = operands(nullptr, nullptr, w, ws, M, N, K, trans_b != 0);
        return trans_b ? launch_rows<true>(fn, in, o, y) : launch_rows<false>(fn, in, o, y);
    }
    if (!keep) {
        const size_t codes = (size_t)codes_len(M, K);
        xq = (uint8_t*)ch::scratch(kHeldSlot, codes + (size_t)scales_len(M, K));
        if (!xq) return CLEAVE_HIP_ERR_OOM;
        xs = xq + codes;
    }
    CH_OK(ch::quantize_fp8<X>(fn, x, xq, xs, M, K, 1));
    return launch<T>(fn, operands(xq, xs, w, ws, M, N, K, trans_b != 0), y, trans_b != 0);
}

// The gradient through a dequantised copy of x (every value is exact in bf16) and
// the library's bf16 product.
int32_t weight_grad_wide(const char* fn, const uint8_t* xq, const uint8_t* xs, const uint16_t* g, float* dw, int B,
                         int D, int H) {
    uint16_t* x = (uint16_t*)ch::scratch(kHeldSlot, (size_t)B * D * 2);
    if (!x) return CLEAVE_HIP_ERR_OOM;
    CH_OK(ch::dequantize_fp8<uint16_t>(fn, xq, xs, x, B, D));
    return cleave_hip_matmul_bf16(x, (int64_t)B * D, g, (int64_t)B * H, dw, (int64_t)D * H, D, H, B, 1, 0);
}

int32_t weight_grad(const char* fn, const uint8_t* xq, const uint8_t* xs, const uint16_t* g, float* dw, int B, int D,
                    int H) {
    const int64_t cus = ch::num_cus();
    // The bf16 product on 256 x 256 tiles is worth a copy of x for more than half a
    // round of those tiles, or for 2^36 products from a sixteenth of a round on (us,
    // copy against in place: 3000^3 72 and 83, 512 x 4096^2 28 and 37, 65536 x 1024 x
    // 4096 410 and 577, 65536 x 1024 x 2048 225 and 295, 16384 x 2048^2 130 and 138;
    // below, 2048 x 4096 x 2048 48 and 43, 20000 x 1024 x 2048 118 and 93, 2048^3 38
    // and 23, 65536 x 512^2 81 and 44, 10000 x 784 x 500 42 and 24).  The slices' sums
    // move 16 bytes at a time.
    const int64_t big = (int64_t)((D + 255) / 256) * ((H + 255) / 256);
    const bool wide = big * 2 > cus || (big * 16 >= cus && (int64_t)D * H >= ((1ll << 36) + B - 1) / B);
    // Rows of g of fewer than 4 values: the kernel's chunks of 8 would reach past g's
    // end from more rows than its last one.
    if (wide || H < 4 || ((uintptr_t)dw & 15) != 0) return weight_grad_wide(fn, xq, xs, g, dw, B, D, H);
    using P = Grad;
    const int tiles_m = (D + P::BM - 1) / P::BM, tiles_n = (H + P::BN - 1) / P::BN;
    const int64_t tiles = (int64_t)tiles_m * tiles_n, n = (int64_t)D * H, stride = (n + 3) / 4 * 4;
    CH_REQUIRE(tiles <= ch::kMaxBlocks, "%s: %d x %d is more than one launch covers", fn, D, H);
    // Slices of the rows: a workgroup per CU, each of its groups at least 4 k-tiles
    // deep, and no more sums than a thread adds in passing.
    int64_t slices = std::min<int64_t>({cus / tiles, (int64_t)B / (4 * P::GROUPS * P::BK), 64});
    int rows = B;
    float* to = dw;
    auto cut = [&](int64_t want) {
        rows = (int)(((B + want - 1) / want + P::BK - 1) / P::BK * P::BK);
        return ((int64_t)B + rows - 1) / rows;
    };
    if (slices > 1) {
        // a count that block_coords can hand out by XCD, if one is near
        const int64_t most = slices;
        while (slices > 1 && slices > most - 8 && cut(slices) * tiles % 8) --slices;
        slices = cut(slices > 1 && cut(slices) * tiles % 8 == 0 ? slices : most);
    }
    if (slices > 1) {
        to = (float*)ch::scratch(kPartSlot, sizeof(float) * (size_t)(slices * stride));
        if (!to) return CLEAVE_HIP_ERR_OOM;
    } else {
        slices = 1;
        rows = B;
    }
    gemm_fp8_grad_kernel<<<(unsigned)(tiles * slices), P::GROUPS * P::THREADS, 0, ch::stream()>>>(
        xq, xs, g, to, B, D, H, tiles_m, tiles_n, (int)slices, rows, stride);
    CH_LAUNCHED(fn);
    return slices > 1 ? ch::sum_slices_f32(to, dw, n, (int)slices, stride) : CLEAVE_HIP_OK;
}

}  // namespace

extern "C" {

#define CH_FP8_MATMUL(T, sfx)                                                                                      \
    int32_t cleave_hip_matmul_fp8_##sfx(const uint8_t* a, int64_t alen, const uint8_t* as, int64_t aslen,         \
                                        const uint8_t* b, int64_t blen, const uint8_t* bs, int64_t bslen, T* c,   \
                                        int64_t clen, int32_t M, int32_t N, int32_t K, int32_t trans_b) {         \
        return run_matmul<T>("cleave_hip_matmul_fp8_" #sfx, a, alen, as, aslen, b, blen, bs, bslen, c, clen, M, N, \
                             K, trans_b);                                                                          \
    }
#define CH_FP8_LINEAR(X, T, xsfx, sfx)                                                                             \
    int32_t cleave_hip_linear_fp8_##xsfx##_##sfx(                                                                  \
        const X* x, int64_t xlen, const uint8_t* w, int64_t wlen, const uint8_t* ws, int64_t wslen, T* y,         \
        int64_t ylen, uint8_t* xq, int64_t xqlen, uint8_t* xs, int64_t xslen, int32_t M, int32_t N, int32_t K,    \
        int32_t trans_b) {                                                                                         \
        return run_linear<X, T>("cleave_hip_linear_fp8_" #xsfx "_" #sfx, x, xlen, w, wlen, ws, wslen, y, ylen, xq, \
                                xqlen, xs, xslen, M, N, K, trans_b);                                               \
    }
CH_FP8_MATMUL(float, f32)
CH_FP8_MATMUL(uint16_t, bf16)
CH_FP8_LINEAR(float, float, f32, f32)
CH_FP8_LINEAR(float, uint16_t, f32, bf16)
CH_FP8_LINEAR(uint16_t, float, bf16, f32)
CH_FP8_LINEAR(uint16_t, uint16_t, bf16, bf16)

int32_t cleave_hip_weight_grad_fp8(const uint8_t* xq, int64_t xqlen, const uint8_t* xs, int64_t xslen,
                                   const uint16_t* g, int64_t glen, float* dw, int64_t dwlen, int32_t B, int32_t D,
                                   int32_t H) {
    const char* fn = "cleave_hip_weight_grad_fp8";
    CH_REQUIRE(B > 0 && D > 0 && H > 0, "%s: B, D and H must be positive (%d, %d, %d)", fn, B, D, H);
    // the ends of up to 64 slices of whole k-tiles, and the k-tile after one, are ints
    CH_REQUIRE(B <= INT32_MAX - 4095, "%s: more than %d rows (%d)", fn, INT32_MAX - 4095, B);
    CH_REQUIRE(D <= kMaxPitch && H <= kMaxPitch, "%s: rows of more than %d elements (%d, %d)", fn, kMaxPitch, D, H);
    CH_HELD(fn, xq, xqlen, xs, xslen, B, D);
    CH_REQUIRE(glen == (int64_t)B * H, "%s: glen %lld != B*H (%d x %d)", fn, (long long)glen, B, H);
    CH_REQUIRE(dwlen == (int64_t)D * H, "%s: dwlen %lld != D*H (%d x %d)", fn, (long long)dwlen, D, H);
    CH_REQUIRE(xq && xs && g && dw, "%s: null buffer", fn);
    CH_INIT_OR_RETURN();
    CH_TILES(fn, xq, xqlen);
    CH_DEVICE(fn, xs, xslen);
    CH_REQUIRE(((uintptr_t)g & 1) == 0 && ((uintptr_t)dw & 3) == 0, "%s: g or dw is not element-aligned", fn);
    CH_DEVICE(fn, g, glen * 2);
    CH_DEVICE(fn, dw, dwlen * 4);
    return weight_grad(fn, xq, xs, g, dw, B, D, H);
}

}  // extern "C"
