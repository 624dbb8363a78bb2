// fp8_maps.hip -- the maps between f32 / bf16 matrices and the 8-bit format of
// fp8.hpp: quantisation, activations that leave 8 bits behind for the next
// product and for the backward pass, and their backward.
//
// One pass each: a row's block of 128 lies in 16 lanes of 8 values, so its
// largest magnitude is four DPP steps, and the values are still in registers
// when the scale is known.  All of it is bound by HBM bytes: bf16 65536 x 4096
// sigmoid with its checkpoint 187 us (1.08 GB, 5.8 TB/s), its backward with both
// results 276 us (1.62 GB, 5.9 TB/s), an f32 8192^2 weight 57 us (0.34 GB, 5.9
// TB/s), each pass on other matrices than the one before; on the same ones again the
// last-level cache still holds a part (the backward 240 us).  1000 x 500 is one
// launch, 3 us of it the kernel.
#include <type_traits>

#include "fp8.hpp"

namespace {

using namespace ch::fp8;

constexpr int kThreads = 256;
constexpr int kRows = kThreads / 16;  // rows a workgroup covers: one row of scale padding

// ---- eight neighbouring elements ------------------------------------------------

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

typedef u32x4 __attribute__((aligned(1))) u32x4_any;
// S: a matrix of whole 128-byte lines that this pass alone needs, past the caches.
template <bool S = false>
__device__ __forceinline__ u32x4 load16(const void* p) {  // any alignment
    if constexpr (S) return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
    else return *reinterpret_cast<const u32x4_any*>(p);
}
template <bool S = false>
__device__ __forceinline__ void store16(void* p, u32x4 v) {
    if constexpr (S) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(p));
    else *reinterpret_cast<u32x4_any*>(p) = v;
}

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }

// p[0 .. n) in v, zeros past n; n >= 8 is the whole eight.
template <bool S = false>
__device__ __forceinline__ void load8(const float* p, int n, float (&v)[8]) {
    if (n >= 8) {
        const u32x4 a = load16<S>(p), b = load16<S>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(a[i]), v[i + 4] = __uint_as_float(b[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.0f;
    }
}
template <bool S = false>
__device__ __forceinline__ void load8(const uint16_t* p, int n, float (&v)[8]) {
    if (n >= 8) {
        const u32x4 a = load16<S>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(a[i] << 16);
            v[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? widen(p[i]) : 0.0f;
    }
}
template <bool S = false>
__device__ __forceinline__ void store8(float* p, int n, const float (&v)[8]) {
    if (n >= 8) {
        u32x4 a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = __float_as_uint(v[i]), b[i] = __float_as_uint(v[i + 4]);
        store16<S>(p, a);
        store16<S>(p + 4, b);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = v[i];
    }
}
template <bool S = false>
__device__ __forceinline__ void store8(uint16_t* p, int n, const float (&v)[8]) {
    u32x4 a;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
    if (n >= 8) {
        store16<S>(p, a);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (uint16_t)(i & 1 ? a[i / 2] >> 16 : a[i / 2]);
    }
}

// ---- blocks to codes -------------------------------------------------------------

// The codes of a block's eight values in each of 16 lanes, and its scale byte.
__device__ __forceinline__ uint2 quantize16(float (&v)[8], int& s) {
    float m = row16_max(amax8(v));
    if (__builtin_isinf(m)) {  // the whole row of 16 lanes agrees
        drop_infinities(v, m);
        m = row16_max(m);
    }
    s = scale_byte(__float_as_uint(m));
    return encode8(v, scale_value(s));
}

// Where h > 0 has the code 0, the least code (2^-9): what relu's mask reads.
__device__ __forceinline__ uint2 keep_positive(uint2 q, const float (&h)[8]) {
    uint32_t w[2] = {q.x, q.y};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t shift = 8 * (i & 3);
        if (h[i] > 0.0f && ((w[i / 4] >> shift) & 0xFF) == 0) w[i / 4] |= 1u << shift;
    }
    return make_uint2(w[0], w[1]);
}

// ---- activations -----------------------------------------------------------------

constexpr float kLog2e = 1.44269504088896340736f;

// fwd_near: act(z) where no |z| is past kNear; fwd: any z, and the same bits for those.
// So which of them a wave takes changes nothing, and a row's codes do not depend on
// its neighbours.
struct Relu {
    static constexpr float kClip = __builtin_inff(), kNear = kClip;
    static __device__ __forceinline__ float fwd_near(float z) { return fwd(z); }
    static __device__ __forceinline__ float fwd(float z) { return z > 0.0f ? z : (z != z ? z : 0.0f); }
    // g where z > 0, whatever g holds elsewhere
    static __device__ __forceinline__ float bwd(float z, float g) { return z > 0.0f ? g : 0.0f; }
};
// 2^t for t <= 0, its subnormals too (the instruction gives none).
__device__ __forceinline__ float exp2_down(float t) {
    const bool low = t < -126.0f;
    const float e = __builtin_amdgcn_exp2f(low ? t + 64.0f : t);
    return low ? e * 0x1.0p-64f : e;
}
struct Sigmoid {
    // past kNear, e^-z or its reciprocal leaves the normal floats; there 1 + e^-z is e^-z
    static constexpr float kClip = 32.0f, kNear = 87.0f;
    static __device__ __forceinline__ float fwd_near(float z) {
        return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
    }
    static __device__ __forceinline__ float fwd(float z) {
        return z < -kNear ? exp2_down(kLog2e * z) : fwd_near(z);
    }
    // q (1 - q), q = 1 - s of |z| = u / (1 + u) in u = e^-|z|: nothing overflows or
    // cancels for a large |z|, and as q - q q it is at most 1/4 however q is rounded
    // (u r r passed it, and the scale of a block whose largest g is 1.75 2^k with it).
    static __device__ __forceinline__ float bwd(float z, float g) {
        const float u = __builtin_amdgcn_exp2f(-kLog2e * __builtin_fabsf(z));
        const float q = u * __builtin_amdgcn_rcpf(1.0f + u);
        return g * __builtin_fmaf(-q, q, q);
    }
};
struct Tanh {
    static constexpr float kClip = 16.0f, kNear = __builtin_inff();
    static __device__ __forceinline__ float fwd_near(float z) { return fwd(z); }
    static __device__ __forceinline__ float fwd(float z) {  // in u = e^-2|z|
        const float a = __builtin_fabsf(z), u = __builtin_amdgcn_exp2f(-2.0f * kLog2e * a);
        const float far = (1.0f - u) * __builtin_amdgcn_rcpf(1.0f + u), w = z * z;
        // 1 - u loses the small ones: the series to z^7, 2e-9 off at 1/8
        const float near = a * (1.0f + w * (-1.0f / 3.0f + w * (2.0f / 15.0f - w * (17.0f / 315.0f))));
        return __builtin_copysignf(a < 0.125f ? near : far, z);
    }
    // 4 q (1 - q), q = (1 - tanh |z|) / 2 = u / (1 + u): at most 1, as above
    static __device__ __forceinline__ float bwd(float z, float g) {
        const float u = __builtin_amdgcn_exp2f(-2.0f * kLog2e * __builtin_fabsf(z));
        const float q = u * __builtin_amdgcn_rcpf(1.0f + u);
        return g * (4.0f * __builtin_fmaf(-q, q, q));
    }
};

// min(max(z, -c), c), NaN kept.
__device__ __forceinline__ float clip(float z, float c) {
    return z > c ? c : (z < -c ? -c : z);
}

// A checkpoint's codes: nobody else reads them soon (writing), or ever again (reading).
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <bool S>
__device__ __forceinline__ void store_codes(uint8_t* p, uint2 w) {
    const u32x2 v = {w.x, w.y};
    if constexpr (S) __builtin_nontemporal_store(v, reinterpret_cast<u32x2*>(p));
    else *reinterpret_cast<u32x2*>(p) = v;
}
template <bool S>
__device__ __forceinline__ uint2 load_codes(const uint8_t* p) {
    u32x2 v;
    if constexpr (S) v = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
    else v = *reinterpret_cast<const u32x2*>(p);
    return make_uint2(v[0], v[1]);
}

// ---- kernels ---------------------------------------------------------------------

// Workgroup: 16 rows x U blocks; 16 lanes take a row's block, lane l the
// columns 8l .. 8l+7 of it.  Sixteen rows make one whole run of scale bytes,
// the padded rows among them.  f(row, c0, n, kb): columns c0 .. of `row`, n of
// them inside the matrix (it may be <= 0); the row may lie past the last.
template <int U, class F>
__device__ __forceinline__ void for_blocks(int cols, F&& f) {
    const int nb = (int)(pitch_of(cols) / kBlock), nu = (nb + U - 1) / U;
    const int strip = (int)(blockIdx.x / (unsigned)nu), first = (int)(blockIdx.x % (unsigned)nu) * U;
    const int row = strip * kRows + (int)(threadIdx.x >> 4), c = (int)(threadIdx.x & 15) * 8;
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int kb = first + i;
        if (kb < nb) f(i, row, kb * kBlock + c, kb);
    }
}

template <class T, class W>
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                                 uint8_t* __restrict__ s, int rows, int cols) {
    const int64_t pitch = pitch_of(cols), sp = scale_pitch(rows);
    float v[W::U][8];
    for_blocks<W::U>(cols, [&](int i, int row, int c, int) {
        load8<W::S>(x + (int64_t)row * cols + c, row < rows ? cols - c : 0, v[i]);
    });
    for_blocks<W::U>(cols, [&](int i, int row, int c, int kb) {
        int sb;
        const uint2 w = quantize16(v[i], sb);
        if (row < rows) *reinterpret_cast<uint2*>(q + row * pitch + c) = w;
        if ((threadIdx.x & 15) == 0) s[kb * sp + row] = (uint8_t)sb;
    });
}

// A weight's 128 x 128 blocks, one a workgroup: each thread holds 8 rows' eight
// values until the block's maximum is known.
template <class T, bool S>
__global__ __launch_bounds__(kThreads) void quantize_tiles_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                                  uint8_t* __restrict__ s, int rows, int cols) {
    __shared__ float wave_max[kThreads / 64];
    const int64_t pitch = pitch_of(cols), sp = scale_pitch(rows);
    const int nb = (int)(pitch / kBlock);
    const int rb = (int)(blockIdx.x / (unsigned)nb) * kBlock, kb = (int)(blockIdx.x % (unsigned)nb);
    const int r0 = rb + (int)(threadIdx.x >> 4), c = kb * kBlock + (int)(threadIdx.x & 15) * 8;
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = r0 + i * kRows;
        load8<S>(x + (int64_t)row * cols + c, row < rows ? cols - c : 0, v[i]);
    }
    auto over_tile = [&](float m) {
        m = row16_max(m);
#pragma unroll
        for (int o = 16; o < 64; o *= 2) {
            const float t = __shfl_xor(m, o);
            m = t > m ? t : m;
        }
        if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) m = wave_max[w] > m ? wave_max[w] : m;
        return m;
    };
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = amax8(v[i]);
        m = t > m ? t : m;
    }
    m = over_tile(m);
    if (__builtin_isinf(m)) {  // uniform over the workgroup
        m = 0.0f;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float t;
            drop_infinities(v[i], t);
            m = t > m ? t : m;
        }
        m = over_tile(m);
    }
    const int sb = scale_byte(__float_as_uint(m));
    const float scale = scale_value(sb);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = r0 + i * kRows;
        if (row < rows) *reinterpret_cast<uint2*>(q + row * pitch + c) = encode8(v[i], scale);
    }
    // each row's copy of the scale, the padded rows' too
    if (threadIdx.x < kBlock && rb + (int)threadIdx.x < sp) s[kb * sp + rb + threadIdx.x] = (uint8_t)sb;
}

template <class T, class W>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint8_t* __restrict__ q,
                                                              const uint8_t* __restrict__ s, T* __restrict__ out,
                                                              int rows, int cols) {
    const int64_t pitch = pitch_of(cols), sp = scale_pitch(rows);
    uint2 w[W::U];
    int sb[W::U];
    for_blocks<W::U>(cols, [&](int i, int row, int c, int kb) {
        w[i] = row < rows ? *reinterpret_cast<const uint2*>(q + row * pitch + c) : make_uint2(0, 0);
        sb[i] = s[kb * sp + row];
    });
    for_blocks<W::U>(cols, [&](int i, int row, int c, int) {
        float v[8];
        decode8(w[i], scale_value(sb[i]), v);
        if (row < rows) store8(out + (int64_t)row * cols + c, cols - c, v);
    });
}

// h = act(z) in 8 bits; KEEP: and z, clipped to where the derivative is not yet nothing.
template <class Act, class T, bool KEEP, class W>
__global__ __launch_bounds__(kThreads) void act_kernel(const T* __restrict__ z, uint8_t* __restrict__ hq,
                                                       uint8_t* __restrict__ hs, uint8_t* __restrict__ zq,
                                                       uint8_t* __restrict__ zs, int rows, int cols) {
    const int64_t pitch = pitch_of(cols), sp = scale_pitch(rows);
    float v[W::U][8];
    for_blocks<W::U>(cols, [&](int i, int row, int c, int) {
        load8<W::S>(z + (int64_t)row * cols + c, row < rows ? cols - c : 0, v[i]);
    });
    for_blocks<W::U>(cols, [&](int i, int row, int c, int kb) {
        const int n = row < rows ? cols - c : 0;
        float h[8];
        // One way for the whole wave; an infinity (or a signalling NaN) is past any bound.
        const float top = amax8(v[i]);
        if (Act::kNear == __builtin_inff() || !__any(!(top <= Act::kNear))) {
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = Act::fwd_near(v[i][e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = Act::fwd(v[i][e]);
        }
        if (n < 8) {  // act(0) may not be 0
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = e < n ? h[e] : 0.0f;
        }
        int sb;
        uint2 w = quantize16(h, sb);
        if constexpr (std::is_same<Act, Relu>::value) w = keep_positive(w, h);
        if (row < rows) *reinterpret_cast<uint2*>(hq + row * pitch + c) = w;
        if ((threadIdx.x & 15) == 0) hs[kb * sp + row] = (uint8_t)sb;
        if constexpr (KEEP) {
            if (__any(!(top <= Act::kClip))) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] = clip(v[i][e], Act::kClip);
            }
            w = quantize16(v[i], sb);
            if (row < rows) store_codes<W::S>(zq + row * pitch + c, w);
            if ((threadIdx.x & 15) == 0) zs[kb * sp + row] = (uint8_t)sb;
        }
    });
}

// dz = g act'(z) from the checkpoint; WIDE: stored as T, HELD: in 8 bits.
template <class Act, class T, bool WIDE, bool HELD, class W>
__global__ __launch_bounds__(kThreads) void act_bwd_kernel(const uint8_t* __restrict__ zq,
                                                           const uint8_t* __restrict__ zs, const T* g, T* dz,
                                                           uint8_t* __restrict__ dq, uint8_t* __restrict__ ds, int rows,
                                                           int cols) {
    const int64_t pitch = pitch_of(cols), sp = scale_pitch(rows);
    float v[W::U][8];
    uint2 w[W::U];
    int sb[W::U];
    for_blocks<W::U>(cols, [&](int i, int row, int c, int kb) {
        w[i] = row < rows ? load_codes<W::S>(zq + row * pitch + c) : make_uint2(0, 0);
        sb[i] = zs[kb * sp + row];
        load8<W::S>(g + (int64_t)row * cols + c, row < rows ? cols - c : 0, v[i]);
    });
    for_blocks<W::U>(cols, [&](int i, int row, int c, int kb) {
        float z[8];
        decode8(w[i], scale_value(sb[i]), z);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = Act::bwd(z[e], v[i][e]);
        if constexpr (WIDE) {
            if (row < rows) store8<W::S>(dz + (int64_t)row * cols + c, cols - c, v[i]);
        }
        if constexpr (HELD) {
            int b;
            const uint2 d = quantize16(v[i], b);
            if (row < rows) *reinterpret_cast<uint2*>(dq + row * pitch + c) = d;
            if ((threadIdx.x & 15) == 0) ds[kb * sp + row] = (uint8_t)b;
        }
    });
}

// ---- launches --------------------------------------------------------------------

// How a kernel walks: U blocks a thread, S: streaming its wide matrices.
template <int U_, bool S_>
struct Walk {
    static constexpr int U = U_;
    static constexpr bool S = S_;
};
template <class T>
bool whole_lines(const T* p, int cols) {
    return ((int64_t)cols * (int64_t)sizeof(T)) % 128 == 0 && ((uintptr_t)p & 127) == 0;
}

// go(Walk, grid of for_blocks<Walk::U>).  Four blocks a thread keep eight loads in
// flight; with fewer workgroups than fill the card, one block each spreads the work
// wider.  `lines`: the wide matrices are whole 128-byte lines and streamed (bf16
// 65536 x 4096, sigmoid and its backward, 189 -> 186 and 287 -> 281 us, 8192 x 4096
// backward 45 -> 37; without whole lines it costs: f32 30000 x 1000, 38 -> 42).
template <bool STREAM = true, class Go>
int32_t by_blocks(const char* fn, int rows, int cols, bool lines, Go go) {
    const int64_t strips = scale_pitch(rows) / kRows, nb = pitch_of(cols) / kBlock;
    const int64_t wide = strips * ((nb + 3) / 4);
    const bool four = wide >= 4 * (int64_t)ch::num_cus();
    const int64_t blocks = four ? wide : strips * nb;
    CH_REQUIRE(blocks <= ch::kMaxBlocks, "%s: %d x %d is more than one launch covers", fn, rows, cols);
    if (!four) {
        go(Walk<1, false>{}, (unsigned)blocks);
    } else if (!STREAM || !lines) {
        go(Walk<4, false>{}, (unsigned)blocks);
    } else {
        if constexpr (STREAM) go(Walk<4, true>{}, (unsigned)blocks);
    }
    CH_LAUNCHED(fn);
    return CLEAVE_HIP_OK;
}

int32_t check_shape(const char* fn, int64_t len, int rows, int cols) {
    CH_REQUIRE(rows >= 0 && cols >= 0, "%s: negative shape (%d x %d)", fn, rows, cols);
    CH_REQUIRE(len == (int64_t)rows * cols, "%s: %lld elements are not %d x %d", fn, (long long)len, rows, cols);
    return CLEAVE_HIP_OK;
}
#define CH_SHAPE(fn, len, rows, cols)                          \
    do {                                                       \
        int32_t _st = check_shape((fn), (len), (rows), (cols)); \
        if (_st != CLEAVE_HIP_OK) return _st;                  \
    } while (0)
// Codes move eight at a time.
#define CH_CODES(fn, q, qlen)                                                                  \
    do {                                                                                       \
        CH_REQUIRE(((uintptr_t)(q) & 7) == 0, "%s: " #q " is not 8-byte aligned", (fn));        \
        CH_DEVICE((fn), (q), (qlen));                                                          \
    } while (0)
#define CH_ELEMENTS(fn, p, len)                                                                          \
    do {                                                                                                 \
        CH_REQUIRE(((uintptr_t)(p) & (sizeof(*(p)) - 1)) == 0, "%s: " #p " is not element-aligned", (fn)); \
        CH_DEVICE((fn), (p), (len) * (int64_t)sizeof(*(p)));                                             \
    } while (0)

template <class T>
int32_t run_quantize(const char* fn, const T* x, int64_t xlen, uint8_t* q, int64_t qlen, uint8_t* s, int64_t slen,
                     int rows, int cols, int block_rows) {
    CH_REQUIRE(block_rows == 1 || block_rows == kBlock, "%s: block_rows is 1 or 128, not %d", fn, block_rows);
    CH_SHAPE(fn, xlen, rows, cols);
    CH_HELD(fn, q, qlen, s, slen, rows, cols);
    if (xlen == 0) return CLEAVE_HIP_OK;
    CH_REQUIRE(x && q && s, "%s: null buffer", fn);
    CH_INIT_OR_RETURN();
    CH_ELEMENTS(fn, x, xlen);
    CH_CODES(fn, q, qlen);
    CH_DEVICE(fn, s, slen);
    return ch::quantize_fp8<T>(fn, x, q, s, rows, cols, block_rows);
}

template <class T>
int32_t run_dequantize(const char* fn, const uint8_t* q, int64_t qlen, const uint8_t* s, int64_t slen, T* out,
                       int64_t outlen, int rows, int cols) {
    CH_SHAPE(fn, outlen, rows, cols);
    CH_HELD(fn, q, qlen, s, slen, rows, cols);
    if (outlen == 0) return CLEAVE_HIP_OK;
    CH_REQUIRE(q && s && out, "%s: null buffer", fn);
    CH_INIT_OR_RETURN();
    CH_CODES(fn, q, qlen);
    CH_DEVICE(fn, s, slen);
    CH_ELEMENTS(fn, out, outlen);
    return ch::dequantize_fp8<T>(fn, q, s, out, rows, cols);
}

template <class Act, class T>
int32_t run_act(const char* fn, const T* z, int64_t zlen, uint8_t* hq, int64_t hqlen, uint8_t* hs, int64_t hslen,
                uint8_t* zq, int64_t zqlen, uint8_t* zs, int64_t zslen, int rows, int cols) {
    CH_SHAPE(fn, zlen, rows, cols);
    CH_HELD(fn, hq, hqlen, hs, hslen, rows, cols);
    const bool keep = zq != nullptr || zs != nullptr;
    if (keep) CH_HELD(fn, zq, zqlen, zs, zslen, rows, cols);
    CH_REQUIRE(!keep || !(std::is_same<Act, Relu>::value), "%s: relu's checkpoint is its result; pass no zq", fn);
    if (zlen == 0) return CLEAVE_HIP_OK;
    CH_REQUIRE(z && hq && hs && (!keep || (zq && zs)), "%s: null buffer", fn);
    CH_INIT_OR_RETURN();
    CH_ELEMENTS(fn, z, zlen);
    CH_CODES(fn, hq, hqlen);
    CH_DEVICE(fn, hs, hslen);
    if (keep) {
        CH_CODES(fn, zq, zqlen);
        CH_DEVICE(fn, zs, zslen);
    }
    return by_blocks(fn, rows, cols, whole_lines(z, cols), [&](auto walk, unsigned grid) {
        using W = decltype(walk);
        if constexpr (!std::is_same<Act, Relu>::value) {
            if (keep) {
                act_kernel<Act, T, true, W><<<grid, kThreads, 0, ch::stream()>>>(z, hq, hs, zq, zs, rows, cols);
                return;
            }
        }
        act_kernel<Act, T, false, W><<<grid, kThreads, 0, ch::stream()>>>(z, hq, hs, nullptr, nullptr, rows, cols);
    });
}

template <class Act, class T>
int32_t run_act_bwd(const char* fn, const uint8_t* zq, int64_t zqlen, const uint8_t* zs, int64_t zslen, const T* g,
                    int64_t glen, T* dz, int64_t dzlen, uint8_t* dq, int64_t dqlen, uint8_t* ds, int64_t dslen,
                    int rows, int cols) {
    CH_SHAPE(fn, glen, rows, cols);
    CH_HELD(fn, zq, zqlen, zs, zslen, rows, cols);
    const bool wide = dz != nullptr, held = dq != nullptr || ds != nullptr;
    if (wide) CH_SHAPE(fn, dzlen, rows, cols);
    if (held) CH_HELD(fn, dq, dqlen, ds, dslen, rows, cols);
    if (glen == 0) return CLEAVE_HIP_OK;
    CH_REQUIRE(zq && zs && g && (wide || held) && (!held || (dq && ds)), "%s: null buffer", fn);
    CH_INIT_OR_RETURN();
    CH_CODES(fn, zq, zqlen);
    CH_DEVICE(fn, zs, zslen);
    CH_ELEMENTS(fn, g, glen);
    if (wide) CH_ELEMENTS(fn, dz, dzlen);
    if (held) {
        CH_CODES(fn, dq, dqlen);
        CH_DEVICE(fn, ds, dslen);
    }
    const bool lines = whole_lines(g, cols) && (!wide || whole_lines(dz, cols));
    return by_blocks(fn, rows, cols, lines, [&](auto walk, unsigned grid) {
        using W = decltype(walk);
        auto go = [&](auto w, auto h) {
            act_bwd_kernel<Act, T, decltype(w)::value, decltype(h)::value, W>
                <<<grid, kThreads, 0, ch::stream()>>>(zq, zs, g, dz, dq, ds, rows, cols);
        };
        using Y = std::true_type;
        using N = std::false_type;
        if (wide && held) go(Y{}, Y{});
        else if (wide) go(Y{}, N{});
        else go(N{}, Y{});
    });
}

}  // namespace

namespace ch {

template <class T>
int32_t quantize_fp8(const char* fn, const T* x, uint8_t* q, uint8_t* s, int rows, int cols, int block_rows) {
    if (block_rows == kBlock) {
        const int64_t tiles = ((int64_t)rows + kBlock - 1) / kBlock * (pitch_of(cols) / kBlock);
        CH_REQUIRE(tiles <= kMaxBlocks, "%s: %d x %d is more than one launch covers", fn, rows, cols);
        if (whole_lines(x, cols)) {
            quantize_tiles_kernel<T, true><<<(unsigned)tiles, kThreads, 0, stream()>>>(x, q, s, rows, cols);
        } else {
            quantize_tiles_kernel<T, false><<<(unsigned)tiles, kThreads, 0, stream()>>>(x, q, s, rows, cols);
        }
        CH_LAUNCHED(fn);
        return CLEAVE_HIP_OK;
    }
    return by_blocks(fn, rows, cols, whole_lines(x, cols), [&](auto walk, unsigned grid) {
        quantize_rows_kernel<T, decltype(walk)><<<grid, kThreads, 0, stream()>>>(x, q, s, rows, cols);
    });
}
template int32_t quantize_fp8<float>(const char*, const float*, uint8_t*, uint8_t*, int, int, int);
template int32_t quantize_fp8<uint16_t>(const char*, const uint16_t*, uint8_t*, uint8_t*, int, int, int);

template <class T>
int32_t dequantize_fp8(const char* fn, const uint8_t* q, const uint8_t* s, T* out, int rows, int cols) {
    // what it writes is read next
    return by_blocks<false>(fn, rows, cols, false, [&](auto walk, unsigned grid) {
        dequantize_kernel<T, decltype(walk)><<<grid, kThreads, 0, stream()>>>(q, s, out, rows, cols);
    });
}
template int32_t dequantize_fp8<float>(const char*, const uint8_t*, const uint8_t*, float*, int, int);
template int32_t dequantize_fp8<uint16_t>(const char*, const uint8_t*, const uint8_t*, uint16_t*, int, int);

}  // namespace ch

extern "C" {

int64_t cleave_hip_fp8_codes_len(int32_t rows, int32_t cols) {
    CH_REQUIRE(rows >= 0 && cols >= 0, "cleave_hip_fp8_codes_len: negative shape (%d x %d)", rows, cols);
    return codes_len(rows, cols);
}
int64_t cleave_hip_fp8_scales_len(int32_t rows, int32_t cols) {
    CH_REQUIRE(rows >= 0 && cols >= 0, "cleave_hip_fp8_scales_len: negative shape (%d x %d)", rows, cols);
    return scales_len(rows, cols);
}

#define CH_FP8_ENTRIES(T, sfx)                                                                                     \
    int32_t cleave_hip_quantize_fp8_##sfx(const T* x, int64_t xlen, uint8_t* q, int64_t qlen, uint8_t* s,         \
                                          int64_t slen, int32_t rows, int32_t cols, int32_t block_rows) {         \
        return run_quantize<T>("cleave_hip_quantize_fp8_" #sfx, x, xlen, q, qlen, s, slen, rows, cols, block_rows); \
    }                                                                                                              \
    int32_t cleave_hip_dequantize_fp8_##sfx(const uint8_t* q, int64_t qlen, const uint8_t* s, int64_t slen,       \
                                            T* out, int64_t outlen, int32_t rows, int32_t cols) {                 \
        return run_dequantize<T>("cleave_hip_dequantize_fp8_" #sfx, q, qlen, s, slen, out, outlen, rows, cols);   \
    }                                                                                                              \
    CH_FP8_ACT(relu, Relu, T, sfx)                                                                                 \
    CH_FP8_ACT(sigmoid, Sigmoid, T, sfx)                                                                           \
    CH_FP8_ACT(tanh, Tanh, T, sfx)
#define CH_FP8_ACT(act, Act, T, sfx)                                                                               \
    int32_t cleave_hip_##act##_fp8_##sfx(const T* z, int64_t zlen, uint8_t* hq, int64_t hqlen, uint8_t* hs,       \
                                         int64_t hslen, uint8_t* zq, int64_t zqlen, uint8_t* zs, int64_t zslen,   \
                                         int32_t rows, int32_t cols) {                                             \
        return run_act<Act, T>("cleave_hip_" #act "_fp8_" #sfx, z, zlen, hq, hqlen, hs, hslen, zq, zqlen, zs,      \
                               zslen, rows, cols);                                                                 \
    }                                                                                                              \
    int32_t cleave_hip_##act##_bwd_fp8_##sfx(const uint8_t* zq, int64_t zqlen, const uint8_t* zs, int64_t zslen,  \
                                             const T* g, int64_t glen, T* dz, int64_t dzlen, uint8_t* dq,          \
                                             int64_t dqlen, uint8_t* ds, int64_t dslen, int32_t rows,              \
                                             int32_t cols) {                                                       \
        return run_act_bwd<Act, T>("cleave_hip_" #act "_bwd_fp8_" #sfx, zq, zqlen, zs, zslen, g, glen, dz, dzlen,  \
                                   dq, dqlen, ds, dslen, rows, cols);                                              \
    }

CH_FP8_ENTRIES(float, f32)
CH_FP8_ENTRIES(uint16_t, bf16)

}  // extern "C"
