// gemm_fp8_rows.hpp -- 8-bit products of a few rows (served tokens): bound by
// the weight's bytes, and below a few MiB by latency, so one launch does it all:
// it quantises x, multiplies, and sums over k within a workgroup.
//
// A workgroup owns a few columns of C over the whole of K, its waves take turns
// at the k-blocks, and their partial sums meet in LDS, in the order of the
// waves.  Codes are widened to bf16, exactly and with their scales, for
// v_mfma_f32_16x16x32_bf16: operand lane l holds 8 values of row (column) l % 16,
// group g = l / 16; the accumulator holds column l % 16, rows 4 (l / 16) + v.
//
// B stored N x K: 16 columns a workgroup.  A k-block of a column is 128 bytes,
//   32 of them in each of four lanes; matrix instruction t takes bytes 8 t .. +7
//   of each, so that group g's k are 32 g + 8 t .. +7, of x as well.
// B stored K x N: 64 columns a workgroup.  Each wave copies 32 k-rows x 64 bytes at
//   a time into its own ring in LDS (2 KiB a stage) and reads them with
//   ds_read_b64_tr_b8, which hands lane l column l % 16 of k-rows 8 g .. +7.
//
// Fewer column groups than CUs take slices of K, summed by a group's last
// workgroup.  Measured, us a call in a loop from Python (5.6 is what a call costs):
// from codes 1 x 4096^2 6.0 (N x K) and 7.0, 1 x 8192^2 13.5 (5.0 TB/s of codes) and
// 14.8, 16 x 8192^2 17.8 and 16.3, 32 x 4096^2 8.7 and 12.1; from a bf16 x 1 x 4096^2
// 6.4 and 7.2, 1 x 8192^2 16.5 and 14.8.
#pragma once

#include "gemm_fp8.hpp"
#include "last_block.hpp"

namespace ch {
namespace fp8 {

typedef float v4f __attribute__((ext_vector_type(4)));

// Where a lane's 8 values of matrix instruction t lie in a k-block.
template <bool NT>
__device__ __forceinline__ int k_of(int g, int t) {
    return NT ? 32 * g + 8 * t : 32 * t + 8 * g;
}

// Eight codes as bf16 times a power of two.
__device__ __forceinline__ tiles::v8bf widen8(uint2 q, float scale) {
    bf16x2 p[4];
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.x, scale, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.x, scale, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.y, scale, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.y, scale, true);
    tiles::v8bf v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// The first operand: x itself (float, or uint16_t for bf16), or codes already.
template <class X>
struct RowsIn {
    const X* x;
    uint8_t* q;  // where x's codes and scales go, or (X = uint8_t) come from; may be null else
    uint8_t* s;
};

// A lane's part of one k-block of a row as it lies in memory, so that the loads
// of several can be in flight.  Rows past M read the last one; k past K zeros.
struct __attribute__((packed)) Packed16 { v4u v; };
__device__ __forceinline__ v4u load16(const void* p) { return reinterpret_cast<const Packed16*>(p)->v; }

template <class X>
struct Raw;
template <>
struct Raw<float> {
    v4u w[4][2];
    template <bool NT>
    __device__ __forceinline__ void load(const RowsIn<float>& in, const Operands& o, int m, int kb, int g) {
        const float* const row = in.x + (int64_t)m * o.K;
        if ((kb + 1) * kBlock <= o.K) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) w[t][h] = load16(row + kb * kBlock + k_of<NT>(g, t) + 4 * h);
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int k = kb * kBlock + k_of<NT>(g, t);
                w[t][0] = w[t][1] = v4u{};
                if (k + 8 <= o.K) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) w[t][h] = load16(row + k + 4 * h);
                } else if (k < o.K) {
#pragma unroll
                    for (int e = 0; e < 7; ++e) w[t][e / 4][e % 4] = k + e < o.K ? __float_as_uint(row[k + e]) : 0u;
                }
            }
        }
    }
    __device__ __forceinline__ void values(int t, float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(w[t][e / 4][e % 4]);
    }
};
template <>
struct Raw<uint16_t> {
    v4u w[4];
    template <bool NT>
    __device__ __forceinline__ void load(const RowsIn<uint16_t>& in, const Operands& o, int m, int kb, int g) {
        const uint16_t* const row = in.x + (int64_t)m * o.K;
        if ((kb + 1) * kBlock <= o.K) {
#pragma unroll
            for (int t = 0; t < 4; ++t) w[t] = load16(row + kb * kBlock + k_of<NT>(g, t));
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int k = kb * kBlock + k_of<NT>(g, t);
                w[t] = v4u{};
                if (k + 8 <= o.K) {
                    w[t] = load16(row + k);
                } else if (k < o.K) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const uint32_t lo = k + e < o.K ? row[k + e] : 0, hi = k + e + 1 < o.K ? row[k + e + 1] : 0;
                        w[t][e / 2] = lo | hi << 16;
                    }
                }
            }
        }
    }
    __device__ __forceinline__ void values(int t, float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = __uint_as_float(w[t][e] << 16);
            v[2 * e + 1] = __uint_as_float(w[t][e] & 0xFFFF0000u);
        }
    }
};
template <>
struct Raw<uint8_t> {  // codes already
    uint2 q[4];
    int sb;
    template <bool NT>
    __device__ __forceinline__ void load(const RowsIn<uint8_t>&, const Operands& o, int m, int kb, int g) {
        const uint8_t* const row = o.a + m * o.pa + (int64_t)kb * kBlock;
#pragma unroll
        for (int t = 0; t < 4; ++t) q[t] = *reinterpret_cast<const uint2*>(row + k_of<NT>(g, t));
        sb = o.as[kb * o.spa + m];
    }
};

// The four operands of a k-block of rows 16 f .. +15, quantised here unless they
// come as codes.
template <bool NT, class X>
__device__ __forceinline__ void rows_operand(const Raw<X>& raw, const RowsIn<X>& in, const Operands& o, int f, int kb,
                                             int lane, bool keep, tiles::v8bf (&a)[4]) {
    uint2 q[4];
    int sb;
    if constexpr (sizeof(X) == 1) {
#pragma unroll
        for (int t = 0; t < 4; ++t) q[t] = raw.q[t];
        sb = raw.sb;
    } else {
        const int m = 16 * f + (lane & 15), g = lane >> 4;
        float v[4][8];
        float top = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            raw.values(t, v[t]);
            const float h = amax8(v[t]);
            top = h > top ? h : top;
        }
        auto over_groups = [&](float h) {  // the four lanes of a row
            float w = __shfl_xor(h, 16);
            h = w > h ? w : h;
            w = __shfl_xor(h, 32);
            return w > h ? w : h;
        };
        top = over_groups(top);
        if (__any(__builtin_isinf(top))) {  // uniform: the lanes stay together for the exchange
            float h[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) drop_infinities(v[t], h[t]);
            top = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t) top = h[t] > top ? h[t] : top;
            top = over_groups(top);
        }
        sb = scale_byte(__float_as_uint(top));
#pragma unroll
        for (int t = 0; t < 4; ++t) q[t] = encode8(v[t], scale_value(sb));
        if (keep) {
            if (m < o.M) {
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    *reinterpret_cast<uint2*>(in.q + m * o.pa + (int64_t)kb * kBlock + k_of<NT>(g, t)) = q[t];
            }
            if (g == 0 && m < o.spa) in.s[kb * o.spa + m] = (uint8_t)(m < o.M ? sb : kOne);
        }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) a[t] = widen8(q[t], scale_value(sb));
}

// Up to four rows: 16 lanes take one row's k-block, 8 values each, where the
// operand's layout would have every lane of a column quantise what 15 others do
// (1 x 8192^2, bf16 x: 22.8 us against 16.5).  The codes and scales reach the
// operand's lanes through LDS of the wave's own.
constexpr int kSegRows = 4;
template <class X>
struct Seg {  // 8 values of row min(lane / 16, M - 1)
    v4u w[sizeof(X) / 2];
    __device__ __forceinline__ void load(const RowsIn<X>& in, const Operands& o, int kb, int lane) {
        constexpr int PER = 16 / sizeof(X);
        const X* const row = in.x + (int64_t)min(lane >> 4, o.M - 1) * o.K;
        const int k = kb * kBlock + 8 * (lane & 15);
        if ((kb + 1) * kBlock <= o.K) {
#pragma unroll
            for (int h = 0; h < 8 / PER; ++h) w[h] = load16(row + k + PER * h);
        } else {
            X t[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = k + e < o.K ? row[k + e] : X(0);
            __builtin_memcpy(w, t, sizeof(w));
        }
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (sizeof(X) == 4) v[e] = __uint_as_float(w[e / 4][e % 4]);
            else v[e] = __uint_as_float(e & 1 ? w[0][e / 2] & 0xFFFF0000u : w[0][e / 2] << 16);
        }
    }
};
struct alignas(16) SegBlock {  // a k-block of the four rows
    uint8_t codes[kSegRows][kBlock];
    int scale[kSegRows];
};
template <class X>
__device__ __forceinline__ void seg_quantise(const Seg<X>& seg, const RowsIn<X>& in, const Operands& o, int kb,
                                             int lane, bool keep, SegBlock& to) {
    float v[8];
    seg.values(v);
    float top = row16_max(amax8(v));
    if (__any(__builtin_isinf(top))) {  // uniform: the lanes stay together for the exchange
        float h;
        drop_infinities(v, h);
        top = row16_max(h);
    }
    const int sb = scale_byte(__float_as_uint(top));
    const uint2 q = encode8(v, scale_value(sb));
    const int m = lane >> 4, c = 8 * (lane & 15);
    *reinterpret_cast<uint2*>(&to.codes[m][c]) = q;
    if (c == 0) to.scale[m] = sb;
    if (keep) {
        if (m < o.M) *reinterpret_cast<uint2*>(in.q + m * o.pa + (int64_t)kb * kBlock + c) = q;
        // each row's first four lanes: its scale, and those of the padded rows m + 4, m + 8, m + 12
        const int r = m + kSegRows * (lane & 15);
        if (r < o.spa && (lane & 15) < 4) in.s[kb * o.spa + r] = (uint8_t)(r < o.M ? sb : kOne);
    }
}
template <bool NT>
__device__ __forceinline__ void seg_operand(const SegBlock& from, int lane, tiles::v8bf (&a)[4]) {
    const int m = min(lane & 15, kSegRows - 1), g = lane >> 4;
    const float scale = scale_value(from.scale[m]);
#pragma unroll
    for (int t = 0; t < 4; ++t) a[t] = widen8(*reinterpret_cast<const uint2*>(&from.codes[m][k_of<NT>(g, t)]), scale);
}

template <bool NT>
struct Rows {
    static constexpr int NW = 8, COLS = NT ? 16 : 64, THREADS = 64 * NW;
    static constexpr int STAGES = 4, STAGE = 32 * 64;  // K x N: k-steps of 32 rows in flight per wave
    static constexpr int RING = NT ? 0 : NW * STAGES * STAGE;
};

constexpr int kMaxSliced = 512;  // column groups of a launch that cuts K
__device__ uint32_t g_rows_counters[kMaxSliced];

// FR: row blocks of 16 (M <= 16 FR), or 0 for up to kSegRows rows of an x that is
// quantised here.  Grid: column groups x slices of K; `part`
// takes a group's sums where there are several, and its last workgroup adds them
// in order.
template <bool NT, int FR_, class X, class T>
__global__ __launch_bounds__(512) void gemm_fp8_rows_kernel(RowsIn<X> in, Operands o, T* __restrict__ C,
                                                            float* part) {
    using P = Rows<NT>;
    constexpr bool SEG = FR_ == 0;
    constexpr int FR = SEG ? 1 : FR_, NW = P::NW, FC = P::COLS / 16;
    constexpr int SUMS = NW * FR * 16 * P::COLS * 4;
    __shared__ __attribute__((aligned(1024))) char smem[P::RING > SUMS ? P::RING : SUMS];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4;
    // K x N: two column groups share each 128-byte line; on one XCD, whose L2 then
    // gets it from memory once (1 x 8192^2 23 -> 15 us, 1 x 4096^2 9.9 -> 7.0)
    int group = (int)blockIdx.x;
    if (!NT && gridDim.x % 16 == 0) group = group / 16 * 16 + group % 8 * 2 + group / 8 % 2;
    const int n0 = group * P::COLS;
    const int nkb = (o.K + kBlock - 1) / kBlock, slices = (int)gridDim.y, slice = (int)blockIdx.y;
    const int kb0 = (int)((int64_t)nkb * slice / slices), kb1 = (int)((int64_t)nkb * (slice + 1) / slices);
    const bool keep = sizeof(X) != 1 && in.q != nullptr && group == 0;

    v4f acc[FR][FC];
#pragma unroll
    for (int f = 0; f < FR; ++f)
#pragma unroll
        for (int c = 0; c < FC; ++c) acc[f][c] = v4f{};

    if constexpr (NT) {
        const int n = min(n0 + (lane & 15), o.N - 1);
        const uint8_t* const row = o.b + n * o.pb + 32 * g;
        // k-blocks in flight: what the registers of a wave hold of x
        constexpr int DEEP = SEG || sizeof(X) * FR <= 2 ? 4 : 2;
        v4u w[DEEP][2];
        std::conditional_t<SEG, Seg<X>, Raw<X>> raw[DEEP][FR];
        __shared__ SegBlock segs[SEG ? NW : 1][DEEP];
        int sb[DEEP];
        auto load = [&](int d, int kb) {
#pragma unroll
            for (int h = 0; h < 2; ++h) w[d][h] = *reinterpret_cast<const v4u*>(row + (int64_t)kb * kBlock + 16 * h);
            sb[d] = o.bs[kb * o.spb + n];
            if constexpr (SEG) {
                raw[d][0].load(in, o, kb, lane);
            } else {
#pragma unroll
                for (int f = 0; f < FR; ++f)
                    raw[d][f].template load<NT>(in, o, min(16 * f + (lane & 15), o.M - 1), kb, g);
            }
        };
        const int own = kb0 + wave;
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
            if (own + d * NW < kb1) load(d, own + d * NW);
        for (int base = own; base < kb1; base += DEEP * NW) {
            if constexpr (SEG) {
#pragma unroll
                for (int d = 0; d < DEEP; ++d) {
                    const int kb = base + d * NW;
                    if (kb < kb1) seg_quantise<X>(raw[d][0], in, o, kb, lane, keep, segs[wave][d]);
                }
                __builtin_amdgcn_wave_barrier();  // the wave's LDS instructions run in order
            }
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                const int kb = base + d * NW;
                if (kb >= kb1) break;
                tiles::v8bf b[4];
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    b[t] = widen8(make_uint2(w[d][t / 2][2 * (t & 1)], w[d][t / 2][2 * (t & 1) + 1]),
                                  scale_value(sb[d]));
#pragma unroll
                for (int f = 0; f < FR; ++f) {
                    tiles::v8bf a[4];
                    if constexpr (SEG) seg_operand<NT>(segs[wave][d], lane, a);
                    else rows_operand<NT, X>(raw[d][f], in, o, f, kb, lane, keep, a);
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        acc[f][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[t], b[t], acc[f][0], 0, 0, 0);
                }
                if (kb + DEEP * NW < kb1) load(d, kb + DEEP * NW);
            }
            if constexpr (SEG) __builtin_amdgcn_wave_barrier();
        }
    } else {
        // Stage s of the wave's ring holds its k-steps s, s + 4, ...; step u is
        // rows 32 (u % 4) .. of its (u / 4)-th k-block: a copy of 16 rows x 64
        // bytes is one instruction.
        const uint32_t ring = lds_addr(smem) + (uint32_t)(wave * P::STAGES * P::STAGE);
        const int own = kb0 + wave, mine = own < kb1 ? (kb1 - own + NW - 1) / NW : 0, steps = 4 * mine;
        auto issue = [&](int u) {
            const int v = min(u, steps - 1), kb = own + (v >> 2) * NW;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int k = min(kb * kBlock + 32 * (v & 3) + 16 * j + (lane >> 2), o.K - 1);
                dma16_far(o.b + k * o.pb + n0 + 16 * (lane & 3), ring + (uint32_t)((u % P::STAGES) * P::STAGE + 1024 * j));
            }
        };
        if (mine > 0) {
#pragma unroll
            for (int u = 0; u < P::STAGES; ++u) issue(u);
        }
        const int nb = n0 / kBlock;
        std::conditional_t<SEG, Seg<X>, Raw<X>> raw[FR];
        __shared__ SegBlock segs[SEG ? NW : 1];
        int sb = 0;
        auto load = [&](int kb) {
            sb = o.bs[nb * o.spb + (int64_t)kb * kBlock];
            if constexpr (SEG) {
                raw[0].load(in, o, kb, lane);
            } else {
#pragma unroll
                for (int f = 0; f < FR; ++f) raw[f].template load<NT>(in, o, min(16 * f + (lane & 15), o.M - 1), kb, g);
            }
        };
        if (mine > 0) load(own);
        for (int i = 0; i < mine; ++i) {
            const int kb = own + i * NW;
            const float scale = scale_value(sb);
            tiles::v8bf a[FR][4];
            if constexpr (SEG) {
                seg_quantise<X>(raw[0], in, o, kb, lane, keep, segs[wave]);
                __builtin_amdgcn_wave_barrier();  // the wave's LDS instructions run in order
                seg_operand<NT>(segs[wave], lane, a[0]);
                __builtin_amdgcn_wave_barrier();
            } else {
#pragma unroll
                for (int f = 0; f < FR; ++f) rows_operand<NT, X>(raw[f], in, o, f, kb, lane, keep, a[f]);
            }
            if (i + 1 < mine) load(kb + NW);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                // this step's two copies are the oldest of the eight in flight
                asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
                uint2 q[FC];
#pragma unroll
                for (int c = 0; c < FC; ++c) {
                    const uint32_t at = ring + (uint32_t)(t * P::STAGE + (8 * g + ((lane & 15) >> 1)) * 64 + 16 * c +
                                                          8 * (lane & 1));
                    const v2i r = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(uintptr_t)at);
                    q[c] = make_uint2((uint32_t)r[0], (uint32_t)r[1]);
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                issue(4 * i + t + P::STAGES);
#pragma unroll
                for (int c = 0; c < FC; ++c) {
                    const tiles::v8bf b = widen8(q[c], scale);
#pragma unroll
                    for (int f = 0; f < FR; ++f)
                        acc[f][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[f][t], b, acc[f][c], 0, 0, 0);
                }
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // the rings become the sums' place
    }

    // The waves' sums, row by row, in their order.
    float* const sums = reinterpret_cast<float*>(smem);
    constexpr int ROW = P::COLS, PART = FR * 16 * P::COLS;
#pragma unroll
    for (int f = 0; f < FR; ++f)
#pragma unroll
        for (int c = 0; c < FC; ++c)
#pragma unroll
            for (int v = 0; v < 4; ++v)
                sums[wave * PART + (16 * f + 4 * g + v) * ROW + 16 * c + (lane & 15)] = acc[f][c][v];
    __syncthreads();
    if (slices > 1) {
        float* const mine = part + ((int64_t)group * slices + slice) * PART;
        for (int e = (int)threadIdx.x; e < PART; e += P::THREADS) {
            float y = sums[e];
#pragma unroll
            for (int w = 1; w < NW; ++w) y += sums[w * PART + e];
            if (e / ROW < o.M) ch::publish(mine + e, y);
        }
        if (!ch::last_block(&g_rows_counters[group], (uint32_t)slices)) return;
    }
    for (int e = (int)threadIdx.x; e < PART; e += P::THREADS) {
        const int m = e / ROW, n = n0 + e % ROW;
        if (m < o.M && n < o.N) {
            float y;
            if (slices > 1) {
                const float* const from = part + (int64_t)group * slices * PART + e;
                y = ch::fetch(from);
                for (int z = 1; z < slices; ++z) y += ch::fetch(from + (int64_t)z * PART);
            } else {
                y = sums[e];
#pragma unroll
                for (int w = 1; w < NW; ++w) y += sums[w * PART + e];
            }
            store_c(C, (int64_t)m * o.N + n, y);
        }
    }
}

}  // namespace fp8
}  // namespace ch
