// gemm_fp8_grad.hpp -- the weight gradient from a layer's saved 8-bit input:
// dw[D x H] = x^T g, x [B x D] codes with a scale per row and block of 128
// columns, g [B x H] bf16.
//
// The sum runs over the rows, along which the scales change, so the scales
// cannot wait for the accumulator: each code is widened to bf16 with its row's
// scale (exact) on its way into LDS, once per tile, and the product is
// v_mfma_f32_32x32x16_bf16's, f32 sums at the bf16 rate.
//
// Tiles of 128 x 128 of dw, k-tiles of 32 rows; two groups of four waves, each
// with two LDS stages and half of the workgroup's k-tiles, whose sums meet in LDS:
// two waves a SIMD, and half the slices' sums of two workgroups on a CU.  A k-tile
// is multiplied from registers while the next one's operands are read and the one
// after that is written; the loads of the next four are in flight to registers.
// LDS holds both operands as [32 rows][columns] (gemm_tiles.hpp's MN layout, read by
// ds_read_b64_tr_b16).  Rows past the last are zeros in both operands (a zero in
// one alone would turn the other's infinity into a NaN), columns past D or H are
// not stored.  With few tiles the rows are cut into slices, whose sums are added
// in order by another launch; a slice's tiles run on one XCD, or each of the eight
// would fetch its rows.
//
// What bounds it: no unit alone.  The LDS is busy 0.48 of 2048^3's cycles and 0.38 of
// 10000 x 784 x 500's (0.09 and 0.07 of them for conflicts), the matrix instructions
// 0.34 and 0.25; the rest is waits of a k-tile's chain and the way in and out: 2048^3
// takes 23 to 25 us (690-750 TFLOP/s), of which 8 do not depend on the rows (256 rows
// take 9.9); 10000 x 784 x 500 23 us with its sums (1.6 MB of dw as 13 MB of slices).  Against one group and
// two workgroups a CU: 2048^3 33 -> 23 us, 4096 x 1024^2 26 -> 24, 65536 x 512^2 47 ->
// 44, 10000 x 784 x 500 22 -> 24, 100 x 2000 x 1000 7 -> 8.
#pragma once

#include <utility>

#include "gemm_fp8.hpp"
#include "gemm_pingpong.hpp"

namespace ch {
namespace fp8 {

struct Grad {
    static constexpr int BM = 128, BN = 128, BK = 32, NW = 4, GROUPS = 2;
    static constexpr int THREADS = 64 * NW;  // of a group
    static constexpr int WM = BM / 64, WN = NW / WM, TN = BN / WN, FM = 2, FN = TN / 32;  // waves of 64 x TN
    static constexpr int A_BYTES = BK * BM * 2, B_BYTES = BK * BN * 2, STAGE = A_BYTES + B_BYTES;
    static constexpr int PF = 4;  // k-tiles whose loads are in flight, in registers
    static constexpr int CHUNKS_A = BK * BM / 16 / THREADS;  // of 16 codes a thread
    static constexpr int CHUNKS_B = BK * BN / 8 / THREADS;   // of 8 values
    static_assert(PF % 2 == 0, "a k-tile's stage follows from its slot");
    static_assert(CHUNKS_A * 16 * THREADS == BK * BM && CHUNKS_B * 8 * THREADS == BK * BN, "whole chunks");
};

typedef float v4f __attribute__((ext_vector_type(4)));
struct __attribute__((packed)) PackedChunk { v4u v; };

static __global__ __launch_bounds__(512, 2) void gemm_fp8_grad_kernel(
    const uint8_t* __restrict__ xq, const uint8_t* __restrict__ xs, const uint16_t* __restrict__ g,
    float* __restrict__ dw, int B, int D, int H, int tiles_m, int tiles_n, int slices, int rows_per_slice,
    int64_t slice_stride) {
    using P = Grad;
    constexpr int BM = P::BM, BN = P::BN, BK = P::BK, FM = P::FM, FN = P::FN, PF = P::PF;
    __shared__ __attribute__((aligned(1024))) char lds[P::GROUPS][2][P::STAGE];
    const int lane = threadIdx.x & 63, tid = (int)threadIdx.x % P::THREADS;
    const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / P::THREADS);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % P::NW;
    char(*const smem)[P::STAGE] = lds[group];
    const int wm = (wave / P::WN) * 64, wn = (wave % P::WN) * P::TN;
    int slice, tm, tn;
    ch::block_coords((int)blockIdx.x, tiles_m, tiles_n, slices, slice, tm, tn);
    const int d0 = tm * BM, h0 = tn * BN;
    const int b0 = slice * rows_per_slice, b1 = min(B, b0 + rows_per_slice);
    // whole k-tiles (without g's last row), half of them each group's; then those left
    const int nk = (b1 - b0 + BK - 1) / BK, whole = min(b1 - b0, B - 1 - b0) / BK / 2;
    const int first = group * whole;
    const int64_t pitch = pitch_of(D), sp = scale_pitch(B);
    dw += (int64_t)slice * slice_stride;

    // A thread's chunks, 16 codes of a row and 8 values of g of a row, as offsets
    // from the k-tile's first row.  A chunk past the columns reads some other one:
    // its columns are not stored.  One across the end of its row reads on in the next
    // rows, which lie in g: H >= 4, and no row of these k-tiles is the last.
    constexpr int CPA = BM / 16, CPB = BN / 8;
    uint32_t oa[P::CHUNKS_A], os[P::CHUNKS_A], ob[P::CHUNKS_B];
#pragma unroll
    for (int j = 0; j < P::CHUNKS_A; ++j) {
        const int e = tid + P::THREADS * j;
        const int64_t col = min((int64_t)d0 + 16 * (e % CPA), pitch - 16);
        oa[j] = (uint32_t)(e / CPA * pitch + col);
        os[j] = (uint32_t)(e / CPA);
    }
    const uint8_t* const scales = xs + (int64_t)min((int64_t)d0 / kBlock, pitch / kBlock - 1) * sp;
#pragma unroll
    for (int j = 0; j < P::CHUNKS_B; ++j) {
        const int e = tid + P::THREADS * j, col = h0 + 8 * (e % CPB);
        ob[j] = (uint32_t)((e / CPB * (int64_t)H + (col < H ? col : 0)) * 2);
    }
    constexpr int LAST = PF;  // the slot of the k-tile after those in pairs
    v4u ra[PF + 1][P::CHUNKS_A], rb[PF + 1][P::CHUNKS_B];
    int sc[PF + 1][P::CHUNKS_A];
    auto load = [&](int slot, int kt) {
        const int64_t row = b0 + (int64_t)(first + kt) * BK;
        const uint8_t* const pa = xq + row * pitch;
        const uint8_t* const ps = scales + row;
        const uint16_t* const pb = g + row * H;
#pragma unroll
        for (int j = 0; j < P::CHUNKS_A; ++j) {
            ra[slot][j] = *reinterpret_cast<const v4u*>(pa + oa[j]);
            sc[slot][j] = ps[os[j]];
        }
#pragma unroll
        for (int j = 0; j < P::CHUNKS_B; ++j)
            rb[slot][j] = reinterpret_cast<const PackedChunk*>(reinterpret_cast<const char*>(pb) + ob[j])->v;
    };
    // A k-tile after those in pairs: an odd one, or that with the slice's last row
    // where it is not a whole one, or g's last row, past which a chunk across the end
    // of it may not reach.  Rows past the slice are zeros.
    // Every load lies inside the slice, without a branch of a lane's own.
    auto load_last = [&](int kt) {
        const int row0 = b0 + kt * BK;
#pragma unroll
        for (int j = 0; j < P::CHUNKS_A; ++j) {
            const int r = row0 + (int)os[j];
            const int64_t row = min(r, b1 - 1);
            ra[LAST][j] = *reinterpret_cast<const v4u*>(xq + row * pitch + (oa[j] - os[j] * (uint32_t)pitch));
            sc[LAST][j] = scales[row];
        }
#pragma unroll
        for (int j = 0; j < P::CHUNKS_B; ++j) {
            const int e = tid + P::THREADS * j, r = row0 + e / CPB, col = h0 + 8 * (e % CPB);
            const uint16_t* const p = g + (int64_t)min(r, b1 - 1) * H;
            if (h0 + BN <= H) {
                rb[LAST][j] = reinterpret_cast<const PackedChunk*>(p + col)->v;
            } else {
                uint32_t v[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] = p[min(col + c, H - 1)];
#pragma unroll
                for (int c = 0; c < 8; c += 2) rb[LAST][j][c / 2] = v[c] | v[c + 1] << 16;
            }
        }
    };
    auto clear_last = [&](int kt) {
        const int row0 = b0 + kt * BK;
#pragma unroll
        for (int j = 0; j < P::CHUNKS_A; ++j)
            if (row0 + (int)os[j] >= b1) ra[LAST][j] = v4u{};
#pragma unroll
        for (int j = 0; j < P::CHUNKS_B; ++j)
            if (row0 + (tid + P::THREADS * j) / CPB >= b1) rb[LAST][j] = v4u{};
    };
    auto put = [&](int stage, int slot) {
        char* const ta = smem[stage];
        char* const tb = ta + P::A_BYTES;
#pragma unroll
        for (int j = 0; j < P::CHUNKS_A; ++j) {
            const int e = tid + P::THREADS * j, kr = e / CPA, c = 2 * (e % CPA);
            const float scale = scale_value(sc[slot][j]);
            bf16x2 w[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(ra[slot][j][i], scale, false);
                w[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(ra[slot][j][i], scale, true);
            }
            v4u lo, hi;
            __builtin_memcpy(&lo, w, 16);
            __builtin_memcpy(&hi, w + 4, 16);
            // chunks c and c + 1 lie side by side: the swizzle flips even bits of the slot alone
            *reinterpret_cast<v4u*>(ta + kr * 256 + tiles::mn_slot<2>(kr, c) * 16) = lo;
            *reinterpret_cast<v4u*>(ta + kr * 256 + tiles::mn_slot<2>(kr, c + 1) * 16) = hi;
        }
#pragma unroll
        for (int j = 0; j < P::CHUNKS_B; ++j) {
            const int e = tid + P::THREADS * j, kr = e / CPB, c = e % CPB;
            *reinterpret_cast<v4u*>(tb + kr * 256 + tiles::mn_slot<2>(kr, c) * 16) = rb[slot][j];
        }
    };

    v16f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v16f{};
    tiles::v8bf fa[2][BK / 16][FM], fb[2][BK / 16][FN];
    auto read = [&](auto set, int stage) {
        constexpr int F = decltype(set)::value;
        const char* const ta = smem[stage];
        const char* const tb = ta + P::A_BYTES;
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[F][kk][i] = tiles::read_frag<false, 128, BK>(ta, wm + 32 * i, kk, lane);
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[F][kk][j] = tiles::read_frag<false, 128, BK>(tb, wn + 32 * j, kk, lane);
        }
    };
    auto multiply = [&](auto set) {
        constexpr int F = decltype(set)::value;
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk)
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[F][kk][i], fb[F][kk][j], acc[i][j], 0, 0, 0);
    };
    // K-tile kt is multiplied from registers while the next one's operands are read
    // from its stage, and the one after that goes to the stage that kt's came from
    // (read by everybody before the barrier).
    auto step = [&](auto slot_, int kt) {
        constexpr int SLOT = decltype(slot_)::value, NEXT = (SLOT + 2) % PF;
        __syncthreads();
        read(std::integral_constant<int, (SLOT + 1) % 2>{}, (SLOT + 1) % 2);
        put(SLOT % 2, NEXT);                      // past the last k-tile nobody reads it
        load(NEXT, min(kt + 2 + PF, whole - 1));  // always: a branch would cost the count of loads in flight
        multiply(std::integral_constant<int, SLOT % 2>{});
        // the LDS's work goes between the first five of the eight matrix instructions:
        // what is done by the barrier costs no wait there
#pragma unroll
        for (int i = 0; i < 5; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // LDS reads
            __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);  // VALU
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // LDS writes
            __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // loads
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 3, 0);
    };
    const bool more = 2 * whole < nk;  // at most one for each group
    if (more) {
        load_last(2 * whole + group);
        asm volatile("" ::: "memory");
    }
    if (whole > 0) {
#pragma unroll
        for (int t = 0; t < PF; ++t) {
            load(t, min(t, whole - 1));
            asm volatile("" ::: "memory");  // in this order, which the loop's waits count on
        }
        put(0, 0);
        put(1, 1);
        load(0, min(PF, whole - 1));
        asm volatile("" ::: "memory");
        load(1, min(PF + 1, whole - 1));
        __syncthreads();
        read(std::integral_constant<int, 0>{}, 0);
        // rounds of PF alone in the loop: a way out of one's middle would have the loop's
        // first wait expect any slot's loads to be the newest
        int kt = 0;
        for (; kt + PF <= whole; kt += PF) pingpong_unrolled<PF, 0>(kt, kt + PF, step, std::make_integer_sequence<int, PF>{});
        pingpong_unrolled<PF, 0>(kt, whole, step, std::make_integer_sequence<int, PF>{});
    }
    if (more) {
        clear_last(2 * whole + group);
        __syncthreads();  // the stage may still be read
        put(0, LAST);
        __syncthreads();
        read(std::integral_constant<int, 0>{}, 0);
        multiply(std::integral_constant<int, 0>{});
    }

    // The groups' sums meet in LDS, a row of blocks at a time, and leave in whole lines.
    constexpr int ROWS = 32 * P::WM;
    static_assert(ROWS * BN * 4 <= 2 * P::STAGE, "a row of blocks fits the group's stages");
    const bool whole4 = H % 4 == 0;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        __syncthreads();
        float* const to = reinterpret_cast<float*>(smem) + (wm / 2 + 4 * (lane >> 5)) * BN + wn + (lane & 31);
#pragma unroll
        for (int v = 0; v < 16; ++v)
#pragma unroll
            for (int j = 0; j < FN; ++j) to[(8 * (v / 4) + v % 4) * BN + 32 * j] = acc[i][j][v];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < ROWS * BN / 4 / (P::GROUPS * P::THREADS); ++q) {
            const int e = (int)threadIdx.x + q * P::GROUPS * P::THREADS;
            const int row = e / (BN / 4), d = d0 + row / 32 * 64 + 32 * i + row % 32, h = h0 + 4 * (e % (BN / 4));
            v4f y = reinterpret_cast<const v4f*>(lds[0])[e] + reinterpret_cast<const v4f*>(lds[1])[e];
            float* const out = dw + (int64_t)d * H + h;
            if (d >= D || h >= H) continue;
            if (whole4) {
                *reinterpret_cast<v4f*>(out) = y;
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (h + c < H) out[c] = y[c];
            }
        }
    }
}

}  // namespace fp8
}  // namespace ch
