// gemm_fp8_pingpong.hpp -- large 8-bit products in bf16: 256 x 256 tiles, two
// groups of waves in alternating phases (as gemm_pingpong.hpp).
//
// Eight waves, each 128 x 64 of C in 4 x 2 blocks of 32 x 32; waves 0-3 and 4-7
// sit one of each on a SIMD, and while one group multiplies (C phase, 8 matrix
// instructions, 512 cycles) the other reads its next operands from LDS and
// starts copies (M phase).  A barrier ends each phase; both groups run one loop,
// group 1 a barrier behind (in a loop each, as pingpong_schedule has it, the
// accumulators' tuples of 16 registers were copied and spilled).
//
// A k-block of 128 takes two phases: phase x = 0, 1 multiplies half x of the
// wave's rows, over the whole k-block, by columns that stay in registers for
// both.  So a k-contiguous operand is copied in whole 128-byte lines (in k-tiles of
// 64 bytes a row, two L2 requests for each line, 8192^3 A.B^T took 454 us).
// One workgroup a CU walks its tiles, so that the stores of one overlap the first
// k-blocks of the next.
// LDS: four units of A (128 rows x 128 bytes, half x of both groups' rows), two
// of B (32 KiB), and the scales of 64 k-blocks, 256 + 256 bytes each; K is
// walked in segments of 8192.
//
// What bounds it: for 8192^3 the matrix cores, busy 0.90 of the cycles in which the
// shader engines are, at the clock that power leaves (1.6-1.7 GHz): 376 us (A.B) and
// 382 (A.B^T) in a loop, 2.9 PFLOP/s.  65536 x 4096 x 1024 keeps them busy 0.56: 8
// k-blocks between a tile's first copies and its stores, 512 MiB of C in all; 273 us in
// a loop, 2.0 PFLOP/s.  Waiting less in the loop gave 8192^3 nothing any more.
// Just past a whole round of tiles the last one is paid in full (4096^2 x 8192 100 us,
// 4352 x 4096 x 8192, 16 tiles more, 157).
#pragma once

#include "gemm_fp8_tiled.hpp"

namespace ch {
namespace fp8 {

struct PingPong {
    static constexpr int BM = 256, BN = 256, BK = 128, NW = 8, WN = 4;
    static constexpr int TM = 128, TN = 64, FM = TM / 32, FN = TN / 32;
    static constexpr int UNITS_A = 4, UNITS_B = 2, UNIT_A = 128 * BK, UNIT_B = 256 * BK;
    static constexpr int B_AT = UNITS_A * UNIT_A, SCALE_AT = B_AT + UNITS_B * UNIT_B;
    static constexpr int SEGMENT = 64;                 // k-blocks whose scales LDS holds
    static constexpr int SCALE_BYTES = SEGMENT * 256;  // of one operand
    static constexpr int LDS_BYTES = SCALE_AT + 2 * SCALE_BYTES;
    static_assert(LDS_BYTES <= 160 * 1024, "LDS per workgroup");
};

// Slot of chunk c (16 bytes) of row r of a 128-byte KC tile row: 16 lanes read a
// chunk of 16 rows, two of which share 256 bytes of banks.
__device__ __forceinline__ int kc128_slot(int r, int c) { return c ^ ((r & 7) ^ ((r >> 3) & 1)); }

// K off 128 (RAGGED) matters to a B stored K x N alone: its last k-block's rows.
template <bool NT, bool RAGGED>
__global__ __launch_bounds__(512) void gemm_fp8_pingpong_kernel(Operands o, uint16_t* __restrict__ C, int tiles_m,
                                                                int tiles_n, int nt_c) {
    using P = PingPong;
    constexpr int FN = P::FN, NW = P::NW, BK = P::BK;
    __shared__ __attribute__((aligned(1024))) char smem[P::LDS_BYTES];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = wave / P::WN, wn = wave % P::WN;
    const int nkb = (o.K + BK - 1) / BK;
    const uint32_t lds0 = lds_addr(smem);

    // ---- copies ----
    const int64_t step_b = NT ? BK : BK * o.pb;
    int m0, n0;
    const char* a0;
    const char* b0;
    uint32_t va[2][2], vb[4], vb_last[4];
    // The lane offsets count from the tile's first row (and column), so that
    // only a tile at an edge, whose rows are held back, has its own.
    bool inside = false;
    auto set_tile = [&](int tile) {
        int tm, tn;
        ch::tile_coords(tile, tiles_m, tiles_n, tm, tn);
        m0 = tm * P::BM;
        n0 = tn * P::BN;
        a0 = reinterpret_cast<const char*>(o.a) + m0 * o.pa;
        b0 = reinterpret_cast<const char*>(o.b) + (NT ? n0 * o.pb : n0);
        const bool was_inside = inside;
        inside = ch::whole_tile(m0, P::BM, o.M) && (NT ? n0 + P::BN <= o.N : n0 + P::BN <= o.pb);
        if (inside && was_inside) return;
#pragma unroll
        for (int j = 0; j < 2; ++j) {  // 8 rows an instruction: unit rows 0-63 are group 0's, 64-127 group 1's
            const int r = (wave + NW * j) * 8 + (lane >> 3);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int row = (r & 63) + 64 * x + 128 * (r >> 6);
                va[x][j] = (uint32_t)(min(row, o.M - 1 - m0) * o.pa + 16 * kc128_slot(r, lane & 7));
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int q = wave + NW * j;
            if constexpr (NT) {
                const int r = q * 8 + (lane >> 3);
                vb[j] = (uint32_t)(min(r, o.N - 1 - n0) * o.pb + 16 * kc128_slot(r, lane & 7));
            } else {
                const int kr = q * 4 + (lane >> 4);
                const int64_t col = min((int64_t)16 * mn_slot<256>(kr, lane & 15), o.pb - 16 - n0);
                vb[j] = (uint32_t)(kr * o.pb + col);
                if constexpr (RAGGED) vb_last[j] = (uint32_t)(min(kr, o.K - 1 - (nkb - 1) * BK) * o.pb + col);
            }
        }
    };
    int first = 0, count = min(nkb, P::SEGMENT);  // the segment's first k-block, and its k-blocks
    // Unit `unit` of A: half x of the rows of k-block first + min(p, count - 1).
    auto issue_a = [&](int unit, int x, int p) {
        const char* const a = a0 + (int64_t)(first + min(p, count - 1)) * BK;
        const uint32_t dst = lds0 + (uint32_t)(unit * P::UNIT_A) + 1024u * (uint32_t)wave;
#pragma unroll
        for (int j = 0; j < 2; ++j) dma16(a, va[x][j], dst + (uint32_t)(1024 * NW * j));
    };
    // Half y of the copies of B's k-block p into unit `unit`.
    auto issue_b = [&](int unit, int y, int p) {
        const int src = first + min(p, count - 1);
        const char* const b = b0 + src * step_b;
        const uint32_t dst = lds0 + (uint32_t)(P::B_AT + unit * P::UNIT_B) + 1024u * (uint32_t)wave;
#pragma unroll
        for (int j = 2 * y; j < 2 * y + 2; ++j) {
            const uint32_t v = !NT && RAGGED && src == nkb - 1 ? vb_last[j] : vb[j];
            dma16(b, v, dst + (uint32_t)(1024 * NW * j));
        }
    };
    // The segment's scales: 16 lanes copy a k-block's 256 bytes.
    auto issue_scales = [&]() {
        for (int q = wave; q < P::SEGMENT / 4 && first + 4 * q < nkb; q += NW) {
            const int kb = min(first + 4 * q + (lane >> 4), nkb - 1);
            const int64_t m = min((int64_t)m0 + 16 * (lane & 15), o.spa - 16);
            int64_t at;
            if constexpr (NT) at = kb * o.spb + min((int64_t)n0 + 16 * (lane & 15), o.spb - 16);
            else at = min((int64_t)(n0 / kBlock + (lane & 15) / 8), o.pb / kBlock - 1) * o.spb + (int64_t)kb * kBlock;
            const uint32_t dst = lds0 + (uint32_t)P::SCALE_AT + 1024u * (uint32_t)q;
            dma16_far(o.as + kb * o.spa + m, dst);
            dma16_far(o.bs + at, dst + P::SCALE_BYTES);
        }
    };

    // ---- fragments ----
    v16f acc[P::FM][FN];
    auto zero_acc = [&]() {
#pragma unroll
        for (int i = 0; i < P::FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = v16f{};
    };
    v8i fa[2][2], fb[FN][2];  // [block][half of the k-block]
    int sa[2], sb[FN];
    // Read addresses, opaque so that each stays one register beside immediates:
    // of chunk 2 (lane / 32) + x, and, where the swizzle mixes in the half of
    // the k-block or the block of columns, of each.
    uint32_t ra[2][2], rb[2][2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int r = lane & 31;
            const uint32_t at = (uint32_t)(r * BK + kc128_slot(r, 4 * s + 2 * (lane >> 5) + x) * 16);
            ra[s][x] = lds0 + (uint32_t)(grp * 64 * BK) + at;
            if constexpr (NT) {
                rb[s][x] = lds0 + (uint32_t)(P::B_AT + wn * P::TN * BK) + at;
            } else {  // one per block of columns x; k-rows 64 apart share a swizzle
                const int col = wn * P::TN + 32 * x + (lane & 16) + 8 * (lane & 1);
                const int kr = 64 * s + 32 * (lane >> 5) + ((lane & 15) >> 1);
                rb[s][x] = lds0 + (uint32_t)(P::B_AT + kr * 256 + mn_slot<256>(kr, col >> 4) * 16 + (col & 15));
            }
            tiles::opaque(ra[s][x]);
            tiles::opaque(rb[s][x]);
        }
    uint32_t rsa = lds0 + (uint32_t)(P::SCALE_AT + grp * P::TM + (lane & 31));
    uint32_t rsb = lds0 + (uint32_t)(P::SCALE_AT + P::SCALE_BYTES + wn * P::TN + (lane & 31));
    tiles::opaque(rsa);
    tiles::opaque(rsb);
    auto read16 = [](uint32_t at) { return *(const lds_v4i*)(uintptr_t)at; };
    auto read_tr = [](uint32_t at) { return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(uintptr_t)at); };
    typedef __attribute__((address_space(3))) uint8_t lds_u8;
    auto read8 = [](uint32_t at) { return (int)*(const lds_u8*)(uintptr_t)at; };

    // M phase 2 p + X of k-block p (parity PB): reads, then the copies of B's
    // k-block (4 instructions a wave over the phases 2 p - 1 and 2 p for k-block
    // p + 1, whose unit was last read in phase 2 p - 2) and of A's unit three
    // phases on.  Each group's wait is for its own copies of the next phase's
    // operands: what may be left in flight is newer.  A segment starts with two
    // k-blocks in LDS: phase 0 has nothing to copy, and phases 0 to 2 (of
    // k-blocks 0 and 1) no copy to wait for, which leaves the stores of the tile
    // before, older than their copies, the time to land.
    auto m_phase = [&](auto block, auto half, int p) {
        constexpr int BLOCK = decltype(block)::value, X = decltype(half)::value;
        constexpr int PB = BLOCK % 2, UA = 2 * PB + X;
#pragma unroll
        for (int i = 0; i < 2; ++i) sa[i] = read8(rsa + (uint32_t)p * 256 + 64 * X + 32 * i);
        if constexpr (X == 0) {
#pragma unroll
            for (int j = 0; j < FN; ++j) sb[j] = read8(rsb + (uint32_t)p * 256 + 32 * j);
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if constexpr (NT) {
                        const v4i lo = read16(rb[s][0] + (uint32_t)(PB * P::UNIT_B + j * 32 * BK));
                        const v4i hi = read16(rb[s][1] + (uint32_t)(PB * P::UNIT_B + j * 32 * BK));
                        fb[j][s] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                    } else {
                        v2i t[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) t[x] = read_tr(rb[s][j] + (uint32_t)(PB * P::UNIT_B + x * 8 * 256));
                        fb[j][s] = v8i{t[0][0], t[0][1], t[1][0], t[1][1], t[2][0], t[2][1], t[3][0], t[3][1]};
                    }
                }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const v4i lo = read16(ra[s][0] + (uint32_t)(UA * P::UNIT_A + i * 32 * BK));
                const v4i hi = read16(ra[s][1] + (uint32_t)(UA * P::UNIT_A + i * 32 * BK));
                fa[i][s] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
        if constexpr (BLOCK != 0 || X != 0) {
            if constexpr (X == 0) issue_b(1 - PB, 1, p + 1);
            else issue_b(PB, 0, p + 2);
            issue_a((UA + 3) % P::UNITS_A, 1 - X, p + 1 + X);
        }
        wait_reads_and_copies<2 * BLOCK + X < 3 ? 63 : (X == 0 ? 8 : 6)>();
    };
    auto c_phase = [&](auto half) {
        constexpr int X = decltype(half)::value;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[2 * X + i][j] = mfma(fa[i][s], fb[j][s], acc[2 * X + i][j], sa[i], sb[j]);
        // the results are wanted here: else some of them are formed past the barrier
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) wanted(acc[2 * X + i][j]);
        __builtin_amdgcn_s_setprio(0);
    };
    auto step = [&](auto block, int p) {
        m_phase(block, std::integral_constant<int, 0>{}, p);
        asm volatile("s_barrier" ::: "memory");
        c_phase(std::integral_constant<int, 0>{});
        asm volatile("s_barrier" ::: "memory");
        m_phase(block, std::integral_constant<int, 1>{}, p);
        asm volatile("s_barrier" ::: "memory");
        c_phase(std::integral_constant<int, 1>{});
        asm volatile("s_barrier" ::: "memory");
    };
    // The first two k-blocks of the segment, and its scales.
    auto prologue = [&]() {
        issue_scales();
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            issue_b(p, 0, p);
            issue_b(p, 1, p);
            issue_a(2 * p, 0, p);
            issue_a(2 * p + 1, 1, p);
        }
    };
    // A segment whose first copies have landed in this wave's part of LDS.
    auto segment = [&]() {
        asm volatile("s_barrier" ::: "memory");
        if (grp == 1) asm volatile("s_barrier" ::: "memory");
        step(std::integral_constant<int, 0>{}, 0);
        if (count > 1) {
            step(std::integral_constant<int, 1>{}, 1);
            for (int p = 2; p < count; p += 2) {
                step(std::integral_constant<int, 2>{}, p);
                if (p + 1 >= count) break;
                step(std::integral_constant<int, 3>{}, p + 1);
            }
        }
        if (grp == 0) asm volatile("s_barrier" ::: "memory");
        // The last barrier has every wave past its LDS reads, and a wave's copies
        // go where only it wrote before.
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };

    // Tiles blockIdx.x, + gridDim.x, ...: the next tile's first copies go out
    // before this one's C, and are waited for after it.
    const int total = tiles_m * tiles_n;
    int tile = (int)blockIdx.x;
    set_tile(tile);
    prologue();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    for (;;) {
        zero_acc();
        segment();
        while (first + count < nkb) {
            first += count;
            count = min(nkb - first, P::SEGMENT);
            prologue();
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            segment();
        }
        first = 0;
        count = min(nkb, P::SEGMENT);
        const int r0 = m0 + grp * P::TM, c0 = n0 + wn * P::TN;
        const bool whole = ch::whole_tile(m0, P::BM, o.M) && n0 + P::BN <= o.N;
        tile += (int)gridDim.x;
        const bool more = tile < total;
        if (more) {
            set_tile(tile);
            prologue();
        }
        if (whole) {
            if (nt_c) store_blocks<P::FM, true, true>(C, o.M, o.N, r0, c0, acc, lane);
            else store_blocks<P::FM, true>(C, o.M, o.N, r0, c0, acc, lane);
            // 64 stores follow the copies: with one of them landed, so have the copies
            asm volatile("s_waitcnt vmcnt(63)" ::: "memory");
        } else {
            store_blocks<P::FM, false>(C, o.M, o.N, r0, c0, acc, lane);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        if (!more) break;
    }
}

}  // namespace fp8
}  // namespace ch
