// gemm_fp8_tiled.hpp -- 8-bit products on tiles small enough for two
// workgroups on a CU, so that one stores C while the other multiplies.
//
// Waves of TM x 64 of C in blocks of 32 x 32; k-tiles of 64 (64 bytes a row) in
// a ring of S LDS stages, one barrier a k-tile.  The scales lie beside the ring,
// a chunk of 8 k-blocks read while the next is copied; a lane reads its own as
// bytes, once a k-block.
#pragma once

#include <utility>

#include "gemm_fp8.hpp"
#include "gemm_pingpong.hpp"

namespace ch {
namespace fp8 {

template <int BM_, int BN_, int TM_, int S_>
struct Tiled {
    static constexpr int BM = BM_, BN = BN_, BK = 64, TM = TM_, TN = 64, S = S_;
    static constexpr int WM = BM / TM, WN = BN / TN, NW = WM * WN, THREADS = 64 * NW;
    static constexpr int FM = TM / 32, FN = TN / 32;
    static constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK;
    static constexpr int PER_A = A_BYTES / 1024 / NW, PER_B = B_BYTES / 1024 / NW, LPW = PER_A + PER_B;
    static constexpr int CHUNK = BM < 128 || BN < 128 ? 16 : 8;  // k-blocks a scale chunk: whole copies
    static constexpr int B_AT = S * A_BYTES, SCALE_A_AT = B_AT + S * B_BYTES;
    static constexpr int SCALE_B_AT = SCALE_A_AT + 2 * CHUNK * BM;
    static constexpr int LDS_BYTES = SCALE_B_AT + 2 * CHUNK * BN;
    static_assert(PER_A * 1024 * NW == A_BYTES && PER_B * 1024 * NW == B_BYTES, "whole copies per wave");
    static_assert(CHUNK * BM % 1024 == 0 && CHUNK * BN % 1024 == 0 && CHUNK * (BM + BN) / 1024 <= NW,
                  "a whole scale copy per wave at most");
    static_assert(LDS_BYTES <= 80 * 1024, "two workgroups on a CU");
};

// Slot of chunk c (16 bytes) of row r of a 64-byte KC tile row: 16 lanes read a
// chunk of 16 rows, four of which share each 64 bytes of banks.
__device__ __forceinline__ int kc64_slot(int r, int c) { return c ^ (((r >> 1) & 3) ^ ((r >> 3) & 1)); }

// From each lane's column of rows v (low half) and v + 1: the even lane gets its
// column and the next of row v, the odd lane the one before and its own of row
// v + 1.
__device__ __forceinline__ uint32_t pair_up(uint32_t p, uint32_t select) {
    const uint32_t q = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)p, 0xB1, 0xF, 0xF, true);  // of lane l ^ 1
    return __builtin_amdgcn_perm(q, p, select);
}
__device__ __forceinline__ uint32_t pair_select(int lane) {
    // bytes 0-3 are p's, 4-7 q's: even lanes (p.lo, q.lo), odd (q.hi, p.hi)
    return lane & 1 ? 0x03020706u : 0x05040100u;
}

// A wave's FM x 2 blocks of 32 x 32 to C from (r0, c0), a row's 64 columns at a
// time.  Rows v and v + 1 of each block are packed, and v_permlane32_swap of the
// two blocks' words pairs their halves: the first then holds 64 columns of rows
// 8 (v/4) + v%4 and the next, the second those 4 below.  Full 128-byte lines in
// bf16, two rows an instruction.  Addresses are a scalar per row and one lane
// offset (formed per element in 64 bits, they took half of the 5300 cycles in
// which a workgroup of 256 x 256 stored its tile).
// WHOLE: all of it lies in C.  NTC: stored non-temporally.
template <int FM, bool WHOLE, bool NTC = false>
__device__ __forceinline__ void store_blocks(uint16_t* __restrict__ C, int M, int N, int r0, int c0,
                                             const v16f (&acc)[FM][2], int lane) {
    typedef uint32_t __attribute__((aligned(2))) u32_2;
    const uint32_t select = pair_select(lane);
    const int c = c0 + (lane & 62);
    const uint32_t at = (uint32_t)(((int64_t)(lane & 1) * N + (lane & 62)) * 2);  // N <= 2^23
    char* const base = reinterpret_cast<char*>(C + (int64_t)r0 * N + c0);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int v = 0; v < 16; v += 2) {
            const auto s = __builtin_amdgcn_permlane32_swap(pack_bf16(acc[i][0][v], acc[i][0][v + 1]),
                                                            pack_bf16(acc[i][1][v], acc[i][1][v + 1]), false, false);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t w = pair_up(h ? s[1] : s[0], select);
                const int row = 32 * i + 8 * (v / 4) + v % 4 + 4 * h, r = r0 + row + (lane & 1);
                u32_2* const p = reinterpret_cast<u32_2*>(base + (int64_t)row * N * 2 + at);
                if constexpr (WHOLE && NTC) __builtin_nontemporal_store(w, p);
                else if (WHOLE || (r < M && c + 1 < N)) *p = w;
                else if (r < M && c < N) *reinterpret_cast<uint16_t*>(p) = (uint16_t)w;
            }
        }
}
template <int FM, bool WHOLE>
__device__ __forceinline__ void store_blocks(float* __restrict__ C, int M, int N, int r0, int c0,
                                             const v16f (&acc)[FM][2], int lane) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const int r = r0 + 32 * i + 8 * (v / 4) + 4 * (lane >> 5) + v % 4;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c = c0 + 32 * j + (lane & 31);
                if (WHOLE || (r < M && c < N)) C[(int64_t)r * N + c] = acc[i][j][v];
            }
        }
}

// Every wave's copies but its N newest have landed.
template <int N>
__device__ __forceinline__ void landed_barrier() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    asm volatile("s_barrier" ::: "memory");
}
// This wave's LDS reads have come, and its copies but the N newest.
template <int N>
__device__ __forceinline__ void wait_reads_and_copies() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
// v is formed by here.
__device__ __forceinline__ void wanted(const v16f& v) { asm volatile("" : : "v"(v)); }

// RAGGED: K off 64, which matters to a B stored K x N: its last k-tile's rows.
// WIDE: codes widened to bf16, for f32 results.  Several slices of K: C is their
// f32 sums, `part` elements apart.
template <bool NT, bool RAGGED, bool WIDE, class T, int BM, int BN, int TM, int S>
__global__ __launch_bounds__(BM / TM * BN, 2) void gemm_fp8_tiled_kernel(Operands o, T* __restrict__ C, int tiles_m,
                                                                         int tiles_n, int slices, int64_t part) {
    using P = Tiled<BM, BN, TM, S>;
    constexpr int FM = P::FM, FN = P::FN, NW = P::NW, BK = P::BK;
    __shared__ __attribute__((aligned(1024))) char smem[P::LDS_BYTES];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = (wave / P::WN) * TM, wn = (wave % P::WN) * P::TN;
    int slice, tm, tn;
    ch::block_coords((int)blockIdx.x, tiles_m, tiles_n, slices, slice, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int all = (o.K + BK - 1) / BK, nkb = (o.K + kBlock - 1) / kBlock;
    // the slice's k-blocks, and its k-tiles (counted from its first)
    const int kb0 = (int)((int64_t)nkb * slice / slices), kb1 = (int)((int64_t)nkb * (slice + 1) / slices);
    const int nk = min(all, kb1 * (kBlock / BK)) - kb0 * (kBlock / BK);
    C += slice * part;
    const uint32_t lds0 = lds_addr(smem);

    // ---- copies ----
    const int64_t step_b = NT ? BK : BK * o.pb;
    const char* const a0 = reinterpret_cast<const char*>(o.a) + m0 * o.pa + (int64_t)kb0 * kBlock;
    const char* const b0 =
        reinterpret_cast<const char*>(o.b) + (NT ? n0 * o.pb : 0) + kb0 * (kBlock / BK) * step_b;
    const bool has_last = kb1 == nkb;
    uint32_t va[P::PER_A], vb[P::PER_B], vb_last[P::PER_B];
#pragma unroll
    for (int j = 0; j < P::PER_A; ++j) {
        const int r = (wave + NW * j) * 16 + (lane >> 2);
        va[j] = (uint32_t)(min(r, o.M - 1 - m0) * o.pa + 16 * kc64_slot(r, lane & 3));
    }
#pragma unroll
    for (int j = 0; j < P::PER_B; ++j) {
        if constexpr (NT) {
            const int r = (wave + NW * j) * 16 + (lane >> 2);
            vb[j] = (uint32_t)(min(r, o.N - 1 - n0) * o.pb + 16 * kc64_slot(r, lane & 3));
        } else {
            constexpr int CPR = BN / 16;
            const int kr = (wave + NW * j) * (64 / CPR) + lane / CPR;
            const int64_t col = min((int64_t)n0 + 16 * mn_slot<BN>(kr, lane % CPR), o.pb - 16);
            vb[j] = (uint32_t)(kr * o.pb + col);
            if constexpr (RAGGED) vb_last[j] = (uint32_t)(min(kr, o.K - 1 - (all - 1) * BK) * o.pb + col);
        }
    }
    auto issue = [&](int stage, int kt) {  // k-tile min(kt, nk - 1)
        const int src = min(kt, nk - 1);
        const uint32_t dst = lds0 + 1024u * (uint32_t)wave;
        const char* const a = a0 + (int64_t)src * BK;
        const char* const b = b0 + src * step_b;
#pragma unroll
        for (int j = 0; j < P::PER_A; ++j) dma16(a, va[j], dst + (uint32_t)(stage * P::A_BYTES + 1024 * NW * j));
#pragma unroll
        for (int j = 0; j < P::PER_B; ++j) {
            const uint32_t v = !NT && RAGGED && has_last && src == nk - 1 ? vb_last[j] : vb[j];
            dma16(b, v, dst + (uint32_t)(P::B_AT + stage * P::B_BYTES + 1024 * NW * j));
        }
    };
    // Scales of the slice's chunk h of k-blocks, a copy by each of the first waves.
    auto issue_scales = [&](int h) {
        constexpr int NA = P::CHUNK * BM / 1024, NB = P::CHUNK * BN / 1024;
        if (wave < NA) {
            const int at = 1024 * wave + 16 * lane;
            const int kb = min(kb0 + h * P::CHUNK + at / BM, nkb - 1);
            const int64_t m = min((int64_t)m0 + at % BM, o.spa - 16);
            dma16_far(o.as + kb * o.spa + m, lds0 + (uint32_t)(P::SCALE_A_AT + (h & 1) * P::CHUNK * BM + 1024 * wave));
        } else if (wave < NA + NB) {
            const int at = 1024 * (wave - NA) + 16 * lane;
            const int kb = min(kb0 + h * P::CHUNK + at / BN, nkb - 1);
            int64_t from;
            if constexpr (NT) from = kb * o.spb + min((int64_t)n0 + at % BN, o.spb - 16);
            else from = min((int64_t)(n0 + at % BN) / kBlock, o.pb / kBlock - 1) * o.spb + (int64_t)kb * kBlock;
            dma16_far(o.bs + from, lds0 + (uint32_t)(P::SCALE_B_AT + (h & 1) * P::CHUNK * BN + 1024 * (wave - NA)));
        }
    };

    // ---- fragments ----
    v16f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v16f{};
    int sa[FM], sb[FN];
    // Read addresses, opaque so that each stays one register beside immediates.
    uint32_t ra[2], rb[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int r = lane & 31;
        const uint32_t at = (uint32_t)(r * BK + kc64_slot(r, 2 * (lane >> 5) + x) * 16);
        ra[x] = lds0 + (uint32_t)(wm * BK) + at;
        if constexpr (NT) {
            rb[x] = lds0 + (uint32_t)(P::B_AT + wn * BK) + at;
        } else {  // one address per block of columns
            const int col = wn + 32 * x + (lane & 16) + 8 * (lane & 1), kr = 32 * (lane >> 5) + ((lane & 15) >> 1);
            rb[x] = lds0 + (uint32_t)(P::B_AT + kr * BN + mn_slot<BN>(kr, col >> 4) * 16 + (col & 15));
        }
        tiles::opaque(ra[x]);
        tiles::opaque(rb[x]);
    }
    uint32_t rsa = lds0 + (uint32_t)(P::SCALE_A_AT + wm + (lane & 31));
    uint32_t rsb = lds0 + (uint32_t)(P::SCALE_B_AT + wn + (lane & 31));
    auto read16 = [](uint32_t at) { return *(const lds_v4i*)(uintptr_t)at; };
    auto read_tr = [](uint32_t at) { return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(uintptr_t)at); };
    typedef __attribute__((address_space(3))) uint8_t lds_u8;
    auto read8 = [](uint32_t at) { return (int)*(const lds_u8*)(uintptr_t)at; };

    auto step = [&](auto stage, int u) {
        constexpr int ST = decltype(stage)::value;
        // k-tile u has landed, and every wave is done with k-tile u - 1, whose stage takes k-tile u + S - 1
        landed_barrier<(S - 2) * P::LPW>();
        if ((u & 1) == 0) {
            const uint32_t kb = (uint32_t)(u >> 1) % (2 * P::CHUNK);
#pragma unroll
            for (int i = 0; i < FM; ++i) sa[i] = read8(rsa + kb * BM + 32 * i);
#pragma unroll
            for (int j = 0; j < FN; ++j) sb[j] = read8(rsb + kb * BN + 32 * j);
        }
        v8i fa[FM], fb[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            if constexpr (NT) {
                const v4i lo = read16(rb[0] + (uint32_t)(ST * P::B_BYTES + j * 32 * BK));
                const v4i hi = read16(rb[1] + (uint32_t)(ST * P::B_BYTES + j * 32 * BK));
                fb[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            } else {
                v2i t[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) t[x] = read_tr(rb[j] + (uint32_t)(ST * P::B_BYTES + x * 8 * BN));
                fb[j] = v8i{t[0][0], t[0][1], t[1][0], t[1][1], t[2][0], t[2][1], t[3][0], t[3][1]};
            }
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const v4i lo = read16(ra[0] + (uint32_t)(ST * P::A_BYTES + i * 32 * BK));
            const v4i hi = read16(ra[1] + (uint32_t)(ST * P::A_BYTES + i * 32 * BK));
            fa[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        // the half of the chunk before this one is free from this chunk's second k-tile on
        if (u % (2 * P::CHUNK) == 2 && u + 2 * P::CHUNK - 2 < nk) issue_scales(u / (2 * P::CHUNK) + 1);
        issue((ST + S - 1) % S, u + S - 1);
        if constexpr (WIDE) {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                tiles::v8bf a[FM], b[FN];
#pragma unroll
                for (int i = 0; i < FM; ++i) a[i] = widen(fa[i], t, sa[i]);
#pragma unroll
                for (int j = 0; j < FN; ++j) b[j] = widen(fb[j], t, sb[j]);
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = mfma(fa[i], fb[j], acc[i][j], sa[i], sb[j]);
        }
        // the results are wanted here: else some of them are formed past the next barrier
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) wanted(acc[i][j]);
    };
    issue_scales(0);
#pragma unroll
    for (int t = 0; t < S - 1; ++t) issue(t, t);
    for (int u = 0; u < nk; u += S) pingpong_unrolled<S, 0>(u, nk, step, std::make_integer_sequence<int, S>{});
    // the copies past the last k-tile must land before the LDS is released
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    if (ch::whole_tile(m0, BM, o.M) && n0 + BN <= o.N) store_blocks<FM, true>(C, o.M, o.N, m0 + wm, n0 + wn, acc, lane);
    else store_blocks<FM, false>(C, o.M, o.N, m0 + wm, n0 + wn, acc, lane);
}

}  // namespace fp8
}  // namespace ch
