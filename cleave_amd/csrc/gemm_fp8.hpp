// gemm_fp8.hpp -- products of 8-bit matrices (fp8.hpp) on the scaled matrix
// instructions of gfx950, v_mfma_scale_f32_32x32x64_f8f6f4.
//
// C[M x N] = A B^T (A: M x K, B: N x K, both with K along their rows) or A B
// (B: K x N, quantised by 128 x 128 blocks).  With a = qa 2^ea and b = qb 2^eb,
// every k-block of 128 has one ea per row of A and one eb per column of C:
//   C[m][n] = sum over blocks of 2^(ea + eb) sum over k of qa qb,
// and the instruction takes ea and eb as a byte per lane, so the sum runs on
// in its f32 accumulator with no other arithmetic.
//
// What the instruction rounds (found by products made for it): of each 8
// consecutive k it aligns the products to the largest and cuts them off, towards
// zero, at 2^-13 of that one's 2^(exponent of a + exponent of b), a subnormal code's
// exponent being -6; it adds the 8's sum to the f32 accumulator, rounding down.  On
// normal data that is 1e-5 of the result, 3e-5 with columns 12 times the rest:
// little beside the rounding of a bf16 result (2e-3; 2% of 8192^3's results take
// the neighbouring value), too much for an f32 one.  So only bf16 results come
// this way.  For f32 ones (WIDE) each code is widened to bf16, exactly and with its
// scale, and v_mfma_f32_32x32x16_bf16 sums in f32 (1e-7 on the same data) at half
// the rate.
//
// v_mfma_scale_f32_32x32x64 operands: lane l holds 32 bytes of row (column)
// l % 32 at k = 32 (l / 32) .. +31, and its scale byte covers those 32; the
// accumulator holds column l % 32, rows 8 (v/4) + 4 (l/32) + v%4.
//
// LDS tiles (16-byte chunks, copied by global_load_lds_dwordx4 as in
// gemm_tiles.hpp, whose per-lane source picks the slot):
//   KC (K along the rows): [R rows][64 bytes], chunk c of row r in slot
//     kc64_slot(r, c): 16 lanes read a chunk of 16 rows, which then fall into 16
//     different slots of the 256 bytes of banks.
//   MN (K across the rows): [64 k-rows][R bytes], read by ds_read_b64_tr_b8:
//     lane 2j + h of a 16-lane group points at k-row kb + j, bytes 8h .. 8h+7
//     of 16 columns; lane i receives column i of k-rows kb .. kb+7.  A half wave
//     reads 8 k-rows x 32 bytes, which XOR-ing 32-byte pairs of chunks with the
//     k-row spreads over the banks.
//
// Ragged shapes: codes are padded with zeros to whole blocks along a row, so
// KC rows are whole; a row past M (N) reads the last one, whose results are
// not stored; a k-row past K reads the last one, which meets A's zero codes.
#pragma once

#include "extents.hpp"
#include "fp8.hpp"
#include "gemm_common.hpp"
#include "gemm_tiles.hpp"

namespace ch {
namespace fp8 {

using tiles::dma16;
using tiles::lds_addr;
using tiles::lds_void;

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i lds_v4i;
typedef __attribute__((address_space(3))) v2i lds_v2i;

// dma16 from any address a lane names.
__device__ __forceinline__ void dma16_far(const void* src, uint32_t lds_dst) {
    asm volatile("global_load_lds_dwordx4 %0, off" : : "v"(src), "{m0}"(lds_dst) : "memory");
}

// Slot of chunk c of k-row r of an MN tile R bytes wide.
template <int R>
__device__ __forceinline__ int mn_slot(int r, int c) {
    static_assert(R == 64 || R == 128 || R == 256, "64, 128 or 256 columns");
    if constexpr (R == 64) return c ^ (((r >> 2) & 1) << 1);  // four k-rows share 256 bytes
    else if constexpr (R == 128) return c ^ (((r >> 1) & 3) << 1);  // two k-rows share 256 bytes
    else return c ^ ((r & 7) << 1);
}

__device__ __forceinline__ v16f mfma(v8i a, v8i b, v16f c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// Codes 8 t .. 8 t + 7 of a lane's 32 as bf16 values, times 2^(s - 127) (exact,
// short of bf16's range): an operand of v_mfma_f32_32x32x16_bf16.  Lane l holds
// k = 32 (l / 32) + 8 t .. +7 of A and of B alike, so the four steps sum the
// same 64 k as the 8-bit instruction.
__device__ __forceinline__ tiles::v8bf widen(v8i q, int t, int s) {
    const float scale = scale_value(s);
    bf16x2 p[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        p[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)q[2 * t + h], scale, false);
        p[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)q[2 * t + h], scale, true);
    }
    tiles::v8bf v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// v as an element of C, f32 or bf16.
__device__ __forceinline__ void store_c(float* C, int64_t at, float v) { C[at] = v; }
__device__ __forceinline__ void store_c(uint16_t* C, int64_t at, float v) {
    C[at] = (uint16_t)(pack_bf16(v, v) & 0xFFFFu);
}

struct Operands {
    const uint8_t* a;
    const uint8_t* as;
    const uint8_t* b;
    const uint8_t* bs;
    int M, N, K;
    int64_t pa, pb;    // code pitches
    int64_t spa, spb;  // scale pitches
};

}  // namespace fp8
}  // namespace ch
