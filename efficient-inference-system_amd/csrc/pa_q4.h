// The 4-bit KV page: its layout, and the kernels' helpers to read it (gfx950, wave64).
//
// A page holds 16 tokens of one KV head, K and V in pools of their own, uint8
// [num_blocks, kv_heads, page_bytes]. 64 consecutive values of a row (a group; one at head_dim 64, two
// at 128) share a half-precision scale s and centre z; code c in 0..15 stands for z + s (c - 7.5).
// The page is its codes, 16 * head_dim / 2 bytes, then the pairs (s low, z high) as 32-bit words
// [group][token].
//
// Codes lie where the lanes of v_mfma_f32_16x16x32_f16 take them, so that a wavefront reads a page's
// codes with one load of 4 * HD / 32 consecutive bytes a lane, and makes fp16 operands of them with
// one AND (and one shift) per two values:
//   K  operand A of S^T = K Q^T, lane (g, r) = (lane / 16, lane % 16), row = token r, contraction slot
//      (g, j) of MFMA w = value d = 32 w + 8 g + j. Word (t, g, w) holds j = 0..7, even j in nibble
//      j / 2, odd j in nibble 4 + j / 2: x & 0x000f000f is the pair j = 0, 1, x & 0x00f000f0 the pair
//      2, 3 times 16, and x >> 8 gives the pairs 4, 5 and 6, 7.
//   V  operand A of O^T = V^T P^T, row r of output tile (a, n) = value d = 64 a + 4 r + n, contraction
//      slot (g, j) = token 4 g + j of the first of two pages (j < 4) or 4 g + j - 4 of the second: the
//      slots where the lanes hold the scores of S^T. Word (g, r, p, a) holds tokens 4 g + 2 p (low
//      half) and 4 g + 2 p + 1 (high half), nibble n of each half the value of tile n; the masks above
//      give the pairs of tiles 0, 1 (times 16), 2 and 3 (times 16).
// A token's bytes are its own in both, so rows are written without regard to their neighbours.
//
// The masked words are fp16 subnormals: code c reads as c 2^-24 (16 c 2^-24 for the odd masks), which
// the matrix cores multiply exactly. The factors are taken out of the other operand or of the sums.
#pragma once

#include "pa_common.h"
#include "paged_hip_q4.h"

namespace pa {

constexpr int kQ4Tokens = 16;  // tokens of a page (the block size)
constexpr int kQ4Group = 64;   // values that share (s, z)

constexpr int q4_codes_bytes(int hd) { return kQ4Tokens * hd / 2; }
constexpr int q4_page_bytes(int hd) { return kQ4Tokens * (hd / 2 + 4 * (hd / kQ4Group)); }

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float q4_scale(uint32_t m) { return (float)__builtin_bit_cast(f16x2, m)[0]; }
__device__ __forceinline__ float q4_centre(uint32_t m) { return (float)__builtin_bit_cast(f16x2, m)[1]; }

// Four words of fp16 pairs as one operand.
__device__ __forceinline__ f16x8 q4_operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(f16x8, u32x4{a, b, c, d});
}
constexpr uint32_t kQ4Even = 0x000f000fu, kQ4Odd = 0x00f000f0u;

// A key's page-table entry as a block of the pool, -1 where it is none.
__device__ __forceinline__ int q4_block(int id, int64_t num_blocks) {
  return id >= 0 && (int64_t)id < num_blocks ? id : -1;
}

}  // namespace pa
