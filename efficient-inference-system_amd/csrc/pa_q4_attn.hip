// Paged attention over 4-bit KV pages on gfx950: decode steps and causal prefill chunks, with grouped
// query heads and, on request, the attention weights added to each slot's running total.
//
// A request's query rows over one KV head are numbered m = i * group + j (query position i, head j of
// the `group` heads that share the KV head) and are columns of 16-column tiles. Per step of 32 keys
// (two pages), wavefront and tile, with v_mfma_f32_16x16x32_f16 (fp32 accumulation):
//   S^T = K Q^T   per page and group of 64 values: A = the codes (exact), B = the q rows, held as fp16 in
//                 registers for the whole walk. s and z enter outside: S = sum_groups s (acc - 7.5 qs) +
//                 z qs, qs = the sum of the group's q as rounded, -7.5 qs the accumulator's start (0 where
//                 the codes are centred, below).
//   softmax       lane (g, c) holds column c's scores of keys 4 g + i of both pages.
//   O^T += V^T P^T  A = the codes, B = w = p s of the value's group, in the lanes that hold p. The rest of
//                 the value, sum_keys p z - 7.5 w, is one fp32 sum per column and group.
// The codes never leave the matrix cores' operands and no cross-lane move feeds them (see pa_q4.h).
//
// Precision. bf16 q is exact in fp16 once scaled by a power of two per row (below 2^-23 of the row's
// largest element bits are lost); w is rounded to fp16 (2^-11), the 7.5 w beside it is the rounded
// one, so the error is that of a code within +-7.5. For fp32 q (PARTS = 2) q and w are each the sum
// of two fp16 values, 2^-23 or better: the columns of a tile are 8 rows twice, column c the high parts
// of row c, column c + 8 the low ones, both parts' products summed with one DPP rotation. The second
// product costs no matrix instruction up to 8 rows per tile.
//
// Range. Weights are kept as p = 2^(S - M), M per column, with M chosen so that p * max(s) is near 2^4 when M
// is set, and set again (accumulators rescaled) when a key's p * max(s, 2^-14) passes 2^15: p s stays
// inside fp16, above its subnormals for keys within 2^-18 of the heaviest. M cancels in O / l.
//
// Kernels:
//   q4_narrow_kernel  a tile of rows: the workgroup's wavefronts split the keys and merge in LDS (decode,
//                     chunks of up to two tiles).
//   q4_wide_kernel    each wavefront has a tile of its own, and the workgroup's walk all keys together,
//                     staged through LDS.
//   Either splits the keys over several workgroups when the grid is small, as records (M, l, O) that
//   q4_finish_kernel merges; it also adds the weights of decode steps up. q4_chunk_weights_kernel does so for
//   chunks: it forms the scores again.
#include <type_traits>
#include <utility>

#include "pa_attention.h"
#include "pa_q4.h"

namespace pa {

struct Q4Args {
  const void* q;
  int64_t q_sb, q_sh, q_st;
  void* out;
  int64_t o_sb, o_sh, o_st;
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  float* weights;  // null: no totals
  int64_t num_blocks;
  const int32_t* page_table;
  int64_t pt_stride;
  int32_t max_pages;
  const int32_t* seq_lens;
  const int32_t* cur_lens;
  int32_t B, H, Hk, group, T;
  float scale_log2;
  int32_t tiles;        // row tiles (workgroups' worth of rows) per (request, KV head)
  int32_t splits;       // key ranges per tile, >= 1
  int32_t split_pages;  // pages per key range, even
  float* rec;           // splits > 1: (M, l, O[HD]) per (split, row)
  f32x2* lse;           // totals: each row's (M, log2 of its denominator beside 2^M)
  float* scores;        // decode totals: log2-domain scores [B, H, score_stride]
  int64_t score_stride;
  f16x8* q_ops;         // chunk totals: the row tiles' operands [tile][HD / 32][64 lanes], and per lane
  f32x4* q_aux;         // (qs of the groups, sc, keys seen)
  int32_t op_tiles;     // tiles of 16 / PARTS rows per (request, KV head) there
};

constexpr float kQ4Start = 4.f;         // log2 of p * max(s) when M is set
constexpr float kQ4Limit = 32768.f;     // p * max(s, 2^-14) beyond which M is set again
constexpr short kQ4LimitBits = 0x7800;    // kQ4Limit as a half
constexpr float kQ4Floor = 6.103515625e-5f;  // 2^-14
// M of a row that has met no key: of all finite floats the lowest, since any finite score may be the first.
constexpr float kQ4None = -3.402823466e+38f;
// Scores (log2) from here on are steep: whole numbers, 1 apart and more. The wide kernel's p is 2^(sc S - M) with
// the product exact, so M, a float, would miss the largest by half of its step, and p leave fp16 from 2^28
// on. A column whose M is steep takes the next power of two for sc: its products are floats, M is one of them, and
// keys that are not the largest keep a weight of 0 as before. (The order of M between columns' parts stays:
// steep ones move away from zero, others stay below kQ4Steep.)
constexpr float kQ4Steep = 16777216.f;
__device__ __forceinline__ bool q4_steep(float M) { return fabsf(M) >= kQ4Steep && M > kQ4None; }
__device__ __forceinline__ float q4_steep_unit(float sc) { return ldexpf(1.f, __builtin_amdgcn_frexp_expf(sc)); }
// A zero that the compiler does not know: half * float + zero is one v_fma_mix_f32, which reads the half in
// place, where a product alone is a conversion and a multiplication.
__device__ __forceinline__ float q4_zero() {
  float z = 0.f;
  asm("" : "+v"(z));
  return z;
}
// Two products of a weight and a pair's scale as fp16: v_fma_mixlo_f16 and v_fma_mixhi_f16. (The empty asm
// keep the two apart, or they become a vector of conversions and multiplications, five instructions, and
// the word whole, or its high half is formed again where it is used next.)
__device__ __forceinline__ f16x2 q4_weights(float p0, uint32_t m0, float p1, uint32_t m1) {
  _Float16 lo = (_Float16)(p0 * q4_scale(m0));
  asm("" : "+v"(lo));
  uint32_t both = __builtin_bit_cast(uint32_t, f16x2{lo, (_Float16)(p1 * q4_scale(m1))});
  asm("" : "+v"(both));
  return __builtin_bit_cast(f16x2, both);
}

// Codes as the matrix cores take them. As fp16 subnormals (c 2^-24) they cost one AND, but the cores align
// a product by its operands' exponents without normalising them, so that a sum keeps 7 to 10 bits fewer
// than fp32, and sums of uncentred codes cancel against 7.5 times their weights: 2^-17 of the largest term,
// enough beside a bf16 result. For fp32 q (PARTS = 2) one v_pk_fma_f16 per pair makes them (c - 7.5) 2^-9,
// normal and centred: 5e-7 for 1024 keys' output where the subnormals left 5e-5.
template <int PARTS> constexpr float kQ4Unit = PARTS == 2 ? 512.f : 16777216.f;  // 1 / the value of code 1
template <int PARTS> constexpr int kQ4UnitLog2 = PARTS == 2 ? 9 : 24;
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef __fp16 h16x2 __attribute__((ext_vector_type(2)));  // v_dot2_f32_f16's operand
template <int PARTS, bool ODD>
__device__ __forceinline__ uint32_t q4_pair(uint32_t word) {
  const uint32_t masked = word & (ODD ? kQ4Odd : kQ4Even);
  if constexpr (PARTS == 1) return masked;
  constexpr _Float16 up = (_Float16)32768.f, mid = (_Float16)((ODD ? -16.f : -1.f) * 7.5f / 512.f);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, masked), f16x2{up, up}, f16x2{mid, mid}));
}

// A wavefront's column tile: operands, sums and running state.
template <int HD, int PARTS>
struct Q4Wave {
  static constexpr int G = HD / kQ4Group, W = HD / 32;
  f16x8 q[W];
  float qs[G];  // sum of the group's q operands (units of code 1)
  float sc;     // log2-domain score of such a unit
  float unit;   // what stands for it: sc, or while M is steep the power of two above
  int n;        // keys the column sees (a column without a row: 0x7fffffff)
  f32x4 o[G][4];
  float y[G], M, l;
  f32x4 yw[G];  // PARTS = 1: -7.5 times the sum of w, every row of the product alike
};

template <typename IO>
__device__ __forceinline__ void q4_load_q(const IO* p, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8 * (int)sizeof(IO) / 16; ++i) {
    float f[Vec16<IO>::EPL];
    u32x4 w;
    __builtin_memcpy(&w, reinterpret_cast<const char*>(p) + 16 * i, 16);
    Vec16<IO>::unpack(w, f);
#pragma unroll
    for (int j = 0; j < Vec16<IO>::EPL; ++j) x[i * Vec16<IO>::EPL + j] = f[j];
  }
}

// The row of column c of a tile, and whether the column holds its low parts.
template <int PARTS>
__device__ __forceinline__ int q4_row(int tile, int c) { return PARTS == 2 ? tile * 8 + (c & 7) : tile * 16 + c; }

// q's row at `src` as operands of lane group g: scaled by a power of two so that its largest element is in
// [2^13, 2^14), the factor taken out of sc; odd-mask slots hold a sixteenth. low: the second fp16 part.
template <typename IO, int HD, int PARTS>
__device__ __forceinline__ void q4_row_operands(const IO* src, bool there, bool low, int g, float scale_log2, f16x8 (&q)[HD / 32],
                                                float (&qs)[HD / kQ4Group], float& sc) {
  constexpr int G = HD / kQ4Group, W = HD / 32;
  float x[W][8];
  float top = 0.f;
#pragma unroll
  for (int s = 0; s < W; ++s) {
    if (there) {
      q4_load_q<IO>(src + 32 * s + 8 * g, x[s]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[s][e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[s][e]));
  }
  top = max_xor32(max_xor16(top));
  // rows of zeros and of infinities stay as they are
  int up = top > 0.f && top < INFINITY ? 14 - (__builtin_amdgcn_frexp_expf(top)) : 0;
  up = up > 120 ? 120 : up;
  up = up < -120 ? -120 : up;
  float sum[G];
#pragma unroll
  for (int k = 0; k < G; ++k) sum[k] = 0.f;
#pragma unroll
  for (int s = 0; s < W; ++s) {
    f16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = ldexpf(x[s][e], up - ((e & 2) ? 4 : 0));
      _Float16 h = (_Float16)f;
      if (PARTS == 2 && low) h = (_Float16)(f - (float)h);
      v[e] = h;
      sum[s / 2] += (e & 2) ? 16.f * (float)h : (float)h;
    }
    q[s] = v;
  }
#pragma unroll
  for (int k = 0; k < G; ++k) qs[k] = sum_xor32(sum_xor16(sum[k])) * (1.f / kQ4Unit<PARTS>);
  sc = fmaxf(fminf(ldexpf(scale_log2, kQ4UnitLog2<PARTS> - up), 1e38f), 1e-37f);  // (0 times a score of -inf is NaN)
}

// Column tile `tile` of (request b, KV head hk).
template <typename IO, int HD, int PARTS>
__device__ __forceinline__ void q4_setup(const Q4Args& a, int b, int hk, int tile, int L, int C, int keys, int lane,
                                         Q4Wave<HD, PARTS>& w) {
  constexpr int G = HD / kQ4Group;
  const int g = lane >> 4, c = lane & 15;
  const int row = q4_row<PARTS>(tile, c);
  const bool there = row < a.T * a.group;
  const int i = row / a.group, j = row - i * a.group;
  const IO* src = static_cast<const IO*>(a.q) + (int64_t)b * a.q_sb + (int64_t)(hk * a.group + j) * a.q_sh + (int64_t)i * a.q_st;
  q4_row_operands<IO, HD, PARTS>(src, there, c >= 16 / PARTS, g, a.scale_log2, w.q, w.qs, w.sc);
  int n = valid_keys(L, C, i);
  n = n < keys ? n : keys;
  w.n = there ? n : 0x7fffffff;
  w.unit = w.sc;
  w.M = kQ4None;
  w.l = 0.f;
#pragma unroll
  for (int k = 0; k < G; ++k) {
    w.y[k] = 0.f;
    w.yw[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 4; ++t) w.o[k][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// Scores (units of code 1) of one page against q's operands: lane (g, c) gets keys 4 g + i of its column.
template <int HD, int PARTS>
__device__ __forceinline__ f32x4 q4_scores(const f16x8 (&kf)[HD / 32], const u32x4 (&km)[HD / kQ4Group], const f16x8 (&q)[HD / 32],
                                           const float (&qs)[HD / kQ4Group]) {
  constexpr int G = HD / kQ4Group;
  const float zero = q4_zero();
  f32x4 S = {zero, zero, zero, zero};
#pragma unroll
  for (int k = 0; k < G; ++k) {
    const float q0 = qs[k], start = PARTS == 2 ? 0.f : -7.5f * q0;  // (PARTS = 2: the codes are centred)
    f32x4 acc = {start, start, start, start};
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[2 * k], q[2 * k], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[2 * k + 1], q[2 * k + 1], acc, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      S[i] = fmaf(q4_scale(km[k][i]), acc[i], fmaf(q4_centre(km[k][i]), q0, S[i]));
  }
  if constexpr (PARTS == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) S[i] += dpp<0x128>(S[i]);
  }
  return S;
}

template <int HD, int PARTS>
__device__ __forceinline__ void q4_k_operands(const uint32_t (&k)[HD / 32], f16x8 (&kf)[HD / 32]) {
#pragma unroll
  for (int s = 0; s < HD / 32; ++s) {
    const uint32_t x = k[s], y = x >> 8;
    kf[s] = q4_operand(q4_pair<PARTS, false>(x), q4_pair<PARTS, true>(x), q4_pair<PARTS, false>(y),
                       q4_pair<PARTS, true>(y));
  }
}

// A page in LDS: K codes, V codes, K pairs, V pairs, as the wide kernel stages them.
template <int HD>
struct Q4Staged {
  static constexpr int G = HD / kQ4Group, W = HD / 32, CODES = q4_codes_bytes(HD), META = kQ4Tokens * 4 * G;
  static constexpr int BYTES = 2 * (CODES + META);
  // head_dim 128: K's 16-byte words come in lane order, so that lane L reads bytes 16 L .. (no bank twice)
  __device__ static __forceinline__ void k_words(const uint8_t* p, int lane, uint32_t (&x)[W]) {
    const int g = lane >> 4, c = lane & 15;
    q4_lds_words(p + (HD == 128 ? lane * 16 : (c * 4 + g) * 8), x);
  }
  __device__ static __forceinline__ void v_words(const uint8_t* p, int lane, uint32_t (&x)[2 * G]) {
    q4_lds_words(p + CODES + lane * 8 * G, x);
  }
  __device__ static __forceinline__ u32x4 k_pairs(const uint8_t* p, int g, int k) {
    return *reinterpret_cast<const u32x4*>(p + 2 * CODES + (k * kQ4Tokens + 4 * g) * 4);
  }
  __device__ static __forceinline__ u32x4 v_pairs(const uint8_t* p, int g, int k) {
    return *reinterpret_cast<const u32x4*>(p + 2 * CODES + META + (k * kQ4Tokens + 4 * g) * 4);
  }
  template <int N>
  __device__ static __forceinline__ void q4_lds_words(const uint8_t* p, uint32_t (&x)[N]) {
    if constexpr (N == 4) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = v[i];
    } else {
      const u32x2 v = *reinterpret_cast<const u32x2*>(p);
      x[0] = v[0];
      x[1] = v[1];
    }
  }
};

// One step: the two pages at pg (in LDS), 32 keys from key `key0` on. masked: the column may not see all of
// them, or a page is missing (live: bit h set where page h is there). What a column does not see takes part
// with score -inf and the pair (0, 0), so that nothing in its place reaches the sums.
template <int HD, int PARTS>
__device__ __forceinline__ void q4_step(const uint8_t* pg, Q4Wave<HD, PARTS>& w, int key0, bool masked, int live, int lane) {
  using P = Q4Staged<HD>;
  constexpr int G = P::G, W = P::W;
  const int g = lane >> 4;
  const bool low = PARTS == 2 && (lane & 15) >= 8;
  f32x4 S[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t kw[W];
    P::k_words(pg + h * P::BYTES, lane, kw);
    f16x8 kf[W];
    q4_k_operands<HD, PARTS>(kw, kf);
    u32x4 km[G];
#pragma unroll
    for (int k = 0; k < G; ++k) km[k] = P::k_pairs(pg + h * P::BYTES, g, k);
    S[h] = q4_scores<HD, PARTS>(kf, km, w.q, w.qs);
  }
  u32x4 vm[2][G];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int k = 0; k < G; ++k) vm[h][k] = P::v_pairs(pg + h * P::BYTES, g, k);
  if (masked) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool see = (live >> h & 1) && key0 + 16 * h + 4 * g + i < w.n;
        S[h][i] = see ? S[h][i] : -INFINITY;
#pragma unroll
        for (int k = 0; k < G; ++k) vm[h][k][i] = see ? vm[h][k][i] : 0u;
      }
  }
  float p[2][4];
  uint32_t pw[G][4];
  // weights and, per group, w = p s as fp16 (PARTS = 2: this column's part of it); again with another M where
  // one is too large (never more than once)
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    float big = 0.f;
    s16x2 top = {0, 0};  // (halves from 0 on are ordered as integers)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[h][i] = fast_exp2(fmaf(S[h][i], w.unit, -w.M));
        big = fmaxf(big, p[h][i]);
      }
#pragma unroll
    for (int k = 0; k < G; ++k) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const int h = e >> 2, i = e & 3;
        f16x2 hi, part;
        if constexpr (PARTS == 1) {
          hi = part = q4_weights(p[h][i], vm[h][k][i], p[h][i + 1], vm[h][k][i + 1]);
        } else {
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            const float x = p[h][i + f] * q4_scale(vm[h][k][i + f]);
            hi[f] = (_Float16)x;
            const _Float16 rest = (_Float16)(x - (float)hi[f]);
            part[f] = low ? rest : hi[f];
          }
        }
        top = __builtin_elementwise_max(top, __builtin_bit_cast(s16x2, hi));
        pw[k][e / 2] = __builtin_bit_cast(uint32_t, part);
      }
    }
    const bool far = top[0] > kQ4LimitBits || top[1] > kQ4LimitBits || big > kQ4Limit / kQ4Floor;
    if (__builtin_expect(!__any(far), 1)) break;
    float sc = w.sc;
    asm volatile("" : "+v"(sc));  // (or what follows is taken before the loop, in every step)
    const float steep_unit = q4_steep_unit(sc);
    float m = kQ4None;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float s = kQ4Floor;
        asm volatile("" : "+v"(s));  // (the same)
#pragma unroll
        for (int k = 0; k < G; ++k) s = fmaxf(s, q4_scale(vm[h][k][i]));
        const float t = S[h][i] * sc, low = fmaf(S[h][i], sc, __builtin_amdgcn_logf(s)) - kQ4Start;
        m = fmaxf(m, fabsf(t) >= kQ4Steep ? S[h][i] * steep_unit : __builtin_amdgcn_fmed3f(low, 1.f - kQ4Steep, kQ4Steep - 1.f));
      }
    m = max_xor32(max_xor16(m));
    const float M = fmaxf(w.M, m), f = fast_exp2(w.M - M);
    w.M = M;
    w.unit = q4_steep(M) ? steep_unit : w.sc;
    w.l *= f;
#pragma unroll
    for (int k = 0; k < G; ++k) {
      w.y[k] *= f;
      if constexpr (PARTS == 1) w.yw[k] *= f;
#pragma unroll
      for (int t = 0; t < 4; ++t) w.o[k][t] *= f;
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) w.l += p[h][i];
#pragma unroll
  for (int k = 0; k < G; ++k) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w.y[k] = fmaf(p[e >> 2][e & 3], q4_centre(vm[e >> 2][k][e & 3]), w.y[k]);
    if constexpr (PARTS == 1) {  // -7.5 w, as rounded: on the matrix cores, which have the time that v_dot2_f32_f16 takes (1%)
      constexpr _Float16 m = (_Float16)-7.5f;
      w.yw[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f16x8{m, m, m, m, m, m, m, m},
                                                       q4_operand(pw[k][0], pw[k][1], pw[k][2], pw[k][3]), w.yw[k], 0, 0, 0);
    }
  }
  uint32_t vw[2][2 * G];
#pragma unroll
  for (int h = 0; h < 2; ++h) P::v_words(pg + h * P::BYTES, lane, vw[h]);
#pragma unroll
  for (int k = 0; k < G; ++k) {
    const f16x8 b = q4_operand(pw[k][0], pw[k][1], pw[k][2], pw[k][3]);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      uint32_t x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // page e / 2, token pair e % 2
        const uint32_t x0 = vw[e >> 1][(e & 1) * G + k], x1 = t & 2 ? x0 >> 8 : x0;
        x[e] = t & 1 ? q4_pair<PARTS, true>(x1) : q4_pair<PARTS, false>(x1);
      }
      w.o[k][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(q4_operand(x[0], x[1], x[2], x[3]), b, w.o[k][t], 0, 0, 0);
    }
  }
}

// A tile's walk is done: the lanes' sums joined. Leaves in lane (g, c) the 16 values d = 64 k + 16 g ..
// + 15 of column c's unnormalised row per group, and l.
template <int HD, int PARTS>
__device__ __forceinline__ void q4_join(Q4Wave<HD, PARTS>& w, float (&o)[HD / kQ4Group][16], float& l) {
  constexpr int G = HD / kQ4Group;
  l = sum_xor32(sum_xor16(w.l));
#pragma unroll
  for (int k = 0; k < G; ++k) {
    float y = sum_xor32(sum_xor16(w.y[k]));
    if constexpr (PARTS == 1) y += w.yw[k][0];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v = w.o[k][t][i];
        if constexpr (PARTS == 2) v += dpp<0x128>(v);
        o[k][4 * i + t] = fmaf(v, (t & 1) ? kQ4Unit<PARTS> / 16.f : kQ4Unit<PARTS>, y);
      }
  }
}

template <typename IO>
__device__ __forceinline__ void q4_store16(IO* p, const float (&o)[16], float f) {
  if constexpr (sizeof(IO) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 v = {o[4 * i] * f, o[4 * i + 1] * f, o[4 * i + 2] * f, o[4 * i + 3] * f};
      __builtin_memcpy(p + 4 * i, &v, 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = pack_bf16x2(o[8 * i + 2 * j] * f, o[8 * i + 2 * j + 1] * f);
      __builtin_memcpy(p + 8 * i, &v, 16);
    }
  }
}

// Record of a row's part: M, l, O[HD].
template <int HD>
__device__ __forceinline__ float* q4_record(const Q4Args& a, int b, int hk, int row, int split) {
  const int64_t rows = (int64_t)a.T * a.group;
  return a.rec + ((((int64_t)b * a.Hk + hk) * rows + row) * a.splits + split) * (HD + 2);
}
__device__ __forceinline__ f32x2* q4_lse(const Q4Args& a, int b, int hk, int row) {
  return a.lse + ((int64_t)b * a.Hk + hk) * a.T * a.group + row;
}

// log2 of a row's denominator as (M, log2 l): a key's weight is 2^(S - M - log2 l), where S - M comes first, since
// the sum of the two would round to M's last digit (a weight off by 1% at scores of 10^5). log2 l is infinite
// (weights of 0) where the row sees no key, NaN where it met one.
__device__ __forceinline__ f32x2 q4_log_sum(float M, float l) {
  return l > 0.f || l != l ? f32x2{M, __builtin_amdgcn_logf(l)} : f32x2{0.f, INFINITY};
}

// Workgroup -> (request, KV head, tile, split): KV heads innermost, so that workgroups of one moment
// read neighbouring slabs of the same blocks; later (longer) tiles first.
struct Q4Unit { int b, hk, tile, split; };
__device__ __forceinline__ Q4Unit q4_unit(const Q4Args& a) {
  int x = blockIdx.x;
  Q4Unit u;
  u.hk = x % a.Hk;
  x /= a.Hk;
  u.split = x % a.splits;
  x /= a.splits;
  u.b = x % a.B;
  u.tile = a.tiles - 1 - x / a.B;
  return u;
}

constexpr int kQ4Waves = 4;
constexpr int kQ4MaxNarrow = 32;  // rows that the narrow kernel takes (two tiles of 16)

// Each wavefront has a column tile of its own, and the workgroup walks the keys together: stages of 64 keys
// go from the pools straight into LDS (global_load_lds, one page per wavefront), two stages ahead in a ring
// of three, with one barrier a stage. Read from memory by each wavefront for itself, the pages' pairs alone
// (16 bytes that 16 lanes share) cost more load instructions than the codes.
//
// Bound by vector instructions: a step of 32 keys takes some 200 (the codes' ANDs and shifts 80, the pairs' scales
// and centres 64, exponentials and sums the rest) to 18 matrix instructions, 82% of the cycles that a CU has
// work (4 x 512 rows of 32 heads x 128 bf16 over 1024 to 4096 keys: 215 to 235 us from one process to another, 420 to 460
// TFLOP/s; 200 rows of 32 over 8 heads over 16k keys: 138 us, 390). Two tiles a wavefront, which share the codes' part, take 256 registers: 240 us.
//
// HALVES = 2, for grids that leave the GPU room: eight wavefronts for the same four tiles, stages of 128 keys,
// each half of the wavefronts taking its half of every stage, joined in LDS at the end. A step is a chain of
// LDS reads, matrix instructions and exponentials that one wavefront a SIMD does not fill (4 x 256 rows of 8
// heads x 64 over up to 1024 keys, fp32: 26 -> 21.5 us; the same keys split over workgroups instead cost a
// merging launch, 31 us).
constexpr int kQ4WideWaves = 4;  // column tiles of a workgroup
constexpr int kQ4Ring = 3;

// The request whose place in the order of falling cached lengths is `place` (equal lengths in the batch's
// order), for batches of up to 64: the longest requests' tiles start first, so that the grid's end is filled
// with short ones.
__device__ __forceinline__ int q4_by_length(const int32_t* lens, int B, int place, int lane) {
  if (B > 64) return place;
  const int mine = lane < B ? lens[lane] : -0x7fffffff;
  int before = 0;
  for (int j = 0; j < B; ++j) {
    const int other = __builtin_amdgcn_readlane(mine, j);
    before += other > mine || (other == mine && j < lane);
  }
  return __builtin_ctzll(__ballot(lane < B && before == place));
}

template <typename IO, int HD, int PARTS, int HALVES>
__global__ __launch_bounds__(64 * kQ4WideWaves * HALVES, HALVES == 2 ? 2 : 3) void q4_wide_kernel(const Q4Args a) {
  using P = Q4Staged<HD>;
  constexpr int G = HD / kQ4Group, PB = q4_page_bytes(HD);
  constexpr int ROWS = 16 / PARTS;  // rows of a column tile
  constexpr int SP = kQ4WideWaves * HALVES;  // pages of a stage
  constexpr uint32_t SPMASK = (1u << SP) - 1;
  constexpr int STAGE = SP * P::BYTES;
  constexpr int JOIN = HALVES == 2 ? kQ4WideWaves * 64 * (16 * G + 2) * 4 : 0;  // the second half's sums
  constexpr int LOADS = HD == 128 ? 3 : 2;  // load instructions of a page
  __shared__ __attribute__((aligned(16))) uint8_t ring[kQ4Ring * STAGE > JOIN ? kQ4Ring * STAGE : JOIN];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int half = HALVES == 2 ? wave / kQ4WideWaves : 0, tile_wave = HALVES == 2 ? wave % kQ4WideWaves : wave;
  const int g = lane >> 4, c = lane & 15;
  Q4Unit u = q4_unit(a);
  u.b = __builtin_amdgcn_readfirstlane(q4_by_length(a.seq_lens, a.B, u.b, lane));
  const int L = a.seq_lens[u.b], C = a.cur_lens[u.b];
  const int rows = a.T * a.group;
  int keys = L < a.max_pages * kQ4Tokens ? L : a.max_pages * kQ4Tokens;
  keys = keys > 0 ? keys : 0;
  auto seen = [&](int row) {  // keys that the row sees
    const int n = valid_keys(L, C, row / a.group);
    return n < keys ? n : keys;
  };
  // what the workgroup's rows see together, and its share of the pages
  const int wg_first = u.tile * kQ4WideWaves * ROWS;
  const int wg_end = wg_first + kQ4WideWaves * ROWS < rows ? wg_first + kQ4WideWaves * ROWS : rows;
  const int pages = (seen(wg_end - 1) + kQ4Tokens - 1) / kQ4Tokens;
  const int p0 = u.split * a.split_pages;
  int p1 = a.splits > 1 ? p0 + a.split_pages : pages;
  p1 = p1 < pages ? p1 : pages;
  if (a.splits > 1 && p0 >= p1) return;  // no record: the merge knows how far each row's pages reach
  // what the wavefront's rows see: all of them, some of them
  const int first = wg_first + tile_wave * ROWS;
  const int end = first + ROWS < rows ? first + ROWS : rows;
  const int all = first < rows ? seen(first) : 0, most = first < rows ? seen(end - 1) : 0;
  Q4Wave<HD, PARTS> w;
  const int tile = first / ROWS;
  q4_setup<IO, HD, PARTS>(a, u.b, u.hk, tile, L, C, keys, lane, w);
  if (a.q_ops != nullptr && u.split == 0 && half == 0) {  // for q4_chunk_weights_kernel
    const int64_t at = ((int64_t)u.b * a.Hk + u.hk) * a.op_tiles + tile;
    // (padding may hold NaN and infinities: as zeros there, and it sees no key, whose values may be NaN too)
    const bool pad = (int64_t)q4_row<PARTS>(tile, c) >= (int64_t)(C < a.T ? C : a.T) * a.group;
#pragma unroll
    for (int s = 0; s < HD / 32; ++s) a.q_ops[(at * (HD / 32) + s) * 64 + lane] = pad ? f16x8{} : w.q[s];
    a.q_aux[at * 64 + lane] = f32x4{pad ? 0.f : w.qs[0], pad ? 0.f : w.qs[G - 1], w.sc, __int_as_float(pad ? 0 : w.n)};
  }

  if (p0 < p1) {
    const int32_t* table = a.page_table + (int64_t)u.b * a.pt_stride;
    const int64_t step = (int64_t)a.Hk * PB;
    const uint8_t* kb = a.k_pool + (int64_t)u.hk * PB;
    const uint8_t* vb = a.v_pool + (int64_t)u.hk * PB;
    int ids = -1, base = p0 - 64;  // blocks of pages base .. base + 63 (-1: none), and which there are
    uint64_t there = 0;
    // per-lane source of what a page's last load fetches: the pairs and, at head_dim 64, the codes of both
    const uint8_t* meta_src = (lane & (4 * G) ? vb : kb) + q4_codes_bytes(HD) + (lane & (4 * G - 1)) * 16;
    const uint8_t* code_src = (lane < 32 ? kb : vb) + (lane & 31) * 16;
    const uint32_t k_off = (uint32_t)(c * 4 + g) * 16, v_off = (uint32_t)lane * 16;
    const int stages = (p1 - p0 + SP - 1) / SP;
    uint32_t live = 0;  // pages of the ring's stages that are there, SP bits a slot
    auto issue = [&](int st, int slot) {
      const int pg = p0 + st * SP;
      if (pg - base >= 64) {
        base = pg;
        ids = pg + lane < p1 ? q4_block(table[pg + lane], a.num_blocks) : -1;
        there = __ballot(ids >= 0);
      }
      live = (live & ~(SPMASK << SP * slot)) |
             ((uint32_t)(there >> (pg - base)) & SPMASK) << SP * slot;
      const int mine = __builtin_amdgcn_readlane(ids, pg - base + wave);
      const int64_t off = (int64_t)(mine >= 0 ? mine : 0) * step;  // (pages that are not there: block 0's bytes, unseen)
      uint8_t* dst = ring + slot * STAGE + wave * P::BYTES;
      if constexpr (HD == 128) {
        stage_load16(kb + off, k_off, dst);
        stage_load16(vb + off, v_off, dst + P::CODES);
      } else {
        stage_load16_at(code_src + off, dst);
      }
      if (lane < 8 * G) stage_load16_at(meta_src + off, dst + 2 * P::CODES);
    };
    auto compute = [&](int st, int slot) {
#pragma unroll 1
      for (int h = half * kQ4WideWaves; h < (half + 1) * kQ4WideWaves; h += 2) {
        const int key0 = (p0 + st * SP + h) * kQ4Tokens;
        const int bits = (int)(live >> (SP * slot + h)) & 3;
        const uint8_t* pg = ring + slot * STAGE + h * P::BYTES;
        if (key0 >= most || bits == 0) continue;
        q4_step<HD, PARTS>(pg, w, key0, bits != 3 || key0 + 32 > all, bits, lane);
      }
    };
    issue(0, 0);
    issue(1, 1);
    for (int st = 0, slot = 0; st < stages; ++st) {
      vm_wait<LOADS>();  // this wavefront's page of stage st has arrived; the barrier: everybody's, and stage
      lds_read_wait();   // st - 1, whose slot is filled next, has been read
      __builtin_amdgcn_s_barrier();
      issue(st + 2, slot == 0 ? 2 : slot - 1);
      compute(st, slot);
      slot = slot == 2 ? 0 : slot + 1;
    }
    vm_wait<0>();  // nothing may still be on its way into LDS when the workgroup ends
  }
  const int row = q4_row<PARTS>(tile, c);
  float o[G][16], l;
  q4_join<HD, PARTS>(w, o, l);
  if constexpr (HALVES == 2) {
    __syncthreads();  // every wavefront has read its last stage
    float* mine = reinterpret_cast<float*>(ring) + (tile_wave * 64 + lane) * (16 * G + 2);
    if (half == 1) {
      mine[0] = w.M;
      mine[1] = l;
#pragma unroll
      for (int k = 0; k < G; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) mine[2 + 16 * k + i] = o[k][i];
    }
    __syncthreads();
    if (half == 1) return;
    const float M = fmaxf(w.M, mine[0]), f0 = fast_exp2(w.M - M), f1 = fast_exp2(mine[0] - M);
    w.M = M;
    l = fmaf(f0, l, f1 * mine[1]);
#pragma unroll
    for (int k = 0; k < G; ++k)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[k][i] = fmaf(f0, o[k][i], f1 * mine[2 + 16 * k + i]);
  }
  if (row >= rows || c >= ROWS) return;
  if (a.splits > 1) {
    float* rec = q4_record<HD>(a, u.b, u.hk, row, u.split);
    if (g == 0) {
      rec[0] = w.M;
      rec[1] = l;
    }
#pragma unroll
    for (int k = 0; k < G; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<f32x2*>(rec + 2 + 64 * k + 16 * g + 2 * i) = f32x2{o[k][2 * i], o[k][2 * i + 1]};
  } else {
    const int i = row / a.group, j = row - i * a.group;
    IO* out = static_cast<IO*>(a.out) + (int64_t)u.b * a.o_sb + (int64_t)(u.hk * a.group + j) * a.o_sh + (int64_t)i * a.o_st;
    const float f = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
    for (int k = 0; k < G; ++k) q4_store16<IO>(out + 64 * k + 16 * g, o[k], f);
    if (a.lse != nullptr && g == 0) *q4_lse(a, u.b, u.hk, row) = q4_log_sum(w.M, l);
  }
}

// ---------------------------------------------------------------------------------------------
// Up to one tile of rows (decode, short chunks). A column tile has 16 / PARTS columns, and a decode step over
// unshared heads would fill one of them, its softmax repeated in all. So GP columns hold rows (GP the
// rows rounded up to 1, 4 or the whole tile), q is repeated in the others, and a batch of pages goes
// through together: page t's scores are kept by the lanes of columns GP t' .. (t' = t % PG, PG = columns / GP), where
// softmax, scales and running sums then cost one page's work for PG pages. For the second product page t's
// weights turn back to the first GP columns by a DPP rotation of the row; the other columns' sums are
// never read.
//
// A batch's loads are all issued before its products, and K's registers are filled again while the second
// product runs: 16 KB and more in flight per wavefront.
//
// Bound by memory: 16 requests of 512 to 32768 keys, 32 heads x 128 bf16, 577 MB read: 106 us, 5.4 TB/s (a page at
// a time, its softmax repeated in every column, took 370 us where pages batched over the columns took 176).
// 64 requests of 32 over 8 heads of 512 to 16384 keys with totals: 339 MB read, 41 MB of scores written, 85 us,
// 4.5 TB/s.
// ---------------------------------------------------------------------------------------------
template <int N>
__device__ __forceinline__ uint32_t row_from(uint32_t x) {  // lane c of a 16-lane row: lane (c + N) % 16
  if constexpr (N % 16 == 0) return x;
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + (16 - N % 16), 0xF, 0xF, false);  // row_ror
}
template <int GP, int N = 8>
__device__ __forceinline__ float row_max(float x) {  // over the lanes c + k GP of a row
  if constexpr (N < GP) return x;
  else return row_max<GP, N / 2>(fmaxf(x, dpp<0x120 + N>(x)));
}
template <int GP, int N = 8>
__device__ __forceinline__ float row_sum(float x) {
  if constexpr (N < GP) return x;
  else return row_sum<GP, N / 2>(x + dpp<0x120 + N>(x));
}

template <int HD, int PARTS, int GP>
struct Q4Batch {
  static constexpr int G = HD / kQ4Group, W = HD / 32;
  // pages that share a softmax: 8 at most, which 213 to 223 registers hold at head_dim 128 (16 spill)
  static constexpr int COLS = 16 / PARTS, PG = COLS / GP < 8 ? COLS / GP : 8;
  static constexpr int PAGES = PG == 1 ? 2 : PG < 4 ? 4 : PG, NB = PAGES / PG;
  uint32_t k[PAGES][W], v[PAGES][2 * G];
  u32x4 km[NB][G], vm[NB][G];
  int live[NB];  // this lane's pages: 1 where the page is there
};

template <int N>
__device__ __forceinline__ void q4_load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = x[i];
  } else {
    const u32x2 x = *reinterpret_cast<const u32x2*>(p);
    w[0] = x[0];
    w[1] = x[1];
  }
}

// O^T += V^T P^T over a batch, two pages per matrix instruction.
template <int HD, int PARTS, int GP, bool LAST, int... PAIRS>
__device__ __forceinline__ void q4_narrow_values(const Q4Batch<HD, PARTS, GP>& r,
                                                 const uint32_t (&w)[Q4Batch<HD, PARTS, GP>::NB][HD / kQ4Group][2],
                                                 f32x4 (&o)[HD / kQ4Group][4], int cnt, std::integer_sequence<int, PAIRS...>) {
  constexpr int G = HD / kQ4Group, PG = Q4Batch<HD, PARTS, GP>::PG;
  auto pair = [&](auto index) {
    constexpr int T0 = 2 * decltype(index)::value, T1 = T0 + 1;
    if (LAST && T0 >= cnt) return;
#pragma unroll
    for (int k = 0; k < G; ++k) {
      const f16x8 b = q4_operand(row_from<(T0 % PG) * GP>(w[T0 / PG][k][0]), row_from<(T0 % PG) * GP>(w[T0 / PG][k][1]),
                                 row_from<(T1 % PG) * GP>(w[T1 / PG][k][0]), row_from<(T1 % PG) * GP>(w[T1 / PG][k][1]));
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t x0 = r.v[e >> 1 ? T1 : T0][(e & 1) * G + k], x1 = t & 2 ? x0 >> 8 : x0;
          x[e] = t & 1 ? q4_pair<PARTS, true>(x1) : q4_pair<PARTS, false>(x1);
        }
        o[k][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(q4_operand(x[0], x[1], x[2], x[3]), b, o[k][t], 0, 0, 0);
      }
    }
  };
  (pair(std::integral_constant<int, PAIRS>()), ...);
}

template <typename IO, int HD, int PARTS, int GP>
__global__ __launch_bounds__(64 * kQ4Waves, 2) void q4_narrow_kernel(const Q4Args a) {
  using Batch = Q4Batch<HD, PARTS, GP>;
  constexpr int G = Batch::G, W = Batch::W, COLS = Batch::COLS, PG = Batch::PG, PAGES = Batch::PAGES, NB = Batch::NB;
  constexpr int PB = q4_page_bytes(HD), CB = q4_codes_bytes(HD);
  __shared__ float part[kQ4Waves * GP * (HD + 2)];
  __shared__ f32x2 lse_of[GP];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15, col = c & (COLS - 1);
  const int row_in = col % GP, page_in = col / GP % PG;  // this lane's row of the tile and page of the batch
  const bool spare = col / GP >= PG;                     // (columns beyond the batch's pages)
  const bool low = PARTS == 2 && c >= COLS;
  const Q4Unit u = q4_unit(a);
  const int L = a.seq_lens[u.b], C = a.cur_lens[u.b];
  const int rows = a.T * a.group, first = u.tile * COLS;
  const int here = rows - first < GP ? rows - first : GP;  // rows of this tile (tiles of one row set have GP = COLS)
  int keys = L < a.max_pages * kQ4Tokens ? L : a.max_pages * kQ4Tokens;
  keys = keys > 0 ? keys : 0;
  int most = valid_keys(L, C, (first + here - 1) / a.group);
  most = most < keys ? most : keys;
  const int pages = (most + kQ4Tokens - 1) / kQ4Tokens;
  int p0 = u.split * a.split_pages, p1 = a.splits > 1 ? p0 + a.split_pages : pages;
  p1 = p1 < pages ? p1 : pages;
  if (a.splits > 1 && p0 >= p1) return;  // no record: the merge knows how far the rows' pages reach
  {  // the wavefronts' shares, an even number of pages each
    const int per = p1 > p0 ? ((p1 - p0 + 2 * kQ4Waves - 1) / (2 * kQ4Waves)) * 2 : 0;
    p0 += per * wave;
    p1 = p0 + per < p1 ? p0 + per : p1;
  }

  // q: the row of this lane's column, scaled by a power of two; see q4_setup for the factors
  const int row = first + row_in;
  const bool there = row_in < here;
  const int qi = row / a.group, qj = row - qi * a.group;
  f16x8 q[W];
  float qs[G], sc;
  {
    const IO* src = static_cast<const IO*>(a.q) + (int64_t)u.b * a.q_sb + (int64_t)(u.hk * a.group + qj) * a.q_sh + (int64_t)qi * a.q_st;
    q4_row_operands<IO, HD, PARTS>(src, there, low, g, a.scale_log2, q, qs, sc);
  }
  int n = valid_keys(L, C, qi);
  n = n < keys ? n : keys;
  n = there ? n : 0;

  f32x4 start[G], o[G][4];
  float y[G], l = 0.f, M = kQ4None;
  const float zero = q4_zero();
#pragma unroll
  for (int k = 0; k < G; ++k) {
    const float s0 = PARTS == 2 ? 0.f : -7.5f * qs[k];
    start[k] = f32x4{s0, s0, s0, s0};
    y[k] = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t) o[k][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  float* scores = nullptr;
  if (a.scores != nullptr && there && !low && !spare)
    scores = a.scores + ((int64_t)u.b * a.H + u.hk * a.group + row) * a.score_stride + 4 * g;

  if (p0 < p1) {
    const int32_t* table = a.page_table + (int64_t)u.b * a.pt_stride;
    const int64_t step = (int64_t)a.Hk * PB;
    const uint8_t* kb = a.k_pool + (int64_t)u.hk * PB;
    const uint8_t* vb = a.v_pool + (int64_t)u.hk * PB;
    const uint32_t k_lane = (uint32_t)(c * 4 + g) * (W * 4), v_lane = (uint32_t)lane * (8 * G);
    int ids = 0, base = p0 - 64;
    Batch r;
    // page ids of a batch: 64 at a time in a register, a batch never crosses them (PAGES divides 64)
    auto next_ids = [&](int p) {
      if (p - base >= 64) {
        base = p;
        const int id = p + lane < p1 ? table[p + lane] : -1;
        ids = q4_block(id, a.num_blocks);
      }
    };
    // (a last batch of fewer pages reads its last one again: loads under branches would make every wait for
    // one a wait for all)
    auto id_at = [&](int p, int t) {
      const int at = p + t < p1 ? p + t : p1 - 1;
      const int id = __builtin_amdgcn_readlane(ids, at - base);
      return id >= 0 ? id : 0;
    };
    auto load_k = [&](int p) {
#pragma unroll
      for (int t = 0; t < PAGES; ++t) q4_load_words(kb + (int64_t)id_at(p, t) * step + k_lane, r.k[t]);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int at = __shfl(ids, p - base + nb * PG + page_in);
        const bool live = p + nb * PG + page_in < p1 && at >= 0 && !spare;
        r.live[nb] = live;
#pragma unroll
        for (int k = 0; k < G; ++k) {
          const int64_t off = (int64_t)(live ? at : 0) * step + CB + (k * kQ4Tokens + 4 * g) * 4;
          r.km[nb][k] = *reinterpret_cast<const u32x4*>(kb + off);
          r.vm[nb][k] = *reinterpret_cast<const u32x4*>(vb + off);
        }
      }
    };
    auto load_v = [&](int p) {
#pragma unroll
      for (int t = 0; t < PAGES; ++t) q4_load_words(vb + (int64_t)id_at(p, t) * step + v_lane, r.v[t]);
    };
    auto batch = [&](int p, auto is_last) {
      constexpr bool LAST = decltype(is_last)::value;
      const int cnt = LAST ? p1 - p : PAGES;
      f32x4 acc[NB][G];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int k = 0; k < G; ++k) acc[nb][k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < PAGES; ++t) {
        if (LAST && t >= cnt) continue;
        f16x8 kf[W];
        q4_k_operands<HD, PARTS>(r.k[t], kf);
#pragma unroll
        for (int k = 0; k < G; ++k) {
          f32x4 x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[2 * k], q[2 * k], start[k], 0, 0, 0);
          x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[2 * k + 1], q[2 * k + 1], x, 0, 0, 0);
          if (t % PG == 0) {
            acc[t / PG][k] = x;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t / PG][k][i] = page_in == t % PG ? x[i] : acc[t / PG][k][i];
          }
        }
      }
      // what a row does not see takes part with score -inf and the pair (0, 0)
      f32x4 S[NB];
      u32x4 vm[NB][G];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        f32x4 x = {zero, zero, zero, zero};
#pragma unroll
        for (int k = 0; k < G; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x[i] = fmaf(q4_scale(r.km[nb][k][i]), acc[nb][k][i], fmaf(q4_centre(r.km[nb][k][i]), qs[k], x[i]));
        const int key = (p + nb * PG + page_in) * kQ4Tokens + 4 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (PARTS == 2) x[i] += dpp<0x128>(x[i]);
          const bool see = r.live[nb] && key + i < n;
          S[nb][i] = see ? x[i] * sc : -INFINITY;
#pragma unroll
          for (int k = 0; k < G; ++k) vm[nb][k][i] = see ? r.vm[nb][k][i] : 0u;
        }
        if (scores != nullptr && p + nb * PG + page_in < p1)
          *reinterpret_cast<f32x4*>(scores + (p + nb * PG + page_in) * kQ4Tokens) = S[nb];
      }
      if constexpr (!LAST) {
        next_ids(p + PAGES);
        load_k(p + PAGES);
      }
      float pr[NB][4];
      uint32_t w[NB][G][2];
#pragma unroll 1
      for (int pass = 0; pass < 2; ++pass) {  // (as in q4_step)
        float big = 0.f;
        s16x2 top = {0, 0};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            pr[nb][i] = fast_exp2(S[nb][i] - M);
            big = fmaxf(big, pr[nb][i]);
          }
#pragma unroll
          for (int k = 0; k < G; ++k)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              f16x2 hi, part;
              if constexpr (PARTS == 1) {
                hi = part = q4_weights(pr[nb][i], vm[nb][k][i], pr[nb][i + 1], vm[nb][k][i + 1]);
              } else {
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                  const float x = pr[nb][i + f] * q4_scale(vm[nb][k][i + f]);
                  hi[f] = (_Float16)x;
                  const _Float16 rest = (_Float16)(x - (float)hi[f]);
                  part[f] = low ? rest : hi[f];
                }
              }
              top = __builtin_elementwise_max(top, __builtin_bit_cast(s16x2, hi));
              w[nb][k][i / 2] = __builtin_bit_cast(uint32_t, part);
            }
        }
        const bool far = top[0] > kQ4LimitBits || top[1] > kQ4LimitBits || big > kQ4Limit / kQ4Floor;
        if (__builtin_expect(!__any(far), 1)) break;
        float m = kQ4None;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float s = kQ4Floor;
            asm volatile("" : "+v"(s));
#pragma unroll
            for (int k = 0; k < G; ++k) s = fmaxf(s, q4_scale(vm[nb][k][i]));
            m = fmaxf(m, S[nb][i] + __builtin_amdgcn_logf(s) - kQ4Start);
          }
        m = row_max<GP>(max_xor32(max_xor16(m)));
        const float now = fmaxf(M, m), f = fast_exp2(M - now);
        M = now;
        l *= f;
#pragma unroll
        for (int k = 0; k < G; ++k) {
          y[k] *= f;
#pragma unroll
          for (int t = 0; t < 4; ++t) o[k][t] *= f;
        }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) l += pr[nb][i];
#pragma unroll
        for (int k = 0; k < G; ++k) {
#pragma unroll
          for (int i = 0; i < 4; ++i) y[k] = fmaf(pr[nb][i], q4_centre(vm[nb][k][i]), y[k]);
          if constexpr (PARTS == 1) {
            const h16x2 mid = {(__fp16)-7.5f, (__fp16)-7.5f};
            y[k] = __builtin_amdgcn_fdot2(__builtin_bit_cast(h16x2, w[nb][k][0]), mid, y[k], false);
            y[k] = __builtin_amdgcn_fdot2(__builtin_bit_cast(h16x2, w[nb][k][1]), mid, y[k], false);
          }
        }
      }
      q4_narrow_values<HD, PARTS, GP, LAST>(r, w, o, cnt, std::make_integer_sequence<int, PAGES / 2>());
      if constexpr (!LAST) load_v(p + PAGES);
    };
    next_ids(p0);
    load_k(p0);
    load_v(p0);
    int p = p0;
    for (; p + PAGES < p1; p += PAGES) batch(p, std::false_type());
    batch(p, std::true_type());
  }

  // the lanes' sums joined, the wavefronts' parts merged
  l = row_sum<GP>(sum_xor32(sum_xor16(l))) * (1.f / PARTS);
#pragma unroll
  for (int k = 0; k < G; ++k) y[k] = row_sum<GP>(sum_xor32(sum_xor16(y[k]))) * (1.f / PARTS);
  {
    float* mine = part + (wave * GP + row_in) * (HD + 2);
    if (c < GP) {
      if (g == 0) {
        mine[0] = M;
        mine[1] = l;
      }
    }
#pragma unroll
    for (int k = 0; k < G; ++k)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = o[k][t][i];
          if constexpr (PARTS == 2) v += dpp<0x128>(v);
          v = fmaf(v, (t & 1) ? kQ4Unit<PARTS> / 16.f : kQ4Unit<PARTS>, y[k]);
          if (c < GP) mine[2 + 64 * k + 16 * g + 4 * i + t] = v;
        }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < here * HD; x += 64 * kQ4Waves) {
    const int r = x / HD, d = x - r * HD, m = first + r;
    float top = kQ4None;
#pragma unroll
    for (int v = 0; v < kQ4Waves; ++v) top = fmaxf(top, part[(v * GP + r) * (HD + 2)]);
    float den = 0.f, s = 0.f;
#pragma unroll
    for (int v = 0; v < kQ4Waves; ++v) {
      const float* rec = part + (v * GP + r) * (HD + 2);
      const float f = fast_exp2(rec[0] - top);
      den = fmaf(f, rec[1], den);
      s = fmaf(f, rec[2 + d], s);
    }
    if (a.splits > 1) {
      float* rec = q4_record<HD>(a, u.b, u.hk, m, u.split);
      if (d == 0) {
        rec[0] = top;
        rec[1] = den;
      }
      rec[2 + d] = s;
    } else {
      const int i = m / a.group, j = m - i * a.group;
      IO* out = static_cast<IO*>(a.out) + (int64_t)u.b * a.o_sb + (int64_t)(u.hk * a.group + j) * a.o_sh + (int64_t)i * a.o_st;
      Elem<IO>::store(out + d, den > 0.f || den != den ? s / den : 0.f);
      if (a.lse != nullptr && d == 0) {
        const f32x2 e = q4_log_sum(top, den);
        lse_of[r] = e;
        *q4_lse(a, u.b, u.hk, m) = e;
      }
    }
  }
  // one workgroup has seen all keys of all the head's rows: the totals without another launch
  if (a.scores != nullptr && a.splits == 1 && a.tiles == 1 && C > 0) {
    __syncthreads();
    const float* mine = a.scores + ((int64_t)u.b * a.H + u.hk * a.group) * a.score_stride;
    for (int t = threadIdx.x; t < most; t += 64 * kQ4Waves) {
      const int id = q4_block(a.page_table[(int64_t)u.b * a.pt_stride + t / kQ4Tokens], a.num_blocks);
      if (id < 0) continue;
      float sum = 0.f;
      for (int j = 0; j < here; ++j) sum += fast_exp2(mine[j * a.score_stride + t] - lse_of[j][0] - lse_of[j][1]);
      atomicAdd(a.weights + ((int64_t)id * a.Hk + u.hk) * kQ4Tokens + (t & (kQ4Tokens - 1)), sum);
    }
  }
}

// Key ranges that hold keys of query position i.
__device__ __forceinline__ int q4_splits_of(const Q4Args& a, int b, int i) {
  int n = valid_keys(a.seq_lens[b], a.cur_lens[b], i);
  n = n < a.max_pages * kQ4Tokens ? n : a.max_pages * kQ4Tokens;
  return (n + a.split_pages * kQ4Tokens - 1) / (a.split_pages * kQ4Tokens);
}

// A row's splits: lane s reads (M, l) of split s (of 64 at a time); their weights 2^(M_s - M) stay in the lanes.
// Returns M and l.
template <int HD>
__device__ __forceinline__ void q4_row_state(const float* rec, int splits, int lane, float& M, float& l) {
  M = kQ4None;
  for (int s = lane; s < splits; s += 64) M = fmaxf(M, rec[(int64_t)s * (HD + 2)]);
  M = wave_max(M);
  l = 0.f;
  for (int s = lane; s < splits; s += 64) {
    const f32x2 r = *reinterpret_cast<const f32x2*>(rec + (int64_t)s * (HD + 2));
    l = fmaf(fast_exp2(r[0] - M), r[1], l);
  }
  l = wave_sum(l);
}

// Records of the splits -> outputs and, for decode totals, the keys' weights from the scores that the first
// kernel left in the workspace. The first `merges` workgroups merge, one wavefront per row; of the others each
// adds kQ4FinishKeys keys' weights of one KV head, having formed its rows' denominators from the records by itself (a
// launch less than in two steps). A block that two rows of the page table share is added to by both, hence
// the atomic; otherwise each slot gets one addition. 64 requests of 32 over 8 heads of 512 to 16384 keys: 42 MB of
// scores and 10 MB of totals, 21 us, 2.4 TB/s, with the vector units busy 31% of the time: latency, of the lengths, the
// records and the denominators that each workgroup takes one after the other before its scores.
constexpr int kQ4FinishKeys = 1024;  // (256, a key per thread, repeated the denominators too often: 34 -> 20 us)

template <typename IO, int HD>
__global__ __launch_bounds__(256) void q4_finish_kernel(const Q4Args a, int64_t total, int merges, int chunks) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int rows = a.T * a.group;
  if ((int)blockIdx.x < merges) {
    const int64_t x = (int64_t)blockIdx.x * 4 + wave;
    if (x >= total) return;
    const int row = (int)(x % rows);
    const int hk = (int)(x / rows % a.Hk), b = (int)(x / rows / a.Hk);
    const float* rec = q4_record<HD>(a, b, hk, row, 0);
    const int i = row / a.group, j = row - i * a.group;
    const int splits = q4_splits_of(a, b, i);
    float M, l;
    q4_row_state<HD>(rec, splits, lane, M, l);
    constexpr int E = HD / 64;
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
      const float* p = rec + (int64_t)s * (HD + 2);
      const float f = fast_exp2(p[0] - M);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(f, p[2 + lane + 64 * e], o[e]);
    }
    IO* out = static_cast<IO*>(a.out) + (int64_t)b * a.o_sb + (int64_t)(hk * a.group + j) * a.o_sh + (int64_t)i * a.o_st;
#pragma unroll
    for (int e = 0; e < E; ++e) Elem<IO>::store(out + lane + 64 * e, l > 0.f || l != l ? o[e] / l : 0.f);
    if (a.lse != nullptr && lane == 0) *q4_lse(a, b, hk, row) = q4_log_sum(M, l);
    return;
  }
  __shared__ f32x2 lse[kQ4MaxNarrow];
  int x = (int)blockIdx.x - merges;
  const int hk = x % a.Hk;
  x /= a.Hk;
  const int chunk = x % chunks, b = x / chunks;
  const int L = a.seq_lens[b], C = a.cur_lens[b];
  int n = valid_keys(L, C, 0);
  n = n < a.max_pages * kQ4Tokens ? n : a.max_pages * kQ4Tokens;
  const int t0 = chunk * kQ4FinishKeys;
  if (t0 >= n || C < 1) return;
  if (a.splits > 1) {
    const int splits = q4_splits_of(a, b, 0);
    for (int j = wave; j < a.group; j += 4) {
      float M, l;
      q4_row_state<HD>(q4_record<HD>(a, b, hk, j, 0), splits, lane, M, l);
      if (lane == 0) lse[j] = q4_log_sum(M, l);
    }
  } else if ((int)threadIdx.x < a.group) {
    lse[threadIdx.x] = *q4_lse(a, b, hk, threadIdx.x);
  }
  __syncthreads();
  const float* mine = a.scores + ((int64_t)b * a.H + hk * a.group) * a.score_stride;
  const int t1 = t0 + kQ4FinishKeys < n ? t0 + kQ4FinishKeys : n;
#pragma unroll 4
  for (int t = t0 + threadIdx.x; t < t1; t += 256) {
    const int id = q4_block(a.page_table[(int64_t)b * a.pt_stride + t / kQ4Tokens], a.num_blocks);
    float sum = 0.f;
#pragma unroll 4
    for (int j = 0; j < a.group; ++j) sum += fast_exp2(mine[j * a.score_stride + t] - lse[j][0] - lse[j][1]);
    if (id >= 0) atomicAdd(a.weights + ((int64_t)id * a.Hk + hk) * kQ4Tokens + (t & (kQ4Tokens - 1)), sum);
  }
}

// Totals of a chunk: the scores formed again, PG pages per workgroup whose operands and pairs stay in registers;
// the workgroup's wavefronts take the row tiles in turn, the next tile's operands on their way, and their
// sums meet in LDS in a fixed order; or (EACH) every wavefront has pages of its own and takes all tiles. READY:
// the tiles' q operands are in the workspace, left by the wide kernel (formed here they cost as much as the
// scores). A block that two rows of the page table share is added to by both, hence the atomic; otherwise
// each slot gets one addition. Bound by vector instructions, 170 to 16 matrix instructions a tile: 200 rows of 32
// over 8 heads x 128 bf16 over 16.5k keys 73 us (370 TFLOP/s).
constexpr int kQ4SumWaves = 8;

template <typename IO, int HD, int PARTS, bool READY, int PG, bool EACH>
__global__ __launch_bounds__(64 * kQ4SumWaves) void q4_chunk_weights_kernel(const Q4Args a) {
  constexpr int G = HD / kQ4Group, W = HD / 32, PB = q4_page_bytes(HD);
  constexpr int ROWS = 16 / PARTS;
  constexpr int STEP = EACH ? 1 : kQ4SumWaves;  // from one row tile of a wavefront to its next
  __shared__ float part[kQ4SumWaves][PG * kQ4Tokens];
  const int b = blockIdx.z, hk = blockIdx.y;
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int p0 = PG * (EACH ? (int)blockIdx.x * kQ4SumWaves + wave : (int)blockIdx.x), key0 = p0 * kQ4Tokens;
  const int L = a.seq_lens[b], C = a.cur_lens[b];
  const int keys = L < a.max_pages * kQ4Tokens ? L : a.max_pages * kQ4Tokens;
  if (key0 >= keys || C < 1) return;
  const int rows = a.T * a.group, real = (C < a.T ? C : a.T) * a.group;  // rows behind `real` are padding
  // the first row that sees the first of these keys: key0 < L - C + 1 + i. Where none does (more new tokens
  // claimed than there are keys and rows), its tile's operands need not be there.
  int64_t i0 = (int64_t)key0 - ((int64_t)L - C);
  i0 = i0 > 0 ? i0 : 0;
  if (i0 >= a.T) return;
  const int32_t* table = a.page_table + (int64_t)b * a.pt_stride;
  int id[PG];
  f16x8 kf[PG][W];
  u32x4 km[PG][G];
#pragma unroll
  for (int h = 0; h < PG; ++h) {
    id[h] = p0 + h < a.max_pages ? q4_block(__builtin_amdgcn_readfirstlane(table[p0 + h]), a.num_blocks) : -1;
    const uint8_t* kp = a.k_pool + ((int64_t)(id[h] >= 0 ? id[h] : 0) * a.Hk + hk) * PB;
    uint32_t kw[W];
    q4_load_words(kp + (c * 4 + g) * (4 * W), kw);
    q4_k_operands<HD, PARTS>(kw, kf[h]);
#pragma unroll
    for (int k = 0; k < G; ++k)
      km[h][k] = *reinterpret_cast<const u32x4*>(kp + q4_codes_bytes(HD) + (k * kQ4Tokens + 4 * g) * 4);
  }
  float sum[PG][4];
#pragma unroll
  for (int h = 0; h < PG; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[h][i] = 0.f;
  // (the next tile's operands are loaded while this one's scores are formed; past the last one, its own)
  f16x8 next[W];
  f32x4 next_aux;
  f32x2 next_lse;
  const int last = (real - 1) / ROWS;
  auto load = [&](int tile) {
    tile = tile < last ? tile : last;
    const int row = q4_row<PARTS>(tile, c);
    next_lse = row < real && c < ROWS ? *q4_lse(a, b, hk, row < rows ? row : rows - 1) : f32x2{0.f, INFINITY};  // (2^-inf: 0)
    if constexpr (READY) {
      const int64_t at = ((int64_t)b * a.Hk + hk) * a.op_tiles + tile;
#pragma unroll
      for (int s = 0; s < W; ++s) next[s] = a.q_ops[(at * W + s) * 64 + lane];
      next_aux = a.q_aux[at * 64 + lane];
    }
  };
  int tile = (int)(i0 * a.group / ROWS) + (EACH ? 0 : wave);
  if (tile * ROWS < real) load(tile);
  for (; tile * ROWS < real; tile += STEP) {
    f16x8 q[W];
    float qs[G], sc;
    int n;
    const float M = next_lse[0], log_l = next_lse[1], lse = M + log_l;
    if constexpr (READY) {
#pragma unroll
      for (int s = 0; s < W; ++s) q[s] = next[s];
#pragma unroll
      for (int k = 0; k < G; ++k) qs[k] = next_aux[k];
      sc = next_aux[2];
      n = __float_as_int(next_aux[3]);
      load(tile + STEP);
    } else {
      Q4Wave<HD, PARTS> w;
      q4_setup<IO, HD, PARTS>(a, b, hk, tile, L, C, keys, lane, w);
      const bool pad = q4_row<PARTS>(tile, c) >= real;
#pragma unroll
      for (int s = 0; s < W; ++s) q[s] = pad ? f16x8{} : w.q[s];
#pragma unroll
      for (int k = 0; k < G; ++k) qs[k] = pad ? 0.f : w.qs[k];
      sc = w.sc;
      n = pad ? 0 : w.n;
      load(tile + STEP);
    }
    // masked: some columns do not see all the keys, or have scores that M + log2 l in one float would blur
    auto add = [&](auto masked) {
      const float unit = READY && q4_steep(M) ? q4_steep_unit(sc) : sc;
#pragma unroll
      for (int h = 0; h < PG; ++h) {
        const f32x4 S = q4_scores<HD, PARTS>(kf[h], km[h], q, qs);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = S[i] * unit;
          if (!READY) asm("" : "+v"(x));  // (the narrow kernel's scores are rounded, the wide one's products exact)
          const float p = fast_exp2(decltype(masked)::value ? (READY ? fmaf(S[i], unit, -M) : x - M) - log_l : fmaf(S[i], sc, -lse));
          sum[h][i] += decltype(masked)::value && key0 + h * kQ4Tokens + 4 * g + i >= n ? 0.f : p;
        }
      }
    };
    if (__any(n < key0 + PG * kQ4Tokens || !(fabsf(M) < 256.f))) add(std::true_type()); else add(std::false_type());
  }
#pragma unroll
  for (int h = 0; h < PG; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float s = group_sum<16>(sum[h][i]);
      if (c != i) continue;
      const int t = h * kQ4Tokens + 4 * g + i;
      if constexpr (!EACH)
        part[wave][t] = s;
      else if (id[h] >= 0 && key0 + t < keys)
        atomicAdd(a.weights + ((int64_t)id[h] * a.Hk + hk) * kQ4Tokens + 4 * g + i, s);
    }
  if constexpr (EACH) return;
  __syncthreads();
  const int t = threadIdx.x;
  if (t < PG * kQ4Tokens && key0 + t < keys) {
    const int block = q4_block(table[p0 + t / kQ4Tokens], a.num_blocks);
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kQ4SumWaves; ++w) s += part[w][t];
    if (block >= 0) atomicAdd(a.weights + ((int64_t)block * a.Hk + hk) * kQ4Tokens + (t & (kQ4Tokens - 1)), s);
  }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
struct Q4Plan {
  int parts, rows_per_tile;
  bool wide, halves, four;
  int tiles, splits, split_pages;
  int64_t rows;
  size_t rec, lse, scores, score_stride, ops, aux, bytes;  // (the parts in floats)
  int op_tiles;
};

// Which kernel, how many row tiles and key ranges, and the workspace.
static Q4Plan q4_plan(int io_dtype, int32_t batch, int32_t heads, int32_t kv_heads, int32_t query_len, int32_t head_dim,
                      int32_t max_pages, bool weights) {
  Q4Plan p{};
  p.parts = io_dtype == PA_DTYPE_F32 ? 2 : 1;
  const int rpt = p.parts == 2 ? 8 : 16;
  p.rows = (int64_t)query_len * (heads / kv_heads);
  // More rows than two tiles: the wide kernel. Up to there the narrow one, whose tiles each read the keys for
  // themselves, but for bf16 at head_dim 128, where more than four rows leave it batches of two pages: there the
  // wide one from 512 keys on, for one tile while it gives a CU at most one workgroup. Narrow -> wide in us:
  //   8 requests x 4 KV heads x 8 rows, 512 / 2048 / 8192 keys   13.9 / 22.9 / 31.0 -> 13.7 / 14.2 / 22.5
  //   64 x 8 x 6 rows                                           26.8 / 66.9 / 161 -> 19.8 / 57.8 / 208
  //   8 x 8 x 24 rows, 512 / 1024 / 8192 (128: 7.8 -> 8.3)       20.7 / 25.3 / 64.2 -> 15.6 / 17.4 / 41.3
  //   the same at head_dim 64                                  7.5 / 10.3 / 28.0 -> 12.5 / 13.5 / 27.2
  //   8 x 8 x 16 rows, fp32                                    11.4 / 16.7 / 60.8 -> 17.4 / 18.9 / 53.8
  // A decode step's totals come from the narrow kernel's scores at a lower price than from scores formed again,
  // once there are many: 64 x 1 x 16 rows, 2048 / 8192 keys 38 / 50 -> 27 / 54.
  const int64_t heads_of_all = (int64_t)batch * kv_heads;
  const bool early = p.parts == 1 && head_dim == 128 && p.rows > 4 && max_pages >= 32 &&
                     (p.rows > rpt || heads_of_all <= pa_host::device_cu_count()) &&
                     (!weights || query_len > 1 || heads_of_all * max_pages <= 16384);
  p.wide = p.rows > 2 * rpt || early;
  p.rows_per_tile = p.wide ? kQ4WideWaves * rpt : rpt;
  p.tiles = (int)((p.rows + p.rows_per_tile - 1) / p.rows_per_tile);
  const int64_t units = (int64_t)batch * kv_heads * p.tiles;
  // workgroups that the GPU holds; more ranges than fit would wait for a second round
  const int64_t target = (p.wide ? (head_dim == 64 ? 4 : 3) : 2) * (int64_t)pa_host::device_cu_count();
  const int64_t want = units <= 0 ? 1 : p.wide ? (target / units > 1 ? target / units : 1) : (target + units - 1) / units;
  int pages = (int)((max_pages + want - 1) / want);
  // A second launch merges ranges: 64 pages (one batch or two per wavefront) are not worth it, 128 are; nor
  // are they for the wide kernel where its row tiles alone give every CU a workgroup.
  const int least = p.wide ? (units >= pa_host::device_cu_count() ? 64 : 16) : max_pages <= 64 ? 64 : 32;
  if (!p.wide && pages > 96) pages = 96;  // requests of very different lengths: ranges end together
  pages = pages < least ? least : pages;
  pages = (pages + 7) / 8 * 8;
  p.split_pages = pages;
  p.splits = max_pages > pages ? (max_pages + pages - 1) / pages : 1;
  // One row: 8 (fp32) or 16 pages of columns to it, but four for many pages of bf16 at head_dim 128, whose batches
  // are half the size (2 x 32 heads over 1024 / 4096 / 16384 keys 8.5 / 11.8 / 27.4 -> 9.1 / 12.2 / 25.9 us, 16 x 32
  // 12.5 / 43.1 / 154 -> 13.0 / 40.1 / 145; fp32 53 -> 66).
  p.four = p.parts == 1 && head_dim == 128 && units * max_pages >= 49152;
  // eight wavefronts to a workgroup while there are fewer than two workgroups a CU
  p.halves = p.wide && units * p.splits < 2 * (int64_t)pa_host::device_cu_count();
  p.rec = p.splits > 1 ? (size_t)batch * kv_heads * p.rows * p.splits * (head_dim + 2) : 0;
  p.lse = weights ? (size_t)batch * kv_heads * p.rows * 2 : 0;
  p.score_stride = (size_t)(max_pages + (max_pages & 1)) * kQ4Tokens;
  p.scores = weights && query_len == 1 && !p.wide ? (size_t)batch * heads * p.score_stride : 0;
  p.op_tiles = p.tiles * kQ4WideWaves;
  const size_t ops = weights && p.wide ? (size_t)batch * kv_heads * p.op_tiles * 64 : 0;
  p.ops = ops * (head_dim / 32) * (sizeof(f16x8) / sizeof(float));
  p.aux = ops * (sizeof(f32x4) / sizeof(float));
  auto up = [](size_t n) { return (n + 63) / 64 * 64; };
  p.rec = up(p.rec);
  p.lse = up(p.lse);
  p.scores = up(p.scores);
  p.bytes = (p.rec + p.lse + p.scores + p.ops + p.aux) * sizeof(float);
  return p;
}

template <typename IO, int HD, int PARTS>
static void launch_q4(const Q4Args& a, const Q4Plan& p, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.B * a.Hk * p.tiles * p.splits));
  if (p.wide && p.halves)
    q4_wide_kernel<IO, HD, PARTS, 2><<<grid, 2 * 64 * kQ4WideWaves, 0, stream>>>(a);
  else if (p.wide)
    q4_wide_kernel<IO, HD, PARTS, 1><<<grid, 64 * kQ4WideWaves, 0, stream>>>(a);
  else if (p.rows == 1 && !p.four)
    q4_narrow_kernel<IO, HD, PARTS, 1><<<grid, 64 * kQ4Waves, 0, stream>>>(a);
  else if (p.rows <= 4)
    q4_narrow_kernel<IO, HD, PARTS, 4><<<grid, 64 * kQ4Waves, 0, stream>>>(a);
  else
    q4_narrow_kernel<IO, HD, PARTS, 16 / PARTS><<<grid, 64 * kQ4Waves, 0, stream>>>(a);
  // totals of decode steps that one workgroup saw whole are done in place
  const bool totals = a.scores != nullptr && !(p.splits == 1 && p.tiles == 1);
  if (p.splits > 1 || totals) {
    const int64_t total = (int64_t)a.B * a.Hk * a.T * a.group;
    const int merges = p.splits > 1 ? (int)((total + 3) / 4) : 0, chunks = (a.max_pages * kQ4Tokens + kQ4FinishKeys - 1) / kQ4FinishKeys;
    const int64_t wgs = merges + (totals ? (int64_t)chunks * a.Hk * a.B : 0);
    q4_finish_kernel<IO, HD><<<(unsigned)wgs, 256, 0, stream>>>(a, total, merges, chunks);
  }
  if (a.weights != nullptr && a.scores == nullptr) {
    // PG: a page while four would leave CUs without a workgroup (3 x 61 rows of 24 over 3 heads x 64: 9.2 -> 5.9 us),
    // otherwise four, which read the row tiles' operands the least often (two: 72 -> 84 us at the size above).
    // EACH: for few tiles, and for up to 32 where the pages fill the GPU (8 x 4 rows of 32 over 8 heads x 128 over
    // 2048 keys, 32 x 12 of 32 heads, 4 x 200 of 32 heads, whole calls: 41 -> 25, 746 -> 194, 146 -> 119 us; but
    // 3 x 61 as above 15 -> 28).
    auto sum = [&](auto ready, auto pages, auto each) {
      const int per = pages * (each ? kQ4SumWaves : 1);
      const dim3 wg((unsigned)((a.max_pages + per - 1) / per), a.Hk, a.B);
      q4_chunk_weights_kernel<IO, HD, PARTS, decltype(ready)::value, decltype(pages)::value, decltype(each)::value>
          <<<wg, 64 * kQ4SumWaves, 0, stream>>>(a);
    };
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 4> four;
    constexpr std::true_type yes;
    constexpr std::false_type no;
    const int64_t units = (int64_t)a.Hk * a.B * a.max_pages, cus = pa_host::device_cu_count();
    const int64_t tiles = (p.rows + 16 / PARTS - 1) / (16 / PARTS);
    if (tiles <= 4 || (tiles <= 32 && units >= 8 * cus)) {
      const bool small = units < 4 * 4 * kQ4SumWaves * cus;
      if (a.q_ops == nullptr)
        small ? sum(no, one, yes) : sum(no, four, yes);
      else
        small ? sum(yes, one, yes) : sum(yes, four, yes);
    } else {
      units < 4 * cus ? sum(yes, one, no) : sum(yes, four, no);
    }
  }
}

}  // namespace pa

using namespace pa;

namespace {
// The bytes of [batch, heads, tokens] rows: sizes, strides and a row's length.
struct Q4Rows {
  int64_t n[3], stride[3], row;
};

// Whether offset d is a difference of two rows' places, within a row's length: of its dimensions the one of the
// largest stride first, whose multiples that leave a remainder in reach of the others are few.
bool q4_row_apart(const Q4Rows& r, const int (&order)[3], int at, int64_t d) {
  if (at == 3) return d > -r.row && d < r.row;
  int64_t reach = r.row - 1;
  for (int k = at + 1; k < 3; ++k) reach += (r.n[order[k]] - 1) * r.stride[order[k]];
  const int64_t n = r.n[order[at]], s = r.stride[order[at]];
  if (n == 1 || s == 0) return q4_row_apart(r, order, at + 1, d);
  int64_t first = (d - reach) / s - 1, last = (d + reach) / s + 1;
  first = first > 1 - n ? first : 1 - n;
  last = last < n - 1 ? last : n - 1;
  if (last - first > 64) return true;  // (strides that no tensor of separate rows has)
  for (int64_t k = first; k <= last; ++k)
    if (q4_row_apart(r, order, at + 1, d - k * s)) return true;
  return false;
}

// Whether two sets of rows share a byte. Of sets whose extents meet, those of the same strides are compared
// exactly (q and out may be interleaved in one tensor); others count as meeting.
bool q4_rows_meet(const void* a, Q4Rows ra, const void* b, Q4Rows rb) {
  const auto extent = [](const void* p, const Q4Rows& r, int64_t& lo, int64_t& hi) {
    lo = hi = (int64_t)reinterpret_cast<uintptr_t>(p);
    for (int k = 0; k < 3; ++k) (r.stride[k] < 0 ? lo : hi) += (r.n[k] - 1) * r.stride[k];
    hi += r.row;
  };
  int64_t a0, a1, b0, b1;
  extent(a, ra, a0, a1);
  extent(b, rb, b0, b1);
  if (a1 <= b0 || b1 <= a0) return false;
  for (int k = 0; k < 3; ++k)
    if (ra.n[k] > 1 && (ra.stride[k] != rb.stride[k] || ra.stride[k] < 0)) return true;
  int order[3] = {0, 1, 2};
  for (int i = 0; i < 2; ++i)
    for (int k = 0; k < 2; ++k)
      if (ra.stride[order[k]] < ra.stride[order[k + 1]]) {
        const int t = order[k];
        order[k] = order[k + 1];
        order[k + 1] = t;
      }
  return q4_row_apart(ra, order, 0, (int64_t)reinterpret_cast<uintptr_t>(b) - (int64_t)reinterpret_cast<uintptr_t>(a));
}
}  // namespace

extern "C" size_t pa_q4_attention_workspace_size(int io_dtype, int32_t batch, int32_t num_heads, int32_t kv_heads,
                                                 int32_t query_len, int32_t head_dim, int32_t max_pages, int32_t weights) {
  if (batch <= 0 || num_heads <= 0 || kv_heads <= 0 || num_heads % kv_heads || query_len <= 0 || max_pages <= 0 ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  return q4_plan(io_dtype, batch, num_heads, kv_heads, query_len, head_dim, max_pages, weights != 0).bytes;
}

extern "C" int pa_q4_attention(const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t,
                               void* out, int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_t, int io_dtype,
                               const void* k_pool, const void* v_pool, int64_t num_blocks,
                               const int32_t* page_table, int64_t pt_stride, int32_t max_pages,
                               const int32_t* seq_lens, const int32_t* cur_lens, float* weights,
                               int32_t batch, int32_t num_heads, int32_t kv_heads, int32_t query_len, int32_t head_dim,
                               float scale, void* workspace, size_t workspace_bytes, void* stream_) {
  pa_host::clear_error();
  PA_CHECK_ARG(batch >= 0 && num_heads > 0 && kv_heads > 0 && query_len >= 0 && max_pages >= 0,
               "pa_q4_attention: bad sizes: batch=%d heads=%d kv_heads=%d query_len=%d max_pages=%d", batch, num_heads,
               kv_heads, query_len, max_pages);
  PA_CHECK_ARG(num_heads % kv_heads == 0, "pa_q4_attention: %d query heads are no multiple of %d KV heads", num_heads, kv_heads);
  PA_CHECK_ARG(io_dtype == PA_DTYPE_F32 || io_dtype == PA_DTYPE_BF16, "pa_q4_attention: bad io dtype %d", io_dtype);
  PA_CHECK_ARG(scale > 0.f && scale < INFINITY, "pa_q4_attention: scale must be positive and finite");
  if (head_dim != 64 && head_dim != 128)
    PA_FAIL(PA_ERR_UNSUPPORTED, "pa_q4_attention: no 4-bit pages for head_dim %d (64 and 128)", head_dim);
  if (batch == 0 || query_len == 0) return PA_OK;
  PA_CHECK_ARG(q && out && seq_lens && cur_lens, "pa_q4_attention: null q/out/seq_lens/cur_lens");
  if (max_pages > 0) {
    PA_CHECK_ARG(page_table != nullptr && pt_stride >= max_pages, "pa_q4_attention: page table missing or stride < max_pages");
    PA_CHECK_ARG(k_pool && v_pool && num_blocks > 0, "pa_q4_attention: KV pool missing or empty");
    PA_CHECK_ARG(((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15) == 0,
                 "pa_q4_attention: the pools must be 16-byte aligned");
  }
  PA_CHECK_ARG(max_pages <= (1 << 26) && (int64_t)query_len * (num_heads / kv_heads) <= (1 << 26) && kv_heads <= 65535 &&
                   batch <= 65535, "pa_q4_attention: sizes beyond the kernels' 32-bit indices");
  const Q4Plan p = q4_plan(io_dtype, batch, num_heads, kv_heads, query_len, head_dim, max_pages, weights != nullptr && max_pages > 0);
  PA_CHECK_ARG((int64_t)batch * kv_heads * p.tiles * p.splits <= 0x7fffffffLL &&
                   (int64_t)batch * kv_heads * (p.rows / 4 + 1 + max_pages / 16 + 1) <= 0x7fffffffLL,
               "pa_q4_attention: grid too large");
  if (p.bytes && (workspace == nullptr || workspace_bytes < p.bytes))
    PA_FAIL(PA_ERR_WORKSPACE, "pa_q4_attention: workspace too small: need %zu bytes, have %zu", p.bytes, workspace_bytes);
  PA_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "pa_q4_attention: the workspace must be 16-byte aligned");
  const int64_t elem = io_dtype == PA_DTYPE_F32 ? 4 : 2;
  const Q4Rows rows_q{{batch, num_heads, query_len}, {q_stride_b * elem, q_stride_h * elem, q_stride_t * elem}, head_dim * elem};
  const Q4Rows rows_out{{batch, num_heads, query_len}, {out_stride_b * elem, out_stride_h * elem, out_stride_t * elem},
                        head_dim * elem};
  PA_CHECK_ARG(!q4_rows_meet(q, rows_q, out, rows_out),
               "pa_q4_attention: out must not be q or overlap it (other rows, and a chunk's totals, read q after a row is written)");

  Q4Args a{};
  a.q = q; a.q_sb = q_stride_b; a.q_sh = q_stride_h; a.q_st = q_stride_t;
  a.out = out; a.o_sb = out_stride_b; a.o_sh = out_stride_h; a.o_st = out_stride_t;
  a.k_pool = static_cast<const uint8_t*>(k_pool); a.v_pool = static_cast<const uint8_t*>(v_pool);
  a.weights = max_pages > 0 ? weights : nullptr;
  a.num_blocks = num_blocks;
  a.page_table = page_table; a.pt_stride = pt_stride; a.max_pages = max_pages;
  a.seq_lens = seq_lens; a.cur_lens = cur_lens;
  a.B = batch; a.H = num_heads; a.Hk = kv_heads; a.group = num_heads / kv_heads; a.T = query_len;
  a.scale_log2 = scale * kLog2e;
  a.tiles = p.tiles; a.splits = p.splits; a.split_pages = p.split_pages;
  float* ws = static_cast<float*>(workspace);
  a.rec = p.splits > 1 ? ws : nullptr;
  a.lse = p.lse ? reinterpret_cast<f32x2*>(ws + p.rec) : nullptr;
  a.scores = p.scores ? ws + p.rec + p.lse : nullptr;
  a.score_stride = (int64_t)p.score_stride;
  float* ops = ws + p.rec + p.lse + p.scores;
  a.q_ops = p.ops && a.weights ? reinterpret_cast<f16x8*>(ops) : nullptr;
  a.q_aux = reinterpret_cast<f32x4*>(ops + p.ops);
  a.op_tiles = p.op_tiles;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const std::lock_guard<std::mutex> whole(pa_host::workspace_mutex(workspace));
  if (io_dtype == PA_DTYPE_F32) {
    if (head_dim == 64) launch_q4<float, 64, 2>(a, p, stream); else launch_q4<float, 128, 2>(a, p, stream);
  } else {
    if (head_dim == 64) launch_q4<uint16_t, 64, 1>(a, p, stream); else launch_q4<uint16_t, 128, 1>(a, p, stream);
  }
  PA_CHECK_LAUNCH("pa_q4_attention");
  return PA_OK;
}
