// The 4-bit paged KV cache: rows quantised into their slots, slots read back as values (gfx950).
#include "pa_q4.h"

namespace pa {

struct Q4RowArgs {
  const void* k_new;  // append: rows in; read: rows out
  const void* v_new;
  int64_t sb, sh, st;
  uint8_t* k_pool;
  uint8_t* v_pool;
  float* weights;  // append: the slots' running totals, cleared; may be null
  int64_t num_blocks;
  const int32_t* slots;
  int32_t B, H, T;
};

// The row of a lane, HD / 8 lanes a row. CHUNK (calls of 16 tokens and more): a workgroup takes 256 / (HD / 8)
// consecutive tokens of one head, K and V, so that the row's place is scalar arithmetic but for the token,
// and a page, whose bytes interleave its tokens, is written by one workgroup or two. Otherwise (decode steps)
// rows follow each other, and K and V are the halves of the grid's y axis (in that order, with its divisions in
// every lane, 4 x 512 rows of 32 heads x 128 bf16 are read in 12.6 us, not 9.8).
struct Q4Row {
  int h, e;        // head, and which eight values
  uint32_t b, j;   // request and token; j >= T: no row
};
template <int HD, bool CHUNK>
__device__ __forceinline__ Q4Row q4_row_of(int H, int T) {
  constexpr uint32_t LPR = HD / 8, TOKENS = 256 / LPR;
  Q4Row r;
  r.e = (int)(threadIdx.x % LPR);
  if constexpr (CHUNK) {
    uint32_t x = blockIdx.x;
    r.h = (int)(x % (uint32_t)H);
    x /= (uint32_t)H;
    const uint32_t groups = ((uint32_t)T + TOKENS - 1) / TOKENS;
    r.b = x / groups;
    r.j = (x - r.b * groups) * TOKENS + threadIdx.x / LPR;
  } else {
    uint32_t x = (blockIdx.x * 256u + threadIdx.x) / LPR;
    r.h = (int)(x % (uint32_t)H);
    x /= (uint32_t)H;
    r.b = x / (uint32_t)T;
    r.j = x - r.b * (uint32_t)T;
  }
  return r;
}

// Eight lanes share a group of 64 values, lane i of them values 8 i .. 8 i + 7: the eight of one K
// word, and two n-quadruples of V.
template <int HD>
__device__ __forceinline__ void q4_row_place(int h, int H, int64_t blk, int tok, int e, uint32_t& kw, uint32_t& vw,
                                             uint32_t& meta, int64_t& page) {
  constexpr int G = HD / kQ4Group, W = HD / 32;
  page = (blk * H + h) * q4_page_bytes(HD);
  const int w = e >> 2, g = e & 3;               // values 8 e = 32 w + 8 g of the row
  kw = (uint32_t)((tok * 4 + g) * W + w) * 4u;   // byte of the K word
  const int a = e >> 3, r = (e & 7) * 2;         // V: group a, quadruples r and r + 1
  vw = (uint32_t)((((tok >> 2) * 16 + r) * 2 + ((tok >> 1) & 1)) * G + a) * 4u + (uint32_t)(tok & 1) * 2u;
  meta = (uint32_t)q4_codes_bytes(HD) + (uint32_t)(a * kQ4Tokens + tok) * 4u;
}

template <typename T>
__device__ __forceinline__ void q4_load8(const T* p, bool vec, float (&x)[8]) {
  if (vec) {
    constexpr int V = 8 * (int)sizeof(T) / 16;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const u32x4 w = reinterpret_cast<const u32x4*>(p)[i];
      float f[Vec16<T>::EPL];
      Vec16<T>::unpack(w, f);
#pragma unroll
      for (int j = 0; j < Vec16<T>::EPL; ++j) x[i * Vec16<T>::EPL + j] = f[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = Elem<T>::load(p + j);
  }
}

// The codes of a lane's eight values: (x - z) / s + 7.5 of fp64 to the nearest, ties to even, in 0..15, formed as
// x / s + (7.5 - z / s) in one fma a value. Where the quotient is below 16 the fp32 value is within
// 2.5e-6 + |z / s| 2^-24 of the real one (8 x 2^-23 of the reciprocal, 2^-24 each of the sum, below 16, and
// of its constant), so it decides unless it lies that close (taken twice as wide) to a border between two
// codes. Larger quotients are clamped whatever their error. Next to a border x - z = m s exactly is a tie,
// which fp32 proves (half the groups of eight rows of bf16 hold one); what is left, about one value in
// 10^5 of fp32 rows whose centre is a few steps at most, is divided in fp64.
__device__ __forceinline__ void q4_codes(const float (&x)[8], float z, float s, uint32_t (&c)[8]) {
  const float rs = __builtin_amdgcn_rcpf(s), mid = fmaf(-z, rs, 7.5f);
  float y[8], far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = fmaf(x[i], rs, mid);
    const float n = rintf(y[i]);
    far = fmaxf(far, fabsf(y[i] - n));
    c[i] = (uint32_t)(int)__builtin_amdgcn_fmed3f(n, 0.f, 15.f);
  }
  const float sure = 0.5f - fmaf(fabsf(mid), 0x1p-23f, 6e-6f);
  if (__builtin_expect(far > sure, 0)) {
    bool hard = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (fabsf(y[i] - rintf(y[i])) <= sure) continue;
      const float below = floorf(y[i]), d = x[i] - z, dx = d - x[i];
      const float lost = (x[i] - (d - dx)) - (z + dx);  // d's rounding error
      const bool tie = lost == 0.f && fmaf(7.f - below, s, d) == 0.f;
      c[i] = tie ? (uint32_t)(int)__builtin_amdgcn_fmed3f(2.f * rintf(0.5f * below + 0.25f), 0.f, 15.f) : c[i];
      hard |= !tie;
    }
    if (__builtin_expect(hard, 0)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double d = ((double)x[i] - (double)z) / (double)s + 7.5;
        c[i] = (uint32_t)(int)fmin(fmax(rint(d), 0.0), 15.0);
      }
    }
  }
}

// Scale and centre of a group. The products round to fp32 before they round to halves: left to itself the
// compiler forms product and conversion as one v_fma_mixlo_f16, which rounds once, and a scale next to a
// border differs.
__device__ __forceinline__ void q4_pair_of(float hi, float lo, _Float16& s, _Float16& z) {
  float sf = (hi - lo) * (float)(1.0 / 15.0), zf = (hi + lo) * 0.5f;
  asm("" : "+v"(sf), "+v"(zf));
  s = (_Float16)sf;
  z = (_Float16)zf;
}

// One row's eight values of K or V into its slot: per group s = half((hi - lo) / 15), z = half((hi + lo) / 2) of
// the values clamped to half's range, then the codes.
template <int HD>
__device__ __forceinline__ void q4_put(uint8_t* p, float (&x)[8], bool is_v, int e, uint32_t kw, uint32_t vw, uint32_t meta) {
  float odd = 0.f;  // NaN where a value is NaN (or infinite)
#pragma unroll
  for (int i = 0; i < 8; ++i) odd = fmaf(x[i], 0.f, odd);
  float hi = x[0], lo = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    hi = fmaxf(hi, x[i]);
    lo = fminf(lo, x[i]);
  }
  bool nan = false;
  if (__builtin_expect(!(odd == 0.f && hi <= 65504.f && lo >= -65504.f), 0)) {
    hi = -65504.f;
    lo = 65504.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      nan |= x[i] != x[i];
      x[i] = x[i] != x[i] ? 0.f : __builtin_amdgcn_fmed3f(x[i], -65504.f, 65504.f);
      hi = fmaxf(hi, x[i]);
      lo = fminf(lo, x[i]);
    }
  }
  hi = group_max<8>(nan ? INFINITY : hi);  // a group with a NaN: (NaN, NaN)
  lo = -group_max<8>(-lo);
  _Float16 sh, zh;
  q4_pair_of(hi, lo, sh, zh);
  const bool bad = hi == INFINITY;
  const float s = (float)sh, z = (float)zh;
  uint32_t c[8];
  if (bad || !(s > 0.f)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = 0;
  } else {
    q4_codes(x, z, s, c);
  }
  if (!is_v) {
    *reinterpret_cast<uint32_t*>(p + kw) = c[0] | c[2] << 4 | c[4] << 8 | c[6] << 12 | c[1] << 16 | c[3] << 20 |
                                           c[5] << 24 | c[7] << 28;
  } else {
    constexpr int G = HD / kQ4Group;
    *reinterpret_cast<uint16_t*>(p + vw) = (uint16_t)(c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12);
    *reinterpret_cast<uint16_t*>(p + vw + 8 * G) = (uint16_t)(c[4] | c[5] << 4 | c[6] << 8 | c[7] << 12);
  }
  if ((e & 7) == 0) {
    const uint32_t su = bad ? 0x7e00u : (uint32_t)__builtin_bit_cast(uint16_t, sh);
    uint32_t zu = bad ? 0x7e00u : (uint32_t)__builtin_bit_cast(uint16_t, zh);
    zu = zu == 0x8000u ? 0u : zu;  // a centre of zero is +0, whatever zeros the row holds
    *reinterpret_cast<uint32_t*>(p + meta) = su | zu << 16;
  }
}

// Quantising append. 4 x 512 rows of 32 heads x 128 bf16, 43 MB: 14.8 us, 2.9 TB/s, bound by the 390 vector
// instructions that a wavefront's 1024 values take (10.5 us); with fp64 for every tie 19.9. A decode step is
// latency (8 rows of 8 heads x 64: 2.5 us).
template <typename T, int HD, bool CHUNK>
__global__ __launch_bounds__(256) void q4_append_kernel(const Q4RowArgs a, uint32_t total, int vec) {
  if (!CHUNK && blockIdx.x * 256u + threadIdx.x >= total) return;  // (whole rows: 8 or 16 lanes each)
  const Q4Row at = q4_row_of<HD, CHUNK>(a.H, a.T);
  if (CHUNK && at.j >= (uint32_t)a.T) return;
  const int h = at.h, e = at.e;
  const int32_t slot = a.slots[at.b * (uint32_t)a.T + at.j];
  const int64_t src = (int64_t)at.b * a.sb + (int64_t)h * a.sh + (int64_t)at.j * a.st + 8 * e;
  const bool first_v = !CHUNK && blockIdx.y != 0;
  float x[2][8];
  q4_load8(static_cast<const T*>(first_v ? a.v_new : a.k_new) + src, vec, x[0]);
  if constexpr (CHUNK) q4_load8(static_cast<const T*>(a.v_new) + src, vec, x[1]);
  if (slot < 0) return;
  const int64_t blk = (uint32_t)slot / kQ4Tokens;
  if (blk >= a.num_blocks) return;
  const int tok = slot & (kQ4Tokens - 1);
  uint32_t kw, vw, meta;
  int64_t page;
  q4_row_place<HD>(h, a.H, blk, tok, e, kw, vw, meta, page);
  q4_put<HD>((first_v ? a.v_pool : a.k_pool) + page, x[0], first_v, e, kw, vw, meta);
  if constexpr (CHUNK) q4_put<HD>(a.v_pool + page, x[1], true, e, kw, vw, meta);
  if (!first_v && e == 0 && a.weights != nullptr) a.weights[(blk * a.H + h) * kQ4Tokens + tok] = 0.f;
}

// One row's eight values of K or V, z + s (c - 7.5) rounded once to T.
template <typename T, int HD>
__device__ __forceinline__ void q4_get(const uint8_t* p, T* out, bool there, bool is_v, uint32_t kw, uint32_t vw, uint32_t meta) {
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (there) {
    uint32_t c;  // nibble i: value i
    if (!is_v) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(p + kw);
      c = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) c |= (w >> (4 * ((i >> 1) + 4 * (i & 1))) & 15u) << (4 * i);
    } else {
      constexpr int G = HD / kQ4Group;
      c = (uint32_t)*reinterpret_cast<const uint16_t*>(p + vw) |
          (uint32_t)*reinterpret_cast<const uint16_t*>(p + vw + 8 * G) << 16;
    }
    const uint32_t m = *reinterpret_cast<const uint32_t*>(p + meta);
    const float s = q4_scale(m), z = q4_centre(m);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf(s, (float)(c >> (4 * i) & 15u) - 7.5f, z);
  }
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<f32x4*>(out)[0] = f32x4{x[0], x[1], x[2], x[3]};
    reinterpret_cast<f32x4*>(out)[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<u32x4*>(out) = w;
  }
}

// The values that slots stand for; rows without a slot are zeros. Bound by memory: 4 x 512 rows of 32 heads x
// 128 bf16, 43 MB: 9.8 us, 4.4 TB/s.
template <typename T, int HD, bool CHUNK>
__global__ __launch_bounds__(256) void q4_read_kernel(const Q4RowArgs a, uint32_t total) {
  if (!CHUNK && blockIdx.x * 256u + threadIdx.x >= total) return;
  const Q4Row at = q4_row_of<HD, CHUNK>(a.H, a.T);
  if (CHUNK && at.j >= (uint32_t)a.T) return;
  const int32_t slot = a.slots[at.b * (uint32_t)a.T + at.j];
  const int64_t blk = (uint32_t)slot / kQ4Tokens;
  const bool there = slot >= 0 && blk < a.num_blocks;
  uint32_t kw, vw, meta;
  int64_t page;
  q4_row_place<HD>(at.h, a.H, there ? blk : 0, slot & (kQ4Tokens - 1), at.e, kw, vw, meta, page);
  const int64_t dst = (int64_t)at.b * a.sb + (int64_t)at.h * a.sh + (int64_t)at.j * a.st + 8 * at.e;
  const bool first_v = !CHUNK && blockIdx.y != 0;
  q4_get<T, HD>((first_v ? a.v_pool : a.k_pool) + page, static_cast<T*>(const_cast<void*>(first_v ? a.v_new : a.k_new)) + dst,
                there, first_v, kw, vw, meta);
  if constexpr (CHUNK) q4_get<T, HD>(a.v_pool + page, static_cast<T*>(const_cast<void*>(a.v_new)) + dst, there, true, kw, vw, meta);
}

// Workgroups of a call in either order.
constexpr int kChunkTokens = 16;
static int64_t row_workgroups(int32_t B, int32_t T, int32_t H, int32_t HD) {
  const int per = 256 / (HD / 8);  // rows of a workgroup
  return T >= kChunkTokens ? (int64_t)B * ((T + per - 1) / per) * H : ((int64_t)B * T * H + per - 1) / per;
}

template <typename T, int HD>
static void launch_append(const Q4RowArgs& a, int vec, hipStream_t stream) {
  const unsigned n = (unsigned)row_workgroups(a.B, a.T, a.H, HD);
  if (a.T >= kChunkTokens)
    q4_append_kernel<T, HD, true><<<n, 256, 0, stream>>>(a, 0, vec);
  else
    q4_append_kernel<T, HD, false><<<dim3(n, 2), 256, 0, stream>>>(a, (uint32_t)((int64_t)a.B * a.T * a.H * (HD / 8)), vec);
}

template <typename T, int HD>
static void launch_read(const Q4RowArgs& a, hipStream_t stream) {
  const unsigned n = (unsigned)row_workgroups(a.B, a.T, a.H, HD);
  if (a.T >= kChunkTokens)
    q4_read_kernel<T, HD, true><<<n, 256, 0, stream>>>(a, 0);
  else
    q4_read_kernel<T, HD, false><<<dim3(n, 2), 256, 0, stream>>>(a, (uint32_t)((int64_t)a.B * a.T * a.H * (HD / 8)));
}

static int check_rows(const char* what, const void* k, const void* v, int dtype, const void* k_pool, const void* v_pool,
                      int64_t num_blocks, const int32_t* slots, int32_t batch, int32_t heads, int32_t rows,
                      int32_t head_dim, bool& empty) {
  PA_CHECK_ARG(batch >= 0 && rows >= 0 && heads > 0 && num_blocks >= 0, "%s: bad sizes: batch=%d rows=%d heads=%d", what,
               batch, rows, heads);
  PA_CHECK_ARG(dtype == PA_DTYPE_F32 || dtype == PA_DTYPE_BF16, "%s: bad dtype %d", what, dtype);
  if (head_dim != 64 && head_dim != 128) PA_FAIL(PA_ERR_UNSUPPORTED, "%s: no 4-bit pages for head_dim %d (64 and 128)", what, head_dim);
  empty = batch == 0 || rows == 0;
  if (empty) return PA_OK;
  PA_CHECK_ARG(k && v && slots, "%s: null rows or slots", what);
  PA_CHECK_ARG(num_blocks == 0 || (k_pool && v_pool), "%s: null pool", what);
  PA_CHECK_ARG(((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15) == 0,
               "%s: the pools must be 16-byte aligned", what);
  PA_CHECK_ARG((int64_t)batch * rows <= 0x7fffffffLL && row_workgroups(batch, rows, heads, head_dim) <= 0x7fffff00LL / 256,
               "%s: too many rows in one call", what);
  return PA_OK;
}

}  // namespace pa

using namespace pa;

extern "C" size_t pa_q4_page_bytes(int32_t head_dim) {
  return head_dim == 64 || head_dim == 128 ? (size_t)q4_page_bytes(head_dim) : 0;
}

extern "C" int pa_q4_append(const void* k_new, const void* v_new, int64_t new_stride_b, int64_t new_stride_h,
                            int64_t new_stride_t, int new_dtype, void* k_pool, void* v_pool, int64_t num_blocks,
                            float* weights, const int32_t* slot_mapping, int32_t batch, int32_t kv_heads,
                            int32_t query_len, int32_t head_dim, void* stream) {
  pa_host::clear_error();
  bool empty = false;
  if (const int st = check_rows("pa_q4_append", k_new, v_new, new_dtype, k_pool, v_pool, num_blocks, slot_mapping, batch,
                                kv_heads, query_len, head_dim, empty))
    return st;
  if (empty || num_blocks == 0) return PA_OK;
  Q4RowArgs a{k_new, v_new, new_stride_b, new_stride_h, new_stride_t, static_cast<uint8_t*>(k_pool),
              static_cast<uint8_t*>(v_pool), weights, num_blocks, slot_mapping, batch, kv_heads, query_len};
  const int64_t per = new_dtype == PA_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
  const int vec = ((reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new)) & 15) == 0 &&
                  new_stride_b % per == 0 && new_stride_h % per == 0 && new_stride_t % per == 0;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (new_dtype == PA_DTYPE_F32)
    head_dim == 64 ? launch_append<float, 64>(a, vec, st) : launch_append<float, 128>(a, vec, st);
  else
    head_dim == 64 ? launch_append<uint16_t, 64>(a, vec, st) : launch_append<uint16_t, 128>(a, vec, st);
  PA_CHECK_LAUNCH("pa_q4_append");
  return PA_OK;
}

extern "C" int pa_q4_read(const void* k_pool, const void* v_pool, int64_t num_blocks, const int32_t* slot_mapping,
                          void* k_out, void* v_out, int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_t,
                          int out_dtype, int32_t batch, int32_t kv_heads, int32_t query_len, int32_t head_dim,
                          void* stream) {
  pa_host::clear_error();
  bool empty = false;
  if (const int st = check_rows("pa_q4_read", k_out, v_out, out_dtype, k_pool, v_pool, num_blocks, slot_mapping, batch,
                                kv_heads, query_len, head_dim, empty))
    return st;
  if (empty) return PA_OK;
  const int64_t per = out_dtype == PA_DTYPE_F32 ? 4 : 8;
  PA_CHECK_ARG(((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) == 0 &&
                   out_stride_b % per == 0 && out_stride_h % per == 0 && out_stride_t % per == 0,
               "pa_q4_read: the outputs must start, and their rows follow each other, at multiples of 16 bytes");
  Q4RowArgs a{k_out, v_out, out_stride_b, out_stride_h, out_stride_t, static_cast<uint8_t*>(const_cast<void*>(k_pool)),
              static_cast<uint8_t*>(const_cast<void*>(v_pool)), nullptr, num_blocks, slot_mapping, batch, kv_heads, query_len};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (out_dtype == PA_DTYPE_F32)
    head_dim == 64 ? launch_read<float, 64>(a, st) : launch_read<float, 128>(a, st);
  else
    head_dim == 64 ? launch_read<uint16_t, 64>(a, st) : launch_read<uint16_t, 128>(a, st);
  PA_CHECK_LAUNCH("pa_q4_read");
  return PA_OK;
}
