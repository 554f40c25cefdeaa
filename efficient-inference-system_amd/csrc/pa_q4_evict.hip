// Eviction from the 4-bit paged KV cache by accumulated attention weight (gfx950).
//
// Per (request, KV head) of n > keep cached keys: the newest `window` stay, and of the others the keep -
// window of the largest totals (equal totals: the lower index; NaN above every number, as torch's
// sort and argmax have it). The kept rows move, in their order and bit for bit, into the request's new
// pages, their totals with them. Two launches: the choice, a radix select over the totals with one
// workgroup per (request, head), and the move, one wavefront per new page.
#include "pa_q4.h"

namespace pa {

struct Q4EvictArgs {
  uint8_t* k_pool;
  uint8_t* v_pool;
  float* weights;
  int64_t num_blocks;
  const int32_t* page_table;
  int64_t pt_stride;
  int32_t max_pages;
  const int32_t* seq_lens;
  const int32_t* new_table;
  int64_t new_stride;
  int32_t new_pages;
  int32_t keep, window;
  int32_t* kept;      // [B, Hk, keep], -1 behind the last
  int32_t* new_lens;  // [B]
  int32_t B, Hk;
  int32_t held;       // totals that fit the choice's LDS
};

// Totals as unsigned words of the same order: NaN highest, -0 = +0; a key without a page is lowest.
__device__ __forceinline__ uint32_t q4_rank(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kSelHists = 8, kSelPitch = 257;  // 16k totals and these leave room for two workgroups a CU
constexpr int kSelHeld = 32768;  // totals in LDS (128 KB); longer requests read them from memory in every pass

__device__ __forceinline__ int wave_total(int x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// Inclusive sums over the lanes.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // row_shr:1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return x;
}

// The choice. Passes of 8 bits narrow the (keep - window)-th largest total down until 64 or fewer share its
// bits (two passes as a rule), which are compared with each other. Eight histograms for the lanes to take
// turns at: totals share their high bits, and a wavefront's 64 additions to one address run one after the
// other. Then each wavefront walks its contiguous part of the keys, the counts of the parts before it
// known, and writes the places of the kept ones in order. No atomics reach memory, so the choice is exact.
// 8 requests x 8 heads of 600 to 1000 keys 7.4 us, 16 x 32 heads of 2500 to 16384 keys 27.5 us (17 MB of totals
// in 64-byte pieces: 11 us of it): latency, of two dependent loads and of the passes' barriers. Four passes
// with a histogram per wavefront, which left 16k keys one workgroup a CU: 8.7 and 32.6 us.
__global__ __launch_bounds__(kSelThreads) void q4_choose_kernel(const Q4EvictArgs a) {
  extern __shared__ uint32_t held[];  // the first a.held totals
  __shared__ int hist[kSelHists][kSelPitch];
  __shared__ int sums[2][kSelWaves];
  __shared__ int counts[2][256];
  __shared__ uint32_t few[64];  // the totals left once there are so few
  __shared__ uint32_t found;
  __shared__ int few_count, found_want;
  const int hk = blockIdx.x % a.Hk, b = blockIdx.x / a.Hk;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t* table = a.page_table + (int64_t)b * a.pt_stride;
  int L = a.seq_lens[b];
  L = L < a.max_pages * kQ4Tokens ? L : a.max_pages * kQ4Tokens;
  L = L > 0 ? L : 0;
  const int count = L < a.keep ? L : a.keep;
  int32_t* kept = a.kept + ((int64_t)b * a.Hk + hk) * a.keep;
  for (int i = count + tid; i < a.keep; i += kSelThreads) kept[i] = -1;
  if (hk == 0 && tid == 0) a.new_lens[b] = count;
  if (L <= a.keep) {  // all stay
    for (int i = tid; i < L; i += kSelThreads) kept[i] = i;
    return;
  }
  const int cand = L - a.window;  // > 0: keep >= window
  auto total_at = [&](int t) -> uint32_t {
    const int id = q4_block(table[t / kQ4Tokens], a.num_blocks);
    return id < 0 ? 0u : q4_rank(a.weights[((int64_t)id * a.Hk + hk) * kQ4Tokens + (t & (kQ4Tokens - 1))]);
  };
  const int in_lds = cand < a.held ? cand : a.held;
  int want = a.keep - a.window;  // of the candidates
  uint32_t prefix = 0;
  int* const mine = hist[lane % kSelHists];
  for (int i = tid; i < kSelHists * kSelPitch; i += kSelThreads) (&hist[0][0])[i] = 0;
  __syncthreads();
  if (want > 0) {  // the totals come from memory, eight at a time on their way
    for (int t0 = tid; t0 < cand; t0 += 8 * kSelThreads) {
      int id[8];
      uint32_t u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = t0 + i * kSelThreads;
        id[i] = t < cand ? q4_block(table[t / kQ4Tokens], a.num_blocks) : -1;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        u[i] = id[i] < 0 ? 0u : q4_rank(a.weights[((int64_t)id[i] * a.Hk + hk) * kQ4Tokens + (t0 & (kQ4Tokens - 1))]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = t0 + i * kSelThreads;
        if (t < in_lds) held[t] = u[i];
        if (t < cand) atomicAdd(&mine[u[i] >> 24], 1);
      }
    }
  }
  for (int shift = 24, turn = 0; shift >= 0 && want > 0; shift -= 8, turn ^= 1) {
    const uint32_t seen = shift < 24 ? 0xffffffffu << (shift + 8) : 0u;
    if (shift < 24)
      for (int t = tid; t < cand; t += kSelThreads) {
        const uint32_t u = t < in_lds ? held[t] : total_at(t);
        if ((u & seen) == prefix) atomicAdd(&mine[u >> shift & 255], 1);
      }
    __syncthreads();
    if (tid < 256) {
      int n = 0;
#pragma unroll
      for (int w = 0; w < kSelHists; ++w) {
        n += hist[w][tid];
        hist[w][tid] = 0;  // for the next pass
      }
      counts[turn][255 - tid] = n;  // the highest digit first
    }
    if (tid == 0) few_count = 0;
    __syncthreads();
    // the digit where the count from above passes `want`: every wavefront finds it, four digits a lane
    int n[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      n[i] = counts[turn][4 * lane + i];
      sum += n[i];
    }
    int above = wave_scan(sum) - sum, digit = -1, left = 0, before = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (above < want && above + n[i] >= want) {
        digit = 255 - 4 * lane - i;
        before = above;
        left = n[i];
      }
      above += n[i];
    }
    const int at = __builtin_ctzll(__ballot(digit >= 0));  // (one lane: want is at most the candidates left)
    prefix |= (uint32_t)__builtin_amdgcn_readlane(digit, at) << shift;
    want -= __builtin_amdgcn_readlane(before, at);
    left = __builtin_amdgcn_readlane(left, at);
    if (left <= 64 && shift > 0) {  // each compared with all, four by every wavefront
      const uint32_t mask = 0xffffffffu << shift;
      for (int t = tid; t < cand; t += kSelThreads) {
        const uint32_t u = t < in_lds ? held[t] : total_at(t);
        if ((u & mask) == prefix) few[atomicAdd(&few_count, 1)] = u;
      }
      __syncthreads();
      const uint32_t u = lane < left ? few[lane] : 0u;
      for (int j = wave; j < left; j += kSelWaves) {
        const uint32_t it = __builtin_amdgcn_readlane(u, j);
        const int more = __popcll(__ballot(lane < left && u > it)), same = __popcll(__ballot(lane < left && u == it));
        if (more < want && more + same >= want && lane == 0) {  // (equal ones write the same)
          found = it;
          found_want = want - more;
        }
      }
      __syncthreads();
      prefix = found;
      want = found_want;
      break;
    }
  }
  auto rank = [&](int t) { return t < in_lds ? held[t] : total_at(t); };
  // kept: totals above `prefix`, and the first `want` equal to it (none where nothing was wanted)
  const bool any = a.keep > a.window;
  const int per = ((cand + kSelWaves - 1) / kSelWaves + 63) / 64 * 64;
  const int t0 = wave * per, t1 = t0 + per < cand ? t0 + per : cand;
  int gt = 0, eq = 0;
  if (any)
    for (int t = t0 + lane; t < t1; t += 64) {
      const uint32_t u = rank(t);
      gt += u > prefix;
      eq += u == prefix;
    }
  gt = wave_total(gt);
  eq = wave_total(eq);
  if (lane == 0) {
    sums[0][wave] = gt;
    sums[1][wave] = eq;
  }
  __syncthreads();
  int gt_before = 0, eq_before = 0;
  for (int w = 0; w < wave; ++w) {
    gt_before += sums[0][w];
    eq_before += sums[1][w];
  }
  if (any)
    for (int t = t0; t < t1; t += 64) {
      const bool in = t + lane < t1;
      const uint32_t u = in ? rank(t + lane) : 0u;
      const bool is_gt = in && u > prefix, is_eq = in && u == prefix;
      const uint64_t mg = __ballot(is_gt), me = __ballot(is_eq);
      const uint64_t below = (1ull << lane) - 1;
      const int g = gt_before + __popcll(mg & below), e = eq_before + __popcll(me & below);
      if (is_gt || (is_eq && e < want)) kept[g + (e < want ? e : want)] = t + lane;
      gt_before += __popcll(mg);
      eq_before += __popcll(me);
    }
  for (int i = tid; i < a.window; i += kSelThreads) kept[a.keep - a.window + i] = cand + i;
}

// The move: lane (g, c) = (lane / 16, lane % 16) takes the K words (c, g) and the V words (g, c) of the new
// page, from wherever each token was. A page's rows behind the last kept one stay as they were. Bound by
// memory: 16 x 32 heads x 128 cut to 2048 of up to 16384 keys, 337 MB read (163 MB of them kept: a token's V codes
// are halves of words that three neighbours share) and 155 MB written: 106 us, 4.6 TB/s, the rate of a copy.
template <int HD>
__global__ __launch_bounds__(256) void q4_move_kernel(const Q4EvictArgs a, int pages, uint32_t total) {
  constexpr int G = HD / kQ4Group, W = HD / 32, PB = q4_page_bytes(HD), CB = q4_codes_bytes(HD);
  const uint32_t x = blockIdx.x * 4u + (threadIdx.x >> 6);
  if (x >= total) return;
  const int hk = (int)(x % (uint32_t)a.Hk);
  const int p = (int)(x / (uint32_t)a.Hk % (uint32_t)pages), b = (int)(x / (uint32_t)a.Hk / (uint32_t)pages);
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int id = q4_block(a.new_table[(int64_t)b * a.new_stride + p], a.num_blocks);
  if (id < 0) return;
  const int at = p * kQ4Tokens + c;
  const int t = at < a.keep ? a.kept[((int64_t)b * a.Hk + hk) * a.keep + at] : -1;
  const int from = t >= 0 ? q4_block(a.page_table[(int64_t)b * a.pt_stride + t / kQ4Tokens], a.num_blocks) : -1;
  const int tok = t & (kQ4Tokens - 1);
  const int64_t head = (int64_t)hk * PB, stride = (int64_t)a.Hk * PB;
  const int64_t src = (int64_t)from * stride + head, dst = (int64_t)id * stride + head;
  // K: a token without a page moves as zeros
  uint32_t k[W];
  const uint32_t* ks = reinterpret_cast<const uint32_t*>(a.k_pool + src) + (tok * 4 + g) * W;
#pragma unroll
  for (int i = 0; i < W; ++i) k[i] = from >= 0 ? ks[i] : 0u;
  if (t >= 0) {
    uint32_t* kd = reinterpret_cast<uint32_t*>(a.k_pool + dst) + (c * 4 + g) * W;
    if constexpr (W == 4)
      *reinterpret_cast<u32x4*>(kd) = u32x4{k[0], k[1], k[2], k[3]};
    else
      *reinterpret_cast<u32x2*>(kd) = u32x2{k[0], k[1]};
  }
  // pairs and total
  if (t >= 0 && g < G) {
    const int so = CB + (g * kQ4Tokens + tok) * 4, to = CB + (g * kQ4Tokens + c) * 4;
    *reinterpret_cast<uint32_t*>(a.k_pool + dst + to) = from >= 0 ? *reinterpret_cast<const uint32_t*>(a.k_pool + src + so) : 0u;
    *reinterpret_cast<uint32_t*>(a.v_pool + dst + to) = from >= 0 ? *reinterpret_cast<const uint32_t*>(a.v_pool + src + so) : 0u;
  }
  if (t >= 0 && g == 3)
    a.weights[((int64_t)id * a.Hk + hk) * kQ4Tokens + c] =
        from >= 0 ? a.weights[((int64_t)from * a.Hk + hk) * kQ4Tokens + tok] : 0.f;
  // V: halves of tokens 4 g .. 4 g + 3
  uint32_t v[2][G];
  uint32_t ok = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int te = __shfl(t, 4 * g + e), fe = __shfl(from, 4 * g + e);
    const int ke = te & (kQ4Tokens - 1);
    // word p of the token's quadruple, both groups; its half is the token's
    const uint32_t* vs = reinterpret_cast<const uint32_t*>(a.v_pool + (int64_t)fe * stride + head) +
                         (((ke >> 2) * 16 + c) * 2 + (ke >> 1 & 1)) * G;
    uint32_t word[G];
    if (te >= 0 && fe >= 0) {
      if constexpr (G == 2) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(vs);
        word[0] = x[0];
        word[1] = x[1];
      } else {
        word[0] = vs[0];
      }
    } else {
#pragma unroll
      for (int i = 0; i < G; ++i) word[i] = 0;
    }
    ok |= (uint32_t)(te >= 0) << e;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const uint32_t w = ke & 1 ? word[i] >> 16 : word[i] & 0xffffu;
      v[e >> 1][i] = e & 1 ? v[e >> 1][i] | w << 16 : w;
    }
  }
  uint32_t* vd = reinterpret_cast<uint32_t*>(a.v_pool + dst) + (g * 16 + c) * 2 * G;
  if (ok == 15u) {
    if constexpr (G == 2)
      *reinterpret_cast<u32x4*>(vd) = u32x4{v[0][0], v[0][1], v[1][0], v[1][1]};
    else
      *reinterpret_cast<u32x2*>(vd) = u32x2{v[0][0], v[1][0]};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (ok >> e & 1)
#pragma unroll
        for (int i = 0; i < G; ++i)
          reinterpret_cast<uint16_t*>(vd)[((e >> 1) * G + i) * 2 + (e & 1)] = (uint16_t)(v[e >> 1][i] >> (e & 1 ? 16 : 0));
  }
}

}  // namespace pa

using namespace pa;

extern "C" int pa_q4_evict(void* k_pool, void* v_pool, float* weights, int64_t num_blocks,
                           const int32_t* page_table, int64_t pt_stride, int32_t max_pages, const int32_t* seq_lens,
                           const int32_t* new_page_table, int64_t new_pt_stride, int32_t new_max_pages,
                           int32_t keep, int32_t window, int32_t* kept, int32_t* new_seq_lens,
                           int32_t batch, int32_t kv_heads, int32_t head_dim, void* stream_) {
  pa_host::clear_error();
  PA_CHECK_ARG(batch >= 0 && kv_heads > 0 && max_pages >= 0 && new_max_pages >= 0 && num_blocks >= 0,
               "pa_q4_evict: bad sizes: batch=%d kv_heads=%d max_pages=%d new_max_pages=%d", batch, kv_heads, max_pages,
               new_max_pages);
  PA_CHECK_ARG(keep > 0 && window >= 0 && window <= keep, "pa_q4_evict: keep (%d) must be positive and hold the window (%d)",
               keep, window);
  if (head_dim != 64 && head_dim != 128)
    PA_FAIL(PA_ERR_UNSUPPORTED, "pa_q4_evict: no 4-bit pages for head_dim %d (64 and 128)", head_dim);
  PA_CHECK_ARG(max_pages <= (1 << 26) && keep <= (1 << 30), "pa_q4_evict: sizes beyond the kernels' 32-bit indices");
  if (batch == 0) return PA_OK;
  PA_CHECK_ARG(seq_lens && kept && new_seq_lens, "pa_q4_evict: null seq_lens, kept or new_seq_lens");
  const int64_t most = (int64_t)max_pages * kQ4Tokens < keep ? (int64_t)max_pages * kQ4Tokens : keep;
  PA_CHECK_ARG((int64_t)new_max_pages * kQ4Tokens >= most, "pa_q4_evict: %d new pages do not hold the %lld kept keys",
               new_max_pages, (long long)most);
  if (max_pages > 0) {
    PA_CHECK_ARG(k_pool && v_pool && weights && num_blocks > 0, "pa_q4_evict: pools or weights missing or empty");
    PA_CHECK_ARG(((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15) == 0,
                 "pa_q4_evict: the pools must be 16-byte aligned");
    PA_CHECK_ARG(page_table && pt_stride >= max_pages && new_page_table && new_pt_stride >= new_max_pages,
                 "pa_q4_evict: page table missing or stride below its width");
  }
  // what a workgroup writes, others still read
  const auto meet = [](const int32_t* x, int64_t nx, const int32_t* y, int64_t ny) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
    return a < b + 4 * (uintptr_t)ny && b < a + 4 * (uintptr_t)nx;
  };
  const int64_t n_kept = (int64_t)batch * kv_heads * keep, n_old = max_pages > 0 ? (batch - 1) * pt_stride + max_pages : 0,
                n_new = max_pages > 0 ? (batch - 1) * new_pt_stride + new_max_pages : 0;
  PA_CHECK_ARG(!meet(new_seq_lens, batch, seq_lens, batch) && !meet(new_seq_lens, batch, page_table, n_old) &&
                   !meet(new_seq_lens, batch, new_page_table, n_new) && !meet(new_seq_lens, batch, kept, n_kept) &&
                   !meet(kept, n_kept, seq_lens, batch) && !meet(kept, n_kept, page_table, n_old) &&
                   !meet(kept, n_kept, new_page_table, n_new),
               "pa_q4_evict: kept and new_seq_lens must not overlap each other, the lengths or the page tables");
  PA_CHECK_ARG(max_pages == 0 || page_table != new_page_table, "pa_q4_evict: the new pages must be none of the old ones");
  const int pages = (int)((most + kQ4Tokens - 1) / kQ4Tokens);
  PA_CHECK_ARG((int64_t)batch * kv_heads * (pages + 1) <= 0x7fffff00LL, "pa_q4_evict: grid too large");
  Q4EvictArgs a{};
  a.k_pool = static_cast<uint8_t*>(k_pool); a.v_pool = static_cast<uint8_t*>(v_pool); a.weights = weights;
  a.num_blocks = num_blocks; a.page_table = page_table; a.pt_stride = pt_stride; a.max_pages = max_pages;
  a.seq_lens = seq_lens; a.new_table = new_page_table; a.new_stride = new_pt_stride; a.new_pages = new_max_pages;
  a.keep = keep; a.window = window; a.kept = kept; a.new_lens = new_seq_lens; a.B = batch; a.Hk = kv_heads;
  const int64_t longest = (int64_t)max_pages * kQ4Tokens;
  a.held = (int32_t)(longest < kSelHeld ? longest : kSelHeld);
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const size_t lds = (size_t)a.held * sizeof(uint32_t);
  if (lds > (32u << 10)) {  // past the default limit of 64 KB with the static part
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(q4_choose_kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, kSelHeld * (int)sizeof(uint32_t));
    if (e != hipSuccess) PA_FAIL(PA_ERR_HIP, "pa_q4_evict: %s", hipGetErrorString(e));
  }
  q4_choose_kernel<<<(unsigned)(batch * kv_heads), kSelThreads, lds, stream>>>(a);
  PA_CHECK_LAUNCH("pa_q4_evict choice");
  if (pages > 0) {
    const uint32_t total = (uint32_t)((int64_t)batch * kv_heads * pages);
    if (head_dim == 64)
      q4_move_kernel<64><<<(total + 3) / 4, 256, 0, stream>>>(a, pages, total);
    else
      q4_move_kernel<128><<<(total + 3) / 4, 256, 0, stream>>>(a, pages, total);
    PA_CHECK_LAUNCH("pa_q4_evict move");
  }
  return PA_OK;
}
