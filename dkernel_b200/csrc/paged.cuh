// Paged K/V cache: what the attention kernels share.  A request's query and key ranges, page look-ups,
// and one attention row on the CUDA cores, straight from the definition in include/bsa.h.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace bsa {

// first query row, drafted tokens, context tokens; false: nothing is stored, whatever pages the block table names
struct PagedRequest { int t0, n, L; bool stored = true; };

// Query rows stay inside [0, total_q) whatever cu_q holds.  A request that stores nothing has rows that attend nothing
// (batches are padded with such requests); one that stores some tokens, but fewer than it queries, counts as one without
// context.
// Tables, lengths and mask words are loaded as data that may have changed since the launch (no __ldg): the tensor-core
// kernel may be resident before the step's kernel in front of it has written them.
__device__ __forceinline__ PagedRequest paged_request(const bsa_paged_params& p, int b) {
  PagedRequest r;
  if (p.cu_q) {
    r.t0 = min(max(p.cu_q[b], 0), p.total_q);
    r.n = min(max(p.cu_q[b + 1] - r.t0, 0), p.total_q - r.t0);
  } else {
    r.t0 = b;
    r.n = 1;
  }
  const int stored = p.seqlens[b];
  r.stored = stored > 0;
  r.L = max(stored - r.n, 0);
  return r;
}

__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : (1ull << n) - 1ull; }

// The drafts (of the n of its request) that draft i attends, as far as a word can name them.
__device__ __forceinline__ uint64_t draft_word(const bsa_paged_params& p, const PagedRequest& r, int i) {
  return (uint64_t)p.tree_mask[r.t0 + i] & low_bits(r.n);
}
__device__ __forceinline__ int draft_depth(uint64_t word, int i) {
  return __popcll(i < 64 ? word & ~(1ull << i) : word);
}

// Page of logical token s, or -1.
__device__ __forceinline__ int page_of(const int32_t* table, int64_t page_index, int max_pages, int num_pages) {
  if (page_index >= max_pages) return -1;
  const int pg = table[page_index];
  return pg >= 0 && pg < num_pages ? pg : -1;
}

template <typename T> __device__ __forceinline__ float cache_to_f(T x) { return Elem<T>::to_f(x); }
template <> __device__ __forceinline__ float cache_to_f<uint8_t>(uint8_t x) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(x, __NV_E4M3)));
}

// Query row t0 + i of head h, by one warp: 32 keys at a time, one per lane for the logits, then the head dim
// over the lanes for the products with V.  Only attended keys are touched.  T: q, o; C: the cache.
// This is every row of the calls that the tensor-core kernel does not serve, and the rows that it cannot finish:
// where P V meets an infinity or NaN, a weight of 0 no longer leaves a row alone.
template <typename T, typename C>
__device__ __noinline__ void paged_row(const bsa_paged_params& p, int b, PagedRequest r, int i, int h, int lane) {
  constexpr int kDims = 8;   // head dims up to 256
  const int kvh = h / (p.hq / p.hkv), d = p.d, bs = p.block_size;
  const T* q = static_cast<const T*>(p.q) + (int64_t)(r.t0 + i) * p.q_st + (int64_t)h * p.q_sh;
  const C* kc = static_cast<const C*>(p.k_cache) + (int64_t)kvh * p.kc_sh;
  const C* vc = static_cast<const C*>(p.v_cache) + (int64_t)kvh * p.vc_sh;
  const int32_t* table = p.block_tables + (int64_t)b * p.table_stride;
  const bool tree = p.tree_mask != nullptr;
  const uint64_t word = tree ? draft_word(p, r, i) : 0ull;
  const int pos = r.L + (tree ? draft_depth(word, i) : i);
  const int hp = pattern_head(h, p.h_pat, p.hq, p.hkv);
  const int32_t* crow = p.crow + (int64_t)hp * p.crow_sh;
  const int32_t* cols = p.col + (int64_t)hp * p.col_sh;
  const int row = pos / bs;
  const int c_beg = row < p.n_rows ? __ldg(crow + row) : 0, c_end = row < p.n_rows ? __ldg(crow + row + 1) : 0;
  const bool fp8 = sizeof(C) == 1;
  const float scale2 = p.sm_scale * (fp8 ? p.k_scale : 1.f) * kLog2e;

  float m = -INFINITY, l = 0.f, acc[kDims];
#pragma unroll
  for (int x = 0; x < kDims; ++x) acc[x] = 0.f;
  // keys s (one per lane); those that count are attended
  auto keys = [&](int64_t s, bool on) {
    int64_t vrow = 0;
    float x = -INFINITY;
    if (on) {
      const int pg = page_of(table, s / p.page_size, r.stored ? p.max_pages : 0, p.num_pages);
      on = pg >= 0;
      if (on) {
        const int slot = (int)(s % p.page_size);
        const C* kr = kc + (int64_t)pg * p.kc_sp + (int64_t)slot * p.kc_ss;
        vrow = (int64_t)pg * p.vc_sp + (int64_t)slot * p.vc_ss;
        float dot = 0.f;
        for (int e = 0; e < d; ++e) dot = fmaf(Elem<T>::to_f(q[e]), cache_to_f<C>(kr[e]), dot);
        x = dot * scale2;
      }
    }
    float mx = x;
    bool nan = on && x != x;
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    nan = __any_sync(0xffffffffu, nan);
    const float m_new = nan ? NAN : fmaxf(m, mx);
    uint32_t live = __ballot_sync(0xffffffffu, on);
    if (!live || m_new == -INFINITY) return;
    const float alpha = m == -INFINITY ? 0.f : exp2f(m - m_new);
    const float w = on ? exp2f(x - m_new) : 0.f;
    float sum = w;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = l * alpha + sum;
    m = m_new;
#pragma unroll
    for (int x2 = 0; x2 < kDims; ++x2) acc[x2] *= alpha;
    while (live) {
      const int src = __ffs(live) - 1;
      live &= live - 1;
      const float ws = __shfl_sync(0xffffffffu, w, src);
      const C* vr = vc + __shfl_sync(0xffffffffu, vrow, src);
#pragma unroll
      for (int x2 = 0; x2 < kDims; ++x2)
        if (lane + 32 * x2 < d) acc[x2] = fmaf(ws, cache_to_f<C>(vr[lane + 32 * x2]), acc[x2]);
    }
  };
  // columns ascend, so the drafts' membership test can search
  auto has = [&](int c) {
    int lo = c_beg, hi = c_end;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(cols + mid) < c) lo = mid + 1; else hi = mid;
    }
    return lo < c_end && __ldg(cols + lo) == c;
  };
  for (int c = c_beg; c < c_end; ++c) {
    const int64_t s0 = (int64_t)__ldg(cols + c) * bs;
    if (s0 < 0) continue;
    if (s0 >= r.L) break;
    for (int k = 0; k < bs; k += 32) {
      const int64_t s = s0 + k + lane;
      if (s0 + k < r.L) keys(s, k + lane < bs && s < r.L);
    }
  }
  for (int j0 = 0; j0 < r.n; j0 += 32) {
    const int j = j0 + lane;
    bool on = j < r.n;
    if (on) on = tree ? j < 64 && ((word >> j) & 1ull) : j <= i;
    if (on) on = has((r.L + (tree ? draft_depth(draft_word(p, r, j), j) : j)) / bs);
    keys((int64_t)r.L + j, on);
  }
  const float inv = (l == 0.f ? 0.f : 1.f / l) * (fp8 ? p.v_scale : 1.f);
  T* o = static_cast<T*>(p.o) + (int64_t)(r.t0 + i) * p.o_st + (int64_t)h * p.o_sh;
#pragma unroll
  for (int x = 0; x < kDims; ++x)
    if (lane + 32 * x < d) o[lane + 32 * x] = Elem<T>::from_f(l == 0.f ? 0.f : acc[x] * inv);
  if (p.lse && lane == 0)
    p.lse[(int64_t)h * p.lse_sh + r.t0 + i] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

bool paged_sm100_supported(const bsa_paged_params* p, const char** why);
size_t paged_sm100_workspace(const bsa_paged_params* p);
int paged_sm100(const bsa_paged_params* p, cudaStream_t s);

}  // namespace bsa
