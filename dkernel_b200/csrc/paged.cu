// Paged K/V cache: a step's bookkeeping, cache writes, committed branches, and the CUDA-core form of the
// attention (the tcgen05 form is in paged_sm100.cu).  Semantics: include/bsa.h.
#include <algorithm>

#include "paged.cuh"

namespace bsa {
namespace {

// ------------------------------------------------------------------ a step's tables
// Bound by latency: a few dependent loads.  One cluster makes the tables: each CTA scans all requests (a few loads per
// thread; a scan spread over CTAs would cost the exchange of its sums instead) and keeps offsets in shared memory; pages
// are then shared out.  The barrier between pushing surplus pages and popping missing ones is the cluster's own, so a
// step is one launch, with the slots of up to 4096 tokens (16 requests, 88 tokens: 4.6 us).  Slots of more tokens are a
// second launch over the whole machine (768 requests, 230 thousand tokens: 9.9 us; by the one cluster 33).
constexpr int kStepThreads = 1024;

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// inclusive scan over the block's threads; total = sum of all
__device__ __forceinline__ long long block_scan(long long x, long long* warp_sums, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += up;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    long long s = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += up;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  x += warp ? warp_sums[warp - 1] : 0;
  *total = warp_sums[kStepThreads / 32 - 1];
  __syncthreads();
  return x;
}

// Slots and positions of the step's tokens, by the warp `w` of `warps`, U tokens of a lane at a time.  The 32 * U tokens of
// a warp are consecutive: the requests of its first and last one bound the others' searches, to nothing where one request
// has them all.  page(b, i): page i of request b.
constexpr int kStepTokens = 4096;      // up to so many the tables' kernel does them itself
template <typename F>
__device__ __forceinline__ void step_tokens(const bsa_paged_step_params& p, const int* cu, int w, int warps, int lane, F page) {
  constexpr int U = 4;
  const int B = p.batch, P = p.page_size, T = p.max_tokens, real = cu[B];
  auto request_of = [&](int t, int lo, int hi) {     // cu[b] <= t < cu[b + 1] with lo <= b < hi
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
  };
  const int per = T <= 32 * warps ? 1 : U;           // few tokens: spread over the warps
  for (int tw = w * (32 * per); tw < T; tw += warps * (32 * per)) {
    const int b_first = tw < real ? request_of(tw, 0, B) : 0;
    const int b_last = tw < real ? request_of(min(tw + 32 * per, real) - 1, b_first, B) + 1 : 1;
    long long slot[U];
    int pos[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = tw + u * 32 + lane;
      slot[u] = -1;
      pos[u] = 0;
      if (u < per && t < real) {
        const int b = request_of(t, b_first, b_last), i = t - cu[b];
        const long long ctx = max(__ldg(p.context_lens + b), 0), at = ctx + i;
        // tokens past 2^31 have no page: a table holds fewer
        const int pi = at > 0x7fffffffll ? 0x7fffffff : (int)at / P, pg = page(b, pi);
        if (pg >= 0) slot[u] = (long long)pg * P + ((int)at - pi * P);
        int depth = i;
        if (p.tree_mask) depth = draft_depth((uint64_t)__ldg(p.tree_mask + t) & low_bits(cu[b + 1] - cu[b]), i);
        pos[u] = (int)min(ctx + depth, 0x7fffffffll);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = tw + u * 32 + lane;
      if (u < per && t < T) {
        p.slots[t] = slot[u];
        p.positions[t] = pos[u];
      }
    }
  }
}

// The same for many tokens, over the whole machine, from the finished tables.
__global__ void __launch_bounds__(256) paged_slots_kernel(const bsa_paged_step_params p) {
  extern __shared__ int slots_smem[];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int b = threadIdx.x; b <= p.batch; b += 256) slots_smem[b] = p.cu_seqlen_q[b];
  __syncthreads();
  step_tokens(p, slots_smem, blockIdx.x * 8 + (threadIdx.x >> 5), gridDim.x * 8, threadIdx.x & 31, [&](int b, int pi) {
    return pi < p.page_counts[b] ? p.block_tables[(int64_t)b * p.table_stride + pi] : -1;
  });
}

__global__ void __launch_bounds__(kStepThreads) paged_step_kernel(bsa_paged_step_params p, int ctas) {
  extern __shared__ int step_smem[];
  __shared__ long long warp_sums[32];
  const int B = p.batch, P = p.page_size, W = p.max_pages;
  const int T = p.max_tokens;
  int* cu = step_smem;            // [B + 1]
  int* held = cu + B + 1;         // [B] pages before the step
  int* target = held + B;         // [B] pages after it
  int* off = target + B;          // [B] first push (target < held) or first pop
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int n_free = min(max(*p.num_free, 0), p.free_capacity);     // this and the counts are written below: no __ldg
  long long new_before = 0, moved_before = 0;
  if (tid == 0) cu[0] = 0;
  for (int b0 = 0; b0 < B; b0 += kStepThreads) {
    const int b = b0 + tid;
    const int want = b < B ? max(__ldg(p.new_lens + b), 0) : 0;
    const int ctx = b < B ? max(__ldg(p.context_lens + b), 0) : 0;
    const int h = b < B ? min(max(p.page_counts[b], 0), W) : 0;
    long long total;
    const long long incl = block_scan(want, warp_sums, &total) + new_before;
    const int c1 = (int)min(incl, (long long)T), c0 = (int)min(incl - want, (long long)T);
    const long long len = (long long)ctx + (c1 - c0);
    const int tg = b < B ? (int)min((len + P - 1) / P, (long long)W) : 0;
    // pushes in the low half, pops in the high half: W * B < 2^31 is checked by the host
    const long long moved = tg < h ? (long long)(h - tg) : (long long)(tg - h) << 32;
    long long total2;
    const long long mincl = block_scan(moved, warp_sums, &total2) + moved_before;
    if (b < B) {
      cu[b + 1] = c1;
      held[b] = h;
      target[b] = tg;
      off[b] = tg < h ? (int)((mincl - moved) & 0xffffffffll) : (int)((mincl - moved) >> 32);
      if (rank == 0) {
        p.cu_seqlen_q[b + 1] = c1;
        p.seqlens[b] = (int)min(len, 0x7fffffffll);
      }
    }
    new_before += total;
    moved_before += total2;
  }
  __syncthreads();
  const int pushes = (int)(moved_before & 0xffffffffll), pops = (int)(moved_before >> 32);
  if (rank == 0 && tid == 0) p.cu_seqlen_q[0] = 0;

  // surplus pages go on the stack, a warp per request
  const int warps = ctas * (kStepThreads / 32);
  if (pushes)
    for (int b = rank * (kStepThreads / 32) + warp; b < B; b += warps)
      for (int i = target[b] + lane; i < held[b]; i += 32) {
        const long long at = (long long)n_free + off[b] + i - target[b];
        int32_t* entry = p.block_tables + (int64_t)b * p.table_stride + i;
        if (at < p.free_capacity) p.free_pages[at] = *entry;
        *entry = -1;
      }
  if (ctas > 1) cluster_sync_all(); else __syncthreads();

  const int avail = (int)min((long long)n_free + pushes, (long long)p.free_capacity);
  // page `nth` (in the order of request and page) of the missing ones; not through the read-only cache, the
  // stack has just been written
  auto popped = [&](int nth) { return nth < avail ? *(volatile int32_t*)(p.free_pages + (avail - 1 - nth)) : -1; };
  if (pops)
    for (int b = rank * (kStepThreads / 32) + warp; b < B; b += warps)
      for (int i = held[b] + lane; i < target[b]; i += 32)
        p.block_tables[(int64_t)b * p.table_stride + i] = popped(off[b] + i - held[b]);
  if (rank == 0) {
    for (int b = tid; b < B; b += kStepThreads) {
      // written where it stays, too: a count outside [0, W] has been clamped, and the slots' kernel reads it here
      const int h = held[b], tg = target[b];
      p.page_counts[b] = tg <= h ? tg : h + min(max(avail - off[b], 0), tg - h);
    }
    if (tid == 0) {
      *p.num_free = max(avail - pops, 0);
      *p.short_pages = max(pops - avail, 0);
    }
  }

  if (p.max_tokens <= kStepTokens)
    step_tokens(p, cu, rank * (kStepThreads / 32) + warp, ctas * (kStepThreads / 32), lane, [&](int b, int pi) {
      if (pi >= target[b]) return -1;
      return pi < held[b] ? *(volatile int32_t*)(p.block_tables + (int64_t)b * p.table_stride + pi)
                          : popped(off[b] + pi - held[b]);
    });
  if (ctas > 1) cluster_sync_all();   // no CTA leaves while another may still need the cluster's barrier
}

// ------------------------------------------------------------------ cache writes
// n / d for n < 2^31 by a multiplication (Granlund and Montgomery): a thread's index arithmetic costs less than its 32 bytes.
struct FastDiv {
  uint32_t d, m;
  int s;
  explicit FastDiv(uint32_t x) : d(x), s(0) {
    while ((1ull << s) < x) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - x)) / x + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

// x / scale, correctly rounded, from the correctly rounded reciprocal (Markstein: one residual step); where the
// quotient is too large for the residual it is past e4m3's end anyway, and too small below its half step.  A true
// division: k * (1 / scale) alone would decide ties the other way now and then.  (IEEE division took 92 of the 149 us
// of 65000 tokens x 8 heads x 128.)
__device__ __forceinline__ float quotient(float x, float scale, float rcp) {
  const float q = x * rcp;
  const float r = fmaf(fmaf(-q, scale, x), rcp, q);
  return fabsf(q) < 1e30f ? r : q;
}
template <typename T> __device__ __forceinline__ uint16_t to_e4m3x2(T x, T y, float scale, float rcp, bool divide) {
  float2 f;
  f.x = Elem<T>::to_f(x);
  f.y = Elem<T>::to_f(y);
  if (divide) {
    f.x = __fdiv_rn(f.x, scale);
    f.y = __fdiv_rn(f.y, scale);
  } else {
    f.x = quotient(f.x, scale, rcp);
    f.y = quotient(f.y, scale, rcp);
  }
  return (uint16_t)__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
}

// Both caches in one grid: blockIdx.y = 0 for K, 1 for V.  Bound by HBM: each element is read and written once.  A
// thread moves VEC elements (16 bytes of the cache, or of the input where that is wider, if everything is aligned; else
// one), 64 bytes at a time so that enough loads are in flight; consecutive threads are consecutive in (token, head, dim).
// 65000 tokens x 8 heads x 128 from bf16 into e4m3: 80 us, 5.0 TB/s (119 with 124 registers, two CTAs per SM; 84 to 100
// with more CTAs than are resident).
template <typename T, typename C, int VEC>
__global__ void __launch_bounds__(256, 4) paged_write_kernel(const __grid_constant__ bsa_paged_write_params p, const FastDiv per_token,
                                                          const FastDiv pieces, const FastDiv page, uint32_t total) {
  constexpr int kIn = VEC * (int)sizeof(T), kOut = VEC * (int)sizeof(C);
  constexpr int U = kIn > 16 ? 2 : 4;
  const bool is_v = blockIdx.y != 0;
  const T* src = static_cast<const T*>(is_v ? p.v : p.k);
  C* dst = static_cast<C*>(is_v ? p.v_cache : p.k_cache);
  const int64_t st = is_v ? p.v_st : p.k_st, sh = is_v ? p.v_sh : p.k_sh;
  const int64_t cp = is_v ? p.vc_sp : p.kc_sp, cs = is_v ? p.vc_ss : p.kc_ss, ch = is_v ? p.vc_sh : p.kc_sh;
  const float scale = is_v ? p.v_scale : p.k_scale, rcp = __frcp_rn(scale);
  const bool divide = !(rcp >= 1.17549435e-38f && rcp < INFINITY);      // a reciprocal that is no normal number
  const int64_t slots = (int64_t)p.num_pages * p.page_size;
  for (uint64_t x0 = (uint64_t)blockIdx.x * (256 * U) + threadIdx.x; x0 < total; x0 += (uint64_t)gridDim.x * (256 * U)) {
    int64_t slot[U];
    uint32_t tok[U], head[U], el[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t x = x0 + u * 256;
      slot[u] = -1;
      if (x < total) {
        tok[u] = per_token.div((uint32_t)x);
        const uint32_t rem = (uint32_t)x - tok[u] * per_token.d;
        head[u] = pieces.div(rem);
        el[u] = (rem - head[u] * pieces.d) * VEC;
        slot[u] = __ldg(p.slots + tok[u]);
        if (slot[u] >= slots) slot[u] = -1;
      }
    }
    alignas(16) T in[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (slot[u] < 0) continue;
      const T* s = src + (int64_t)tok[u] * st + (int64_t)head[u] * sh + el[u];
      if constexpr (VEC == 1) in[u][0] = *s;
      else
#pragma unroll
        for (int i = 0; i < kIn / 16; ++i) reinterpret_cast<uint4*>(in[u])[i] = __ldcs(reinterpret_cast<const uint4*>(s) + i);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (slot[u] < 0) continue;
      const int64_t pg = slot[u] < 0x7fffffffll ? (int64_t)page.div((uint32_t)slot[u]) : slot[u] / p.page_size;
      C* o = dst + pg * cp + (slot[u] - pg * p.page_size) * cs + (int64_t)head[u] * ch + el[u];
      if constexpr (VEC == 1) {
        if constexpr (sizeof(C) == 1) *o = (uint8_t)to_e4m3x2<T>(in[u][0], in[u][0], scale, rcp, divide);
        else *o = in[u][0];
      } else if constexpr (sizeof(C) == 1) {
        alignas(16) uint16_t out[VEC / 2];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) out[i] = to_e4m3x2<T>(in[u][2 * i], in[u][2 * i + 1], scale, rcp, divide);
        *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(out);
      } else {
#pragma unroll
        for (int i = 0; i < kOut / 16; ++i) reinterpret_cast<uint4*>(o)[i] = reinterpret_cast<const uint4*>(in[u])[i];
      }
    }
  }
}

// ------------------------------------------------------------------ committed branches
// Bound by latency, too: branch and block table are known after three dependent loads, the moves are one more (64 trees:
// 5.5 us).  CTA (x, request): its threads own V-byte pieces of a token's K and V rows.  Draft numbers on a branch ascend,
// so the r-th is at least r: token L + r is written when every branch token that was there has been read.
template <typename V>
__global__ void __launch_bounds__(256) paged_commit_kernel(bsa_paged_commit_params p, int elem_bytes) {
  const int b = blockIdx.y;
  const int t0 = min(max(__ldg(p.cu_q + b), 0), p.total_q);
  const int n = min(max(__ldg(p.cu_q + b + 1) - t0, 0), p.total_q - t0);
  const int a = __ldg(p.accepted + b), L = max(__ldg(p.context_lens + b), 0);
  const bool any = a >= 0 && a < n && (!p.tree_mask || a < 64);
  uint64_t word = 0;
  if (any && p.tree_mask) {
    word = ((uint64_t)__ldg(p.tree_mask + t0 + a) & low_bits(n)) | 1ull << a;
  }
  const int count = !any ? 0 : p.tree_mask ? __popcll(word) : a + 1;
  if (blockIdx.x == 0 && threadIdx.x == 0) p.new_context_lens[b] = (int)min((long long)L + count, 0x7fffffffll);
  if (!p.tree_mask || !any) return;   // a chain is in place already
  const int stay = __ffsll((long long)~word) - 1;   // the first drafts 0, 1, ... are, too (-1: all 64)
  if (stay < 0 || stay >= count) return;
  const int32_t* table = p.block_tables + (int64_t)b * p.table_stride;
  const int pieces = p.d * elem_bytes / (int)sizeof(V), per_cache = p.hkv * pieces;
  for (int x = blockIdx.x * 256 + threadIdx.x; x < 2 * per_cache; x += gridDim.x * 256) {
    const bool is_v = x >= per_cache;
    const int y = is_v ? x - per_cache : x, h = y / pieces, c = y - h * pieces;
    char* base = static_cast<char*>(is_v ? p.v_cache : p.k_cache);
    const int64_t sp = is_v ? p.vc_sp : p.kc_sp, ss = is_v ? p.vc_ss : p.kc_ss, sh = is_v ? p.vc_sh : p.kc_sh;
    // unsigned: L + 63 may pass 2^31, and a negative page would be looked up in front of the table
    auto place = [&](uint32_t at) -> V* {
      const uint32_t pi = at / (uint32_t)p.page_size;
      const int pg = page_of(table, pi, p.max_pages, p.num_pages);
      if (pg < 0) return nullptr;
      return reinterpret_cast<V*>(base + ((int64_t)pg * sp + (int64_t)(at - pi * (uint32_t)p.page_size) * ss + (int64_t)h * sh) * elem_bytes) + c;
    };
    uint64_t left = word & ~low_bits(stay);
    int r = stay;
    while (left) {
      // four at a time: their loads are in flight together
      V val[4];
      const V* src[4];
      int m = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        src[i] = nullptr;
        if (!left) continue;
        src[i] = place((uint32_t)L + (uint32_t)(__ffsll((long long)left) - 1));
        left &= left - 1;
        if (src[i]) val[i] = *src[i];
        ++m;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i >= m) continue;
        V* dst = place((uint32_t)L + (uint32_t)(r + i));
        if (src[i] && dst) *dst = val[i];
      }
      r += m;
    }
  }
}

// ------------------------------------------------------------------ attention on the CUDA cores
template <typename T, typename C>
__global__ void __launch_bounds__(256) paged_rows_kernel(bsa_paged_params p) {
  const int64_t x = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (x >= (int64_t)p.total_q * p.hq) return;
  const int t = (int)(x / p.hq), h = (int)(x % p.hq);
  int b = t;
  if (p.cu_q) {
    if (t < __ldg(p.cu_q) || t >= __ldg(p.cu_q + p.batch)) return;
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(p.cu_q + mid) <= t) lo = mid; else hi = mid;
    }
    b = lo;
  }
  if (b >= p.batch) return;
  const PagedRequest r = paged_request(p, b);
  if (t - r.t0 >= r.n) return;
  paged_row<T, C>(p, b, r, t - r.t0, h, lane);
}

bool known_dtype(int t) { return t == BSA_F16 || t == BSA_BF16 || t == BSA_F32; }

int validate_paged(const bsa_paged_params* p, const char* who) {
  BSA_CHECK_ARG(p, "%s: null params", who);
  BSA_CHECK_ARG(p->q && p->o && ((p->k_cache && p->v_cache) || p->num_pages == 0), "%s: null tensor pointer", who);
  BSA_CHECK_ARG(p->crow && p->col, "%s: null layout pointer", who);
  BSA_CHECK_ARG((p->block_tables || p->max_pages == 0) && p->seqlens, "%s: null block table or lengths", who);
  BSA_CHECK_ARG(p->batch >= 0 && p->hq >= 1 && p->hkv >= 1 && p->d >= 1 && p->total_q >= 0 && p->max_pages >= 0 &&
                    p->page_size >= 1 && p->num_pages >= 0,
                "%s: bad shape batch=%d hq=%d hkv=%d d=%d total_q=%d max_pages=%d page_size=%d num_pages=%d", who,
                p->batch, p->hq, p->hkv, p->d, p->total_q, p->max_pages, p->page_size, p->num_pages);
  BSA_CHECK_ARG(p->hq % p->hkv == 0, "%s: hq=%d is not a multiple of hkv=%d", who, p->hq, p->hkv);
  BSA_CHECK_ARG(p->h_pat == 1 || p->h_pat == p->hkv || p->h_pat == p->hq,
                "%s: pattern has %d heads, expected 1, %d or %d", who, p->h_pat, p->hkv, p->hq);
  const int bs = p->block_size;
  BSA_CHECK_ARG(bs >= 16 && bs <= 128 && (bs & (bs - 1)) == 0,
                "%s: block_size must be a power of two in [16,128], got %d", who, bs);
  BSA_CHECK_ARG(known_dtype(p->dtype), "%s: unknown dtype %d", who, p->dtype);
  BSA_CHECK_ARG(p->kv_dtype == p->dtype || (p->kv_dtype == BSA_F8E4M3 && p->dtype != BSA_F32),
                "%s: the cache has q's type, or is e4m3 under f16/bf16 queries", who);
  BSA_CHECK_ARG(p->cu_q || p->total_q == p->batch, "%s: without cu_q there is one query token per request", who);
  return BSA_OK;
}

template <typename T>
int launch_rows(const bsa_paged_params* p, cudaStream_t s) {
  const int64_t rows = (int64_t)p->total_q * p->hq, grid = (rows + 7) / 8;
  if (grid > 0x7fffffffLL) {
    set_error("bsa_paged_fwd: too many rows for one launch");
    return BSA_E_TOOBIG;
  }
  if (p->kv_dtype == BSA_F8E4M3) {
    if constexpr (sizeof(T) == 2) paged_rows_kernel<T, uint8_t><<<(unsigned)grid, 256, 0, s>>>(*p);
  } else {
    paged_rows_kernel<T, T><<<(unsigned)grid, 256, 0, s>>>(*p);
  }
  return check_launch("paged_rows_kernel");
}

template <typename T, typename C, int VEC>
int launch_write_vec(const bsa_paged_write_params* p, cudaStream_t s) {
  const int64_t per_token = (int64_t)p->hkv * (p->d / VEC), total = per_token * p->tokens;
  if (total > 0x7fffffffLL) {
    set_error("bsa_paged_write: %d tokens of %d heads x %d are too many for one call", p->tokens, p->hkv, p->d);
    return BSA_E_TOOBIG;
  }
  const int64_t per_cta = 256 * (VEC * sizeof(T) > 16 ? 2 : 4);
  const unsigned grid = (unsigned)std::min<int64_t>((total + per_cta - 1) / per_cta, 148 * 2);   // all resident
  paged_write_kernel<T, C, VEC><<<dim3(grid, 2), 256, 0, s>>>(*p, FastDiv((uint32_t)per_token), FastDiv(p->d / VEC),
                                                               FastDiv(p->page_size), (uint32_t)total);
  return check_launch("paged_write_kernel");
}

template <typename T, typename C>
int launch_write(const bsa_paged_write_params* p, cudaStream_t s) {
  constexpr int V = 16 / sizeof(C);      // 16 bytes stored, as many or more read
  const int64_t in[] = {p->k_st, p->k_sh, p->v_st, p->v_sh};
  const int64_t out[] = {p->kc_sp, p->kc_ss, p->kc_sh, p->vc_sp, p->vc_ss, p->vc_sh};
  bool wide = p->d % V == 0 && reinterpret_cast<uintptr_t>(p->k) % 16 == 0 && reinterpret_cast<uintptr_t>(p->v) % 16 == 0 &&
              reinterpret_cast<uintptr_t>(p->k_cache) % 16 == 0 && reinterpret_cast<uintptr_t>(p->v_cache) % 16 == 0;
  for (int64_t x : in) wide = wide && x * (int64_t)sizeof(T) % 16 == 0;
  for (int64_t x : out) wide = wide && x % V == 0;
  return wide ? launch_write_vec<T, C, V>(p, s) : launch_write_vec<T, C, 1>(p, s);
}
}  // namespace
}  // namespace bsa

using namespace bsa;

extern "C" {

int bsa_paged_step(const bsa_paged_step_params* p, void* stream) {
  BSA_CHECK_ARG(p, "bsa_paged_step: null params");
  BSA_CHECK_ARG(p->cu_seqlen_q && p->num_free && p->short_pages, "bsa_paged_step: null pointer");
  BSA_CHECK_ARG(p->batch >= 0 && p->max_pages >= 0 && p->free_capacity >= 0 && p->page_size >= 1 && p->max_tokens >= 0,
                "bsa_paged_step: bad shape batch=%d max_pages=%d free_capacity=%d page_size=%d max_tokens=%d", p->batch,
                p->max_pages, p->free_capacity, p->page_size, p->max_tokens);
  BSA_CHECK_ARG(p->batch == 0 || (p->block_tables && p->page_counts && p->context_lens && p->new_lens && p->seqlens),
                "bsa_paged_step: null pointer");
  BSA_CHECK_ARG((p->free_capacity == 0 || p->free_pages) && (p->max_tokens == 0 || (p->slots && p->positions)),
                "bsa_paged_step: null pointer");
  if (p->batch > BSA_PAGED_STEP_MAX_BATCH || (int64_t)p->batch * p->max_pages > 0x7fffffffLL) {
    set_error("bsa_paged_step: %d requests of %d pages; at most %d requests and 2^31 table entries", p->batch, p->max_pages,
              BSA_PAGED_STEP_MAX_BATCH);
    return BSA_E_TOOBIG;
  }
  const size_t smem = (size_t)(4 * p->batch + 1) * sizeof(int);
  BSA_CHECK_CUDA(cudaFuncSetAttribute(paged_step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const int ctas = p->max_tokens + 16 * (int64_t)p->batch > 4 * kStepThreads ? 8 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kStepThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BSA_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_step_kernel, *p, ctas));
  if (p->max_tokens <= kStepTokens) return check_launch("paged_step_kernel");
  cfg.gridDim = dim3((unsigned)std::min(296, cdiv_i(p->max_tokens, 1024)));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = (size_t)(p->batch + 1) * sizeof(int);
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  BSA_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_slots_kernel, *p));
  return check_launch("paged_slots_kernel");
}

int bsa_paged_write(const bsa_paged_write_params* p, void* stream) {
  BSA_CHECK_ARG(p, "bsa_paged_write: null params");
  BSA_CHECK_ARG(p->tokens >= 0 && p->hkv >= 1 && p->d >= 1 && p->page_size >= 1 && p->num_pages >= 0,
                "bsa_paged_write: bad shape tokens=%d hkv=%d d=%d page_size=%d num_pages=%d", p->tokens, p->hkv, p->d,
                p->page_size, p->num_pages);
  BSA_CHECK_ARG(known_dtype(p->dtype), "bsa_paged_write: unknown dtype %d", p->dtype);
  BSA_CHECK_ARG(p->cache_dtype == p->dtype || p->cache_dtype == BSA_F8E4M3,
                "bsa_paged_write: the cache has k's type or is e4m3");
  BSA_CHECK_ARG(p->cache_dtype != BSA_F8E4M3 || (p->k_scale > 0.f && p->v_scale > 0.f),
                "bsa_paged_write: an e4m3 cache needs positive scales");
  if (p->tokens == 0 || p->num_pages == 0) return BSA_OK;
  BSA_CHECK_ARG(p->k && p->v && p->k_cache && p->v_cache && p->slots, "bsa_paged_write: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f8 = p->cache_dtype == BSA_F8E4M3;
  switch (p->dtype) {
    case BSA_F16: return f8 ? launch_write<__half, uint8_t>(p, s) : launch_write<__half, __half>(p, s);
    case BSA_BF16: return f8 ? launch_write<__nv_bfloat16, uint8_t>(p, s) : launch_write<__nv_bfloat16, __nv_bfloat16>(p, s);
    default: return f8 ? launch_write<float, uint8_t>(p, s) : launch_write<float, float>(p, s);
  }
}

int bsa_paged_commit(const bsa_paged_commit_params* p, void* stream) {
  BSA_CHECK_ARG(p, "bsa_paged_commit: null params");
  BSA_CHECK_ARG(p->batch >= 0 && p->hkv >= 1 && p->d >= 1 && p->total_q >= 0 && p->max_pages >= 0 && p->page_size >= 1 &&
                    p->num_pages >= 0,
                "bsa_paged_commit: bad shape batch=%d hkv=%d d=%d total_q=%d max_pages=%d page_size=%d num_pages=%d",
                p->batch, p->hkv, p->d, p->total_q, p->max_pages, p->page_size, p->num_pages);
  BSA_CHECK_ARG(known_dtype(p->cache_dtype) || p->cache_dtype == BSA_F8E4M3, "bsa_paged_commit: unknown dtype %d",
                p->cache_dtype);
  if (p->batch == 0) return BSA_OK;
  BSA_CHECK_ARG(((p->k_cache && p->v_cache) || p->num_pages == 0) && (p->block_tables || p->max_pages == 0) && p->context_lens && p->cu_q && p->accepted &&
                    p->new_context_lens, "bsa_paged_commit: null pointer");
  if (p->batch > 65535) {
    set_error("bsa_paged_commit: at most 65535 requests");
    return BSA_E_TOOBIG;
  }
  const int eb = p->cache_dtype == BSA_F8E4M3 ? 1 : (int)dtype_size(p->cache_dtype);
  const int64_t strides[] = {p->kc_sp, p->kc_ss, p->kc_sh, p->vc_sp, p->vc_ss, p->vc_sh};
  bool wide = p->d * eb % 16 == 0 && reinterpret_cast<uintptr_t>(p->k_cache) % 16 == 0 &&
              reinterpret_cast<uintptr_t>(p->v_cache) % 16 == 0;
  for (int64_t x : strides) wide = wide && x * eb % 16 == 0;
  const int vb = wide ? 16 : eb;
  const int64_t pieces = (int64_t)2 * p->hkv * (p->d * eb / vb);
  const dim3 grid((unsigned)std::min<int64_t>((pieces + 255) / 256, 64), p->batch);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (wide) paged_commit_kernel<uint4><<<grid, 256, 0, s>>>(*p, eb);
  else if (eb == 4) paged_commit_kernel<uint32_t><<<grid, 256, 0, s>>>(*p, eb);
  else if (eb == 2) paged_commit_kernel<uint16_t><<<grid, 256, 0, s>>>(*p, eb);
  else paged_commit_kernel<uint8_t><<<grid, 256, 0, s>>>(*p, eb);
  return check_launch("paged_commit_kernel");
}

size_t bsa_paged_workspace_bytes(const bsa_paged_params* p) {
  const char* why = nullptr;
  if (validate_paged(p, "bsa_paged_workspace_bytes") || p->impl == BSA_IMPL_GENERIC || !paged_sm100_supported(p, &why)) return 0;
  return paged_sm100_workspace(p);
}

const char* bsa_paged_why_not_sm100(const bsa_paged_params* p) {
  if (validate_paged(p, "bsa_paged_why_not_sm100")) return last_error();
  const char* why = nullptr;
  return paged_sm100_supported(p, &why) ? nullptr : why;
}

int bsa_paged_fwd(const bsa_paged_params* p, void* stream) {
  int rc = validate_paged(p, "bsa_paged_fwd");
  if (rc) return rc;
  if (p->batch == 0 || p->total_q == 0) return BSA_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->impl != BSA_IMPL_GENERIC) {
    const char* why = nullptr;
    if (paged_sm100_supported(p, &why)) {
      BSA_CHECK_ARG(p->ws && reinterpret_cast<uintptr_t>(p->ws) % 256 == 0,
                    "bsa_paged_fwd: needs a workspace of bsa_paged_workspace_bytes(), 256-byte aligned");
      return paged_sm100(p, s);
    }
    if (p->impl == BSA_IMPL_SM100) {
      set_error("bsa_paged_fwd: the tcgen05 kernel does not serve this call: %s", why);
      return BSA_E_UNSUPPORTED;
    }
  }
  if (p->d > 256) {
    set_error("bsa_paged_fwd: head dim %d is above 256", p->d);
    return BSA_E_UNSUPPORTED;
  }
  switch (p->dtype) {
    case BSA_F16: return launch_rows<__half>(p, s);
    case BSA_BF16: return launch_rows<__nv_bfloat16>(p, s);
    default: return launch_rows<float>(p, s);
  }
}

}  // extern "C"
