// Attention of drafted tokens over a paged K/V cache on the tcgen05 tensor cores (f16 / bf16 queries; cache of
// their type or e4m3; head dims that are multiples of 8, 16 for e4m3, up to 128; pattern blocks of 16, 32 or 64
// tokens; pages of a power of two of tokens, 8 or more).  Semantics: include/bsa.h.
//
// What bounds it: every attended K/V byte of a (request, kv head) has to come from HBM once.  A row tile is 128
// rows = the drafted tokens x the q heads of a kv group; an ITEM is up to two tiles, so that a tree of 64 tokens in
// groups of 4 heads reads its keys once.  The items' pattern blocks are shared out over one persistent CTA per SM in
// equal pieces, whatever the requests' lengths: a CTA's piece may begin and end inside an item, whose partial results
// a second kernel then joins.  Two groups of four softmax warps: with two tiles each takes its own, with one they
// take the K/V tiles in turn and add up in shared memory.
//
// A K/V tile is 64 tokens = 1, 2 or 4 pattern blocks, wherever their pages are: one TMA box per page piece.
// Warps (384 threads, 512 with an e4m3 cache): 0-7 softmax and epilogue, 8 TMA producer, 9 and 10 MMA issuers of the
// two groups, 11 planner, 12-15 e4m3 -> 16-bit.  TMEM: S[group][2] 4x64 | O[group] 2x128 columns.
#include "ptx.cuh"
#include "paged.cuh"

namespace bsa {
namespace {

constexpr int kCtas = 148;            // most CTAs of a launch; sizes the workspace
constexpr int kSeg = 64;              // pattern blocks that a plan lists
constexpr int kPagesPerEntry = 8;
constexpr uint32_t kTailFlag = 1u << 31;
constexpr uint32_t kColMask = (1u << 23) - 1u;   // bits 23..30: pages that exist
constexpr int kOverhead = 2;          // an item's fixed cost in K/V tiles
constexpr int kMinTiles = 2;          // least work of a CTA in K/V tiles
constexpr float kRescale = 8.0f;
constexpr int kWProd = 8, kWIssue0 = 9, kWPlan = 11;

// How rows and items are cut; the same for the whole launch.
struct PagedShape {
  int gt;          // q heads of a group that a tile holds
  int chunks;      // pieces of a group
  int tt;          // tokens of a tile
  int shared;      // these heads have equal pattern rows
  int rows_cap;    // rows of a partial result
  int page_shift, box;
  int ctas;
};

// The item that a CTA begins and others finish; written by every CTA, valid = 0 where there is none.
struct PagedRec { int valid, b, kvh, chunk, tile, last; int pad[2]; };

struct PPlan {
  int valid, first, last, two, part;
  int n, nt, tile0;            // listed blocks, K/V tiles, K/V tiles of the item before this plan
  int b, t0, n_new, L, kvh, head0, gcnt;
  int tok0, ntok, Lp, r0, Sp;  // Lp: keys before it are context for every row of the item; r0 = Lp / block; Sp: end of its keys
  uint32_t tb[32];             // by pattern row: which of the blocks r0, r0 + 1, ... it has
  uint64_t dm[8];              // drafts whose position lies in block r0 + y
  uint32_t col[kSeg], fl[kSeg];
  int page[kSeg * kPagesPerEntry];
};

template <int D, bool KV8> struct PGeo {
  static constexpr int kSub = D / 64;
  static constexpr int kQTile = 128 * D * 2;
  static constexpr int kTile = 64 * D * 2;
  static constexpr int kSlots = KV8 ? (D == 64 ? 4 : 2) : (D == 64 ? 8 : 4);   // 16-bit K slots, and V slots
  static constexpr int kRawTile = 64 * D;
  static constexpr int kRaw = KV8 ? (D == 64 ? 8 : 4) : 1;                     // e4m3 K slots, and V slots
  static constexpr int kRawBytes = KV8 ? 2 * kRaw * kRawTile : 0;
  static constexpr size_t kFixed = 1024 + 2 * kQTile + 2 * kSlots * kTile + kRawBytes;
  static constexpr int kThreads = KV8 ? 512 : 384;
};

template <int NS, int NR> struct PTail {
  uint64_t plan_full[2], plan_free[2], q_full, q_free;
  uint64_t k_full[NS], v_full[NS], k_free[NS], v_free[NS];
  uint64_t raw_k_full[NR], raw_v_full[NR], raw_k_free[NR], raw_v_free[NR];
  uint64_t qk_done[2][2], p_full[2][2], pv_done[2][2], o_free[2], mrg_full, mrg_free;
  uint32_t tmem_base;
  int start_e;
  long long start_base, warp_sums[16];
  uint32_t window[kSeg];
  PPlan plan[2];
  float mrg_ml[2][128];
  alignas(16) float mrg[32 * 128];           // one tile's 32 columns, [column][row]
  alignas(16) uint8_t ostage[4][2048];       // 32 rows x 64 bytes per warp; group 1 stages in mrg
};

__device__ __forceinline__ float pex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pmax3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
template <bool BF16> __device__ __forceinline__ uint32_t ppack2(float lo, float hi) {
  if (BF16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}
// two e4m3 -> two 16-bit values, exactly
template <bool BF16> __device__ __forceinline__ uint32_t e4m3x2_to_16(uint16_t x) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(x));
  if (BF16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&b);
  }
  return h;
}

// ------------------------------------------------------------------ items and their weights
__device__ __forceinline__ int item_count(const PagedShape& sh, int n) { return (n + 2 * sh.tt - 1) / (2 * sh.tt); }

// Where an item's keys lie.  In a tree every row sees the same context; in a chain the tokens before the item are
// context for all its rows.
struct ItemKeys { int Lp, Sp, r0; };
__device__ __forceinline__ ItemKeys item_keys(const bsa_paged_params& p, const PagedShape& sh, const PagedRequest& r, int tile) {
  ItemKeys k;
  const int tok0 = tile * 2 * sh.tt;
  k.Lp = p.tree_mask ? r.L : r.L + tok0;
  k.Sp = p.tree_mask ? r.L + r.n : r.L + min(r.n, tok0 + 2 * sh.tt);
  k.r0 = k.Lp / p.block_size;
  return k;
}

// Units of work of an item: blocks of its first head's first pattern row, blocks that hold its drafts, and a fixed
// cost.  An estimate where rows differ; shares are cut in its proportion.
__device__ __forceinline__ int item_weight(const bsa_paged_params& p, const PagedShape& sh, const PagedRequest& r, int kvh,
                                           int chunk, int tile) {
  const ItemKeys k = item_keys(p, sh, r, tile);
  const int hp = pattern_head(kvh * (p.hq / p.hkv) + chunk * sh.gt, p.h_pat, p.hq, p.hkv);
  const int32_t* cr = p.crow + (int64_t)hp * p.crow_sh;
  const int len = k.r0 < p.n_rows ? __ldg(cr + k.r0 + 1) - __ldg(cr + k.r0) : 0;
  return max(len, 0) + (k.Sp - 1) / p.block_size - k.r0 + 1 + kOverhead * (64 / p.block_size);
}
__device__ __forceinline__ long long request_weight(const bsa_paged_params& p, const PagedShape& sh, int e) {
  const PagedRequest r = paged_request(p, e / p.hkv);
  long long w = 0;
  const int nt = item_count(sh, r.n);
  for (int c = 0; c < sh.chunks; ++c)
    for (int t = 0; t < nt; ++t) w += item_weight(p, sh, r, e % p.hkv, c, t);
  return w;
}

// unit u belongs to the CTA c with U c / C <= u < U (c + 1) / C
__device__ __forceinline__ int owner_of(long long u, long long U, int C) { return (int)(((u + 1) * C - 1) / U); }

// ------------------------------------------------------------------ the kernel
// P is kept as the sum of two 16-bit terms side by side in S's columns, as in the decode and the long packed kernels:
// no precision hangs on which weights a 16-bit type holds exactly.
template <bool BF16, int D, int BS, bool KV8>
__global__ void __launch_bounds__(PGeo<D, KV8>::kThreads, 1)
paged_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ Tmap4 tmK, const __grid_constant__ Tmap4 tmV,
                  const __grid_constant__ bsa_paged_params p, const PagedShape sh, PagedRec* __restrict__ recs,
                  float2* __restrict__ part_ml, float* __restrict__ part_o, int* wait_status) {
  using Geo = PGeo<D, KV8>;
  using T16 = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  using C8 = typename std::conditional<KV8, uint8_t, T16>::type;
  constexpr int kSub = Geo::kSub, NS = Geo::kSlots, NR = Geo::kRaw, kTile = Geo::kTile, kThreads = Geo::kThreads;
  constexpr int E = 64 / BS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * Geo::kQTile;
  uint8_t* sV = sK + NS * kTile;
  uint8_t* sRawK = sV + NS * kTile;
  uint8_t* sRawV = sRawK + NR * Geo::kRawTile;
  auto* tl = reinterpret_cast<PTail<NS, NR>*>(sV + NS * kTile + Geo::kRawBytes);

  // the joining kernel reads nothing before this grid has ended; its launch may be prepared
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (*reinterpret_cast<volatile int*>(wait_status) != 0) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x;

  if (tid == 0) {
    constexpr int kFollow = KV8 ? 15 : 11;   // producer, two issuers, eight softmax warps (and four converters)
    for (int i = 0; i < 2; ++i) { mbar_init(&tl->plan_full[i], 1); mbar_init(&tl->plan_free[i], kFollow); }
    mbar_init(&tl->q_full, 1);
    mbar_init(&tl->q_free, 2);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&tl->k_full[i], KV8 ? 4 : 1); mbar_init(&tl->v_full[i], KV8 ? 4 : 1);
      mbar_init(&tl->k_free[i], 2); mbar_init(&tl->v_free[i], 2);
    }
    for (int i = 0; i < NR; ++i) {
      mbar_init(&tl->raw_k_full[i], 1); mbar_init(&tl->raw_v_full[i], 1);
      mbar_init(&tl->raw_k_free[i], 4); mbar_init(&tl->raw_v_free[i], 4);
    }
    for (int w = 0; w < 2; ++w) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&tl->qk_done[w][i], 1); mbar_init(&tl->p_full[w][i], 4); mbar_init(&tl->pv_done[w][i], 1);
      }
      mbar_init(&tl->o_free[w], 4);
    }
    mbar_init(&tl->mrg_full, 4);
    mbar_init(&tl->mrg_free, 4);
    mbar_fence_init();
    tl->start_e = -1;
  } else if (tid == 32) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK.map);
    tma_prefetch_desc(&tmV.map);
  }
  if (warp == kWIssue0) {
    tmem_alloc(&tl->tmem_base, 512);
    tmem_relinquish();
  }
  // ---- this CTA's share [us, ue) of all units, and the request and kv head it begins in
  const int nE = p.batch * p.hkv;
  constexpr int kWarps = kThreads / 32;
  long long first_w = 0, U = 0;
  for (int e = tid; e < nE; e += kThreads) {
    const long long w = request_weight(p, sh, e);
    if (e == tid) first_w = w;
    U += w;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) U += __shfl_xor_sync(0xffffffffu, U, o);
  if (lane == 0) tl->warp_sums[warp] = U;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  U = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) U += tl->warp_sums[w];
  constexpr int kLeast = kMinTiles * E;
  const int C = (int)max(1ll, min((long long)sh.ctas, (U + kLeast - 1) / kLeast));
  const long long us = cta < C ? U * cta / C : U, ue = cta < C ? U * (cta + 1) / C : U;
  if (us < ue) {
    long long base = 0;
    for (int e0 = 0; e0 < nE && base <= us; e0 += kThreads) {
      const int e = e0 + tid;
      const long long w = e0 == 0 ? first_w : (e < nE ? request_weight(p, sh, e) : 0);
      long long incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      __syncthreads();                 // the sums of the pass before have been read
      if (lane == 31) tl->warp_sums[warp] = incl;
      __syncthreads();
      long long before = base, total = 0;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) {
        if (x < warp) before += tl->warp_sums[x];
        total += tl->warp_sums[x];
      }
      if (w > 0 && before + incl - w <= us && us < before + incl) {
        tl->start_e = e;
        tl->start_base = before + incl - w;
      }
      base += total;
    }
  }
  __syncthreads();
  const uint32_t tmem = tl->tmem_base;
  const bool tree = p.tree_mask != nullptr;
  const int G = p.hq / p.hkv;

  if (warp == kWPlan) {
    // ============================================================ planner
    if (lane == 0) recs[cta].valid = 0;
    int k = 0;             // plans so far
    bool ok = true;
    PPlan* pl = nullptr;
    int n = 0, tiles = 0;
    int e = tl->start_e;
    long long base = tl->start_base;
    for (; ok && us < ue && e >= 0 && e < nE && base < ue; ++e) {
      const int b = e / p.hkv, kvh = e % p.hkv;
      const PagedRequest r = paged_request(p, b);
      const int n_items = item_count(sh, r.n);
      const int32_t* table = p.block_tables + (int64_t)b * p.table_stride;
      for (int ci = 0; ok && ci < sh.chunks * n_items && base < ue; ++ci) {
        const int chunk = ci / n_items, tile = ci % n_items;
        const int w = item_weight(p, sh, r, kvh, chunk, tile);
        if (base + w <= us) { base += w; continue; }
        const int ua = (int)max(us - base, 0ll), ub = (int)min(ue - base, (long long)w);
        const int part = ua == 0 && ub == w ? -1 : ua > 0 ? 2 * cta : 2 * cta + 1;
        if (ua == 0 && ub < w && lane == 0) {
          PagedRec rec = {1, b, kvh, chunk, tile, owner_of(base + w - 1, U, C), {0, 0}};
          recs[cta] = rec;
        }
        base += w;
        const ItemKeys ik = item_keys(p, sh, r, tile);
        const int tok0 = tile * 2 * sh.tt, ntok = min(2 * sh.tt, r.n - tok0), r0 = ik.r0;
        const int head0 = kvh * G + chunk * sh.gt, gcnt = min(sh.gt, G - chunk * sh.gt);
        // blocks that the drafts' positions reach into: r0 + y
        uint64_t my_dm = 0;
        int nx;
        if (tree) {
          int ymax = 0;
          uint32_t y0 = 0xffffu, y1 = 0xffffu;      // of drafts lane and lane + 32
          for (int i = lane; i < r.n; i += 32) {
            const int y = (r.L + draft_depth(draft_word(p, r, i), i)) / BS - r0;
            if (i < 32) y0 = y; else if (i < 64) y1 = y;
            if (i >= tok0 && i < tok0 + ntok) ymax = max(ymax, y);
          }
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            const uint64_t m = (uint64_t)__ballot_sync(0xffffffffu, y0 == (uint32_t)y) |
                               (uint64_t)__ballot_sync(0xffffffffu, y1 == (uint32_t)y) << 32;
            if (lane == y) my_dm = m;
          }
          nx = __reduce_max_sync(0xffffffffu, ymax) + 1;
        } else {
          nx = (ik.Lp % BS + ntok - 1) / BS + 1;
        }
        // pattern rows, one per lane: x = row - r0, g = head (one for all where they are equal)
        const int per_x = sh.shared ? 1 : sh.gt, nf = nx * per_x;
        (void)BSA_IN_BOUNDS(nf <= 32, wait_status, 820);
        const int fx = lane / per_x, fg = lane % per_x;
        const int32_t* my_cols = p.col;
        int cur = 0, end = 0;       // CSR entries of columns below r0
        uint32_t my_tb = 0;
        if (lane < nf && fg < gcnt && r0 + fx < p.n_rows) {
          const int hp = pattern_head(head0 + fg, p.h_pat, p.hq, p.hkv);
          const int32_t* cr = p.crow + (int64_t)hp * p.crow_sh + r0 + fx;
          my_cols = p.col + (int64_t)hp * p.col_sh;
          cur = __ldg(cr);
          end = __ldg(cr + 1);
          if (!BSA_IN_BOUNDS(cur >= 0 && cur <= end && (p.col_sh == 0 || end <= p.col_sh), wait_status, 821)) end = cur;
          while (end > cur) {
            const int c = __ldg(my_cols + end - 1);
            if (c < r0) break;
            if (c - r0 < 32) my_tb |= 1u << (c - r0);
            --end;
          }
        }
        const int beg0 = __shfl_sync(0xffffffffu, cur, 0), n0 = __shfl_sync(0xffffffffu, end, 0) - beg0;
        const int32_t* cols0 = p.col + (int64_t)pattern_head(head0, p.h_pat, p.hq, p.hkv) * p.col_sh;
        // the share [ua, ub) of the units as a range of the first row's entries
        const int ia = (int)((long long)ua * n0 / w), ib = ub == w ? n0 : (int)((long long)ub * n0 / w);

        n = tiles = 0;
        bool first = true;
        auto open = [&]() {
          const int pb = k & 1;
          if (!mbar_wait(&tl->plan_free[pb], ((k >> 1) & 1) ^ 1, wait_status, 1001)) { ok = false; return; }
          pl = &tl->plan[pb];
          pl->tb[lane] = my_tb;
          if (lane < 8) pl->dm[lane] = my_dm;
          if (lane == 0) {
            pl->valid = 1;
            pl->first = first;
            pl->two = ntok > sh.tt;
            pl->part = part;
            pl->tile0 = tiles;
            pl->b = b; pl->t0 = r.t0; pl->n_new = r.n; pl->L = r.L; pl->kvh = kvh; pl->head0 = head0; pl->gcnt = gcnt;
            pl->tok0 = tok0; pl->ntok = ntok; pl->Lp = ik.Lp; pl->r0 = r0; pl->Sp = ik.Sp;
          }
          first = false;
          n = 0;
        };
        auto publish = [&](bool last) {
          const int nt = (n + E - 1) / E;
          if (lane == 0) { pl->n = n; pl->nt = nt; pl->last = last; }
          tiles += nt;
          __syncwarp();
          if (lane == 0) mbar_arrive(&tl->plan_full[k & 1]);
          ++k;
        };
        // up to 32 blocks, one per lane, in order
        auto emit = [&](bool on, int col, uint32_t fl, uint32_t tail) {
          const uint32_t who = __ballot_sync(0xffffffffu, on);
          const int cnt = __popc(who);
          if (!cnt || !ok) return;
          if (n + cnt > kSeg) {
            publish(false);
            open();
            if (!ok) return;
          }
          if (on) {
            const int at = n + __popc(who & ((1u << lane) - 1u));
            const long long s0 = (long long)col * BS;
            uint32_t have = 0;
            if (sh.box == BS) {          // a block lies in one page
              const int pg = page_of(table, s0 >> sh.page_shift, p.max_pages, p.num_pages);
              pl->page[at * kPagesPerEntry] = pg;
              have = pg >= 0 ? 0xffu : 0u;
            } else {
              for (int i = 0; i < BS / sh.box; ++i) {
                const int pg = page_of(table, (s0 >> sh.page_shift) + i, p.max_pages, p.num_pages);
                pl->page[at * kPagesPerEntry + i] = pg;
                have |= (pg >= 0 ? 1u : 0u) << i;
              }
            }
            pl->col[at] = (uint32_t)col | have << 23 | tail;
            pl->fl[at] = fl;
          }
          n += cnt;
        };
        open();
        if (!ok) break;
        if (nf == 1) {
          // one pattern row: its entries are the list
          int c = ia + lane < ib ? __ldg(cols0 + beg0 + ia + lane) : 0;
          for (int i = ia; ok && i < ib; i += 32) {
            const int next = i + 32 + lane < ib ? __ldg(cols0 + beg0 + i + 32 + lane) : 0;
            emit(i + lane < ib, c, 1u, 0u);
            c = next;
          }
        } else {
          // several rows: the union of their columns inside the share's range, a window of kSeg columns at a time
          const int clo = ia == 0 ? 0 : __ldg(cols0 + beg0 + ia);
          const int chi = ub == w ? r0 : ib == 0 ? 0 : __ldg(cols0 + beg0 + ib);
          if (clo > 0) {
            int lo = cur, hi = end;
            while (lo < hi) {
              const int mid = (lo + hi) >> 1;
              if (__ldg(my_cols + mid) < clo) lo = mid + 1; else hi = mid;
            }
            cur = lo;
          }
          while (ok) {
            const int next = cur < end ? __ldg(my_cols + cur) : 0x7fffffff;
            const int wc = max(__reduce_min_sync(0xffffffffu, next), 0);
            if (wc >= chi) break;
            const int stop = (int)min((long long)wc + kSeg, (long long)chi);
            for (int i = lane; i < kSeg; i += 32) tl->window[i] = 0u;
            __syncwarp();
            for (int f = 0; f < nf; ++f) {
              const int fe = __shfl_sync(0xffffffffu, end, f);
              int fc = __shfl_sync(0xffffffffu, cur, f);
              const int32_t* fcols = p.col + (int64_t)pattern_head(head0 + min(f % per_x, gcnt - 1), p.h_pat, p.hq, p.hkv) * p.col_sh;
              while (true) {
                const int c = fc + lane < fe ? __ldg(fcols + fc + lane) : 0x7fffffff;
                const bool in = c < stop;
                if (in && BSA_IN_BOUNDS(c >= wc, wait_status, 822)) tl->window[c - wc] |= 1u << f;
                const int cnt = __popc(__ballot_sync(0xffffffffu, in));
                fc += cnt;
                if (cnt < 32) break;
              }
              if (lane == f) cur = fc;
              __syncwarp();
            }
            for (int i = 0; i < kSeg && ok; i += 32) {
              const uint32_t fl = tl->window[i + lane];
              emit(fl != 0u, wc + i + lane, fl, 0u);
            }
            __syncwarp();
          }
        }
        if (ub == w) {
          const int ny = (ik.Sp - 1) / BS - r0 + 1;
          for (int i = 0; ok && i < ny; i += 32) emit(i + lane < ny, r0 + i + lane, 0u, kTailFlag);
        }
        if (ok) publish(true);
      }
    }
    if (ok) {
      const int pb = k & 1;
      if (mbar_wait(&tl->plan_free[pb], ((k >> 1) & 1) ^ 1, wait_status, 1002)) {
        if (lane == 0) {
          tl->plan[pb].valid = -1;
          mbar_arrive(&tl->plan_full[pb]);
        }
      }
    }
  } else if (warp == kWProd) {
    // ============================================================ TMA producer
    // the loads' own ring: the 16-bit tiles, or the e4m3 tiles that the converters read
    constexpr int NL = KV8 ? NR : NS;
    constexpr uint32_t kLoadBytes = KV8 ? Geo::kRawTile : kTile;
    uint64_t* kf = KV8 ? tl->raw_k_full : tl->k_full;
    uint64_t* vf = KV8 ? tl->raw_v_full : tl->v_full;
    uint64_t* ke = KV8 ? tl->raw_k_free : tl->k_free;
    uint64_t* ve = KV8 ? tl->raw_v_free : tl->v_free;
    uint8_t* sk = KV8 ? sRawK : sK;
    uint8_t* sv = KV8 ? sRawV : sV;
    const int per = 64 / sh.box;                       // boxes of a tile's 64 tokens
    const int subs = KV8 ? 1 : kSub;
    const int my_sub = lane / per, my_row = (lane % per) * sh.box;
    const int my_e = my_row / BS, my_off = my_row % BS;
    const int my_page = sh.box == BS ? 0 : my_off / sh.box;
    uint32_t rg = 0;
    int items = 0;
    for (int k = 0;; ++k) {
      const int pb = k & 1;
      if (!mbar_wait(&tl->plan_full[pb], (k >> 1) & 1, wait_status, 1011)) break;
      const PPlan* pl = &tl->plan[pb];
      if (pl->valid < 0) break;
      bool ok = true;
      if (pl->first) {
        if (items > 0 && !mbar_wait(&tl->q_free, (items - 1) & 1, wait_status, 1012)) break;
        ++items;
        if (lane == 0) {
          const int tiles = 1 + pl->two;
          mbar_expect_tx(&tl->q_full, (uint32_t)(tiles * kSub * sh.tt * sh.gt * 128));
          (void)BSA_IN_BOUNDS(pl->t0 + pl->tok0 >= 0 && pl->t0 + pl->tok0 < p.total_q && pl->head0 < p.hq, wait_status, 823);
          for (int w = 0; w < tiles; ++w)
            for (int c = 0; c < kSub; ++c)
              tma_load_3d(sQ + w * Geo::kQTile + c * 16384, &tmQ, &tl->q_full, c * 64, pl->head0, pl->t0 + pl->tok0 + w * sh.tt);
        }
        __syncwarp();
      }
      const int nt = pl->nt, n = pl->n, kvh = pl->kvh;
      auto load = [&](int j, uint8_t* ring, const Tmap4* tm, uint64_t* full, uint64_t* empty, int code) -> bool {
        const uint32_t x = rg + (uint32_t)j;
        const int s = x % NL;
        if (!mbar_wait(&empty[s], ((x / NL) & 1) ^ 1, wait_status, code)) return false;
        if (lane == 0) mbar_expect_tx(&full[s], kLoadBytes);
        __syncwarp();
        if (lane < per * subs) {
          const int idx = j * E + my_e;
          int pg = -1, slot = p.page_size;             // outside the page: the box is filled with zeros
          if (idx < n) {
            const uint32_t c = pl->col[idx];
            pg = pl->page[idx * kPagesPerEntry + my_page];
            if (pg >= 0) slot = (int)(((c & kColMask) * BS + my_off) & (uint32_t)(p.page_size - 1));
          }
          (void)BSA_IN_BOUNDS(pg < p.num_pages && (pg < 0 || slot + sh.box <= p.page_size), wait_status, 824);
          uint8_t* dst = ring + s * kLoadBytes + (KV8 ? my_row * D : my_sub * 8192 + my_row * 128);
          tma_load_tile(dst, tm, &full[s], KV8 ? 0 : my_sub * 64, slot, kvh, max(pg, 0));
        }
        __syncwarp();
        return true;
      };
      // K one tile ahead of V: its slot comes free earlier
      if (nt > 0) ok = load(0, sk, &tmK, kf, ke, 1013);
      for (int j = 0; ok && j < nt; ++j) {
        if (j + 1 < nt) ok = load(j + 1, sk, &tmK, kf, ke, 1013);
        if (ok) ok = load(j, sv, &tmV, vf, ve, 1014);
      }
      if (!ok) break;
      rg += (uint32_t)nt;
      __syncwarp();
      if (lane == 0) mbar_arrive(&tl->plan_free[pb]);
    }
  } else if (warp == kWIssue0 || warp == kWIssue0 + 1) {
    // ============================================================ MMA issuers, one per softmax group
    const int w = warp - kWIssue0;
    uint32_t idesc_qk = umma_idesc(BF16, 128, 64, false, false);
    if (p.sm_scale < 0.f) idesc_qk |= 1u << 13;        // A negated: the maximum of the scaled logits stays a maximum
    const uint32_t idesc_pv = umma_idesc(BF16, 128, D, false, true);
    const uint64_t qdesc = umma_desc_sw128(smem_u32(sQ), 16, 1024);
    const uint64_t kdesc = umma_desc_sw128(smem_u32(sK), 16, 1024);
    const uint64_t vdesc = umma_desc_sw128(smem_u32(sV), 8192, 1024);
    const uint32_t tS = tmem + w * 128, tO = tmem + 256 + w * 128;
    uint32_t rg = 0, gq = 0, gp = 0;     // ring position of the plan's first tile; products issued by this warp
    int items = 0, begun = 0;            // items; those with a tile of this group
    bool ok = true, started = false;
    for (int k = 0; ok; ++k) {
      const int pb = k & 1;
      if (!mbar_wait(&tl->plan_full[pb], (k >> 1) & 1, wait_status, 1021)) break;
      const PPlan* pl = &tl->plan[pb];
      if (pl->valid < 0) break;
      const int nt = pl->nt, two = pl->two, last = pl->last;
      if (pl->first) {
        if (!mbar_wait(&tl->q_full, items & 1, wait_status, 1022)) break;
        ++items;
        started = false;
      }
      const int step = two ? 1 : 2, j0 = two ? 0 : (w ^ pl->tile0) & 1;
      const uint64_t qd = qdesc + (uint64_t)((two ? w * Geo::kQTile : 0) >> 4);
      auto qk = [&](int j) -> bool {
        const uint32_t x = rg + (uint32_t)j;
        const int s = x % NS, sb = gq & 1;
        if (!mbar_wait(&tl->k_full[s], (x / NS) & 1, wait_status, 1023)) return false;
        tc_fence_after();
        const uint64_t kd = kdesc + (uint64_t)((s * kTile) >> 4);
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            tc_mma_ss(tS + sb * 64, qd + (uint64_t)(((i >> 2) * 16384 + (i & 3) * 32) >> 4),
                      kd + (uint64_t)(((i >> 2) * 8192 + (i & 3) * 32) >> 4), idesc_qk, i ? 1u : 0u);
          tc_commit(&tl->qk_done[w][sb]);
          tc_commit(&tl->k_free[s]);
          if (!two) tc_commit(&tl->k_free[s]);         // for the group that does not read this tile, too
        }
        __syncwarp();
        ++gq;
        return true;
      };
      for (int j = j0; ok && j < nt && j < j0 + 2 * step; j += step) ok = qk(j);
      for (int j = j0; ok && j < nt; j += step) {
        const uint32_t x = rg + (uint32_t)j;
        const int s = x % NS, sb = gp & 1;
        if (!mbar_wait(&tl->v_full[s], (x / NS) & 1, wait_status, 1024)) { ok = false; break; }
        if (!mbar_wait(&tl->p_full[w][sb], (gp >> 1) & 1, wait_status, 1025)) { ok = false; break; }
        if (!started && begun > 0 && !mbar_wait(&tl->o_free[w], (begun - 1) & 1, wait_status, 1026)) { ok = false; break; }
        if (!started) ++begun;
        tc_fence_after();
        const uint64_t vd = vdesc + (uint64_t)((s * kTile) >> 4);
        const uint32_t acc0 = started ? 1u : 0u;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)      // 4..7: the low terms of P
            tc_mma_ts(tO, tS + sb * 64 + kk * 8, vd + (uint64_t)(((kk & 3) * 2048) >> 4), idesc_pv, kk ? 1u : acc0);
          tc_commit(&tl->pv_done[w][sb]);
          tc_commit(&tl->v_free[s]);
          if (!two) tc_commit(&tl->v_free[s]);
        }
        __syncwarp();
        started = true;
        ++gp;
        if (j + 2 * step < nt) ok = qk(j + 2 * step);
      }
      if (!ok) break;
      rg += (uint32_t)nt;
      if (last) {
        if (elect_one()) tc_commit(&tl->q_free);
        __syncwarp();
      }
      if (elect_one()) mbar_arrive(&tl->plan_free[pb]);
      __syncwarp();
    }
  } else if (warp < 8) {
    // ============================================================ softmax and epilogue
    const int w = warp >> 2;
    const int r = tid & 127;                  // tile row = TMEM lane
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + w * 128 + lane_off, tO = tmem + 256 + w * 128 + lane_off;
    const float scale2 = fabsf(p.sm_scale) * (KV8 ? p.k_scale : 1.f) * kLog2e;
    const float v_scale = KV8 ? p.v_scale : 1.f;
    constexpr float kShift = kTermShift<BF16>;
    const bool wide = reinterpret_cast<uintptr_t>(p.o) % 16 == 0 && p.o_st % 8 == 0 && p.o_sh % 8 == 0;
    const int tl_row = r / sh.gt, g = r - tl_row * sh.gt;
    uint32_t rg = 0, gs = 0, mc = 0;          // ring position of the plan's first tile; tiles of this group; merge chunks
    bool alive = true;
    // the row's own state over an item
    float m_used = -INFINITY, l = 0.f;
    int f = 0, i_tok = 0, pos = 0, mine = 0;
    uint32_t tbits = 0;
    uint64_t fm = 0;
    bool row_ok = false, warp_live = false;
    for (int k = 0; alive; ++k) {
      const int pb = k & 1;
      if (!mbar_wait(&tl->plan_full[pb], (k >> 1) & 1, wait_status, 1031)) break;
      const PPlan* pl = &tl->plan[pb];
      if (pl->valid < 0) break;
      const int nt = pl->nt, n = pl->n, two = pl->two;
      const int tw = two ? w * sh.tt : 0;
      if (pl->first) {
        row_ok = tl_row < sh.tt && tw + tl_row < pl->ntok && g < pl->gcnt;
        warp_live = __any_sync(0xffffffffu, row_ok);
        i_tok = pl->tok0 + tw + tl_row;
        m_used = -INFINITY;
        l = 0.f;
        mine = 0;
        fm = 0;
        tbits = 0;
        pos = pl->L + i_tok;
        f = 0;
        if (row_ok) {
          PagedRequest rq{pl->t0, pl->n_new, pl->L};
          uint64_t word = 0;
          if (tree) {
            word = draft_word(p, rq, i_tok);
            pos = pl->L + draft_depth(word, i_tok);
          }
          const int x = pos / BS - pl->r0;
          f = sh.shared ? x : x * sh.gt + g;
          tbits = pl->tb[f & 31];
          if (tree) {
#pragma unroll
            for (int y = 0; y < 8; ++y)
              if ((tbits >> y) & 1u) fm |= pl->dm[y];
            fm &= word;
          }
        }
      }
      const int step = two ? 1 : 2, j0 = two ? 0 : (w ^ pl->tile0) & 1;
      for (int j = j0; j < nt; j += step, ++gs) {
        const int sb = gs & 1;
        const uint32_t x = rg + (uint32_t)j;
        const int s = x % NS;
        // ---- which of the tile's 64 keys this row attends, before the logits are there
        uint64_t M = 0;
        int clear0 = 64;                      // rows of V that hold no key of this item, from here to the end of their block
        bool clear = false;
#pragma unroll
        for (int en = 0; en < E; ++en) {
          const int idx = j * E + en;
          if (idx < n) {
            const uint32_t c = pl->col[idx];
            uint64_t me = 0;
            if (!(c & kTailFlag)) {
              if ((pl->fl[idx] >> f) & 1u) me = low_bits(BS);
            } else {
              const int y = (int)(c & kColMask) - pl->r0, s0 = (int)(c & kColMask) * BS;
              const int nc = min(max(pl->Lp - s0, 0), BS);           // context tokens of the block
              if (nc && (tbits >> y) & 1u) me = low_bits(nc);
              if (tree) {
                const int d0 = s0 + nc - pl->L;                      // first draft of the block
                if (d0 < 64) me |= (fm >> d0) << nc;
              } else if ((tbits >> y) & 1u) {
                me |= low_bits(min(max(pos - s0 + 1, 0), BS));
              }
              me &= low_bits(BS);
              const int len = pl->Sp - s0;
              if (len < BS) { clear = true; clear0 = en * BS + len; }
            }
            uint32_t have = (c >> 23) & 0xffu;
            if (me && have != 0xffu) {
              if (sh.box == BS) me = 0;
              else
                for (int i = 0; i < BS / sh.box; ++i)
                  if (!((have >> i) & 1u)) me &= ~(low_bits(sh.box) << (i * sh.box));
            }
            M |= me << (en * BS);
          }
        }
        if (!row_ok) M = 0;
        const bool att = M != 0ull, any_att = __any_sync(0xffffffffu, att);
        if (!mbar_wait(&tl->qk_done[w][sb], (gs >> 1) & 1, wait_status, 1032)) { alive = false; break; }
        tc_fence_after();
        if (clear) {
          // keys behind the item's end: P is 0 there, and 0 times whatever the page holds has to be 0, too
          if (!mbar_wait(&tl->v_full[s], (x / NS) & 1, wait_status, 1033)) { alive = false; break; }
          uint8_t* vt = sV + s * kTile;
          const int cend = (clear0 / BS + 1) * BS;
          for (int q = r; q < (cend - clear0) * kSub * 8; q += 128) {
            const int row = clear0 + q / (kSub * 8), c = (q / 8) % kSub, ch = q & 7;
            *reinterpret_cast<uint4*>(vt + c * 8192 + row * 128 + ch * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async();
        }
        if (warp_live) {
          if (any_att) {
            uint32_t sv[64];
            tmem_ld32(tS + sb * 64, *reinterpret_cast<uint32_t(*)[32]>(&sv[0]));
            tmem_ld32(tS + sb * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(&sv[32]));
            tmem_ld_wait();
            if (__any_sync(0xffffffffu, M != ~0ull)) {
              const uint32_t lo = (uint32_t)M, hi = (uint32_t)(M >> 32);
#pragma unroll
              for (int c = 0; c < 32; ++c) {
                if (!((lo >> c) & 1u)) sv[c] = 0xff800000u;
                if (!((hi >> c) & 1u)) sv[32 + c] = 0xff800000u;
              }
            }
            float m4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              m4[i] = pmax3(__uint_as_float(sv[3 * i]), __uint_as_float(sv[3 * i + 1]), __uint_as_float(sv[3 * i + 2]));
#pragma unroll
            for (int c = 12; c < 60; c += 8)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                m4[i] = pmax3(m4[i], __uint_as_float(sv[c + 2 * i]), __uint_as_float(sv[c + 2 * i + 1]));
            const float mx = pmax3(pmax3(m4[0], m4[1], m4[2]), pmax3(m4[3], __uint_as_float(sv[60]), __uint_as_float(sv[61])),
                                   fmaxf(__uint_as_float(sv[62]), __uint_as_float(sv[63]))) * scale2;
            float alpha = 1.f;
            bool need = false;
            if (mx != -INFINITY) {
              if (m_used == -INFINITY) {
                m_used = mx;                  // O's row is 0 so far
              } else if (mx > m_used + kRescale) {
                alpha = pex2(m_used - mx);
                m_used = mx;
                l *= alpha;
                need = true;
              }
            }
            const bool any = __any_sync(0xffffffffu, need);
            const bool live = att && m_used != -INFINITY;
            const float neg_m = kShift - m_used;
            const uint64_t scale_2 = f32x2(scale2, scale2), neg_m2 = f32x2(neg_m, neg_m);
            uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t pk[16], pq[16];
              if (live) {
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                  float x0, x1;
                  f32x2_split(fma_f32x2(f32x2(sv[h * 32 + 2 * c], sv[h * 32 + 2 * c + 1]), scale_2, neg_m2), x0, x1);
                  const float p0 = pex2(x0), p1 = pex2(x1);
                  sum2[c & 1] = add_f32x2(sum2[c & 1], f32x2(p0, p1));
                  two_terms<BF16, !KV8>(p0, p1, pk[c], pq[c]);
                }
              } else {
#pragma unroll
                for (int c = 0; c < 16; ++c) pk[c] = pq[c] = 0u;
              }
              tmem_st16(tS + sb * 64 + h * 16, pk);
              tmem_st16(tS + sb * 64 + 32 + h * 16, pq);
            }
            float s4[4];
            f32x2_split(sum2[0], s4[0], s4[1]);
            f32x2_split(sum2[1], s4[2], s4[3]);
            l += (s4[0] + s4[1]) + (s4[2] + s4[3]);
            if (any && mine > 0) {
              // rows whose maximum moved: rescale their O once the product before has landed
              if (!mbar_wait(&tl->pv_done[w][(gs - 1) & 1], ((gs - 1) >> 1) & 1, wait_status, 1034)) { alive = false; break; }
              tc_fence_after();
#pragma unroll
              for (int ch = 0; ch < D / 32; ++ch) {
                uint32_t o[32];
                tmem_ld32(tO + ch * 32, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                tmem_st32(tO + ch * 32, o);
              }
            }
          } else {
            uint32_t z[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) z[c] = 0u;
            tmem_st32(tS + sb * 64, z);
            tmem_st32(tS + sb * 64 + 32, z);
          }
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tl->p_full[w][sb]);
        ++mine;
      }
      if (!alive) break;
      rg += (uint32_t)nt;
      if (pl->last) {
        // ---- the item's result
        if (mine > 0) {
          if (!mbar_wait(&tl->pv_done[w][(gs - 1) & 1], ((gs - 1) >> 1) & 1, wait_status, 1035)) break;
          tc_fence_after();
        }
        const bool joins = !two && pl->tile0 + nt > 1;        // one tile: both groups have a part of it
        if (joins && w == 1) {
          // hand this group's part over, 32 columns at a time
          tl->mrg_ml[0][r] = m_used;
          tl->mrg_ml[1][r] = l;
#pragma unroll 1
          for (int ch = 0; ch < D / 32; ++ch, ++mc) {
            uint32_t o[32];
            tmem_ld32(tO + ch * 32, o);
            tmem_ld_wait();
            if (ch && !mbar_wait(&tl->mrg_free, (mc - 1) & 1, wait_status, 1036)) { alive = false; break; }
#pragma unroll
            for (int i = 0; i < 32; ++i) tl->mrg[i * 128 + r] = __uint_as_float(o[i]);
            __syncwarp();
            if (lane == 0) mbar_arrive(&tl->mrg_full);
          }
          if (!alive) break;
          // the buffers are this item's until group 0 has read the last columns
          if (!mbar_wait(&tl->mrg_free, (mc - 1) & 1, wait_status, 1037)) break;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tl->o_free[w]);
        } else if (two || w == 0) {
          float a0 = 1.f, a1 = 0.f, m = m_used, lsum = l;
          bool bad = false;
          const int head = pl->head0 + g, t = pl->t0 + i_tok;
          const int item_row = (tw + tl_row) * sh.gt + g;
          const int part = pl->part;
          float inv = 0.f;
          uint8_t* orow = reinterpret_cast<uint8_t*>(p.o) + ((int64_t)t * p.o_st + (int64_t)head * p.o_sh) * 2;
          uint8_t* stg = w == 0 ? tl->ostage[warp & 3] : reinterpret_cast<uint8_t*>(tl->mrg) + (warp & 3) * 2048;
#pragma unroll 1
          for (int ch = 0; ch < D / 32; ++ch) {
            uint32_t o[32];
            if (mine > 0) {
              tmem_ld32(tO + ch * 32, o);
              tmem_ld_wait();
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = 0u;
            }
            if (ch == D / 32 - 1) {
              // O has been read: the next item's first product may overwrite it.  Only items that this group had a
              // tile of count here: a group without one does not wait for its issuer and could run ahead by phases
              tc_fence_before();
              __syncwarp();
              if (lane == 0 && mine > 0) mbar_arrive(&tl->o_free[w]);
            }
            if (joins) {
              if (!mbar_wait(&tl->mrg_full, mc & 1, wait_status, 1038)) { alive = false; break; }
              if (ch == 0) {
                const float m1 = tl->mrg_ml[0][r], l1 = tl->mrg_ml[1][r];
                m = fmaxf(m_used, m1);
                a0 = l == 0.f ? 0.f : pex2(m_used - m);
                a1 = l1 == 0.f ? 0.f : pex2(m1 - m);
                lsum = l * a0 + l1 * a1;
                if (!(l >= 0.f) || !(l1 >= 0.f)) lsum = NAN;
              }
              // a part without weight is left out, not multiplied by 0
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                float v = a0 != 0.f ? __uint_as_float(o[i]) * a0 : 0.f;
                if (a1 != 0.f) v = fmaf(tl->mrg[i * 128 + r], a1, v);
                o[i] = __float_as_uint(v);
              }
              ++mc;
              __syncwarp();
              if (lane == 0) mbar_arrive(&tl->mrg_free);
            }
            if (ch == 0) inv = lsum > 0.f ? v_scale / lsum : 0.f;
            if (part >= 0) {
              if (row_ok && BSA_IN_BOUNDS(item_row < sh.rows_cap && part < 2 * sh.ctas, wait_status, 825)) {
                float* dst = part_o + ((int64_t)part * sh.rows_cap + item_row) * D + ch * 32;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  reinterpret_cast<uint4*>(dst)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
              }
              continue;
            }
            uint32_t wd[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float x0 = __uint_as_float(o[2 * i]) * inv, x1 = __uint_as_float(o[2 * i + 1]) * inv;
              bad |= !(fabsf(x0) < INFINITY) || !(fabsf(x1) < INFINITY);
              wd[i] = ppack2<BF16>(x0, x1);
            }
            if (lsum == 0.f) {
#pragma unroll
              for (int i = 0; i < 16; ++i) wd[i] = 0u;
            }
            if (wide) {
              // rows -> 64-byte pieces: 16-byte words swizzled by the row pair, then lane L stores word L % 4 of rows
              // L / 4, L / 4 + 8, ...
#pragma unroll
              for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint4*>(stg + lane * 64 + ((i ^ ((lane >> 1) & 3)) * 16)) =
                    make_uint4(wd[4 * i], wd[4 * i + 1], wd[4 * i + 2], wd[4 * i + 3]);
              __syncwarp();
              const int pc = lane & 3;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int sr = i * 8 + (lane >> 2);
                const uint4 val = *reinterpret_cast<const uint4*>(stg + sr * 64 + ((pc ^ ((sr >> 1) & 3)) * 16));
                const long long dst = __shfl_sync(0xffffffffu, (long long)reinterpret_cast<uintptr_t>(orow), sr);
                const int okr = __shfl_sync(0xffffffffu, (int)row_ok, sr);
                if (okr && ch * 32 + pc * 8 < p.d)
                  *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(dst) + ch * 64 + pc * 16) = val;
              }
              __syncwarp();
            } else if (row_ok) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                if (ch * 32 + 2 * i < p.d) reinterpret_cast<uint16_t*>(orow)[ch * 32 + 2 * i] = (uint16_t)wd[i];
                if (ch * 32 + 2 * i + 1 < p.d) reinterpret_cast<uint16_t*>(orow)[ch * 32 + 2 * i + 1] = (uint16_t)(wd[i] >> 16);
              }
            }
          }
          if (!alive) break;
          if (part >= 0) {
            if (row_ok) part_ml[(int64_t)part * sh.rows_cap + item_row] = make_float2(m, lsum);
          } else {
            if (row_ok && p.lse)
              p.lse[(int64_t)head * p.lse_sh + t] = lsum > 0.f ? (m - kShift + log2f(lsum)) * kLn2 : -INFINITY;
            // an infinity or NaN got into the row: attended or not, the definition says what it is
            uint32_t redo = __ballot_sync(0xffffffffu, row_ok && lsum != 0.f && (bad || !(lsum > 0.f)));
            while (redo) {
              const int src = __ffs(redo) - 1;
              redo &= redo - 1;
              const int ri = __shfl_sync(0xffffffffu, i_tok, src), rh = __shfl_sync(0xffffffffu, head, src);
              paged_row<T16, C8>(p, pl->b, PagedRequest{pl->t0, pl->n_new, pl->L}, ri, rh, lane);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&tl->plan_free[pb]);
    }
  } else if (KV8) {
    // ============================================================ e4m3 -> 16-bit tiles in the layout of the products
    const int ct = tid - 384;
    uint32_t rg = 0;
    for (int k = 0;; ++k) {
      const int pb = k & 1;
      if (!mbar_wait(&tl->plan_full[pb], (k >> 1) & 1, wait_status, 1041)) break;
      const PPlan* pl = &tl->plan[pb];
      if (pl->valid < 0) break;
      const int nt = pl->nt;
      auto convert = [&](int j, const uint8_t* raw, uint8_t* tile, uint64_t* rf, uint64_t* re, uint64_t* full, uint64_t* empty,
                         int code) -> bool {
        const uint32_t x = rg + (uint32_t)j;
        const int rs = x % NR, s = x % NS;
        if (!mbar_wait(&rf[rs], (x / NR) & 1, wait_status, code)) return false;
        if (!mbar_wait(&empty[s], ((x / NS) & 1) ^ 1, wait_status, code + 1)) return false;
        const uint8_t* src = raw + rs * Geo::kRawTile;
        uint8_t* dst = tile + s * kTile;
        constexpr int kPieces = D / 16;        // 16 values each
#pragma unroll
        for (int q = 0; q < 64 * kPieces / 128; ++q) {
          const int at = q * 128 + ct, row = at / kPieces, pc = at % kPieces;
          const uint4 v = *reinterpret_cast<const uint4*>(src + at * 16);
          uint32_t out[8];
          const uint32_t in[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            out[2 * i] = e4m3x2_to_16<BF16>((uint16_t)in[i]);
            out[2 * i + 1] = e4m3x2_to_16<BF16>((uint16_t)(in[i] >> 16));
          }
          uint8_t* base = dst + (pc >> 2) * 8192 + row * 128;
          const int c0 = (pc & 3) * 2, odd = pc >> 2;      // upper sub-tiles store their odd half first: no bank twice
          const uint4 lo = make_uint4(out[0], out[1], out[2], out[3]), hi = make_uint4(out[4], out[5], out[6], out[7]);
          *reinterpret_cast<uint4*>(base + ((c0 + odd) ^ (row & 7)) * 16) = odd ? hi : lo;
          *reinterpret_cast<uint4*>(base + ((c0 + 1 - odd) ^ (row & 7)) * 16) = odd ? lo : hi;
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&full[s]);
          mbar_arrive(&re[rs]);
        }
        return true;
      };
      bool ok = true;
      if (nt > 0) ok = convert(0, sRawK, sK, tl->raw_k_full, tl->raw_k_free, tl->k_full, tl->k_free, 1042);
      for (int j = 0; ok && j < nt; ++j) {
        if (j + 1 < nt) ok = convert(j + 1, sRawK, sK, tl->raw_k_full, tl->raw_k_free, tl->k_full, tl->k_free, 1042);
        if (ok) ok = convert(j, sRawV, sV, tl->raw_v_full, tl->raw_v_free, tl->v_full, tl->v_free, 1044);
      }
      if (!ok) break;
      rg += (uint32_t)nt;
      __syncwarp();
      if (lane == 0) mbar_arrive(&tl->plan_free[pb]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWIssue0) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------ joining
// CTA (c, y): the item that CTA c of the kernel above began and did not finish; a warp per row.
template <typename T16, typename C8, int D>
__global__ void __launch_bounds__(256) paged_join_kernel(bsa_paged_params p, PagedShape sh, const PagedRec* recs,
                                                         const float2* __restrict__ part_ml, const float* __restrict__ part_o,
                                                         float shift, const int* wait_status) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (*reinterpret_cast<const volatile int*>(wait_status) != 0) return;
  const int c = blockIdx.x, lane = threadIdx.x & 31;
  const PagedRec rec = recs[c];
  if (!rec.valid) return;
  const PagedRequest r = paged_request(p, rec.b);
  const int G = p.hq / p.hkv, tok0 = rec.tile * 2 * sh.tt, ntok = min(2 * sh.tt, r.n - tok0);
  const int head0 = rec.kvh * G + rec.chunk * sh.gt, gcnt = min(sh.gt, G - rec.chunk * sh.gt);
  const int parts = rec.last - c + 1;
  const float v_scale = sizeof(C8) == 1 ? p.v_scale : 1.f;
  constexpr int V = D / 32;
  for (int row = blockIdx.y * 8 + (threadIdx.x >> 5); row < ntok * sh.gt; row += gridDim.y * 8) {
    const int tok = row / sh.gt, g = row % sh.gt;
    if (g >= gcnt) continue;
    auto at = [&](int i) { return (int64_t)(i == 0 ? 2 * c + 1 : 2 * (c + i)) * sh.rows_cap + row; };
    float m = -INFINITY;
    bool nan = false;
    for (int i = lane; i < parts; i += 32) {
      const float2 ml = part_ml[at(i)];
      if (ml.y != 0.f) m = fmaxf(m, ml.x);
      nan |= !(ml.y >= 0.f);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    nan = __any_sync(0xffffffffu, nan);
    float l = 0.f, acc[V];
#pragma unroll
    for (int x = 0; x < V; ++x) acc[x] = 0.f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
      const float2 ml = part_ml[at(i)];
      float o[V];
      const float* src = part_o + at(i) * D + lane * V;
      if constexpr (V == 4) *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(src);
      else *reinterpret_cast<float2*>(o) = *reinterpret_cast<const float2*>(src);
      if (ml.y == 0.f) continue;             // left out, whatever its columns hold
      const float wgt = pex2(ml.x - m);
      l = fmaf(ml.y, wgt, l);
#pragma unroll
      for (int x = 0; x < V; ++x) acc[x] = fmaf(o[x], wgt, acc[x]);
    }
    const int t = r.t0 + tok0 + tok, h = head0 + g;
    const float inv = l > 0.f ? v_scale / l : 0.f;
    T16* orow = static_cast<T16*>(p.o) + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + lane * V;
    bool bad = nan;
#pragma unroll
    for (int x = 0; x < V; ++x) {
      const float y = acc[x] * inv;
      bad |= !(fabsf(y) < INFINITY);
      if (lane * V + x < p.d) orow[x] = Elem<T16>::from_f(l == 0.f ? 0.f : y);
    }
    if (p.lse && lane == 0) p.lse[(int64_t)h * p.lse_sh + t] = l > 0.f ? (m - shift + log2f(l)) * kLn2 : -INFINITY;
    if (__any_sync(0xffffffffu, bad) && l != 0.f) paged_row<T16, C8>(p, rec.b, r, tok0 + tok, h, lane);
  }
}

// Heads per tile: as many of a group as their pattern rows fit in 32 flags (one per block row that the item's
// positions may reach into, and per head where heads differ).
void plan_shape(const bsa_paged_params* p, PagedShape* sh) {
  const int G = p->hq / p->hkv, bs = p->block_size;
  sh->shared = p->h_pat != p->hq || p->heads_share || G == 1;
  int gt = G < 128 ? G : 128;
  if (!sh->shared) {
    auto rows = [&](int g) {
      return p->tree_mask ? (bs - 1 + 64) / bs + 1 : (bs - 1 + 2 * (128 / g) - 1) / bs + 1;
    };
    while (gt > 1 && gt * rows(gt) > 32) --gt;
  }
  sh->gt = gt;
  sh->chunks = cdiv_i(G, gt);
  sh->tt = 128 / gt;
  const int most = p->cu_q ? (p->total_q < 2 * sh->tt ? p->total_q : 2 * sh->tt) : 1;
  sh->rows_cap = most * gt;
  sh->box = p->page_size < bs ? p->page_size : bs;
  sh->page_shift = 0;
  while ((1 << sh->page_shift) < p->page_size) ++sh->page_shift;
  sh->ctas = kCtas;
}

size_t ml_bytes(const PagedShape& sh) { return ((size_t)2 * sh.ctas * sh.rows_cap * sizeof(float2) + 255) / 256 * 256; }
constexpr size_t kRecBytes = (kCtas * sizeof(PagedRec) + 255) / 256 * 256;

template <bool BF16, int D, int BS, bool KV8>
int launch_paged(const bsa_paged_params* p, const PagedShape& shape, cudaStream_t s) {
  using Geo = PGeo<D, KV8>;
  using T16 = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  using C8 = typename std::conditional<KV8, uint8_t, T16>::type;
  PagedShape sh = shape;
  CUtensorMap tmQ;
  Tmap4 tmK, tmV;
  int rc = make_tmap_rows(&tmQ, p->q, p->d, p->hq, p->total_q, p->q_sh * 2, p->q_st * 2, sh.gt, sh.tt, BF16);
  if (rc) return rc;
  constexpr int eb = KV8 ? 1 : 2;
  const uint32_t box_d = KV8 ? D : 64;
  rc = make_tmap_4d(&tmK, p->k_cache, eb, p->d, p->page_size, p->hkv, p->num_pages, p->kc_ss * eb, p->kc_sh * eb, p->kc_sp * eb,
                    box_d, sh.box, !KV8, BF16);
  if (rc) return rc;
  rc = make_tmap_4d(&tmV, p->v_cache, eb, p->d, p->page_size, p->hkv, p->num_pages, p->vc_ss * eb, p->vc_sh * eb, p->vc_sp * eb,
                    box_d, sh.box, !KV8, BF16);
  if (rc) return rc;
  int dev = 0, sms = 0;
  BSA_CHECK_CUDA(cudaGetDevice(&dev));
  BSA_CHECK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  if (sms < sh.ctas) sh.ctas = sms;
  int* status = wait_status_ptr();
  if (!status) return BSA_E_CUDA;
  auto* recs = static_cast<PagedRec*>(p->ws);
  auto* ml = reinterpret_cast<float2*>(static_cast<char*>(p->ws) + kRecBytes);
  auto* po = reinterpret_cast<float*>(static_cast<char*>(p->ws) + kRecBytes + ml_bytes(shape));
  constexpr size_t smem = Geo::kFixed + sizeof(PTail<Geo::kSlots, Geo::kRaw>);
  static_assert(smem <= 227 * 1024, "shared memory");
  auto kern = paged_attn_kernel<BF16, D, BS, KV8>;
  BSA_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kern<<<sh.ctas, Geo::kThreads, smem, s>>>(tmQ, tmK, tmV, *p, sh, recs, ml, po, status);
  rc = check_launch("paged_attn_kernel");
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sh.ctas, cdiv_i(sh.rows_cap, 8) < 8 ? cdiv_i(sh.rows_cap, 8) : 8);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BSA_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_join_kernel<T16, C8, D>, *p, sh, (const PagedRec*)recs, (const float2*)ml,
                                    (const float*)po, kTermShift<BF16>, (const int*)status));
  return check_launch("paged_join_kernel");
}

template <bool BF16, int D, bool KV8>
int launch_paged_bs(const bsa_paged_params* p, const PagedShape& sh, cudaStream_t s) {
  if (p->block_size == 16) return launch_paged<BF16, D, 16, KV8>(p, sh, s);
  if (p->block_size == 32) return launch_paged<BF16, D, 32, KV8>(p, sh, s);
  return launch_paged<BF16, D, 64, KV8>(p, sh, s);
}
template <bool BF16>
int launch_paged_d(const bsa_paged_params* p, const PagedShape& sh, cudaStream_t s) {
  if (p->kv_dtype == BSA_F8E4M3)
    return p->d <= 64 ? launch_paged_bs<BF16, 64, true>(p, sh, s) : launch_paged_bs<BF16, 128, true>(p, sh, s);
  return p->d <= 64 ? launch_paged_bs<BF16, 64, false>(p, sh, s) : launch_paged_bs<BF16, 128, false>(p, sh, s);
}
}  // namespace

bool paged_sm100_supported(const bsa_paged_params* p, const char** why) {
  auto no = [&](const char* w) { *why = w; return false; };
  if (!(p->dtype == BSA_F16 || p->dtype == BSA_BF16)) return no("dtype is not f16/bf16");
  const bool f8 = p->kv_dtype == BSA_F8E4M3;
  if (p->d > 128 || p->d % (f8 ? 16 : 8)) return no("head dim is not a multiple of 8 (16 for an e4m3 cache) up to 128");
  if (p->block_size > 64) return no("pattern blocks of 128 tokens (refine them to 64)");
  if (p->page_size < 8 || (p->page_size & (p->page_size - 1))) return no("page size is not a power of two from 8 on");
  if (p->num_pages < 1 || p->max_pages < 1) return no("no pages");
  if ((int64_t)p->max_pages * p->page_size > (int64_t)kColMask * p->block_size) return no("block table is too wide");
  const int eb = f8 ? 1 : 2;
  if (!tma_compatible(p->k_cache, eb, p->kc_ss, p->kc_sh, p->kc_sp) || !tma_compatible(p->v_cache, eb, p->vc_ss, p->vc_sh, p->vc_sp))
    return no("the caches need 16-byte aligned bases and strides that are multiples of 16 bytes");
  if (reinterpret_cast<uintptr_t>(p->q) % 16 || (p->hq > 1 && (p->q_sh % 8 || p->q_sh <= 0)) ||
      (p->total_q > 1 && (p->q_st % 8 || p->q_st <= 0 || (p->hq > 1 && p->q_st < p->q_sh))))
    return no("q needs a 16-byte aligned base, strides that are multiples of 16 bytes and heads inside tokens");
  if (!(p->sm_scale != 0.f)) return no("sm_scale is 0 or NaN");
  if (f8 && !(p->k_scale > 0.f)) return no("k_scale is not positive");
  return true;
}

size_t paged_sm100_workspace(const bsa_paged_params* p) {
  PagedShape sh;
  plan_shape(p, &sh);
  return kRecBytes + ml_bytes(sh) + (size_t)2 * sh.ctas * sh.rows_cap * (p->d <= 64 ? 64 : 128) * sizeof(float);
}

int paged_sm100(const bsa_paged_params* p, cudaStream_t s) {
  PagedShape sh;
  plan_shape(p, &sh);
  return p->dtype == BSA_BF16 ? launch_paged_d<true>(p, sh, s) : launch_paged_d<false>(p, sh, s);
}

}  // namespace bsa
