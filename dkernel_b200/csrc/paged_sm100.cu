// Attention of drafted tokens over a paged K/V cache on the tcgen05 tensor cores (f16 / bf16 queries; cache of
// their type or e4m3; head dims that are multiples of 8, 16 for e4m3, up to 128; pattern blocks of 16, 32 or 64
// tokens; pages of a power of two of tokens, 8 or more).  Semantics: include/bsa.h.
//
// What it cannot do without: every attended K/V byte of a (request, kv head) has to come from HBM once.  An ITEM is a tile of
// 128 rows = drafted tokens x q heads of a kv group, and the pattern blocks that any of them attends.  The items' blocks
// are shared out over two persistent CTAs per SM in equal pieces, whatever the requests' lengths: a CTA's piece may begin
// and end inside an item, whose partial results a second kernel then joins.  Requests with more rows than a tile have
// their even and odd tiles in two halves of the line of work, so that two CTAs come to the same keys at about the same
// time and one of them finds them in L2.
// Up to 16 rows (a token's heads, small trees) are repeated down the 128 rows of the tile, twice in each softmax warp's 32.
// Each warp weighs its own quarter of the keys, so that all four have a share of the exponentials, and its second
// repetition holds the low terms of the weights that the first holds the high terms of; what the repetitions have is added
// up in shared memory at the item's end.
//
// A K/V tile is 64 tokens = 1, 2 or 4 pattern blocks, wherever their pages are: one TMA box per page piece.
// Warps (192 threads, 256 with an e4m3 cache): 0-3 softmax and epilogue, 4 planner and TMA producer, 5 MMA issuer,
// 6 and 7 e4m3 -> f16.  TMEM: S 2x64 | O 128 columns.
//
// Measured (bf16, 32 / 8 heads of 128, blocks of 64, band of 16 + one column in 8; one call after another, which brings the
// card to its power limit and 1.6 GHz): 64 single tokens over 1024..8192 tokens 91 us (4.3 TB/s of attended bytes, 84 us before
// the limit is reached), 64 trees of 15..29 drafts 126 us, 48 trees of 30..60 on an e4m3 cache 203 us, one token over 4000
// 22 us.  A launch's first 9 us go by until its first tile is there: tables and lists, each instruction met for the first
// time; then single tokens run at what HBM gives, wide trees at the pace of the softmax warps (two per scheduler: 1850
// cycles a tile against 1024 of exponentials), with shared memory three quarters busy (Q, K and twice V as operands).
// That pace is two thirds of the trees' time and half of the e4m3 trees'; what the rest waits for is not known.  An e4m3 cache
// makes calls slower, not faster: the same 64 single tokens 103 us against 84, the trees 150 against 108, the wide trees 201
// against 142; two warps expand each of its tiles in shared memory before the products.  The cost of a join: 2 to 8 us.  K/V
// tiles pass through L2 evict-first: without that this code and the tables are fetched from DRAM again, launch after launch,
// and trees take 10 % more.
#include <type_traits>

#include "ptx.cuh"
#include "paged.cuh"

namespace bsa {
namespace {

constexpr int kCtas = 296;            // most CTAs of a launch, two per SM; sizes the workspace
constexpr int kSeg = 64;              // pattern blocks that a plan lists at most
constexpr int kSegPages = 128;        // and pages of theirs
constexpr int kWindow = 128;          // columns whose union is formed at a time
constexpr uint32_t kTailFlag = 1u << 31;
constexpr uint32_t kColMask = (1u << 23) - 1u;   // bits 23..30: pages that exist
constexpr int kOverhead = 3;          // an item's fixed cost in K/V tiles (2: trees 1 % slower; 4, 6: single tokens 1, 2 %)
constexpr float kRescale = 8.0f;
constexpr int kWPlan = 4, kWIssue = 5, kWConv = 6;

// How rows and items are cut; the same for the whole launch.  A tile's rows come in chunks of cr (16, 32, 64 or 128) rows
// for ct tokens x gt heads, what one TMA box brings.
struct PagedShape {
  int gt;          // q heads of a group that a tile holds
  int chunks;      // pieces of a group
  int cr, ct;
  int tt;          // tokens of a tile
  int shared;      // these heads have equal pattern rows
  int rows_cap;    // rows of a partial result
  int page_shift, box;
  int least;       // least units of a CTA's share
  int ctas;
  int rr_hint;     // rows of a repetition that most items will have
  float inv_hkv, inv_gt;
};

// The item that a CTA begins and others finish; written by every CTA, valid = 0 where there is none.
struct PagedRec { int valid, b, t0, n, L, tok0, ntok, head0, gcnt, last; };

struct PPlanHead {
  int valid, first, last, part;
  int n, nt;                   // listed blocks, K/V tiles
  int rr;                      // rows of a repetition: 16, or 128 = none
  int b, t0, n_new, L, kvh, head0, gcnt;
  int tok0, ntok, Lp, r0, Sp;  // Lp: keys before it are context for every row of the item; r0 = Lp / block; Sp: end of its keys
};
struct PPlan : PPlanHead {
  uint32_t tb[32];             // by pattern row: which of the blocks r0, r0 + 1, ... it has
  uint64_t dm[8];              // drafts whose position lies in block r0 + y
  uint32_t special[2];         // listed blocks that hold drafts, miss a page, or are not attended by every pattern row
  uint32_t col[kSeg], fl[kSeg];
  int page[kSegPages];
};

template <int D, bool KV8> struct PGeo {
  static constexpr int kSub = D / 64;
  static constexpr int kQTile = 128 * D * 2;
  static constexpr int kTile = 64 * D * 2;
  // 16-bit K and V slots.  With an e4m3 cache K's is free again when Q K^T is done, V's only behind the softmax: V has two
  static constexpr int kKSlots = KV8 ? (D == 64 ? 2 : 1) : (D == 64 ? 4 : 2);
  static constexpr int kVSlots = D == 64 && !KV8 ? 4 : 2;
  static constexpr int kRawTile = 64 * D;
  static constexpr int kRaw = KV8 ? (D == 64 ? 4 : 1) : 1;                     // e4m3 K slots, and V slots
  static constexpr int kRawBytes = KV8 ? 2 * kRaw * kRawTile : 0;
  static constexpr size_t kFixed = 1024 + kQTile + (kKSlots + kVSlots) * kTile + kRawBytes;
  static constexpr int kThreads = KV8 ? 256 : 192;
};

template <int NK, int NV, int NR> struct PTail {
  uint64_t plan_full[2], plan_free[2], q_full, q_free;
  uint64_t k_full[NK], v_full[NV], k_free[NK], v_free[NV];
  uint64_t raw_k_full[NR], raw_v_full[NR], raw_k_free[NR], raw_v_free[NR];
  uint64_t qk_done[2], p_full[2], pv_done[2], o_free, met, q_ready;
  uint32_t tmem_base;
  int start_e;
  long long start_base, warp_sums[16];
  uint32_t window[kWindow];
  PPlan plan[2];
  PPlanHead warm;
  // joining the repetitions of a tile's rows: maxima, sums, weights; per row the joined maximum and sum
  float jm[64], jl[64], jw[64], rm[16], rl[16];
  int jbad[16];
  alignas(16) float stage[2048];             // parts of some columns; without repetitions: 32 rows x 64 bytes per warp
};

// Bounded like every wait, but by 10 s: a warp that recomputes the rows that a NaN got into (32 of them, 6 ms each over
// 64 thousand attended keys) keeps the others waiting that long.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, int* status, int code) {
  return mbar_wait(bar, parity, status, code, 10000000000ull);
}

__device__ __forceinline__ float pex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// NaN if one of them is: a tile whose attended logits are all NaN must not look like one without attended keys
__device__ __forceinline__ float pmax3(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
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
// p = hi + lo, hi cut off: it leaves at most 2^-7 of p in bf16, 2^-10 in f16, and lo's rounding 2^-16 and 2^-22 of p.  As
// two_terms, but without its least low term: an infinity in V meets a low term of 0 here and gives NaN; such rows are
// computed again.
template <bool BF16> __device__ __forceinline__ void psplit(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  float h0, h1, l0, l1;
  if (BF16) {
    asm("prmt.b32 %0, %1, %2, 0x7632;" : "=r"(hi) : "r"(__float_as_uint(p0)), "r"(__float_as_uint(p1)));
    h0 = __uint_as_float(hi << 16);
    h1 = __uint_as_float(hi & 0xffff0000u);
  } else {
    asm("cvt.rz.f16x2.f32 %0, %2, %1;" : "=r"(hi) : "f"(p0), "f"(p1));
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    h0 = h.x;
    h1 = h.y;
  }
  f32x2_split(fma_f32x2(f32x2(h0, h1), f32x2(-1.f, -1.f), f32x2(p0, p1)), l0, l1);
  lo = ppack2<BF16>(l0, l1);
}
// two e4m3 -> two f16, exactly
__device__ __forceinline__ uint32_t e4m3x2_to_f16(uint16_t x) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(x));
  return h;
}

// ------------------------------------------------------------------ items and their weights
// Item s of a request and kv head: piece s % chunks of the group's heads, tile s / chunks of the tokens.
__device__ __forceinline__ int item_count(const PagedShape& sh, int n) {
  return n <= 0 ? 0 : (n <= sh.tt ? 1 : (n + sh.tt - 1) / sh.tt) * sh.chunks;
}

// Where an item's keys lie.  In a tree every row sees the same context; in a chain the tokens before the item are
// context for all its rows.
struct ItemKeys { int tok0, chunk, Lp, Sp, r0; };
template <int BS>
__device__ __forceinline__ ItemKeys item_keys(const bsa_paged_params& p, const PagedShape& sh, const PagedRequest& r, int s) {
  ItemKeys k;
  const int tile = sh.chunks == 1 ? s : s / sh.chunks;
  k.chunk = s - tile * sh.chunks;
  k.tok0 = tile * sh.tt;
  k.Lp = p.tree_mask ? r.L : r.L + k.tok0;
  k.Sp = p.tree_mask ? r.L + r.n : r.L + min(r.n, k.tok0 + sh.tt);
  k.r0 = k.Lp / BS;
  return k;
}

// Units of work of an item: blocks of its first head's first pattern row, blocks that hold its drafts, and a fixed
// cost.  An estimate where rows differ; shares are cut in its proportion.
template <int BS>
__device__ __forceinline__ int item_weight(const bsa_paged_params& p, const PagedShape& sh, const PagedRequest& r, int kvh, int s) {
  const ItemKeys k = item_keys<BS>(p, sh, r, s);
  const int hp = p.h_pat == 1 ? 0 : p.h_pat == p.hkv ? kvh : kvh * (p.hq / p.hkv) + k.chunk * sh.gt;
  const int32_t* cr = p.crow + (int64_t)hp * p.crow_sh;
  const int len = k.r0 < p.n_rows ? __ldg(cr + k.r0 + 1) - __ldg(cr + k.r0) : 0;
  return max(len, 0) + (k.Sp - 1) / BS - k.r0 + 1 + kOverhead * (64 / BS);
}

// The line of work: request and kv head by request and kv head, first their even items, then the odd ones.
struct Entry { int b, kvh, half; };
__device__ __forceinline__ Entry entry_of(const PagedShape& sh, int e, int nE, int hkv) {
  Entry x;
  x.half = e >= nE;
  const int y = x.half ? e - nE : e;
  // exact: (y + 1/2) / hkv is 1 / (2 hkv) off an integer at least; the product's error is 2^-23 of less than 2^20 / hkv
  x.b = nE < (1 << 20) ? (int)((y + 0.5f) * sh.inv_hkv) : y / hkv;
  x.kvh = y - x.b * hkv;
  return x;
}

// ------------------------------------------------------------------ the kernel
// P is kept as the sum of two 16-bit terms in S's columns, as in the decode and the long packed kernels: no precision
// hangs on which weights a 16-bit type holds exactly (the output is as far from 64 bits as its own rounding makes it; one
// term would add as much again, for a few percent of time: with half of the products left out, trees take 119 us, not 126).
template <bool BF16, int D, int BS, bool KV8>
__global__ void __launch_bounds__(PGeo<D, KV8>::kThreads, 2)
paged_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ Tmap4 tmK, const __grid_constant__ Tmap4 tmV,
                  const __grid_constant__ bsa_paged_params p, const __grid_constant__ PagedShape sh, PagedRec* __restrict__ recs,
                  float2* __restrict__ part_ml, float* __restrict__ part_o, int* wait_status) {
  using Geo = PGeo<D, KV8>;
  using T16 = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  using C8 = typename std::conditional<KV8, uint8_t, T16>::type;
  // An e4m3 cache is multiplied in f16: e4m3 -> f16 is one instruction for two values, -> bf16 four.  bf16 queries are
  // converted row by row with a power of two of their own (their largest value comes to 2^13 .. 2^14; what f16 then
  // cannot hold is below 2^-38 of that), which the row's logits are divided by again.
  constexpr bool BE = BF16 && !KV8, QCONV = BF16 && KV8;
  constexpr int kSub = Geo::kSub, NK = Geo::kKSlots, NV = Geo::kVSlots, NR = Geo::kRaw, kTile = Geo::kTile, kThreads = Geo::kThreads;
  constexpr int E = 64 / BS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + Geo::kQTile;
  uint8_t* sV = sK + NK * kTile;
  uint8_t* sRawK = sV + NV * kTile;
  uint8_t* sRawV = sRawK + NR * Geo::kRawTile;
  auto* tl = reinterpret_cast<PTail<NK, NV, NR>*>(sV + NV * kTile + Geo::kRawBytes);

  // the joining kernel reads nothing before this grid has ended; its launch may be prepared
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (*reinterpret_cast<volatile int*>(wait_status) != 0) {
    // what follows in the stream follows the kernel in front of this one, too (which may have let this one start early)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int tid = threadIdx.x, lane = tid & 31;
  const int cta = blockIdx.x;
  const int warp = tid >> 5;

  if (tid == 0) {
    constexpr int kFollow = KV8 ? 7 : 5;       // issuer, four softmax warps (and two converters)
    for (int i = 0; i < 2; ++i) { mbar_init(&tl->plan_full[i], 1); mbar_init(&tl->plan_free[i], kFollow); }
    mbar_init(&tl->q_full, 1);
    mbar_init(&tl->q_free, 1);
    for (int i = 0; i < NK; ++i) { mbar_init(&tl->k_full[i], KV8 ? 2 : 1); mbar_init(&tl->k_free[i], 1); }
    for (int i = 0; i < NV; ++i) { mbar_init(&tl->v_full[i], KV8 ? 2 : 1); mbar_init(&tl->v_free[i], 1); }
    for (int i = 0; i < NR; ++i) {
      mbar_init(&tl->raw_k_full[i], 1); mbar_init(&tl->raw_v_full[i], 1);
      mbar_init(&tl->raw_k_free[i], 2); mbar_init(&tl->raw_v_free[i], 2);
    }
    for (int i = 0; i < 2; ++i) { mbar_init(&tl->qk_done[i], 1); mbar_init(&tl->p_full[i], 4); mbar_init(&tl->pv_done[i], 1); }
    mbar_init(&tl->o_free, 4);
    mbar_init(&tl->met, 4);
    mbar_init(&tl->q_ready, 4);
    mbar_fence_init();
    tl->start_e = -1;
    tl->warm = PPlanHead{1, 1, 1, -1, 0, 1, sh.rr_hint, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  } else if (warp == kWPlan) {
    if (lane == 0) tma_prefetch_desc(&tmQ);
    else if (lane == 1) tma_prefetch_desc(&tmK.map);
    else if (lane == 2) tma_prefetch_desc(&tmV.map);
  } else if (warp == kWIssue) {
    tmem_alloc(&tl->tmem_base, 256);
    tmem_relinquish();
  }
  // Rows that no box brings are zeros: products with them cost least power, and this kernel runs into the power limit
  if (warp < 4) {
#pragma unroll 4
    for (int i = tid; i < Geo::kQTile / 16; i += 128) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async();
  }
  // What is above may overlap the joining kernel of the call before; what is below reads and writes memory.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // ---- this CTA's share [us, ue) of all units, and the entry it begins in
  const int nE = p.batch * p.hkv, nE2 = 2 * nE;
  constexpr int kWarps = kThreads / 32, kKeep = 2048;
  int* kept = reinterpret_cast<int*>(tl->stage);          // weights of the first entries; nobody stages anything yet
  auto div = [](long long x, int y) { return x < 0x7fffffffll ? (long long)((uint32_t)x / (uint32_t)y) : x / y; };   // 64-bit: a microsecond
  long long U = 0, share = 0, us = 0, ue = 0;
  // One copy of the loop for both passes, here and wherever code is first met on the way to the first load: a cold
  // instruction costs some 35 cycles when all SMs fetch the same lines.
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    long long base = 0;
#pragma unroll 1
    for (int e0 = 0; e0 < nE2 && (pass == 0 || base <= us); e0 += kThreads) {
      const int e = e0 + tid;
      int w = 0;
      if (e < nE2) {
        if (pass == 0 || e >= kKeep) {
          const Entry x = entry_of(sh, e, nE, p.hkv);
          const PagedRequest r = paged_request(p, x.b);
          const int ns = item_count(sh, r.n);
#pragma unroll 1
          for (int s = x.half; s < ns; s += 2) w += item_weight<BS>(p, sh, r, x.kvh, s);
          if (e < kKeep) kept[e] = w;
        } else {
          w = kept[e];
        }
      }
      if (pass == 0) {
        U += w;
        continue;
      }
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
    if (pass) break;
#pragma unroll
    for (int o = 16; o; o >>= 1) U += __shfl_xor_sync(0xffffffffu, U, o);
    if (lane == 0) tl->warp_sums[warp] = U;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    U = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) U += tl->warp_sums[w];
    // CTA c has the units [c * share, (c + 1) * share)
    share = max((long long)sh.least, div(U + sh.ctas - 1, sh.ctas));
    us = min(U, cta * share);
    ue = min(U, us + share);
    if (us >= ue) break;
  }
  __syncthreads();
  const uint32_t tmem = tl->tmem_base, tS = tmem, tO = tmem + 128;
  const bool tree = p.tree_mask != nullptr;
  const int G = p.hq / p.hkv;

  if (warp == kWPlan) {
    // ============================================================ planner and TMA producer
    // One warp lists the next blocks and loads them: while it lists, the tiles it has loaded last are being computed.
    if (lane == 0) recs[cta].valid = 0;
    int k = 0;             // plans so far
    bool ok = true;
    PPlan* pl = nullptr;
    int n = 0;
    int e = tl->start_e;
    const int per_entry = sh.box == BS ? 1 : BS / sh.box;      // pages of a block
    const int most = min(kSeg, kSegPages / per_entry), batch = min(most, 32);
    const uint32_t all_pages = (1u << per_entry) - 1u;
    long long base = tl->start_base;
    // the loads' own ring: the 16-bit tiles, or the e4m3 tiles that the converters read
    constexpr int NLK = KV8 ? NR : NK, NLV = KV8 ? NR : NV;
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
    // the caches pass through L2 once; what else is there (this code, the tables) had better stay
    uint64_t policy;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    uint32_t rg = 0;       // tiles loaded
    int items = 0;
    for (; ok && us < ue && e >= 0 && e < nE2 && base < ue; ++e) {
      const Entry x = entry_of(sh, e, nE, p.hkv);
      const int b = x.b, kvh = x.kvh;
      const PagedRequest r = paged_request(p, b);
      const int n_items = item_count(sh, r.n);
      const int32_t* table = p.block_tables + (int64_t)b * p.table_stride;
      for (int si = x.half; ok && si < n_items && base < ue; si += 2) {
        const int w = item_weight<BS>(p, sh, r, kvh, si);
        if (base + w <= us) { base += w; continue; }
        const int ua = (int)max(us - base, 0ll), ub = (int)min(ue - base, (long long)w);
        const long long item0 = base;
        base += w;
        const ItemKeys ik = item_keys<BS>(p, sh, r, si);
        const int tok0 = ik.tok0, ntok = min(sh.tt, r.n - tok0), r0 = ik.r0;
        const int head0 = kvh * G + ik.chunk * sh.gt, gcnt = min(sh.gt, G - ik.chunk * sh.gt);
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
        int ahead = 0;              // one pattern row: the first blocks of this share
        bool simple = nf == 1 && r0 < p.n_rows;
        if (simple) {
          // its last 32 entries and the share's first ones in one round of loads
          const int hp = p.h_pat == 1 ? 0 : p.h_pat == p.hkv ? kvh : head0;
          const int32_t* cr = p.crow + (int64_t)hp * p.crow_sh + r0;
          my_cols = p.col + (int64_t)hp * p.col_sh;
          cur = __ldg(cr);
          end = __ldg(cr + 1);
          if (!BSA_IN_BOUNDS(cur >= 0 && cur <= end && (p.col_sh == 0 || end <= p.col_sh), wait_status, 821)) end = cur;
          const int c = end - 1 - lane >= cur ? __ldg(my_cols + end - 1 - lane) : -1;
          ahead = cur + ua + lane < end ? __ldg(my_cols + cur + ua + lane) : 0;
          const uint32_t past = __ballot_sync(0xffffffffu, c >= r0);
          my_tb = __reduce_or_sync(0xffffffffu, c >= r0 && c - r0 < 32 ? 1u << (c - r0) : 0u);
          end -= __popc(past);
          while (past == 0xffffffffu && end > cur && __ldg(my_cols + end - 1) >= r0) {     // no causal pattern's row
            const int z = __ldg(my_cols + --end) - r0;
            if (z < 32) my_tb |= 1u << z;
          }
        } else if (lane < nf && fg < gcnt && r0 + fx < p.n_rows) {
          const int hp = pattern_head(head0 + fg, p.h_pat, p.hq, p.hkv);
          const int32_t* cr = p.crow + (int64_t)hp * p.crow_sh + r0 + fx;
          my_cols = p.col + (int64_t)hp * p.col_sh;
          cur = __ldg(cr);
          end = __ldg(cr + 1);
          if (!BSA_IN_BOUNDS(cur >= 0 && cur <= end && (p.col_sh == 0 || end <= p.col_sh), wait_status, 821)) end = cur;
          // from the end: a row of a causal pattern ends with its diagonal.  Two loads at a time
          while (end > cur) {
            const int c1 = __ldg(my_cols + end - 1), c2 = __ldg(my_cols + max(end - 2, cur));
            if (c1 < r0) break;
            if (c1 - r0 < 32) my_tb |= 1u << (c1 - r0);
            if (--end == cur || c2 < r0) break;
            if (c2 - r0 < 32) my_tb |= 1u << (c2 - r0);
            --end;
          }
        }
        const int beg0 = __shfl_sync(0xffffffffu, cur, 0), n0 = __shfl_sync(0xffffffffu, end, 0) - beg0;
        const int32_t* cols0 = p.col + (int64_t)pattern_head(head0, p.h_pat, p.hq, p.hkv) * p.col_sh;
        // Units 0 .. n0 - 1 stand for the first row's blocks; who has unit n0 has the drafts, too, and what is behind
        // it is nobody's (n0 < w)
        if (ua > n0) continue;
        const bool owns_tail = ub > n0;
        const int ia = ua, ib = min(ub, n0);
        const int part = ua == 0 && owns_tail ? -1 : ua > 0 ? 2 * cta : 2 * cta + 1;
        if (ua == 0 && !owns_tail && lane == 0) {
          PagedRec rec = {1, b, r.t0, r.n, r.L, tok0, ntok, head0, gcnt, (int)div(item0 + n0, (int)min(share, 0x7fffffffll))};
          recs[cta] = rec;
        }
        // up to 16 rows are repeated (repetitions of 32 and 64 rows, with more to add up at the item's end, were not built)
        const int rr = sh.cr == 16 && ntok <= sh.ct ? 16 : 128;
        n = 0;
        bool first = true, begins = true;
        auto open = [&]() {
          const int pb = k & 1;
          if (!wait_for(&tl->plan_free[pb], ((k >> 1) & 1) ^ 1, wait_status, 1001)) { ok = false; return; }
          pl = &tl->plan[pb];
          pl->tb[lane] = my_tb;
          if (lane < 8) pl->dm[lane] = my_dm;
          if (lane < 2) pl->special[lane] = 0u;
          if (lane == 0) {
            pl->valid = 1;
            pl->first = first;
            pl->part = part;
            pl->rr = rr;
            pl->b = b; pl->t0 = r.t0; pl->n_new = r.n; pl->L = r.L; pl->kvh = kvh; pl->head0 = head0; pl->gcnt = gcnt;
            pl->tok0 = tok0; pl->ntok = ntok; pl->Lp = ik.Lp; pl->r0 = r0; pl->Sp = ik.Sp;
          }
          first = false;
          n = 0;
          __syncwarp();
        };
        auto publish = [&](bool last) {
          const int nt = (n + E - 1) / E;
          if (lane == 0) { pl->n = n; pl->nt = nt; pl->last = last; }
          __syncwarp();
          if (lane == 0) mbar_arrive(&tl->plan_full[k & 1]);
          ++k;
          // K one tile ahead of V: its slot comes free earlier
          for (int t = 0; ok && t < 2 * nt; ++t) {
            const bool is_v = t == 2 * nt - 1 || (t > 0 && !(t & 1));
            const int j = t == 2 * nt - 1 ? nt - 1 : is_v ? t / 2 - 1 : (t + 1) / 2;
            const uint32_t x = rg + (uint32_t)j;
            const int s = is_v ? x % NLV : x % NLK;
            uint64_t* full = (is_v ? vf : kf) + s;
            if (!wait_for((is_v ? ve : ke) + s, ((is_v ? x / NLV : x / NLK) & 1) ^ 1, wait_status, is_v ? 1014 : 1013)) { ok = false; break; }
            if (lane == 0) mbar_expect_tx(full, kLoadBytes);
            __syncwarp();
            if (lane < per * subs) {
              const int idx = j * E + my_e;
              int pg = -1, slot = p.page_size;             // outside the page: the box is filled with zeros
              if (idx < n) {
                const uint32_t c = pl->col[idx];
                pg = pl->page[idx * per_entry + my_page];
                if (pg >= 0) slot = (int)(((c & kColMask) * BS + my_off) & (uint32_t)(p.page_size - 1));
              }
              (void)BSA_IN_BOUNDS(pg < p.num_pages && (pg < 0 || slot + sh.box <= p.page_size), wait_status, 824);
              uint8_t* dst = (is_v ? sv : sk) + s * kLoadBytes + (KV8 ? my_row * D : my_sub * 8192 + my_row * 128);
              tma_load_tile_hint(dst, is_v ? &tmV : &tmK, full, KV8 ? 0 : my_sub * 64, slot, kvh, max(pg, 0), policy);
            }
            __syncwarp();
            if (t == 0 && begins) {
              // Q behind the first K
              if (items > 0 && !wait_for(&tl->q_free, (items - 1) & 1, wait_status, 1012)) { ok = false; break; }
              ++items;
              const int pos = 128 / sh.cr, boxes = kSub * pos;
              if (lane == 0) mbar_expect_tx(&tl->q_full, (uint32_t)(boxes * sh.ct * sh.gt * 128));
              __syncwarp();
              if (lane < boxes) {
                const int at = lane & (pos - 1), c = lane / pos;      // at most 16 boxes
                (void)BSA_IN_BOUNDS(r.t0 + tok0 >= 0 && r.t0 + tok0 < p.total_q && head0 < p.hq, wait_status, 823);
                tma_load_3d(sQ + c * 16384 + at * sh.cr * 128, &tmQ, &tl->q_full, c * 64, head0,
                            r.t0 + tok0 + (rr == 128 ? at : 0) * sh.ct);
              }
              __syncwarp();
            }
          }
          begins = false;
          rg += (uint32_t)nt;
        };
        open();
        if (!ok) break;
        bool windows = nf > 1;
        // flags of a block that all rows attend (those that there are: heads of the last piece, rows of the pattern)
        const uint32_t all_rows = windows ? __ballot_sync(0xffffffffu, lane < nf && fg < gcnt) : 1u;
        const int ny = owns_tail ? (ik.Sp - 1) / BS - r0 + 1 : 0;
        int clo = 0, chi = 0, wc = 0, wi = kWindow;
        if (windows) {
          // several rows: the union of their columns inside the share's range, a window of columns at a time
          // (a share's end is the next one's beginning; behind the first row's last block there is only the context's end)
          auto border = [&](int at) { return at == 0 ? 0 : at < n0 ? __ldg(cols0 + beg0 + at) : r0; };
          clo = border(ia);
          chi = owns_tail ? r0 : border(ib);
          if (clo > 0) {
            int lo = cur, hi = end;
            while (lo < hi) {
              const int mid = (lo + hi) >> 1;
              if (__ldg(my_cols + mid) < clo) lo = mid + 1; else hi = mid;
            }
            cur = lo;
          }
        }
        // then, and with one pattern row at once: its entries [ia, ib), behind them the blocks that hold drafts
        int i = ia;
        while (ok) {
          bool on, done = false;
          int col;
          uint32_t fl, tail = 0u;
          if (windows) {
            if (wi >= kWindow) {
              const int next = cur < end ? __ldg(my_cols + cur) : 0x7fffffff;
              wc = max(__reduce_min_sync(0xffffffffu, next), 0);
              if (wc >= chi) {
                windows = false;
                i = ib;
                continue;
              }
              const int stop = (int)min((long long)wc + kWindow, (long long)chi);
              for (int z = lane; z < kWindow; z += 32) tl->window[z] = 0u;
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
              wi = 0;
            }
            fl = wi + lane < kWindow ? tl->window[wi + lane] : 0u;
            on = fl != 0u;
            col = wc + wi + lane;
          } else {
            done = i >= ib + ny;
            on = i + lane < ib + ny;
            fl = 1u;
            col = ahead;
            if (i + lane >= ib) { col = r0 + i + lane - ib; tail = kTailFlag; }
            if (i + batch + lane < ib) ahead = __ldg(cols0 + beg0 + i + batch + lane);
          }
          on = on && lane < batch;
          wi += batch;
          i += batch;
          // ---- up to `batch` blocks, one per lane, in order
          const uint32_t who = __ballot_sync(0xffffffffu, on);
          const int cnt = __popc(who);
          if (done || n + cnt > most) {
            publish(done);
            if (done || !ok) break;
            open();
            if (!ok) break;
          }
          if (on) {
            const int at = n + __popc(who & ((1u << lane) - 1u));
            const long long s0 = ((long long)col * BS) >> sh.page_shift;
            uint32_t have = 0;
#pragma unroll 1
            for (int z = 0; z < per_entry; ++z) {
              const int pg = page_of(table, s0 + z, r.stored ? p.max_pages : 0, p.num_pages);
              pl->page[at * per_entry + z] = pg;
              have |= (pg >= 0 ? 1u : 0u) << z;
            }
            pl->col[at] = ((uint32_t)col & kColMask) | have << 23 | tail;
            pl->fl[at] = fl;
            if (tail || have != all_pages || fl != all_rows) atomicOr(&pl->special[at >> 5], 1u << (at & 31));
          }
          n += cnt;
        }
      }
    }
    if (ok) {
      const int pb = k & 1;
      if (wait_for(&tl->plan_free[pb], ((k >> 1) & 1) ^ 1, wait_status, 1002)) {
        if (lane == 0) {
          tl->plan[pb].valid = -1;
          mbar_arrive(&tl->plan_full[pb]);
        }
      }
    }
  } else if (warp == kWIssue) {
    // ============================================================ MMA issuer
    uint32_t idesc_qk = umma_idesc(BE, 128, 64, false, false);
    if (p.sm_scale < 0.f) idesc_qk |= 1u << 13;        // A negated: the maximum of the scaled logits stays a maximum
    const uint32_t idesc_pv = umma_idesc(BE, 128, D, false, true);
    const uint64_t qdesc = umma_desc_sw128(smem_u32(sQ), 16, 1024);
    const uint64_t kdesc = umma_desc_sw128(smem_u32(sK), 16, 1024);
    const uint64_t vdesc = umma_desc_sw128(smem_u32(sV), 8192, 1024);
    uint32_t g = 0;                      // tiles before this plan
    int items = 0;
    bool ok = true, started = false;
    for (int k = 0; ok; ++k) {
      const int pb = k & 1;
      if (!wait_for(&tl->plan_full[pb], (k >> 1) & 1, wait_status, 1021)) break;
      const PPlan* pl = &tl->plan[pb];
      if (pl->valid < 0) break;
      const int nt = pl->nt, last = pl->last;
      const bool split = pl->rr == 128;       // both terms of P in a row; else they have rows of their own
      if (pl->first) {
        if (!wait_for(QCONV ? &tl->q_ready : &tl->q_full, items & 1, wait_status, 1022)) break;
        ++items;
        started = false;
      }
      auto qk = [&](int j) -> bool {
        const uint32_t x = g + (uint32_t)j;
        const int s = x % NK, sb = x & 1;
        if (!wait_for(&tl->k_full[s], (x / NK) & 1, wait_status, 1023)) return false;
        tc_fence_after();
        const uint64_t kd = kdesc + (uint64_t)((s * kTile) >> 4);
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            tc_mma_ss(tS + sb * 64, qdesc + (uint64_t)(((i >> 2) * 16384 + (i & 3) * 32) >> 4),
                      kd + (uint64_t)(((i >> 2) * 8192 + (i & 3) * 32) >> 4), idesc_qk, i ? 1u : 0u);
          tc_commit(&tl->qk_done[sb]);
          tc_commit(&tl->k_free[s]);
          if (last && j == nt - 1) tc_commit(&tl->q_free);
        }
        __syncwarp();
        return true;
      };
      for (int j = 0; ok && j < nt && j < 2; ++j) ok = qk(j);
      for (int j = 0; ok && j < nt; ++j) {
        const uint32_t x = g + (uint32_t)j;
        const int s = x % NV, sb = x & 1;
        if (!wait_for(&tl->v_full[s], (x / NV) & 1, wait_status, 1024)) { ok = false; break; }
        if (!wait_for(&tl->p_full[sb], (x >> 1) & 1, wait_status, 1025)) { ok = false; break; }
        // the item before has read O
        if (!started && items > 1 && !wait_for(&tl->o_free, (items - 2) & 1, wait_status, 1026)) { ok = false; break; }
        tc_fence_after();
        const uint64_t vd = vdesc + (uint64_t)((s * kTile) >> 4);
        const uint32_t acc0 = started ? 1u : 0u;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc_mma_ts(tO, tS + sb * 64 + (split ? (kk >> 1) * 32 + (kk & 1) * 8 : kk * 8), vd + (uint64_t)((kk * 2048) >> 4),
                      idesc_pv, kk ? 1u : acc0);
          if (split) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)    // the low terms of P, 16 columns behind the high ones of the same 32 keys
              tc_mma_ts(tO, tS + sb * 64 + (kk >> 1) * 32 + 16 + (kk & 1) * 8, vd + (uint64_t)((kk * 2048) >> 4), idesc_pv, 1u);
          }
          tc_commit(&tl->pv_done[sb]);
          tc_commit(&tl->v_free[s]);
        }
        __syncwarp();
        started = true;
        if (j + 2 < nt) ok = qk(j + 2);
      }
      if (!ok) break;
      g += (uint32_t)nt;
      if (elect_one()) mbar_arrive(&tl->plan_free[pb]);
      __syncwarp();
    }
  } else if (warp < 4) {
    // ============================================================ softmax and epilogue
    const int r = tid;                        // tile row = TMEM lane
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    const uint32_t tSl = tS + lane_off, tOl = tO + lane_off;
    const float scale2_all = fabsf(p.sm_scale) * (KV8 ? p.k_scale : 1.f) * kLog2e;
    float scale2 = scale2_all;
    const float v_scale = KV8 ? p.v_scale : 1.f;
    constexpr float kShift = kTermShift<BE>;
    const bool wide = reinterpret_cast<uintptr_t>(p.o) % 16 == 0 && p.o_st % 8 == 0 && p.o_sh % 8 == 0;
    uint32_t gs = 0, meets = 0;               // tiles so far; joint waits
    bool alive = true;
    // all four warps
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(&tl->met);
      return wait_for(&tl->met, meets++ & 1, wait_status, 1036);
    };
    // the row's own state over an item
    float m_used = -INFINITY, l = 0.f;
    int f = 0, i_tok = 0, head = 0, pos = 0, mine = 0, rep = 0;
    uint32_t tbits = 0;
    uint64_t fm = 0;
    bool row_ok = false, warp_live = false;
    int q_items = 0;
    // Round -1 is a rehearsal: a tile and an item's end without a valid row, on O's columns and no barrier but the warps'
    // own, so that the code has been fetched by the time the first tile comes.
    for (int k = -1; alive; ++k) {
      const bool dry = k < 0;
      const int pb = k & 1;
      if (!dry && !wait_for(&tl->plan_full[pb], (k >> 1) & 1, wait_status, 1031)) break;
      const PPlan* pl = dry ? static_cast<const PPlan*>(&tl->warm) : &tl->plan[pb];   // nothing behind the head is read then
      if (pl->valid < 0) break;
      const int nt = pl->nt, n = pl->n, rr = pl->rr;
      if (pl->first) {
        const int q = r & (rr - 1), qq = q & (sh.cr - 1);
        const int tl_row = q / sh.cr * sh.ct + qq / sh.gt, g = qq % sh.gt, tok = tl_row;
        rep = warp;
        row_ok = qq < sh.ct * sh.gt && tok < pl->ntok && g < pl->gcnt;
        warp_live = __any_sync(0xffffffffu, row_ok);
        i_tok = pl->tok0 + tok;
        head = pl->head0 + g;
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
          f = (sh.shared ? x : x * sh.gt + g) & 31;
          tbits = pl->tb[f];
          if (tree) {
#pragma unroll
            for (int y = 0; y < 8; ++y)
              if ((tbits >> y) & 1u) fm |= pl->dm[y];
            fm &= word;
          }
        }
        if (QCONV && !dry) {
          // this thread's row of Q from bf16 to f16, where it lies
          if (!wait_for(&tl->q_full, q_items & 1, wait_status, 1038)) break;
          ++q_items;
          uint32_t big = 0;
#pragma unroll 1
          for (int c = 0; c < kSub * 8; ++c) {
            const uint4 v = *reinterpret_cast<const uint4*>(sQ + (c >> 3) * 16384 + r * 128 + ((c ^ r) & 7) * 16);
            big = __vmaxu2(big, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
          }
          const int ex = (int)(max(big & 0xffffu, big >> 16) >> 7);
          const int up = ex == 255 ? 0 : min(max(140 - ex, -126), 126);
          const float by = __int_as_float((127 + up) << 23);
          scale2 = scale2_all * __int_as_float((127 - up) << 23);
#pragma unroll 1
          for (int c = 0; c < kSub * 8; ++c) {
            uint4* at = reinterpret_cast<uint4*>(sQ + (c >> 3) * 16384 + r * 128 + ((c ^ r) & 7) * 16);
            uint4 v = *at;
            auto conv = [&](uint32_t x) {
              return ppack2<false>(__uint_as_float(x << 16) * by, __uint_as_float(x & 0xffff0000u) * by);
            };
            v.x = conv(v.x); v.y = conv(v.y); v.z = conv(v.z); v.w = conv(v.w);
            *at = v;
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tl->q_ready);
        }
      }
      // blocks past the last one of a tile that is not full are as special as any
      const uint64_t special = dry ? 0ull : ((uint64_t)pl->special[1] << 32 | pl->special[0]) | ~low_bits(n);
      // ---- one K/V tile; this repetition weighs CW of its 64 keys
      auto softmax_tile = [&](auto cw, uint64_t M, uint32_t tSb) -> bool {
        constexpr int CW = decltype(cw)::value;
        static_assert(CW == 64 || CW == 16, "whole tiles or quarters");
        // 32 logits at a time, read once for the maximum and once more for the weights: half the code of all 64 at once
        // (instruction fetch is a fifth of this kernel's stalls) and half the registers
        constexpr int BL = CW == 64 ? 32 : 16;
        const int c0 = CW == 64 ? 0 : rep * CW;
        const uint64_t mc = CW == 64 ? M : (M >> c0) & low_bits(CW);
        const bool att = mc != 0ull, masked = __any_sync(0xffffffffu, mc != low_bits(CW));
        uint32_t sv[BL];
        auto logits = [&](int h) {
          if constexpr (CW == 64) tmem_ld32(tSb + h * 32, sv);
          else tmem_ld16(tSb + c0, sv);
          tmem_ld_wait();
          if (masked) {
            const uint32_t m32 = (uint32_t)(mc >> (h * 32));
#pragma unroll
            for (int c = 0; c < BL; ++c)
              if (!((m32 >> c) & 1u)) sv[c] = 0xff800000u;
          }
        };
        float mt[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int h = 0; h < CW / BL; ++h) {
          logits(h);
#pragma unroll
          for (int c = 0; c < BL; c += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i) mt[i] = pmax3(mt[i], __uint_as_float(sv[c + 2 * i]), __uint_as_float(sv[c + 2 * i + 1]));
        }
        const float mx = pmax3(pmax3(mt[0], mt[1], mt[2]), mt[3], mt[3]) * scale2;     // NaN stays in m_used and in l
        float alpha = 1.f;
        bool need = false;
        if (mx != -INFINITY) {
          if (m_used == -INFINITY) {
            m_used = mx;                      // O's row is 0 so far
          } else if (row_ok && mx > m_used + kRescale) {
            alpha = pex2(m_used - mx);
            m_used = mx;
            l *= alpha;
            need = true;
          }
        }
        const bool any = __any_sync(0xffffffffu, need);
        const bool live = att && row_ok && m_used != -INFINITY;
        const float neg_m = kShift - m_used;
        const uint64_t scale_2 = f32x2(scale2, scale2), neg_m2 = f32x2(neg_m, neg_m);
        uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll 1
        for (int h = 0; h < CW / BL; ++h) {
          if (CW == 64) logits(h);            // a quarter's are still there
          uint32_t pk[BL / 2], pq[BL / 2];
          if (live) {
#pragma unroll
            for (int c = 0; c < BL / 2; ++c) {
              float x0, x1;
              f32x2_split(fma_f32x2(f32x2(sv[2 * c], sv[2 * c + 1]), scale_2, neg_m2), x0, x1);
              const float p0 = pex2(x0), p1 = pex2(x1);
              sum2[c & 1] = add_f32x2(sum2[c & 1], f32x2(p0, p1));
              psplit<BE>(p0, p1, pk[c], pq[c]);
            }
          } else {
#pragma unroll
            for (int c = 0; c < BL / 2; ++c) pk[c] = pq[c] = 0u;
          }
          if constexpr (CW == 64) {
            // both terms over the logits that they come from, so that the other half is still there
            tmem_st16(tSb + h * 32, pk);
            tmem_st16(tSb + h * 32 + 16, pq);
          } else {
            // this repetition's keys, and no weight on the others'
            uint32_t z[BL / 2];
#pragma unroll
            for (int c = 0; c < BL / 2; ++c) {
              z[c] = 0u;
              if (lane >= 16) pk[c] = pq[c];
            }
#pragma unroll
            for (int i = 0; i < 64 / CW; ++i) {
              const uint32_t at = (uint32_t)(i * (CW / 2));
              if (i == rep) tmem_st8(tSb + at, pk);
              else tmem_st8(tSb + at, z);
            }
          }
        }
        float s4[4];
        f32x2_split(sum2[0], s4[0], s4[1]);
        f32x2_split(sum2[1], s4[2], s4[3]);
        l += (s4[0] + s4[1]) + (s4[2] + s4[3]);
        if (any && mine > 0) {
          // rows whose maximum moved: rescale their O once the product before has landed
          if (!wait_for(&tl->pv_done[(gs - 1) & 1], ((gs - 1) >> 1) & 1, wait_status, 1034)) return false;
          tc_fence_after();
#pragma unroll 1
          for (int ch = 0; ch < D / 16; ++ch) {
            uint32_t o[16];
            tmem_ld16(tOl + ch * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st16(tOl + ch * 16, o);
          }
        }
        return true;
      };
      for (int j = 0; j < nt; ++j, gs += dry ? 0 : 1) {
        const int sb = gs & 1, s = gs % NV;
        // ---- which of the tile's 64 keys this row attends, before the logits are there
        uint64_t M = ~0ull;
        int clear0 = 64;                      // rows of V that hold no key of this item, from here to the end of their block
        bool clear = false, any_att = warp_live;
        if ((special >> (j * E)) & low_bits(E)) {
          M = 0;
#pragma unroll 1
          for (int en = 0; en < E; ++en) {
            const int idx = j * E + en;
            uint64_t me = 0;
            if (idx < n) {
              const uint32_t c = pl->col[idx];
              if (!(c & kTailFlag)) {
                if ((pl->fl[idx] >> f) & 1u) me = low_bits(BS);
              } else {
                const int y = (int)(c & kColMask) - pl->r0, s0 = (int)(c & kColMask) * BS;
                const int nc = min(max(pl->Lp - s0, 0), BS);           // context tokens of the block
                if (nc && (tbits & 1u)) me = low_bits(nc);             // only block r0 holds any
                if (tree) {
                  const int d0 = s0 + nc - pl->L;                      // first draft of the block
                  if (d0 < 64) me |= (fm >> d0) << nc;
                } else if (y < 32 && ((tbits >> y) & 1u)) {
                  me |= low_bits(min(max(pos - s0 + 1, 0), BS));
                }
                me &= low_bits(BS);
                const int len = pl->Sp - s0;
                if (len < BS) { clear = true; clear0 = en * BS + len; }
              }
              const uint32_t have = (c >> 23) & 0xffu;
              if (me && have != low_bits(BS / sh.box))
                for (int i = 0; i < BS / sh.box; ++i)
                  if (!((have >> i) & 1u)) me &= ~(low_bits(sh.box) << (i * sh.box));
            }
            M |= me << (en * BS);
          }
          any_att = __any_sync(0xffffffffu, row_ok && M != 0ull);
          if (!row_ok) M = ~0ull;             // nobody reads these rows: nothing to mask
        }
        if (!dry && !wait_for(&tl->qk_done[sb], (gs >> 1) & 1, wait_status, 1032)) { alive = false; break; }
        tc_fence_after();
        if (clear) {
          // keys behind the item's end: P is 0 there, and 0 times whatever the page holds has to be 0, too
          // (two V slots at least: this tile's barrier cannot still be in the phase of the tile before in its slot, whose
          // product was over before this tile's logits were there)
          if (!wait_for(&tl->v_full[s], (gs / NV) & 1, wait_status, 1033)) { alive = false; break; }
          uint8_t* vt = sV + s * kTile;
          const int cend = (clear0 / BS + 1) * BS;
          for (int q = r; q < (cend - clear0) * kSub * 8; q += 128) {
            const int row = clear0 + q / (kSub * 8), c = (q / 8) % kSub, ch = q & 7;
            *reinterpret_cast<uint4*>(vt + c * 8192 + row * 128 + ch * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async();
        }
        if (warp_live || dry) {
          const uint32_t tSb = dry ? tOl : tSl + sb * 64;
          if (any_att || dry) {
            const bool fine = rr == 128 ? softmax_tile(std::integral_constant<int, 64>{}, M, tSb)
                                        : softmax_tile(std::integral_constant<int, 16>{}, M, tSb);
            if (!fine) { alive = false; break; }
          } else {
            uint32_t z[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) z[c] = 0u;
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_st16(tSb + c * 16, z);
          }
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0 && !dry) mbar_arrive(&tl->p_full[sb]);
        ++mine;
      }
      if (!alive) break;
      if (pl->last) {
        // ---- the item's result
        if (!dry && !wait_for(&tl->pv_done[(gs - 1) & 1], ((gs - 1) >> 1) & 1, wait_status, 1035)) break;
        tc_fence_after();
        const int part = pl->part;
        const int item_row = (i_tok - pl->tok0) * sh.gt + head - pl->head0;
        // where the row goes: the output, or its place among the parts
        (void)BSA_IN_BOUNDS(!row_ok || part < 0 || (item_row < sh.rows_cap && part < 2 * sh.ctas), wait_status, 825);
        uint8_t* orow = part < 0 ? reinterpret_cast<uint8_t*>(p.o) + ((int64_t)(pl->t0 + i_tok) * p.o_st + (int64_t)head * p.o_sh) * 2
                                 : reinterpret_cast<uint8_t*>(part_o + ((int64_t)part * sh.rows_cap + item_row) * D);
        auto release_o = [&]() {               // the next item's first product may overwrite O
          tc_fence_before();
          __syncwarp();
          if (lane == 0 && !dry) mbar_arrive(&tl->o_free);
        };
        const PagedRequest rq{pl->t0, pl->n_new, pl->L};
        if (rr == 128) {
          // rows straight from the accumulator
          float check = 0.f;
          const float inv = l > 0.f ? v_scale / l : 0.f;
          uint8_t* stg = reinterpret_cast<uint8_t*>(tl->stage) + warp * 2048;
#pragma unroll 1
          for (int ch = 0; ch < D / 32; ++ch) {
            uint32_t o[32];
            tmem_ld32(tOl + ch * 32, o);
            tmem_ld_wait();
            if (ch == D / 32 - 1) release_o();
            uint32_t wd[16];
            if (part < 0) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float x0 = __uint_as_float(o[2 * i]) * inv, x1 = __uint_as_float(o[2 * i + 1]) * inv;
                check = fmaf(x0, 0.f, fmaf(x1, 0.f, check));      // NaN once one of them is no finite number
                wd[i] = l == 0.f ? 0u : ppack2<BF16>(x0, x1);
              }
            }
            if (part >= 0 || wide) {
              // 64-byte pieces of the warp's 32 rows (32 columns in 16 bits, or twice 16 in fp32): 16-byte words swizzled by
              // the row pair, then lane L stores word L % 4 of rows L / 4, L / 4 + 8, ...  (Stored by its own thread, a part's
              // row took 32 separate sectors an instruction: 18 thousand cycles an item.)
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
                if (part < 0 && hf) break;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  uint4 v = make_uint4(wd[4 * i], wd[4 * i + 1], wd[4 * i + 2], wd[4 * i + 3]);
                  if (part >= 0) v = make_uint4(o[hf * 16 + 4 * i], o[hf * 16 + 4 * i + 1], o[hf * 16 + 4 * i + 2], o[hf * 16 + 4 * i + 3]);
                  *reinterpret_cast<uint4*>(stg + lane * 64 + ((i ^ ((lane >> 1) & 3)) * 16)) = v;
                }
                __syncwarp();
                const int pc = lane & 3;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int sr = i * 8 + (lane >> 2);
                  const uint4 val = *reinterpret_cast<const uint4*>(stg + sr * 64 + ((pc ^ ((sr >> 1) & 3)) * 16));
                  const long long dst = __shfl_sync(0xffffffffu, (long long)reinterpret_cast<uintptr_t>(orow), sr);
                  const int okr = __shfl_sync(0xffffffffu, (int)row_ok, sr);
                  if (okr && (part >= 0 || ch * 32 + pc * 8 < p.d))
                    *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(dst) + (part >= 0 ? ch * 128 + hf * 64 : ch * 64) + pc * 16) = val;
                }
                __syncwarp();
              }
            } else if (row_ok) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                if (ch * 32 + 2 * i < p.d) reinterpret_cast<uint16_t*>(orow)[ch * 32 + 2 * i] = (uint16_t)wd[i];
                if (ch * 32 + 2 * i + 1 < p.d) reinterpret_cast<uint16_t*>(orow)[ch * 32 + 2 * i + 1] = (uint16_t)(wd[i] >> 16);
              }
            }
          }
          if (part >= 0) {
            if (row_ok) part_ml[(int64_t)part * sh.rows_cap + item_row] = make_float2(m_used, l);
          } else {
            if (row_ok && p.lse)
              p.lse[(int64_t)head * p.lse_sh + pl->t0 + i_tok] = l > 0.f ? (m_used - kShift + log2f(l)) * kLn2 : -INFINITY;
            // an infinity or NaN got into the row: attended or not, the definition says what it is
            uint32_t redo = __ballot_sync(0xffffffffu, row_ok && l != 0.f && (check != 0.f || !(l > 0.f)));
            __syncwarp();                     // other lanes write the row again
            while (redo) {
              const int src = __ffs(redo) - 1;
              redo &= redo - 1;
              paged_row<T16, C8>(p, pl->b, rq, __shfl_sync(0xffffffffu, i_tok, src), __shfl_sync(0xffffffffu, head, src), lane);
            }
          }
        } else {
          // the repetitions' parts are weighed and added, some columns at a time, by all four warps.  Rows in use are the
          // first nr (at most 16) of a part.  Parts: the warps' high terms, and their low terms under the same weight
          constexpr int P = 4;
          const int nr = dry ? 4 : pl->ntok * sh.gt;
          const int q = lane & 15;
          if (lane < nr) {
            tl->jm[rep * nr + q] = m_used;
            tl->jl[rep * nr + q] = l;
          }
          if (!meet()) break;
          if (r < nr) {
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int i = 0; i < P; ++i)
              if (tl->jl[i * nr + r] != 0.f) M = fmaxf(M, tl->jm[i * nr + r]);
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const float li = tl->jl[i * nr + r], a = li != 0.f ? pex2(tl->jm[i * nr + r] - M) : 0.f;
              tl->jw[i * nr + r] = a;         // a part without weight is left out, not multiplied by 0
              if (li != 0.f) L += li * a;
            }
            tl->rm[r] = M;
            tl->rl[r] = L;
            tl->jbad[r] = !(L >= 0.f);
          }
          int shift = D == 64 ? 6 : 7;        // 2^shift columns at a time, 16 or more: what the stage holds
          while ((2 * P * nr) << shift > 2048) --shift;
          const int cols = 1 << shift;
          bool fine = true;
          for (int c0 = 0; c0 < D; c0 += cols) {
            float* buf = tl->stage;
            if (c0 && !meet()) { fine = false; break; }      // the columns before have been added up
            for (int c = 0; c < cols; c += 16) {
              uint32_t o[16];
              tmem_ld16(tOl + c0 + c, o);
              tmem_ld_wait();
              if (q < nr) {
                float* dst = buf + ((2 * rep + (lane >> 4)) * nr + q) * cols + c;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  reinterpret_cast<uint4*>(dst)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
              }
            }
            if (c0 + cols >= D) release_o();
            if (!meet()) { fine = false; break; }
            for (int i = r; i < nr << (shift - 1); i += 128) {
              const int row = i >> (shift - 1), c2 = (i & ((1 << (shift - 1)) - 1)) * 2;
              float x0 = 0.f, x1 = 0.f;
#pragma unroll
              for (int pp = 0; pp < P; ++pp) {
                const float a = tl->jw[pp * nr + row];
                const float2 v = *reinterpret_cast<const float2*>(buf + (2 * pp * nr + row) * cols + c2);
                const float2 u = *reinterpret_cast<const float2*>(buf + ((2 * pp + 1) * nr + row) * cols + c2);
                if (a != 0.f) {
                  x0 = fmaf(v.x + u.x, a, x0);
                  x1 = fmaf(v.y + u.y, a, x1);
                }
              }
              const int tok = (int)((row + 0.5f) * sh.inv_gt), g = row - tok * sh.gt;
              if (tok >= pl->ntok || g >= pl->gcnt) continue;
              if (part >= 0) {
                const int ir = tok * sh.gt + g;
                if (BSA_IN_BOUNDS(ir < sh.rows_cap && part < 2 * sh.ctas, wait_status, 826))
                  *reinterpret_cast<float2*>(part_o + ((int64_t)part * sh.rows_cap + ir) * D + c0 + c2) = make_float2(x0, x1);
                continue;
              }
              const float L = tl->rl[row], inv = L > 0.f ? v_scale / L : 0.f;
              x0 *= inv;
              x1 *= inv;
              if (L != 0.f && (!(fabsf(x0) < INFINITY) || !(fabsf(x1) < INFINITY))) tl->jbad[row] = 1;
              const uint32_t wd = L == 0.f ? 0u : ppack2<BF16>(x0, x1);
              uint16_t* dst = reinterpret_cast<uint16_t*>(p.o) + (int64_t)(pl->t0 + pl->tok0 + tok) * p.o_st +
                              (int64_t)(pl->head0 + g) * p.o_sh + c0 + c2;
              if (wide) {
                if (c0 + c2 < p.d) *reinterpret_cast<uint32_t*>(dst) = wd;
              } else {
                if (c0 + c2 < p.d) dst[0] = (uint16_t)wd;
                if (c0 + c2 + 1 < p.d) dst[1] = (uint16_t)(wd >> 16);
              }
            }
          }
          if (!fine || !meet()) break;        // the flags are complete
          for (int row = warp; row < nr; row += 4) {
            const int tok = (int)((row + 0.5f) * sh.inv_gt), g = row - tok * sh.gt;
            if (tok >= pl->ntok || g >= pl->gcnt) continue;
            const int t = pl->t0 + pl->tok0 + tok, h = pl->head0 + g;
            const float M = tl->rm[row], L = tl->rl[row];
            if (part >= 0) {
              if (lane == 0) part_ml[(int64_t)part * sh.rows_cap + tok * sh.gt + g] = make_float2(M, L);
            } else {
              if (p.lse && lane == 0) p.lse[(int64_t)h * p.lse_sh + t] = L > 0.f ? (M - kShift + log2f(L)) * kLn2 : -INFINITY;
              if (tl->jbad[row]) paged_row<T16, C8>(p, pl->b, rq, pl->tok0 + tok, h, lane);
            }
          }
          if (!meet()) break;                 // before the next item writes rm, rl and the flags
        }
      }
      __syncwarp();
      if (lane == 0 && !dry) mbar_arrive(&tl->plan_free[pb]);
    }
  } else if (KV8 && warp >= kWConv) {
    // ============================================================ e4m3 -> 16-bit tiles in the layout of the products
    uint32_t rg = 0;
    for (int k = 0;; ++k) {
      const int pb = k & 1;
      if (!wait_for(&tl->plan_full[pb], (k >> 1) & 1, wait_status, 1041)) break;
      const PPlan* pl = &tl->plan[pb];
      if (pl->valid < 0) break;
      const int nt = pl->nt;
      bool ok = true;
      // in the order of the loads: K a tile ahead of V
      for (int t = 0; ok && t < 2 * nt; ++t) {
        const bool is_v = t == 2 * nt - 1 || (t > 0 && !(t & 1));
        const int j = t == 2 * nt - 1 ? nt - 1 : is_v ? t / 2 - 1 : (t + 1) / 2;
        const uint32_t x = rg + (uint32_t)j;
        const int rs = x % NR, s = is_v ? x % NV : x % NK;
        const uint8_t* raw = is_v ? sRawV : sRawK;
        uint8_t* tile = is_v ? sV : sK;
        uint64_t* full = is_v ? tl->v_full : tl->k_full;
        uint64_t* empty = is_v ? tl->v_free : tl->k_free;
        uint64_t* rf = is_v ? tl->raw_v_full : tl->raw_k_full;
        uint64_t* re = is_v ? tl->raw_v_free : tl->raw_k_free;
        if (!wait_for(&rf[rs], (x / NR) & 1, wait_status, is_v ? 1044 : 1042)) { ok = false; break; }
        if (!wait_for(&empty[s], ((is_v ? x / NV : x / NK) & 1) ^ 1, wait_status, is_v ? 1045 : 1043)) { ok = false; break; }
        const uint8_t* src = raw + rs * Geo::kRawTile;
        uint8_t* dst = tile + s * kTile;
        // 16 values a lane and turn, the two warps in turns.  A lane keeps its place in the row, and its rows are 8 apart, so
        // that its addresses are a base and constants.  At D = 128 eight lanes take half of a row and the other half of its
        // neighbour: no bank twice, neither in the loads (rows of 128 bytes) nor in the stores (16-byte pieces 0, 2, 4, 6,
        // exclusive-or the row)
        constexpr int kPieces = D / 16, kRows = 32 / kPieces;          // 4 or 8 rows a turn
        const int set = lane >> 3, low = (lane >> 2) & 1;
        const int row = (warp - kWConv) * kRows + (D == 64 ? lane >> 2 : (set & 2) + ((set ^ low) & 1));
        const int pc = D == 64 ? lane & 3 : low * 4 + (lane & 3), c0 = (pc & 3) * 2;
        const uint8_t* from = src + row * D + pc * 16;
        uint8_t* base = dst + (pc >> 2) * 8192 + row * 128;
        const int a0 = (c0 ^ (row & 7)) * 16, a1 = ((c0 + 1) ^ (row & 7)) * 16;
        // Turns go four at a time, their loads before any store: the compiler cannot tell the tiles apart and would wait
        // for each turn's load (1000 cycles a tile of 64 x 128)
#pragma unroll
        for (int q0 = 0; q0 < 32 / kRows; q0 += 4) {
          uint4 v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] = *reinterpret_cast<const uint4*>(from + (q0 + q) * 2 * kRows * D);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t in[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
            uint32_t out[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              out[2 * i] = e4m3x2_to_f16((uint16_t)in[i]);
              out[2 * i + 1] = e4m3x2_to_f16((uint16_t)(in[i] >> 16));
            }
            *reinterpret_cast<uint4*>(base + (q0 + q) * 2 * kRows * 128 + a0) = make_uint4(out[0], out[1], out[2], out[3]);
            *reinterpret_cast<uint4*>(base + (q0 + q) * 2 * kRows * 128 + a1) = make_uint4(out[4], out[5], out[6], out[7]);
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&full[s]);
          mbar_arrive(&re[rs]);
        }
      }
      if (!ok) break;
      rg += (uint32_t)nt;
      __syncwarp();
      if (lane == 0) mbar_arrive(&tl->plan_free[pb]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWIssue) tmem_dealloc(tmem, 256);
}

// ------------------------------------------------------------------ joining
// CTA (c, y): the item that CTA c of the kernel above began and did not finish.  What bounds it is latency: a warp has
// eight (row, part) pairs in flight, four rows by two parts where there are few parts, one row by eight where there
// are many.
template <typename T16, typename C8, int D, int R>
__device__ __forceinline__ void join_rows(const bsa_paged_params& p, const PagedShape& sh, const PagedRec& rec, int c, int lane,
                                          const float2* __restrict__ part_ml, const float* __restrict__ part_o, float shift) {
  constexpr int V = D / 32, PU = 8 / R;
  const int parts = rec.last - c + 1, rows = rec.ntok * sh.gt;
  const float v_scale = sizeof(C8) == 1 ? p.v_scale : 1.f;
#pragma unroll 1
  for (int row0 = (blockIdx.y * 8 + (threadIdx.x >> 5)) * R; row0 < rows; row0 += gridDim.y * 8 * R) {
    float m[R], l[R], acc[R][V];
#pragma unroll
    for (int x = 0; x < R; ++x) {
      m[x] = -INFINITY;
      l[x] = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) acc[x][v] = 0.f;
    }
#pragma unroll 1
    for (int i0 = 0; i0 < parts; i0 += PU) {
      float2 ml[PU][R];
      float o[PU][R][V];
#pragma unroll
      for (int u = 0; u < PU; ++u) {
        const int i = i0 + u;
        const int64_t at = (int64_t)(i == 0 ? 2 * c + 1 : 2 * (c + i)) * sh.rows_cap + row0;
#pragma unroll
        for (int x = 0; x < R; ++x) {
          ml[u][x] = make_float2(0.f, 0.f);
          if (i < parts && row0 + x < rows) {
            ml[u][x] = __ldcg(part_ml + at + x);
            const float* src = part_o + (at + x) * D + lane * V;
            if constexpr (V == 4) *reinterpret_cast<float4*>(o[u][x]) = __ldcg(reinterpret_cast<const float4*>(src));
            else *reinterpret_cast<float2*>(o[u][x]) = __ldcg(reinterpret_cast<const float2*>(src));
          }
        }
      }
#pragma unroll
      for (int u = 0; u < PU; ++u)
#pragma unroll
        for (int x = 0; x < R; ++x)
          if (ml[u][x].y != 0.f) {                       // a part without weight is left out, whatever its columns hold
            const float mn = fmaxf(m[x], ml[u][x].x);
            const float a = m[x] == -INFINITY ? 0.f : pex2(m[x] - mn), w = pex2(ml[u][x].x - mn);
            m[x] = mn;
            l[x] = fmaf(ml[u][x].y, w, l[x] * a);        // NaN stays
#pragma unroll
            for (int v = 0; v < V; ++v) acc[x][v] = fmaf(o[u][x][v], w, acc[x][v] * a);
          }
    }
    uint32_t redo = 0;
#pragma unroll
    for (int x = 0; x < R; ++x) {
      const int row = row0 + x, tok = (int)((row + 0.5f) * sh.inv_gt), g = row - tok * sh.gt;
      if (row >= rows || g >= rec.gcnt) continue;
      const int t = rec.t0 + rec.tok0 + tok, h = rec.head0 + g;
      const float inv = l[x] > 0.f ? v_scale / l[x] : 0.f;
      T16* orow = static_cast<T16*>(p.o) + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + lane * V;
      alignas(8) T16 w[V];
      bool bad = !(l[x] >= 0.f);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float y = acc[x][v] * inv;
        bad |= !(fabsf(y) < INFINITY);
        w[v] = Elem<T16>::from_f(l[x] == 0.f ? 0.f : y);
      }
      if (reinterpret_cast<uintptr_t>(orow) % (2 * V) == 0 && lane * V + V <= p.d) {
        if constexpr (V == 4) *reinterpret_cast<uint2*>(orow) = *reinterpret_cast<const uint2*>(w);
        else *reinterpret_cast<uint32_t*>(orow) = *reinterpret_cast<const uint32_t*>(w);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (lane * V + v < p.d) orow[v] = w[v];
      }
      if (p.lse && lane == 0) p.lse[(int64_t)h * p.lse_sh + t] = l[x] > 0.f ? (m[x] - shift + log2f(l[x])) * kLn2 : -INFINITY;
      if (__any_sync(0xffffffffu, bad) && l[x] != 0.f) redo |= 1u << x;
    }
    __syncwarp();                                        // other lanes write these rows again
    while (redo) {
      const int row = row0 + __ffs(redo) - 1, tok = (int)((row + 0.5f) * sh.inv_gt);
      redo &= redo - 1;
      paged_row<T16, C8>(p, rec.b, PagedRequest{rec.t0, rec.n, rec.L}, rec.tok0 + tok, rec.head0 + row - tok * sh.gt, lane);
    }
  }
}

template <typename T16, typename C8, int D>
__global__ void __launch_bounds__(256, 3) paged_join_kernel(const __grid_constant__ bsa_paged_params p, const __grid_constant__ PagedShape sh,
                                                            const PagedRec* recs, const float2* __restrict__ part_ml,
                                                            const float* __restrict__ part_o, float shift, const int* wait_status) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const PagedRec rec = recs[blockIdx.x];
  if (*reinterpret_cast<const volatile int*>(wait_status) != 0 || !rec.valid) return;
  const int c = blockIdx.x, lane = threadIdx.x & 31;
  if (rec.last - c + 1 > 4) join_rows<T16, C8, D, 1>(p, sh, rec, c, lane, part_ml, part_o, shift);
  else join_rows<T16, C8, D, 4>(p, sh, rec, c, lane, part_ml, part_o, shift);
}

// Heads per tile: as many of a group as their pattern rows fit in 32 flags (one per block row that the item's
// positions may reach into, and per head where heads differ).
void plan_shape(const bsa_paged_params* p, PagedShape* sh) {
  const int G = p->hq / p->hkv, bs = p->block_size;
  sh->shared = p->h_pat != p->hq || p->heads_share || G == 1;
  int gt = G < 128 ? G : 128;
  if (!sh->shared) {
    auto rows = [&](int g) {
      return p->tree_mask ? (bs - 1 + 64) / bs + 1 : (bs - 1 + 128 / g - 1) / bs + 1;   // at least the rows of an item
    };
    while (gt > 1 && gt * rows(gt) > 32) --gt;
  }
  sh->gt = gt;
  sh->chunks = cdiv_i(G, gt);
  // chunks of 16 rows where a tile holds no fewer tokens with them than in chunks of 32.  Single tokens, 64 requests over
  // 1024..8192 tokens: groups of 4 and 8 heads (16 rows, repeated) 84.0 and 87.5 us, of 6 and 10 (32, not repeated) 85.2, 85.8
  sh->cr = gt <= 16 && 2 * (16 / gt) >= 32 / gt ? 16 : gt <= 32 ? 32 : gt <= 64 ? 64 : 128;
  sh->ct = p->cu_q ? sh->cr / gt : 1;      // single tokens: the rows behind them stay zeros
  sh->tt = 128 / sh->cr * sh->ct;
  const int most = p->cu_q ? (p->total_q < sh->tt ? p->total_q : sh->tt) : 1;
  sh->rows_cap = most * gt;
  sh->inv_hkv = 1.f / p->hkv;
  sh->inv_gt = 1.f / gt;
  // of the average request
  const int64_t mean = p->batch > 0 ? (int64_t)p->total_q / p->batch : 1;
  sh->rr_hint = sh->cr == 16 && mean <= sh->ct ? 16 : 128;
  sh->box = p->page_size < bs ? p->page_size : bs;
  sh->page_shift = 0;
  while ((1 << sh->page_shift) < p->page_size) ++sh->page_shift;
  // a part costs its rows' results, written and read, beside the tiles that it saves another CTA
  sh->least = (2 + sh->rows_cap / 32) * (64 / bs);
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
  int rc = make_tmap_rows(&tmQ, p->q, p->d, p->hq, p->total_q, p->q_sh * 2, p->q_st * 2, sh.gt, sh.ct, BF16);
  if (rc) return rc;
  constexpr int eb = KV8 ? 1 : 2;
  const uint32_t box_d = KV8 ? D : 64;
  // no more than a head's row at once: what lies behind it is another head's, for another CTA and time (with 256 bytes for
  // rows of 128, an e4m3 cache's DRAM reads doubled)
  const int promotion = p->d * eb >= 256 ? 256 : p->d * eb >= 128 ? 128 : 64;
  rc = make_tmap_4d(&tmK, p->k_cache, eb, p->d, p->page_size, p->hkv, p->num_pages, p->kc_ss * eb, p->kc_sh * eb, p->kc_sp * eb,
                    box_d, sh.box, !KV8, BF16, promotion);
  if (rc) return rc;
  rc = make_tmap_4d(&tmV, p->v_cache, eb, p->d, p->page_size, p->hkv, p->num_pages, p->vc_ss * eb, p->vc_sh * eb, p->vc_sp * eb,
                    box_d, sh.box, !KV8, BF16, promotion);
  if (rc) return rc;
  int dev = 0, sms = 0;
  BSA_CHECK_CUDA(cudaGetDevice(&dev));
  BSA_CHECK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  if (2 * sms < sh.ctas) sh.ctas = 2 * sms;
  int* status = wait_status_ptr();
  if (!status) return BSA_E_CUDA;
  auto* recs = static_cast<PagedRec*>(p->ws);
  auto* ml = reinterpret_cast<float2*>(static_cast<char*>(p->ws) + kRecBytes);
  auto* po = reinterpret_cast<float*>(static_cast<char*>(p->ws) + kRecBytes + ml_bytes(shape));
  constexpr size_t smem = Geo::kFixed + sizeof(PTail<Geo::kKSlots, Geo::kVSlots, Geo::kRaw>);
  static_assert(smem <= 113 * 1024, "two CTAs per SM");
  auto kern = paged_attn_kernel<BF16, D, BS, KV8>;
  BSA_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sh.ctas);
  cfg.blockDim = dim3(Geo::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BSA_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, tmQ, tmK, tmV, *p, sh, recs, ml, po, status));
  cfg.gridDim = dim3(sh.ctas, cdiv_i(sh.rows_cap, 16));     // 8 warps of four rows, or of one: twice over
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  BSA_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_join_kernel<T16, C8, D>, *p, sh, (const PagedRec*)recs, (const float2*)ml,
                                    (const float*)po, kTermShift<BF16 && !KV8>, (const int*)status));
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
