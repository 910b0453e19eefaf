// Attention over the 16-bit paged cache behind a prefix that the batch shares, on the 5th-generation tensor cores.
//
//   out[b, t, head] = softmax_p(scale q . k_p) v_p,  p over the prefix and own positions <= lens[b] + t
//
// The softmax over a row's positions is cut into parts, each (sum of weights x values, reference, sum of weights), that a
// finishing kernel joins.  A part is an item of work: up to 128 or 256 query rows of a KV head that read the same keys and
// values.  Of the prefix these are rows of ALL sequences, row = (b * tokens + t) * G + g, so that a key is read once for
// the whole batch (once for 256 rows) and the products are full tiles; of a sequence's own part they are its tokens x G
// rows.  Items of few rows, or of long positions, are cut along the positions so that every SM has some.
//
// A CTA takes one item.  Eight warps a row tile: softmax, two threads a row.  The next warp brings K and V
// by tensor copies, the last one issues S = Q K^T (both from shared memory, K-major) and O += P V (P in tensor memory, V
// MN-major), of the two row tiles in turn so that one's products run under the other's softmax.  P, rounded to the cache's
// type, overwrites its scores.  With one row tile two CTAs share an SM to the same end.  Pages are copied as they lie,
// 16 to 128 rows a copy; positions without a page are copied from behind the pool's end, which gives zeros.
//
// Softmax.  A row's reference follows its maximum lazily: it moves when a weight would pass 2^KA_MOST, so outputs in
// tensor memory are seldom rescaled.  Weights of fp16 are at most 2^8, the largest at least 1, held to 2^-11 and below 2^-14
// to 2^-25; of bf16 at most 1, the largest at least 2^-8.  Score x scale less the reference is rounded once, so whatever the
// reference was rounded to, a part's sums go with it exactly.  Its rounding stays in every weight's exponent, half a step of it
// at most: beyond 2^24 that is more than weights have room for.  A row that meets such a reference is marked (no number for a
// reference), and the joining kernel forms it again by itself, score x scale rounded first.  (To do that in the softmax cost 3
// to 8 % of every call: 81 us -> 84 to 88, a second pass over the item in the same kernel 2 to 8 %.  128 sequences of 64 heads
// behind 16384 positions, all rows marked, take 10 ms.)
//
// What lies behind the last position anyone sees may be anything: scores are masked, and those rows of V are zeroed in
// shared memory before the product (zero weight times NaN is NaN).  Rows of V that some rows of the item see and others
// do not (tokens of the same call) are zeroed where they are not finite; rows that see them add them by themselves.
//
// Bound by the chain of a tile rather than by bytes or the tensor pipe: 128 sequences of 64 heads x 128 behind 16384
// positions take 82 us in all (69 GFLOP, 840 TFLOP/s; 41 us at the tensor cores' measured rate), a tile 4.1k cycles, of
// which the softmax is 2.2k, the products 1.0k and hand-offs the rest.  32 of 28 heads behind 8131: 24 us, 6 of them the
// bytes of K and V.
//
// Every wait for an mbarrier is bounded; one that runs out sets the workspace's status word, ends the CTA's work and still
// frees the tensor memory.  The named barriers of a row's two warps have no limit of their own: a warp that gives up arrives
// once for its partner, which then finds the abort flag at its next wait.
#include <algorithm>
#include <cmath>
#include <mutex>

#include <cuda.h>
#include <cudaTypedefs.h>

#include "kv16.h"
#include "tcgen05.cuh"

namespace n730 {

constexpr int KA_KEYS = 128;       // positions of a tile
// log2 of where a new reference puts the largest weight, and of how large a weight may grow before the reference moves.  fp16
// has room above 1 and little below; bf16 has as much below, and values whose multiples by 2^8 fp32 does not hold.
template <bool BF> constexpr float KA_NEW = BF ? -8.f : 0.f;
template <bool BF> constexpr float KA_MOST = BF ? 0.f : 8.f;
constexpr float KA_FAR = 0x1p24f;  // references beyond this leave nothing of a score behind its own rounding
constexpr int KA_RING = 4;         // tiles whose masks are kept
constexpr int KA_BAD = 256;        // positions of an item that some of its rows see and others do not: fewer than its rows

template <int HD, int NT>
struct KACfg {
  static constexpr int NB = HD / 64;                               // 64-channel blocks
  static constexpr int ROWS = NT * 128;
  static constexpr int QB = ROWS * 128, KB = KA_KEYS * 128;        // bytes of a block of Q, of K or V
  static constexpr int KV = NB * KB;                               // bytes of a tile of K or V
  static constexpr int STAGES = NT == 2 || HD == 64 ? 2 : 1;       // one row tile of 128 channels: 96 KB, two CTAs an SM
  static constexpr int COPY_WARP = NT * 8, MMA_WARP = NT * 8 + 1, THREADS = (NT * 8 + 2) * 32;
  static constexpr uint32_t TMEM = NT == 1 ? 256u : 512u;
  static constexpr uint32_t S0 = 0, O0 = NT * KA_KEYS;             // columns: scores, outputs
};
// kind::f16: D fp32, A and B of the cache's type, M = 128
template <bool BF>
constexpr uint32_t ka_idesc(int n, bool mn_major) {
  return (1u << 4) | (BF ? (1u << 7) | (1u << 10) : 0u) | (mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

template <int HD, int NT>
struct KASmem {
  using Cfg = KACfg<HD, NT>;
  uint8_t q[Cfg::NB * Cfg::QB];
  uint8_t k[Cfg::STAGES][Cfg::KV];
  uint8_t v[Cfg::STAGES][Cfg::KV];
  uint32_t pages[KA_RING];   // bit i: positions 16 i .. 16 i + 15 of the tile have a page
  uint64_t qready, kfull[2], vfull[2], kfree[2], vfree[2], sfull[2], pready[2], odone[2], drain;
  uint32_t tmem;
  int abort;
  int n_bad, bad[KA_BAD];
  float half[2][NT][2][128];  // by tile's parity, row tile, half: what the two threads of a row tell each other
  uint8_t far[Cfg::ROWS];     // whether a row has met a reference beyond KA_FAR
};

// Parts of one kind (the prefix's or the sequences' own): [unit][split][4 channels][rows of a unit], a unit being a KV
// head, or a sequence and a KV head.  Rows lie side by side: a warp writes and reads its rows' 16 bytes as one piece
// (written as rows of head_dim floats by a thread each, 256 rows took 10k cycles, half as long as the rest of the item).
struct KAParts {
  int tiles, splits, rows;   // row tiles of a unit, shares of the positions, rows in memory
  int tile_rows;             // rows of a tile
  float4* o;
  float2* ml;                // [unit][split][row]: reference (log2) and sum of weights
};
struct KAArgs {
  N730KV16Cache c;
  const void* q; void* out;
  int64_t ldq, ldo;
  int batch, tokens, heads, group;
  int prefix_items, box;
  bool qvec, ovec;
  float scale_log2e;         // its absolute value, and 1 for a scale of 0: both go with the queries, whose bits are
  uint32_t sign, keep;       // taken as (q ^ sign) & keep
  const int* lens; const int* n_new;
  int* status;
  KAParts pre, own;
  FastDiv by_group, by_tokens;
};

// shares of the positions that are used: the plan knows the tables' widths alone
__device__ __forceinline__ int ka_used(int n, int splits) { return min(splits, (n + KA_KEYS - 1) / KA_KEYS); }

template <bool BF>
__device__ __forceinline__ float2 ka_wide(uint32_t x) {
  return BF ? make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)) : __half22float2(u2h(x));
}
template <bool BF>
__device__ __forceinline__ uint32_t ka_pack(float a, float b) {
  if (!BF) return h2u(__floats2half2_rn(a, b));
  const __nv_bfloat162 y = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&y);
}

// 2-D tensor copy of a box of the pool into shared memory (channel c0, row c1 of the pool)
__device__ __forceinline__ void ka_copy(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               :: "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar))
               : "memory");
}

// The two threads of a row, in warps w and w + 4 of a row tile, meet: each its half's maximum, both the row's.
__device__ __forceinline__ float ka_row_max(float y, float* mine, const float* other, int bar) {
  *mine = y;
  asm volatile("bar.sync %0, 64;" :: "r"(bar) : "memory");
  return fmaxf(y, *other);
}
// Moves a row's reference to where its tile's maximum y asks for it, if that is further up; the thread's sum and, when there are any, its
// half of the outputs (at to) follow.  far: the row's mark.
template <int HD, bool BF>
__device__ __forceinline__ void ka_move(uint32_t to, bool outputs, float y, float& m, float& l, uint8_t* far) {
  const float mn = fmaxf(m, y - KA_NEW<BF>), f = mn == m ? 1.f : ex2(m - mn);
  m = mn;
  l *= f;
  if (fabsf(mn) > KA_FAR && fabsf(mn) < INFINITY) *far = 1;
  if (!outputs) return;
#pragma unroll 1
  for (int cc = 0; cc < HD / 2; cc += 8) tc_scale8(to + cc, f);
}

// A thread's half of one tile of a row whose positions are all seen: weights over the scores, their sum to l.  ts: the
// half's scores; tp: its weights, which lie over the first half's scores.
template <int HD, bool BF>
__device__ __forceinline__ void ka_softmax(uint32_t ts, uint32_t tp, uint32_t to, float c, bool outputs, float* mine,
                                           const float* other, int bar, uint8_t* far, float& m, float& l) {
  float v[64];
  tc_ld64(ts, v);
  float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int i = 4; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], v[i]);
  const float y = ka_row_max(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c, mine, other, bar);
  if (__any_sync(0xffffffffu, y > m + KA_MOST<BF>)) ka_move<HD, BF>(to, outputs, y, m, l, far);
  const float ms = m == -INFINITY ? 0.f : m;
  const float2 c2 = both(c), m2 = both(-ms);
  float2 sum[2] = {both(0.f), both(0.f)};
  uint32_t w[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float2 x = fma2(make_float2(v[2 * i], v[2 * i + 1]), c2, m2);
    const float2 p = make_float2(ex2(x.x), ex2(x.y));
    sum[i & 1] = add2(sum[i & 1], p);
    w[i] = ka_pack<BF>(p.x, p.y);
  }
  tc_st32(tp, w);
  const float2 s = add2(sum[0], sum[1]);
  l += s.x + s.y;
}
// The same where the row sees the first `sees` positions of the half, of those the ones that have a page.
template <int HD, bool BF>
__device__ __forceinline__ void ka_softmax_some(uint32_t ts, uint32_t tp, uint32_t to, float c, int sees, uint32_t pages, bool outputs,
                                                float* mine, const float* other, int bar, uint8_t* far, float& m, float& l) {
  float v[64], mx = -INFINITY;
  tc_ld64(ts, v);
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    v[i] = i < sees && (pages >> (i / 16) & 1) ? v[i] : -INFINITY;
    mx = fmaxf(mx, v[i]);
  }
  const float y = ka_row_max(mx * c, mine, other, bar);
  if (__any_sync(0xffffffffu, y > m + KA_MOST<BF>)) ka_move<HD, BF>(to, outputs, y, m, l, far);
  const float ms = m == -INFINITY ? 0.f : m;
  uint32_t w[32];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 64; i += 2) {
    const float p0 = i < sees && (pages >> (i / 16) & 1) ? ex2(fmaf(v[i], c, -ms)) : 0.f;
    const float p1 = i + 1 < sees && (pages >> (i / 16) & 1) ? ex2(fmaf(v[i + 1], c, -ms)) : 0.f;
    sum += p0 + p1;
    w[i / 2] = ka_pack<BF>(p0, p1);
  }
  l += sum;
  tc_st32(tp, w);
}

template <int HD, bool BF, int NT>
__global__ void __launch_bounds__(KACfg<HD, NT>::THREADS, NT == 1 ? 2 : 1)
kv16_attention_kernel(const KAArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using Cfg = KACfg<HD, NT>;
  constexpr int ST = Cfg::STAGES;
  extern __shared__ __align__(1024) uint8_t ka_raw[];
  KASmem<HD, NT>& sm = *reinterpret_cast<KASmem<HD, NT>*>(aligned_smem(ka_raw));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const N730KV16Cache& c = a.c;
  const int cap = c.max_pages * c.page_size, G = a.group;

  // the item: rows [f0, f0 + nrow) of KV head h, positions [0, sees) of which every row sees the first sees_all
  int i = (int)blockIdx.x;
  const bool pre = i < a.prefix_items;
  if (!pre) i -= a.prefix_items;
  const KAParts& part = pre ? a.pre : a.own;
  const int tile = part.tiles - 1 - i % part.tiles;
  i /= part.tiles;
  const int h = i % c.n_kv;
  i /= c.n_kv;
  const int b = pre ? 0 : i % a.batch, split = pre ? i : i / a.batch;
  const int f0 = tile * Cfg::ROWS;
  int L = 0, nrow, sees, sees_all;
  if (pre) {
    nrow = min(Cfg::ROWS, a.batch * a.tokens * G - f0);
    sees = sees_all = kv16_prefix(c);
  } else {
    L = kv8_len(a.lens, b, cap);
    nrow = min(Cfg::ROWS, kv8_new(a.n_new, b, a.tokens) * G - f0);
    sees = min(L + (f0 + nrow - 1) / G + 1, cap);
    sees_all = min(L + f0 / G + 1, cap);
  }
  const int used = ka_used(sees, part.splits);
  if (nrow <= 0 || split >= used) {
    if (blockIdx.x == 0) pdl_wait();
    return;
  }
  const int all_tiles = (sees + KA_KEYS - 1) / KA_KEYS;
  const int j0 = (int)((int64_t)all_tiles * split / used), nt = (int)((int64_t)all_tiles * (split + 1) / used) - j0;
  const int* table = pre ? c.prefix_table : c.block_table + (int64_t)b * c.max_pages;

  // the queries are asked for first: 16 rows of a softmax warp, 16 bytes a lane
  constexpr int QR = 32 / (HD / 8), QU = 16 / QR;  // rows an instruction, instructions
  const int qsub = lane / (HD / 8), qch = lane % (HD / 8);
  // where row f of the item lies: its token's row, its head
  auto query = [&](int f) {
    const int t = (int)a.by_group.div(f);
    return (int64_t)((pre ? 0 : b * a.tokens) + t) * a.ldq + (int64_t)(h * G + f - t * G) * HD;
  };
  uint4 qx[QU];
  if (warp < NT * 8) {
#pragma unroll
    for (int u = 0; u < QU; ++u) {
      const int r = warp * 16 + u * QR + qsub;
      qx[u] = make_uint4(0, 0, 0, 0);
      if (r >= nrow) continue;
      const uint16_t* p = reinterpret_cast<const uint16_t*>(a.q) + query(f0 + r) + qch * 8;
      if (a.qvec) qx[u] = *reinterpret_cast<const uint4*>(p);
      else qx[u] = make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16, p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16);
    }
  } else if (warp == Cfg::COPY_WARP && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(&kmap)) : "memory");
    asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(&vmap)) : "memory");
  }
  if (tid == 0) {
    mbar_init(&sm.qready, NT * 8);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sm.kfull[s], 1);
      mbar_init(&sm.vfull[s], 1);
      mbar_init(&sm.kfree[s], 1);
      mbar_init(&sm.vfree[s], 1);
      mbar_init(&sm.sfull[s], 1);
      mbar_init(&sm.pready[s], 8);
      mbar_init(&sm.odone[s], 1);
    }
    mbar_init(&sm.drain, 1);
    fence_mbar_init();
    sm.abort = 0;
    sm.n_bad = 0;
  }
  if (warp == Cfg::MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_u32(&sm.tmem)), "r"(Cfg::TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  const uint32_t tmem = sm.tmem;
  volatile int* abortf = &sm.abort;

  if (warp == Cfg::COPY_WARP) {
    // ---------------- K and V: a lane a copy, its page looked up by itself ----------------
    const int chunks = KA_KEYS / a.box, chunk = lane / Cfg::NB, blk = lane % Cfg::NB;
    const bool mine = chunk < chunks;
    const int none = c.n_pages * c.n_kv * c.page_size;  // the first row behind the pool
    auto row_of = [&](int j) {
      const int p = (j0 + j) * KA_KEYS + chunk * a.box;
      if (!mine || p >= sees) return none;
      const int page = table[p / c.page_size];
      return (unsigned)page < (unsigned)c.n_pages ? (page * c.n_kv + h) * c.page_size + p % c.page_size : none;
    };
    const int at = blk * Cfg::KB + chunk * a.box * 128;
    int row = row_of(0), nk = 0, nv = 0;  // tiles asked for
    for (int j = 0; j < nt; ++j) {
      const int s = j % ST;
      const uint32_t ph = (uint32_t)((j / ST - 1) & 1);
      // the tile's pages, 16 positions a bit (positions behind the last count as none)
      const uint32_t has = __ballot_sync(0xffffffffu, row != none && blk == 0);
      const int next = j + 1 < nt ? row_of(j + 1) : none;
      if (j >= ST && !kp_wait_warp(&sm.kfree[s], ph, abortf)) break;
      if (lane == 0) {
        uint32_t m = 0;
        for (int k = 0; k < chunks; ++k)
          if (has >> (k * Cfg::NB) & 1) m |= ((1u << (a.box / 16)) - 1) << (k * (a.box / 16));
        sm.pages[j % KA_RING] = m;
        mbar_arrive_expect_tx(&sm.kfull[s], Cfg::KV);
      }
      __syncwarp();
      if (mine) ka_copy(sm.k[s] + at, &kmap, blk * 64, row, &sm.kfull[s]);
      nk = j + 1;
      if (j >= ST && !kp_wait_warp(&sm.vfree[s], ph, abortf)) break;
      if (lane == 0) mbar_arrive_expect_tx(&sm.vfull[s], Cfg::KV);
      __syncwarp();
      if (mine) ka_copy(sm.v[s] + at, &vmap, blk * 64, row, &sm.vfull[s]);
      nv = j + 1;
      row = next;
    }
    // copies in flight land before their memory is given up, whatever else gave up
    for (int j = max(nk - ST, 0); j < nk; ++j) kv8_wait(&sm.kfull[j % ST], (uint32_t)((j / ST) & 1), 2000000000ull);
    for (int j = max(nv - ST, 0); j < nv; ++j) kv8_wait(&sm.vfull[j % ST], (uint32_t)((j / ST) & 1), 2000000000ull);
  } else if (warp == Cfg::MMA_WARP) {
    // ---------------- products ----------------
    const uint64_t qd = umma_desc_sw128(smem_u32(sm.q)), kd = umma_desc_sw128(smem_u32(sm.k[0]));
    const uint64_t vd = umma_desc_mn_sw128(smem_u32(sm.v[0]), Cfg::KB);
    auto scores = [&](int x, int s) {  // S = Q K^T
      const uint64_t q0 = qd + (uint64_t)(x * 128 * 128 / 16), k0 = kd + (uint64_t)(s * Cfg::KV / 16);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          tc_mma_ss<ka_idesc<BF>(KA_KEYS, false)>(tmem + Cfg::S0 + x * KA_KEYS, q0 + (uint64_t)(((k >> 2) * Cfg::QB + (k & 3) * 32) / 16),
                                                  k0 + (uint64_t)(((k >> 2) * Cfg::KB + (k & 3) * 32) / 16), k > 0);
        tc_commit(&sm.sfull[x]);
        if (x == NT - 1) tc_commit(&sm.kfree[s]);
      }
      __syncwarp();
    };
    auto outputs = [&](int x, int s, bool first) {  // O += P V
      const uint64_t v0 = vd + (uint64_t)(s * Cfg::KV / 16);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < KA_KEYS / 16; ++k)
          tc_mma_ts<ka_idesc<BF>(HD, true)>(tmem + Cfg::O0 + x * HD, tmem + Cfg::S0 + x * KA_KEYS + k * 8, v0 + (uint64_t)(k * 2048 / 16),
                                            !(first && k == 0));
        if (x == NT - 1) tc_commit(&sm.vfree[s]);
      }
      __syncwarp();
    };
    bool go = kp_wait_warp(&sm.qready, 0, abortf) && kp_wait_warp(&sm.kfull[0], 0, abortf);
    if (go) {
      tc_fence_after();
#pragma unroll
      for (int x = 0; x < NT; ++x) scores(x, 0);
    }
#pragma unroll 1
    for (int j = 0; go && j < nt; ++j) {
      const int s = j % ST, s1 = (j + 1) % ST;
      go = kp_wait_warp(&sm.vfull[s], (uint32_t)((j / ST) & 1), abortf);
      // with two stages the next tile's K has been there for long: a wait costs 300 cycles, better here than between products
      if (ST > 1 && go && j + 1 < nt) go = kp_wait_warp(&sm.kfull[s1], (uint32_t)(((j + 1) / ST) & 1), abortf);
#pragma unroll 1
      for (int x = 0; go && x < NT; ++x) {
        go = kp_wait_warp(&sm.pready[x], (uint32_t)(j & 1), abortf);
        if (!go) break;
        tc_fence_after();
        outputs(x, s, j == 0);
        if (j + 1 < nt) {
          if (ST == 1 && x == 0) go = kp_wait_warp(&sm.kfull[s1], (uint32_t)(((j + 1) / ST) & 1), abortf);
          if (!go) break;
          tc_fence_after();
          scores(x, s1);
        } else {
          if (elect_one()) tc_commit(&sm.odone[x]);
          __syncwarp();
        }
      }
    }
  } else {
    // ---------------- softmax: two threads a row, 64 positions of a tile each ----------------
#pragma unroll
    for (int u = 0; u < QU; ++u) {
      const int r = warp * 16 + u * QR + qsub;
      *reinterpret_cast<uint4*>(sm.q + (qch >> 3) * Cfg::QB + r * 128 + (((qch & 7) ^ (r & 7)) << 4)) =
          make_uint4((qx[u].x ^ a.sign) & a.keep, (qx[u].y ^ a.sign) & a.keep, (qx[u].z ^ a.sign) & a.keep, (qx[u].w ^ a.sign) & a.keep);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive1(&sm.qready);
    const int x = warp >> 3, half = warp >> 2 & 1, wq = warp & 3, r = x * 128 + wq * 32 + lane, f = f0 + r;
    const bool live = r < nrow, some_live = x * 128 + wq * 32 < nrow;
    const int vis = !live ? 0 : pre ? sees : min(L + (int)a.by_group.div(f) + 1, cap);
    const uint32_t ts = tmem + ((uint32_t)(wq * 32) << 16) + Cfg::S0 + x * KA_KEYS;
    const uint32_t to = tmem + ((uint32_t)(wq * 32) << 16) + Cfg::O0 + x * HD + half * (HD / 2);
    const int bar = 1 + x * 4 + wq;  // named barrier of the row's two warps
    float m = -INFINITY, l = 0.f;
    sm.far[r] = 0;  // by both of its threads, who meet before either may set it
    bool go = true;
    for (int j = 0; j < nt; ++j) {
      if (!kp_wait_warp(&sm.sfull[x], (uint32_t)(j & 1), abortf)) { go = false; break; }
      tc_fence_after();
      const int p0 = (j0 + j) * KA_KEYS;
      const uint32_t pages = sm.pages[j % KA_RING];
      float* mine = &sm.half[j & 1][x][half][wq * 32 + lane];
      const float* other = &sm.half[j & 1][x][half ^ 1][wq * 32 + lane];
      const bool whole = p0 + KA_KEYS <= sees_all && pages == 0xffu;
      if (some_live) {  // rows of nobody keep what is there as their weights
        if (whole) ka_softmax<HD, BF>(ts + half * 64, ts + half * 32, to, a.scale_log2e, j > 0, mine, other, bar, &sm.far[r], m, l);
        else ka_softmax_some<HD, BF>(ts + half * 64, ts + half * 32, to, a.scale_log2e, vis - p0 - half * 64, pages >> (4 * half), j > 0,
                                     mine, other, bar, &sm.far[r], m, l);
      }
      if (!whole) {
        if (x == 0 && half == 0 && p0 + KA_KEYS > sees_all) {  // rows of V that not everyone sees
          if (!kp_wait_warp(&sm.vfull[j % ST], (uint32_t)((j / ST) & 1), abortf)) { go = false; break; }
          const int row = wq * 32 + lane, p = p0 + row;
          uint8_t* v = sm.v[j % ST] + row * 128;
          bool zero = p >= sees;
          if (p >= sees_all && !zero) {
#pragma unroll 1
            for (int e = 0; e < Cfg::NB * 8; ++e) {  // the row's 16 bytes in any order
              const uint4 y = *reinterpret_cast<const uint4*>(v + (e >> 3) * Cfg::KB + (e & 7) * 16);
              const uint32_t inf = BF ? 0x7f80u : 0x7c00u, w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) zero = zero || (w[k] & inf) == inf || (w[k] >> 16 & inf) == inf;
            }
            if (zero) sm.bad[atomicAdd(&sm.n_bad, 1)] = p;
          }
          if (zero)
#pragma unroll
            for (int e = 0; e < Cfg::NB * 8; ++e)
              *reinterpret_cast<uint4*>(v + (e >> 3) * Cfg::KB + (e & 7) * 16) = make_uint4(0, 0, 0, 0);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive1(&sm.pready[x]);
    }
    if (go) {
      go = kp_wait_warp(&sm.odone[x], 0, abortf);
      tc_fence_after();
    }
    // a warp that gave up leaves its partner nothing to wait for: what the partner needs to get further than the barrier it
    // may be at does not come without this warp
    if (!go && some_live) asm volatile("bar.arrive %0, 64;" :: "r"(bar) : "memory");
    if (go) {
      const int n_bad = *reinterpret_cast<volatile int*>(&sm.n_bad);
      const int64_t unit = (int64_t)(pre ? h : b * c.n_kv + h) * part.splits + split;
      if (some_live) {  // the row's sum is its two threads'
        float* sum = &sm.half[nt & 1][x][1][wq * 32 + lane];
        if (half) *sum = l;
        asm volatile("bar.sync %0, 64;" :: "r"(bar) : "memory");
        if (!half && live) part.ml[unit * part.rows + f] = make_float2(sm.far[r] ? NAN : m, l + *sum);
      }
      const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll 1
      for (int cc = 0; some_live && cc < HD / 2; cc += 32) {
        float o[32];
        tc_ld32(to + cc, o);
        if (live && n_bad) {
          for (int k = 0; k < n_bad; ++k) {
            const int p = sm.bad[k], page = table[p / c.page_size];
            if (p >= vis || (unsigned)page >= (unsigned)c.n_pages) continue;
            const int64_t at = (((int64_t)page * c.n_kv + h) * c.page_size + p % c.page_size) * HD;
            const int64_t qa = query(f);
            float dot = 0.f;
            for (int d = 0; d < HD; ++d) dot = fmaf(kv8_load1(a.q, qa + d, c.dtype), kv8_load1(c.k, at + d, c.dtype), dot);
            const float w = ex2(fmaf(!a.keep ? 0.f : a.sign ? -dot : dot, a.scale_log2e, -ms));
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = fmaf(w, kv8_load1(c.v, at + half * (HD / 2) + cc + e, c.dtype), o[e]);
          }
        }
        __syncwarp();
        if (live) {
          float4* dst = part.o + (unit * (HD / 4) + (half * (HD / 2) + cc) / 4) * part.rows + f;
#pragma unroll
          for (int e = 0; e < 8; ++e) dst[(int64_t)e * part.rows] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (sm.abort) {
    if (tid == 0) *a.status = 1;
    if (warp == Cfg::MMA_WARP) {  // products in flight end before tensor and shared memory are given up
      if (elect_one()) tc_commit(&sm.drain);
      __syncwarp();
      kv8_wait(&sm.drain, 0, 2000000000ull);
    }
    __syncthreads();
  }
  if (warp == Cfg::MMA_WARP)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(Cfg::TMEM));
  if (blockIdx.x == 0) pdl_wait();  // the kernel behind this one waits for it alone, and so for the one before
}

// Attention of single tokens and drafts over their own positions: a warp an item (sequence, KV head, 8 NB of its query rows,
// share of the positions), 16 positions at a time.  Positions, and then channels, are the products' 16 rows and the
// queries their columns (mma.m16n8k16): S^T = K Q^T, O^T += V^T P^T, so that nothing is spent on the 128 rows that a
// tensor-memory tile would have; with single tokens this is bound by the bytes of K and V.  P^T's fragments are those of
// S^T transposed, 8 x 8 at a time, in registers.  Rows arrive by asynchronous copies, three blocks of 16 positions deep;
// no warp waits for another, and a CTA is one warp with KOCfg's three stages, so that it finds room beside the CTA of the
// prefix's kernel that is running (1024 items of 64 heads x 128, 144 positions: 46 us by the kernel above, most of that
// hidden here).
template <int HD> struct KOCfg { static constexpr int KB = 16 * HD * 2, STAGE = 2 * KB, STAGES = 3; };

template <bool BF>
__device__ __forceinline__ void ko_mma(float (&c)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
  else
    mma16816(c, x[0], x[1], x[2], x[3], b0, b1);
}
template <bool TRANS>
__device__ __forceinline__ void ko_load(uint32_t (&x)[4], uint32_t addr) {
  if (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t ko_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int HD, bool BF, int NB>
__global__ void __launch_bounds__(32) kv16_own_kernel(const KAArgs a) {
  using Cfg = KOCfg<HD>;
  constexpr int KS = HD / 16, CH = HD / 8;  // steps of 16 channels; 16-byte pieces of a row
  extern __shared__ __align__(128) uint8_t ko_smem[];
  const N730KV16Cache& c = a.c;
  const int lane = threadIdx.x, G = a.group, cap = c.max_pages * c.page_size;
  int i = (int)blockIdx.x;
  const int f0 = i % a.own.tiles * a.own.tile_rows;  // the first of its rows
  i /= a.own.tiles;
  const int h = i % c.n_kv;
  i /= c.n_kv;
  const int b = i % a.batch, split = i / a.batch;
  const int L = kv8_len(a.lens, b, cap), nrow = min(8 * NB, kv8_new(a.n_new, b, a.tokens) * G - f0);
  auto vis_of = [&](int f) { return min(L + (int)a.by_group.div(f) + 1, cap); };
  const int sees = nrow > 0 ? vis_of(f0 + nrow - 1) : 0, sees_all = vis_of(f0);  // of any row, of every one
  const int used = ka_used(sees, a.own.splits);
  pdl_launch_dependents();
  if (split < used) {
    const int blocks = (sees + 15) / 16, i0 = (int)((int64_t)blocks * split / used), n = (int)((int64_t)blocks * (split + 1) / used) - i0;
    const int* table = c.block_table + (int64_t)b * c.max_pages;
    const uint32_t base = smem_u32(ko_smem);
    // the share's blocks in order: the page of the next one to be fetched is known by then, asked for a block ahead
    int at_page = i0 * 16 / c.page_size, at_off = i0 * 16 - at_page * c.page_size, left = n;
    auto next_page = [&] {
      const int page = left > 0 ? table[at_page] : -1;
      --left;
      return page;
    };
    uint32_t here = 0;  // bit s: the block in stage s has a page
    const int piece = lane % CH, row0 = lane / CH;
    uint32_t to[16 * CH / 32];  // where this lane's 16 bytes of its rows go
#pragma unroll
    for (int u = 0; u < 16 * CH / 32; ++u) {
      const int r = row0 + u * (32 / CH);
      to[u] = base + r * (HD * 2) + ((piece ^ (r & 7)) << 4);
    }
    auto fetch = [&](int j, int page, int s) {
      const bool ok = (unsigned)page < (unsigned)c.n_pages;
      here = ok ? here | 1u << s : here & ~(1u << s);
      if (j < n) {
        const int64_t at = ((int64_t)(((ok ? page : 0) * c.n_kv + h) * c.page_size + at_off) + row0) * HD + piece * 8;
        const uint16_t* k = reinterpret_cast<const uint16_t*>(c.k) + at;
        const uint16_t* v = reinterpret_cast<const uint16_t*>(c.v) + at;
        const int rows = ok ? sees - (i0 + j) * 16 - row0 : 0;  // of this lane's; behind the last position: zeros
#pragma unroll
        for (int u = 0; u < 16 * CH / 32; ++u) {
          const uint32_t bytes = u * (32 / CH) < rows ? 16u : 0u;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(to[u] + s * Cfg::STAGE), "l"(k + u * (32 / CH) * HD), "r"(bytes) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(to[u] + s * Cfg::STAGE + Cfg::KB), "l"(v + u * (32 / CH) * HD), "r"(bytes) : "memory");
        }
        at_off += 16;
        if (at_off == c.page_size) { at_off = 0; ++at_page; }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(0, next_page(), 0);
    fetch(1, next_page(), 1);
    int page = next_page();
    // the queries as the products' columns: row lane / 4 (+ 8), channels 16 k + 2 (lane % 4) (+ 8)
    uint32_t q[NB][KS][2];
#pragma unroll
    for (int y = 0; y < NB; ++y) {
      const int r = y * 8 + (lane >> 2), t = (int)a.by_group.div(f0 + r);
      const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(b * a.tokens + t) * a.ldq +
                           (int64_t)(h * G + f0 + r - t * G) * HD + (lane & 3) * 2;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint16_t* at = qp + k * 16 + e * 8;
          q[y][k][e] = r >= nrow ? 0u : ((a.qvec ? *reinterpret_cast<const uint32_t*>(at) : at[0] | (uint32_t)at[1] << 16) ^ a.sign) & a.keep;
        }
    }
    int vis[NB][2];  // of the rows whose scores this lane holds
#pragma unroll
    for (int y = 0; y < NB; ++y)
#pragma unroll
      for (int e = 0; e < 2; ++e) vis[y][e] = vis_of(min(f0 + y * 8 + (lane & 3) * 2 + e, f0 + nrow - 1));
    float o[NB][KS][4] = {}, m[NB][2], l[NB][2] = {};
#pragma unroll
    for (int y = 0; y < NB; ++y) m[y][0] = m[y][1] = -INFINITY;
    // scores x scale less the reference: in one step, as the kernel above; beyond KA_FAR the product in a step of its own
    float c0[NB][2], c1[NB][2];
#pragma unroll
    for (int y = 0; y < NB; ++y)
#pragma unroll
      for (int e = 0; e < 2; ++e) { c0[y][e] = 1.f; c1[y][e] = a.scale_log2e; }
    // where this lane's rows of the four 8 x 8 pieces lie: K's by position and then channels, V's turned
    const int kr = lane & 15, kc = lane >> 4, vr = (lane & 7) + (lane >> 4) * 8, vc = lane >> 3 & 1;
#pragma unroll 1
    for (int j = 0, s = 0; j < n; ++j, s = s == Cfg::STAGES - 1 ? 0 : s + 1) {
      const int p0 = (i0 + j) * 16;
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();  // everyone's rows are here, and everyone is through with the block before
      const bool ok = here >> s & 1;
      fetch(j + 2, page, s == 0 ? Cfg::STAGES - 1 : s - 1);
      page = next_page();
      if (!ok) continue;
      const uint32_t kb = base + s * Cfg::STAGE, vb = kb + Cfg::KB;
      float x[NB][4] = {}, x2[NB][4] = {};  // two sums: half as long a chain of products
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t f[4];
        ko_load<false>(f, kb + kr * (HD * 2) + (((2 * k + kc) ^ (kr & 7)) << 4));
#pragma unroll
        for (int y = 0; y < NB; ++y) ko_mma<BF>(k & 1 ? x2[y] : x[y], f, q[y][k][0], q[y][k][1]);
      }
      uint32_t w[NB][2];
      float e4[NB][4];
#pragma unroll
      for (int y = 0; y < NB; ++y) {
        float big[2];
        const int p = p0 + (lane >> 2);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[y][e] = p < vis[y][e] ? x[y][e] + x2[y][e] : -INFINITY;
          x[y][2 + e] = p + 8 < vis[y][e] ? x[y][2 + e] + x2[y][2 + e] : -INFINITY;
          big[e] = fmaxf(x[y][e], x[y][2 + e]) * a.scale_log2e;
        }
        if (__any_sync(0xffffffffu, big[0] > m[y][0] + KA_MOST<BF> || big[1] > m[y][1] + KA_MOST<BF>)) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) big[e] = fmaxf(big[e], __shfl_xor_sync(0xffffffffu, big[e], d));
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mn = fmaxf(m[y][e], big[e] - KA_NEW<BF>);
            f[e] = mn == m[y][e] ? 1.f : ex2(m[y][e] - mn);
            m[y][e] = mn;
            l[y][e] *= f[e];
            const bool far = fabsf(mn) > KA_FAR && mn > -INFINITY;
            c0[y][e] = far ? a.scale_log2e : 1.f;
            c1[y][e] = far ? 1.f : a.scale_log2e;
          }
#pragma unroll
          for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[y][k][e] *= f[e & 1];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float ms = m[y][e & 1] == -INFINITY ? 0.f : m[y][e & 1];
          e4[y][e] = ex2(fmaf(x[y][e] * c0[y][e & 1], c1[y][e & 1], -ms));
          l[y][e & 1] += e4[y][e];
        }
        w[y][0] = ko_transpose(ka_pack<BF>(e4[y][0], e4[y][1]));
        w[y][1] = ko_transpose(ka_pack<BF>(e4[y][2], e4[y][3]));
      }
      if (p0 + 16 > sees_all && sees > sees_all) {
        // rows of V that some of the rows do not see: zeroed where not finite, added by the rows that see them
        const uint32_t inf = BF ? 0x7f80u : 0x7c00u;
#pragma unroll 1
        for (int p = max(sees_all, p0); p < min(sees, p0 + 16); ++p) {
          uint8_t* row = ko_smem + s * Cfg::STAGE + Cfg::KB + (p - p0) * (HD * 2);
          uint32_t bad = 0;
          for (int e = lane; e < HD / 2; e += 32) {
            const uint32_t y = *reinterpret_cast<const uint32_t*>(row + e * 4);
            bad |= (y & inf) == inf || (y >> 16 & inf) == inf;
          }
          if (!__any_sync(0xffffffffu, bad)) continue;
          for (int e = lane; e < HD / 2; e += 32) *reinterpret_cast<uint32_t*>(row + e * 4) = 0u;
          const int pg = table[p / c.page_size];
          const int64_t at = (((int64_t)pg * c.n_kv + h) * c.page_size + p % c.page_size) * HD + (lane >> 2);
          const int from = ((p - p0) & 7) * 4 + (lane & 3);
#pragma unroll
          for (int y = 0; y < NB; ++y)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float lo = __shfl_sync(0xffffffffu, e4[y][e], from), hi = __shfl_sync(0xffffffffu, e4[y][2 + e], from);
              if (p >= vis[y][e]) continue;
#pragma unroll
              for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                  o[y][k][2 * u + e] = fmaf(p - p0 < 8 ? lo : hi, kv8_load1(c.v, at + k * 16 + u * 8, c.dtype), o[y][k][2 * u + e]);
            }
        }
        __syncwarp();
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t f[4];
        ko_load<true>(f, vb + vr * (HD * 2) + (((2 * k + vc) ^ (vr & 7)) << 4));
#pragma unroll
        for (int y = 0; y < NB; ++y) ko_mma<BF>(o[y][k], f, w[y][0], w[y][1]);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    const int64_t unit = (int64_t)(b * c.n_kv + h) * a.own.splits + split;
    float* dst = reinterpret_cast<float*>(a.own.o + unit * (HD / 4) * a.own.rows);
#pragma unroll
    for (int y = 0; y < NB; ++y)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[y][e] += __shfl_xor_sync(0xffffffffu, l[y][e], d);
        const int r = y * 8 + (lane & 3) * 2 + e;
        if (r >= nrow) continue;
        if (lane < 4) a.own.ml[unit * a.own.rows + f0 + r] = make_float2(m[y][e], l[y][e]);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int ch = k * 16 + u * 8 + (lane >> 2);
            dst[((int64_t)(ch >> 2) * a.own.rows + f0 + r) * 4 + (ch & 3)] = o[y][k][2 * u + e];
          }
      }
  }
  if (blockIdx.x == 0) pdl_wait();
}

// A marked row by itself, by all warps of a CTA: 32 positions at a time each, then a lane its share of the channels for the
// few weights that are left.  CH of the row's channels, from `ch` on.  Inline: a call's stack cost every launch of the joining
// kernel 1 us.
template <int HD, bool BF, int CH, int WARPS>
__device__ __forceinline__ void ka_again(const KAArgs& a, int b, int t, int h, int g, int ch, float (&part)[WARPS][CH + 2]) {
  constexpr int VL = CH / 32, LANES = HD / 8, GROUP = 32 / LANES;  // lanes of a row of K, rows at a time
  const N730KV16Cache& c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cap = c.max_pages * c.page_size, prefix = kv16_prefix(c), all = prefix + min(kv8_len(a.lens, b, cap) + t + 1, cap);
  const int64_t at = (int64_t)(b * a.tokens + t), col = (int64_t)(h * a.group + g) * HD;
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = kv8_load1(a.q, at * a.ldq + col + lane % LANES * 8 + e, c.dtype);
  const float scale = a.sign ? -a.scale_log2e : a.scale_log2e;
  float m = -INFINITY, l = 0.f, o[VL] = {};
#pragma unroll 1
  for (int i0 = warp * 32; i0 < all; i0 += WARPS * 32) {
    const int i = i0 + lane, p = i < prefix ? i : i - prefix;
    const int page = i >= all ? -1 : i < prefix ? c.prefix_table[p / c.page_size] : c.block_table[(int64_t)b * c.max_pages + p / c.page_size];
    const int64_t row = (unsigned)page < (unsigned)c.n_pages ? (((int64_t)page * c.n_kv + h) * c.page_size + p % c.page_size) * HD : -1;
    float x = -INFINITY;
#pragma unroll 4
    for (int k = 0; k < LANES; ++k) {  // GROUP positions at a time
      const int64_t from = max(__shfl_sync(0xffffffffu, row, k * GROUP + lane / LANES), (int64_t)0);  // the pool's first row for none
      const uint4 y = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(c.k) + from + lane % LANES * 8);
      const float2 y0 = ka_wide<BF>(y.x), y1 = ka_wide<BF>(y.y), y2 = ka_wide<BF>(y.z), y3 = ka_wide<BF>(y.w);
      float d = fmaf(q[0], y0.x, q[1] * y0.y);
      d = fmaf(q[2], y1.x, d); d = fmaf(q[3], y1.y, d); d = fmaf(q[4], y2.x, d);
      d = fmaf(q[5], y2.y, d); d = fmaf(q[6], y3.x, d); d = fmaf(q[7], y3.y, d);
#pragma unroll
      for (int e = 1; e < LANES; e <<= 1) d += __shfl_xor_sync(0xffffffffu, d, e);
      d = __shfl_sync(0xffffffffu, d, lane % GROUP * LANES);
      if (lane / GROUP == k && row >= 0) x = d * scale;
    }
    const float mn = fmaxf(m, warp_max(x)), f = mn == m ? 1.f : ex2(m - mn), w = x == -INFINITY ? 0.f : ex2(x - mn);
    m = mn;
    l = l * f + w;
#pragma unroll
    for (int e = 0; e < VL; ++e) o[e] *= f;
    for (unsigned some = __ballot_sync(0xffffffffu, !(w == 0.f)); some; some &= some - 1) {
      const int k = __ffs(some) - 1;
      const int64_t from = __shfl_sync(0xffffffffu, row, k) + ch + lane * VL;
      const float wk = __shfl_sync(0xffffffffu, w, k);
#pragma unroll
      for (int e = 0; e < VL; ++e) o[e] = fmaf(wk, kv8_load1(c.v, from + e, c.dtype), o[e]);
    }
  }
  l = warp_sum(l);
  __syncthreads();  // the row before is through with its parts
#pragma unroll
  for (int e = 0; e < VL; ++e) part[warp][lane * VL + e] = o[e];
  if (lane == 0) { part[warp][CH] = m; part[warp][CH + 1] = l; }
  __syncthreads();
  if ((int)threadIdx.x >= CH) return;
  m = -INFINITY;
  for (int w = 0; w < WARPS; ++w) m = fmaxf(m, part[w][CH]);
  float sum = 0.f, y = 0.f;
  for (int w = 0; w < WARPS; ++w) {
    const float f = part[w][CH] == -INFINITY ? 0.f : ex2(part[w][CH] - m);
    sum += part[w][CH + 1] == 0.f ? 0.f : part[w][CH + 1] * f;
    y = fmaf(part[w][threadIdx.x], f, y);
  }
  kv8_store1(a.out, at * a.ldo + col + ch + threadIdx.x, BF ? N730_BF16 : N730_F16, sum == 0.f ? 0.f : y / sum);
}

// Joins the rows' parts.  A CTA takes 32 rows of a KV head, a lane a row, and PIECES groups of 4 channels; its warps take
// MINE of these each, and every PARTS-th part: with few rows that is 32 channels and a quarter of the parts, so that a
// part's trip to memory is paid for few times in a row (896 rows of 17 parts: 7 us, 11 with a CTA for all channels), with
// many all channels and parts (8192 rows of 5 parts: 10 us, 17 the other way).  Outputs change places in shared memory so
// that they leave as whole rows.
template <int HD, bool BF, int MINE, int COLS, int PARTS>
__global__ void __launch_bounds__(COLS * PARTS * 32) kv16_join_kernel(const __grid_constant__ KAArgs a) {
  constexpr int PIECES = MINE * COLS;
  __shared__ uint2 out[32][PIECES + 1];
  __shared__ float4 other[PARTS > 1 ? PARTS - 1 : 1][PARTS > 1 ? MINE : 1][COLS][32];
  __shared__ float most[PARTS][32], sums[PARTS][32];
  __shared__ int64_t to[32];
  __shared__ float marked[COLS * PARTS][PIECES * 4 + 2];
  const N730KV16Cache& c = a.c;
  const int lane = threadIdx.x & 31, col = (threadIdx.x >> 5) % COLS, turn = threadIdx.x / (COLS * 32);
  const int G = a.group, cap = c.max_pages * c.page_size, h = blockIdx.y, piece = blockIdx.z * PIECES + col * MINE;
  const int64_t r = (int64_t)blockIdx.x * 32 + lane, rows = (int64_t)a.batch * a.tokens * G;  // row of the KV head
  bool live = r < rows;
  const int tok = live ? (int)a.by_group.div((uint32_t)r) : 0, g = (int)(r - (int64_t)tok * G);
  const int b = (int)a.by_tokens.div(tok), t = tok - b * a.tokens;
  const int n_new = live ? kv8_new(a.n_new, b, a.tokens) : 0;
  live = live && t < n_new;
  // the shares of the row's positions: the last row of its tile decides
  const int np = live && a.pre.o ? ka_used(kv16_prefix(c), a.pre.splits) : 0;
  const int f = t * G + g, f0 = f / a.own.tile_rows * a.own.tile_rows;
  const int last = live ? (int)a.by_group.div(min(f0 + a.own.tile_rows, n_new * G) - 1) : 0;
  const int no = live ? ka_used(min(kv8_len(a.lens, b, cap) + last + 1, cap), a.own.splits) : 0;
  const int64_t p0 = (int64_t)h * a.pre.splits, o0 = (int64_t)(b * c.n_kv + h) * a.own.splits;
  const int n = np + no;  // parts: the prefix's, then the own ones
  pdl_wait();
  float big = -INFINITY, sum = 0.f;
  bool again = false;  // a part has no number for a reference
#pragma unroll 4
  for (int i = turn; i < n; i += PARTS) {
    const float m = (i < np ? a.pre.ml[(p0 + i) * a.pre.rows + r] : a.own.ml[(o0 + i - np) * a.own.rows + f]).x;
    big = fmaxf(big, m);
    again = again || m != m;
  }
  if (col == 0) most[turn][lane] = again ? NAN : big;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PARTS; ++k) {
    big = fmaxf(big, most[k][lane]);
    again = again || most[k][lane] != most[k][lane];
  }
  float4 acc[MINE];
#pragma unroll
  for (int e = 0; e < MINE; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = turn; i < n; i += PARTS) {
    const bool of_prefix = i < np;
    const KAParts& part = of_prefix ? a.pre : a.own;
    const int64_t unit = of_prefix ? p0 + i : o0 + i - np, row = of_prefix ? r : f;
    const float2 ml = part.ml[unit * part.rows + row];
    const float4* src = part.o + (unit * (HD / 4) + piece) * part.rows + row;
    const float w = ml.x == -INFINITY ? 0.f : ex2(ml.x - big);
    sum += ml.y == 0.f ? 0.f : ml.y * w;  // a part without a seen position has no sum either; a NaN stays one
#pragma unroll
    for (int e = 0; e < MINE; ++e) {
      const float4 x = src[(int64_t)e * part.rows];
      acc[e].x = fmaf(w, x.x, acc[e].x); acc[e].y = fmaf(w, x.y, acc[e].y);
      acc[e].z = fmaf(w, x.z, acc[e].z); acc[e].w = fmaf(w, x.w, acc[e].w);
    }
  }
  if (PARTS > 1 && turn) {
#pragma unroll
    for (int e = 0; e < MINE; ++e) other[turn - 1][e][col][lane] = acc[e];
  }
  if (col == 0) sums[turn][lane] = sum;
  if (threadIdx.x < 32) to[lane] = live && !again ? (int64_t)tok * a.ldo + (int64_t)(h * G + g) * HD + blockIdx.z * (PIECES * 4) : -1;
  __syncthreads();
  if (!turn) {
#pragma unroll
    for (int k = 1; k < PARTS; ++k) {
      sum += sums[k][lane];
#pragma unroll
      for (int e = 0; e < MINE; ++e) {
        const float4 x = other[k - 1][e][col][lane];
        acc[e] = make_float4(acc[e].x + x.x, acc[e].y + x.y, acc[e].z + x.z, acc[e].w + x.w);
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int e = 0; e < MINE; ++e)
      out[lane][col * MINE + e] = make_uint2(ka_pack<BF>(acc[e].x * inv, acc[e].y * inv), ka_pack<BF>(acc[e].z * inv, acc[e].w * inv));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * PIECES; i += COLS * PARTS * 32) {
    const int row = i / PIECES, e = i % PIECES;
    if (to[row] < 0) continue;
    uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + to[row] + e * 4;
    const uint2 y = out[row][e];
    if (a.ovec) {
      *reinterpret_cast<uint2*>(dst) = y;
    } else {
      dst[0] = (uint16_t)y.x; dst[1] = (uint16_t)(y.x >> 16); dst[2] = (uint16_t)y.y; dst[3] = (uint16_t)(y.y >> 16);
    }
  }
  for (unsigned marks = __ballot_sync(0xffffffffu, again); marks; marks &= marks - 1) {  // the same in every warp
    const int k = __ffs(marks) - 1;
    ka_again<HD, BF, PIECES * 4, COLS * PARTS>(a, __shfl_sync(0xffffffffu, b, k), __shfl_sync(0xffffffffu, t, k), h,
                                               __shfl_sync(0xffffffffu, g, k), blockIdx.z * (PIECES * 4), marked);
  }
}

// ----------------------------------------------------------------------------- plan
constexpr int KO_ROWS = 16, KO_MOST = 32;  // query rows of a KV head that a warp of the own kernel takes, and that it is used for
struct KAPlan {
  int pre_nt, own_nt;              // row tiles of a CTA; own_nt 0: the kernel for single tokens
  int pre_tiles, pre_splits, own_tiles, own_splits, own_rows;
  int64_t pre_items, own_items;
  int64_t pre_o, pre_ml, own_o, own_ml, bytes;  // in the workspace
};

static KAPlan ka_plan(const N730KV16Cache& c, int batch, int tokens, int heads) {
  KAPlan p{};
  const int G = heads / c.n_kv, sms = num_sms();
  const int64_t pre_rows = (int64_t)batch * tokens * G, own_rows = (int64_t)tokens * G, own_units = (int64_t)batch * c.n_kv;
  auto shape = [&](int64_t rows, int64_t units, int64_t positions, int& nt, int& tiles, int& splits) {
    nt = rows > 128 ? 2 : 1;
    tiles = (int)((rows + nt * 128 - 1) / (nt * 128));
    const int64_t items = units * tiles, slots = (int64_t)sms * (nt == 1 ? 2 : 1);
    const int64_t pos = (positions + KA_KEYS - 1) / KA_KEYS;
    // a share's time in us: its tiles and what it costs to begin and end; the parts' way through memory
    double best = 1e30;
    splits = 1;
    for (int s = 1; s <= std::min<int64_t>(pos, 64); ++s) {
      const double waves = (double)((items * s + slots - 1) / slots);
      const double us = waves * ((double)((pos + s - 1) / s) * 1.9 + 4.5) + s * 0.10 + (double)s * units * rows * c.head_dim * 8 / 1e7;
      if (us < best * 0.98) { best = us; splits = s; }
    }
  };
  if (c.prefix_pages) {
    shape(pre_rows, c.n_kv, (int64_t)c.prefix_pages * c.page_size, p.pre_nt, p.pre_tiles, p.pre_splits);
    p.pre_items = (int64_t)c.n_kv * p.pre_tiles * p.pre_splits;
  }
  const int64_t cap = (int64_t)c.max_pages * c.page_size;
  shape(own_rows, own_units, cap, p.own_nt, p.own_tiles, p.own_splits);
  p.own_rows = p.own_tiles * p.own_nt * 128;
  // few rows: warps of 16 where they fill a share of the SMs (128 sequences of 64 heads, 8 rows each: 82 us for 117; with 3
  // groups of rows, 16 sequences of 5 tokens and 28 heads, 35.1 for 34.8), in one grid with the prefix's items otherwise (one
  // launch less: 4 sequences of 14 heads 10.2 us for 10.5)
  if (own_rows <= KO_MOST && own_units >= sms / 4) {
    p.own_nt = 0;
    p.own_tiles = (int)((own_rows + KO_ROWS - 1) / KO_ROWS);
    p.own_rows = p.own_tiles * KO_ROWS;
    p.own_splits = (int)std::max<int64_t>(1, std::min<int64_t>({(cap + KA_KEYS - 1) / KA_KEYS, 8ll * sms / (own_units * p.own_tiles), 32}));
  }
  p.own_items = own_units * p.own_tiles * p.own_splits;
  auto room = [&](int64_t bytes) { const int64_t at = p.bytes; p.bytes += (bytes + 255) / 256 * 256; return at; };
  room(256);
  const int64_t pr = (int64_t)p.pre_tiles * p.pre_splits * p.pre_nt * 128 * c.n_kv;
  const int64_t orows = own_units * p.own_splits * p.own_rows;
  p.pre_o = room(pr * c.head_dim * 4);
  p.pre_ml = room(pr * 8);
  p.own_o = room(orows * c.head_dim * 4);
  p.own_ml = room(orows * 8);
  return p;
}

static int kv16_attention_check(const N730KV16Cache* c, int batch, int tokens, int heads) {
  const char* what = "kv16_attention";
  if (int rc = kv16_check(c, batch, what)) return rc;
  N730_REQUIRE(batch <= KV8_MAX_BATCH && tokens >= 1 && tokens <= (1 << 20), N730_BAD_ARG, "%s: batch %d, tokens %d", what, batch, tokens);
  N730_REQUIRE(heads >= c->n_kv && heads % c->n_kv == 0 && heads <= 65535, N730_BAD_ARG, "%s: %d heads over %d KV heads", what,
               heads, c->n_kv);
  N730_REQUIRE((int64_t)batch * tokens * heads < (1ll << 30), N730_BAD_ARG, "%s: 2^30 or more query rows", what);
  return N730_OK;
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (no libcuda link).
static PFN_cuTensorMapEncodeTiled_v12000 ka_encoder() {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    else
      cudaGetLastError();
  });
  return fn;
}
// A pool as a 2-D tensor, one row per position and KV head of a page; a copy takes 64 channels of `box` rows,
// swizzled over 128 bytes (x is 0 or 64, a multiple of 16 bytes).
static int ka_map(const N730KV16Cache& c, const void* pool, int box, CUtensorMap* out) {
  auto enc = ka_encoder();
  N730_REQUIRE(enc, N730_CUDA_ERR, "kv16_attention: cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[2] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.n_pages * c.n_kv * c.page_size};
  const cuuint64_t strides[1] = {(cuuint64_t)c.head_dim * 2};
  const cuuint32_t boxes[2] = {64, (cuuint32_t)box}, es[2] = {1, 1};
  N730_REQUIRE(enc(out, c.dtype == N730_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                   const_cast<void*>(pool), dims, strides, boxes, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS,
               N730_CUDA_ERR, "kv16_attention: cuTensorMapEncodeTiled failed");
  return N730_OK;
}

template <int HD, bool BF, int NT>
static int ka_launch_one(const KAArgs& a, const CUtensorMap& km, const CUtensorMap& vm, int64_t grid, bool pdl, cudaStream_t st) {
  const size_t smem = sizeof(KASmem<HD, NT>) + 1024;
  if (int rc = smem_attr_once<kv16_attention_kernel<HD, BF, NT>>((int)smem)) return rc;
  return kv8_launch(kv16_attention_kernel<HD, BF, NT>, dim3((unsigned)grid), dim3(KACfg<HD, NT>::THREADS), smem, st, pdl, a, km, vm);
}

template <int HD, bool BF>
static int ka_launch(KAArgs& a, const KAPlan& p, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
  auto one = [&](int nt, int64_t pre, int64_t own, bool pdl) {
    a.prefix_items = (int)pre;
    return nt == 1 ? ka_launch_one<HD, BF, 1>(a, km, vm, pre + own, pdl, st) : ka_launch_one<HD, BF, 2>(a, km, vm, pre + own, pdl, st);
  };
  // items of the same shape in one grid, the prefix's (longer) first; otherwise the own ones' grid follows on its heels
  if (p.own_nt == 0) {
    if (p.pre_items)
      if (int rc = one(p.pre_nt, p.pre_items, 0, false)) return rc;
    const int smem = KOCfg<HD>::STAGE * KOCfg<HD>::STAGES;
    auto own = [&](auto kernel) { return kv8_launch(kernel, dim3((unsigned)p.own_items), dim3(32), smem, st, p.pre_items > 0, a); };
    if (int rc = a.group * a.tokens <= 8 ? own(kv16_own_kernel<HD, BF, 1>) : own(kv16_own_kernel<HD, BF, 2>)) return rc;
  } else if (!p.pre_items || p.pre_nt == p.own_nt) {
    if (int rc = one(p.own_nt, p.pre_items, p.own_items, false)) return rc;
  } else {
    if (int rc = one(p.pre_nt, p.pre_items, 0, false)) return rc;
    if (int rc = one(p.own_nt, 0, p.own_items, true)) return rc;
  }
  const int64_t rows = (int64_t)a.batch * a.tokens * a.group;
  const unsigned blocks = (unsigned)((rows + 31) / 32);
  if ((int64_t)blocks * a.c.n_kv >= num_sms())
    return kv8_launch(kv16_join_kernel<HD, BF, 4, HD / 16, 1>, dim3(blocks, a.c.n_kv), dim3(HD / 16 * 32), 0, st, true, a);
  return kv8_launch(kv16_join_kernel<HD, BF, 2, 4, 4>, dim3(blocks, a.c.n_kv, HD / 32), dim3(512), 0, st, true, a);
}

}  // namespace n730

using namespace n730;

N730_API int64_t n730_kv16_attention_ws(const N730KV16Cache* c, int batch, int tokens, int n_heads) {
  if (int rc = kv16_attention_check(c, batch, tokens, n_heads)) return rc;
  return ka_plan(*c, batch, tokens, n_heads).bytes;
}

N730_API int n730_kv16_attention(const N730KV16Cache* c, const void* d_q, int64_t ldq, int batch, int tokens, int n_heads,
                                 float scale, const int32_t* d_lens, const int32_t* d_new, void* d_out, int64_t ldo,
                                 void* d_ws, int64_t ws_bytes, void* stream) {
  const char* what = "kv16_attention";
  if (int rc = kv16_attention_check(c, batch, tokens, n_heads)) return rc;
  N730_REQUIRE(d_q && d_out && d_lens && d_ws, N730_NULL, "%s: null pointer", what);
  const int64_t row = (int64_t)n_heads * c->head_dim;
  N730_REQUIRE(ldq >= row && ldo >= row, N730_BAD_ARG, "%s: row strides %lld, %lld < %d heads x %d", what, (long long)ldq,
               (long long)ldo, n_heads, c->head_dim);
  N730_REQUIRE(kv8_aligned(2, (const char*)d_q, (const char*)d_out) && kv8_aligned(4, d_lens, d_new), N730_BAD_ARG,
               "%s: pointers must lie on whole elements", what);
  const float scale_log2e = scale * 1.4426950408889634f;
  N730_REQUIRE(std::isfinite(scale_log2e), N730_BAD_ARG, "%s: scale %g", what, scale);
  N730_REQUIRE(((uintptr_t)d_ws & 15) == 0, N730_BAD_ARG, "%s: the workspace must be 16-byte aligned", what);
  const KAPlan p = ka_plan(*c, batch, tokens, n_heads);
  N730_REQUIRE(ws_bytes >= p.bytes, N730_BAD_ARG, "%s: workspace of %lld bytes, %lld needed", what, (long long)ws_bytes,
               (long long)p.bytes);
  N730_REQUIRE(p.pre_items + p.own_items < (1ll << 31), N730_BAD_ARG, "%s: 2^31 or more pieces of work", what);
  uint8_t* ws = reinterpret_cast<uint8_t*>(d_ws);
  KAArgs a{};
  a.c = *c;
  a.q = d_q; a.out = d_out; a.ldq = ldq; a.ldo = ldo;
  a.batch = batch; a.tokens = tokens; a.heads = n_heads; a.group = n_heads / c->n_kv;
  a.box = 16;
  while (a.box < KA_KEYS && c->page_size % (2 * a.box) == 0) a.box *= 2;
  a.qvec = ((uintptr_t)d_q & 15) == 0 && ldq % 8 == 0;
  a.ovec = ((uintptr_t)d_out & 7) == 0 && ldo % 4 == 0;
  a.scale_log2e = scale_log2e == 0.f ? 1.f : std::fabs(scale_log2e);
  a.keep = scale_log2e == 0.f ? 0u : ~0u;
  a.sign = scale < 0 ? 0x80008000u : 0u;
  a.lens = d_lens; a.n_new = d_new;
  a.status = reinterpret_cast<int*>(ws);
  if (p.pre_items)
    a.pre = KAParts{p.pre_tiles, p.pre_splits, p.pre_tiles * p.pre_nt * 128, p.pre_nt * 128, reinterpret_cast<float4*>(ws + p.pre_o),
                    reinterpret_cast<float2*>(ws + p.pre_ml)};
  a.own = KAParts{p.own_tiles, p.own_splits, p.own_rows, p.own_nt ? p.own_nt * 128 : KO_ROWS, reinterpret_cast<float4*>(ws + p.own_o),
                  reinterpret_cast<float2*>(ws + p.own_ml)};
  a.by_group = FastDiv(a.group);
  a.by_tokens = FastDiv(tokens);
  CUtensorMap km, vm;
  int rc = ka_map(*c, c->k, a.box, &km);
  if (!rc) rc = ka_map(*c, c->v, a.box, &vm);
  if (rc) return rc;
  const bool bf = c->dtype == N730_BF16;
  cudaStream_t st = (cudaStream_t)stream;
  if (c->head_dim == 128) return bf ? ka_launch<128, true>(a, p, km, vm, st) : ka_launch<128, false>(a, p, km, vm, st);
  return bf ? ka_launch<64, true>(a, p, km, vm, st) : ka_launch<64, false>(a, p, km, vm, st);
}
