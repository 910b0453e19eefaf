// Attention over the 8-bit paged key/value cache.
//
//   out[b, t, head] = softmax_p(scale q . k_p) v_p,  positions p <= lens[b] + t of KV head head / G
//
// Split kernel (single tokens and few rows).  The rows of an item (sequence, KV head) are its
// tokens x G query heads, 8 or 16 at a time.  All items' 32-position tiles form one line that the
// CTAs cut into equal runs, so ragged lengths and few sequences load every SM alike; a run that
// covers part of an item leaves its (max, sum, output) in the workspace, and the finishing kernel
// joins an item's parts in run order, with as many CTAs as there are items.  Within a
// CTA each warp takes every fourth tile.  An item counts for KD_ITEM_COST tiles more than it has, the
// time that starting and ending one takes: without that the CTAs that meet many short sequences were
// the last to finish.  The next run's first tile is asked for before this one's outputs are joined.
//
// The products are transposed, so that a key or a channel is a row of mma.m16n8k16's A and the few
// query rows are its 8 columns: no half of an instruction works on rows that are not there.
//   S^T = K Q^T: the order of the channels in the sum is free, so lane (g, t) feeds 16 contiguous
//      bytes of keys g and g + 8, each 4 of them one k-step's slots.
//   O^T = V^T P^T: lane (g, t) feeds 16 contiguous channels of keys 2t, 2t+1, 2t+8, 2t+9,
//      interleaved by byte permutes; P^T comes from S^T by an 8x8 transposition between lanes.
// Each warp fills its own two tile buffers with tensor copies (no barrier between warps in the loop).
// Rows of 128 (64) bytes lie swizzled, and the order of the 16 keys of a product is chosen so that
// the lanes of one shared-memory wavefront meet no bank twice in either product (key_of).  Copies
// of 16 bytes per lane (cp.async) in fragment order reached 4.1 TB/s even without any arithmetic.
// int8 codes become fp16 exactly (1024 + 128 + q by a byte permute, then one subtraction), e4m3
// codes by a conversion.  K's scale multiplies the scores, V's scale the weights.
//
// Softmax.  Weights are kept against a reference that follows the maximum only when a score is more
// than 2^8 above it, so a tile costs one vote and no reduction; a second reference does the same for
// weight x V scale (P), which has to fit fp16 whatever the scales are: the largest P so far lies between 2^KV8_P_NEW
// (fp32 rows: 2^KD_P_NEW_LO), where a new reference puts it, and 2^KV8_P_MOST, where the reference moves.
//
// Numerics.  Queries are scaled by a power of two per row so that a 16-bit query is exact in fp16; an
// fp32 query is split into two fp16 terms, and so is P, which loses 2^-22 of each down to 2^-16 of a warp's largest P and
// 2^-38 of that largest below (fp16's smallest step under 2^13).  For 16-bit calls P is rounded to fp16: 2^-11 of each,
// below the rounding of the output, down to 2^-21 of the largest, 2^-32 of the largest below.  Maxima, sums and outputs
// are fp32.
//
// Bound by HBM: 2 head_dim code bytes and 8 / block of scales a position and KV head.  Whole calls: 128 sequences
// ragged to 4096, 64 / 8 heads x 128, e4m3, 116.5 us (5.2 TB/s); one of 65501 positions 36.5 us, of which 5 start
// and 5 join; 32 ragged to 8192 of 28 / 4 heads with weights 53.7 us, 31 here and 13 in the finishing kernel.  fp32 rows
// take two products for each one: 64 sequences of 2048, 28 / 4 heads, 45.6 us for 39.6 of 16-bit rows, and a prompt of
// 300 behind 724 499 us, every 8 rows reading the context.
#include <algorithm>
#include <mutex>

#include <cuda.h>
#include <cudaTypedefs.h>

#include "kv8.h"

namespace n730 {

constexpr int KD_WARPS = 4;
constexpr int KD_THREADS = KD_WARPS * 32;
constexpr int KD_STAGES = 2;     // tile buffers of a warp
constexpr int KD_TILE = 32;      // positions
constexpr int KD_CTAS_PER_SM = 3;
// What starting and ending an item counts for on the line, in tiles.  Batch of 128 ragged sequences up to 4096 (72B
// heads): 3 131.8 us, 6 124.9, 10 120.5, 16 116.1, 24 117.1, 40 121.1; batch of 32 with weights 55.6, 53.9, 53.4,
// 52.7, 53.2, 54.7.
constexpr int KD_ITEM_COST = 16;
constexpr int KD_MIN_UNITS = 4;  // tiles of a run: fewer would leave warps idle and joins to do
constexpr float KD_SLACK = 8.f;  // log2 of how far a weight in the sum (fp32) may exceed its reference
constexpr float KD_P_NEW_LO = 13.f;  // as KV8_P_NEW for two-term P, whose second term runs out of fp16's range first
constexpr uint64_t KD_WAIT_NS = 1000000000;  // bound of a wait for copies

struct KDArgs {
  N730KV8Cache c;
  const void* q; void* out;
  int64_t ldq, ldo;
  int dtype, odtype, batch, tokens, heads, group, rows, nrg;  // rows = chunk * group; nrg row groups of RG
  int t0, chunk;       // the call's tokens [t0, t0 + chunk) of each sequence
  float scale_log2e;
  const int* lens; const int* n_new;
  int* status;         // set when a wait ran out
  int2* parts;         // [batch][n_kv][nrg] first CTA and number of parts of an item, for the finishing kernel
  float* part;         // [2 * n_cta][RG][HD]
  float* part_ml;      // [2 * n_cta][RG][4]: reference of the output, max, sum
  float* lse;          // [batch][n_kv][rows] log2 of the softmax sum, +inf for an empty row (items of one run)
  float* scores;       // [batch][n_kv][rows][cap] base-2 scores (weights only)
  int n_cta, log_block, box;  // box: rows of a copy, 32, or 16 where pages are no multiples of 32
};

template <int HD>
struct KDGeom {
  static constexpr int KCH = HD / 64;                 // 16-byte K chunks per lane and key
  static constexpr int VB = HD / 8;                   // V bytes per lane and key
  static constexpr int KV_BYTES = KD_TILE * HD;       // K (or V) codes of a tile
  static constexpr int TILE_BYTES = 2 * KV_BYTES;
  // byte of 16-byte chunk c of row r: the copies' 128-byte (64-byte) swizzle
  static __device__ __forceinline__ int chunk(int r, int c) {
    return HD == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  }
  // row of the i-th key of the first 8 of a product (the second 8: + 8)
  static __device__ __forceinline__ int key_of(int i) {
    const int e = HD == 128 ? i & 6 : ((i >> 1) & 1) + ((i >> 2) << 2);  // even i: 0 2 4 6, or 0 1 4 5
    return (i & 1) == 0 ? e : HD == 128 ? (e ^ 4) + 1 : e ^ 3;
  }
};

// one CTA's run through one item
struct KDSeg {
  int valid;
  int b, h, rg;         // sequence, KV head, row group
  int ta, te, units;    // tiles [ta, te) of the item's `units`
  int L, total;         // positions cached before the call, with the new rows
  int f0, nrow;         // first row, rows
};

template <int HD>
struct KDSmem {
  uint8_t ring[KD_WARPS][KD_STAGES][KDGeom<HD>::TILE_BYTES];
  uint2 qf[2][HD / 16][32];        // Q^T as the B operand by k-step and lane: rows 8-15 or low terms second
  uint64_t full[KD_WARPS][KD_STAGES];
  float sc[KD_WARPS][KD_STAGES][4];  // scales of K, V of the tile's two halves
  int ok[KD_WARPS][KD_STAGES];     // bit i: half i has a page
  float rowmul[16];
  float wm[KD_WARPS][16], wmo[KD_WARPS][16], wl[KD_WARPS][16];
  float tot[16][4];
  int out_at[KD_WARPS];            // buffer of each warp's outputs
  KDSeg seg[3];                    // this run, the next, and the last one's, which slow warps may still read
  int pre[1];                      // [batch + 1] prefix sums of the line, then [batch] lengths, [batch] new rows
};

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) { return h2_bits(__floats2half2_rn(lo, hi)); }
__device__ __forceinline__ void mma16816(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// 8x8 matrix of 16-bit elements, one row of two columns a lane: transposed between the lanes
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// 2-D tensor copy (no multicast) of the box whose first row is `row`, completing on `bar`
__device__ __forceinline__ void copy_rows(uint32_t dst, const CUtensorMap* map, int row, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(smem_u32(bar)) : "memory");
}
// 4 bytes, or zeros
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool pred) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" :: "r"(dst), "l"(src), "r"(pred ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

// a sequence's new rows among tokens [t0, t0 + chunk), and the positions cached before them
__device__ __forceinline__ int kd_new(const KDArgs& a, int b) {
  return min(max(kv8_new(a.n_new, b, a.tokens) - a.t0, 0), a.chunk);
}
__device__ __forceinline__ int kd_len(const KDArgs& a, int b, int cap) {
  return (int)min((int64_t)kv8_len(a.lens, b, cap) + a.t0, (int64_t)cap);
}
// tiles of a sequence with new rows
__device__ __forceinline__ int kd_units(int L, int n_new, int cap) {
  return (int)((min((int64_t)L + n_new, (int64_t)cap) + KD_TILE - 1) / KD_TILE);
}

// a / b for 0 <= a, 0 < b: by 32 bits where that is enough (a 64-bit division is a long sequence)
__device__ __forceinline__ int64_t kd_div(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
// the CTA of N whose part of the line of U holds tile u
__device__ __forceinline__ int kd_owner(int64_t u, int64_t U, int64_t N) { return (int)kd_div((u + 1) * N - 1, U); }

// The answer of row f, channels d..d + 3: sums of weight x V against Mo, of weights l against M.
template <int HD>
__device__ __forceinline__ void kd_answer(const KDArgs& a, int b, int h, int f, int d, const float4& num, float Mo, float M, float l) {
  // by two factors, whose product may leave fp32's normal range when the answer does not; a NaN query: NaN
  const float s = l == 0.f ? 0.f : 1.f / l, f2 = l == 0.f || Mo == -INFINITY ? 0.f : ex2(Mo - M);
  const int64_t at = ((int64_t)b * a.tokens + a.t0 + f / a.group) * a.ldo + (int64_t)(h * a.group + f % a.group) * HD + d;
  kv8_store1(a.out, at, a.odtype, num.x * s * f2);
  kv8_store1(a.out, at + 1, a.odtype, num.y * s * f2);
  kv8_store1(a.out, at + 2, a.odtype, num.z * s * f2);
  kv8_store1(a.out, at + 3, a.odtype, num.w * s * f2);
}

// NB: 8-row groups of an item's rows worked on together; LO: fp32 rows in two fp16 terms.
template <int HD, int CODE, int NB, bool LO>
__global__ void __launch_bounds__(KD_THREADS, KD_CTAS_PER_SM) kv8_split_kernel(const KDArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using G = KDGeom<HD>;
  constexpr int RG = 8 * NB, KS = HD / 16, MT = HD / 16, ST = KD_STAGES;
  constexpr float P_NEW = LO ? KD_P_NEW_LO : KV8_P_NEW;
  constexpr int TT = NB == 1 ? 2 : 1;  // halves of a tile worked on together: independent chains for the tensor cores
  extern __shared__ __align__(1024) uint8_t kd_raw[];
  KDSmem<HD>& sm = *reinterpret_cast<KDSmem<HD>*>(aligned_smem(kd_raw));
  static_assert(ST == 2 && sizeof(float) * RG * HD <= G::TILE_BYTES, "a warp's outputs fit the buffer that is not being filled");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const N730KV8Cache& c = a.c;
  const int cap = c.max_pages * c.page_size;
  if (lane == 0) {
    for (int s = 0; s < ST; ++s) mbar_init(&sm.full[warp][s], 1);
    fence_mbar_init();
  }
  bool lost = false;   // a wait of the warp ran out: it asks for nothing more
  uint32_t fills = 0;  // tiles this warp has asked for, and used: buffer and phase go by them
  uint32_t uses = 0;
  pdl_wait();

  // ---- the line: prefix sums of items x (tiles + KD_ITEM_COST) / items ----
  int* const len_of = sm.pre + a.batch + 1;
  int* const new_of = len_of + a.batch;
  if (warp == 0) {
    int run = 0;
    if (lane == 0) sm.pre[0] = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      const int b = b0 + lane;
      int v = 0;
      if (b < a.batch) {
        const int n = kd_new(a, b), L = kd_len(a, b, cap);
        len_of[b] = L;
        new_of[b] = n;
        v = n ? kd_units(L, n, cap) + KD_ITEM_COST : 0;
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
      }
      if (b < a.batch) sm.pre[b + 1] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  pdl_launch_dependents();  // the finishing kernel waits for this grid's end
  const int items = c.n_kv * a.nrg;  // per sequence
  const int64_t U = (int64_t)sm.pre[a.batch] * items;
  const int64_t N = min((int64_t)a.n_cta, (U + KD_MIN_UNITS - 1) / KD_MIN_UNITS);
  const int cta = blockIdx.x;
  if (cta >= N) return;
  // one thread walks the CTA's part [u, u1) of the line
  int64_t u = kd_div(U * cta, N);
  const int64_t u1 = kd_div(U * (cta + 1), N);
  int at_b = -1;
  auto next_run = [&](KDSeg& s) {
    s.valid = 0;
    if (at_b < 0) {
      int lo = 0, hi = a.batch - 1;  // the last b with pre[b] * items <= u
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((int64_t)sm.pre[mid] * items <= u) lo = mid; else hi = mid - 1;
      }
      at_b = lo;
    }
    while (u < u1) {
      while ((int64_t)sm.pre[at_b + 1] * items <= u) ++at_b;  // past sequences without tiles
      const int b = at_b, span = sm.pre[b + 1] - sm.pre[b];
      const int64_t base = (int64_t)sm.pre[b] * items, ub = u - base;
      const int item = (int)kd_div(ub, span), off = (int)(ub - (int64_t)item * span);
      const int end = (int)min((int64_t)span, off + (u1 - u));
      u += end - off;
      s.f0 = item % a.nrg * RG;
      s.nrow = min(RG, new_of[b] * a.group - s.f0);
      s.ta = max(0, off - KD_ITEM_COST);
      s.te = end - KD_ITEM_COST;
      if (s.te <= s.ta || s.nrow <= 0) continue;  // only the item's cost, or rows behind the sequence's new ones
      s.valid = 1;
      s.b = b; s.h = item / a.nrg; s.rg = item % a.nrg;
      s.units = span - KD_ITEM_COST;
      s.L = len_of[b];
      s.total = (int)min((int64_t)s.L + new_of[b], (int64_t)cap);
      if (s.ta == 0)
        a.parts[((int64_t)b * c.n_kv + s.h) * a.nrg + s.rg] =
            make_int2(cta, kd_owner(base + (int64_t)(item + 1) * span - 1, U, N) - cta + 1);
      break;
    }
  };
  constexpr int WALKER = KD_THREADS - 32;  // its first lane walks
  if (tid == WALKER) next_run(sm.seg[0]);
  __syncthreads();

  // ---- the warp's tiles of a run: every KD_WARPS-th ----
  auto tiles_of = [&](const KDSeg& s) { return s.te - s.ta > warp ? (s.te - s.ta - warp + KD_WARPS - 1) / KD_WARPS : 0; };
  // pool row of half tile q0 + lane (-1: no page), looked up 16 tiles at a time
  auto lookup = [&](const KDSeg& s, int q0) {
    const int p = (s.ta + warp + ((q0 + lane) >> 1) * KD_WARPS) * KD_TILE + (lane & 1) * 16;
    if (p >= min(s.total, s.te * KD_TILE)) return -1;
    const int page = c.block_table[(int64_t)s.b * c.max_pages + p / c.page_size];
    return (unsigned)page < (unsigned)c.n_pages ? (page * c.n_kv + s.h) * c.page_size + p % c.page_size : -1;
  };
  // ask for a tile whose half rows are lanes 2 i, 2 i + 1 of `rows`
  auto issue = [&](int rows, int i) {
    if (lost) return;
    const int st = fills % ST;
    ++fills;
    const int row0 = __shfl_sync(0xffffffffu, rows, 2 * i), row1 = __shfl_sync(0xffffffffu, rows, 2 * i + 1);
    if (lane == 0) {
      const uint32_t dst = smem_u32(sm.ring[warp][st]);
      uint64_t* bar = &sm.full[warp][st];
      sm.ok[warp][st] = (row0 >= 0 ? 1 : 0) | (row1 >= 0 ? 2 : 0);
      if (a.box == KD_TILE) {
        mbar_arrive_expect_tx(bar, row0 >= 0 ? G::TILE_BYTES : 0);
        if (row0 >= 0) {
          copy_rows(dst, &kmap, row0, bar);
          copy_rows(dst + G::KV_BYTES, &vmap, row0, bar);
        }
      } else {
        mbar_arrive_expect_tx(bar, (row0 >= 0 ? G::KV_BYTES : 0) + (row1 >= 0 ? G::KV_BYTES : 0));
        if (row0 >= 0) {
          copy_rows(dst, &kmap, row0, bar);
          copy_rows(dst + G::KV_BYTES, &vmap, row0, bar);
        }
        if (row1 >= 0) {
          copy_rows(dst + G::KV_BYTES / 2, &kmap, row1, bar);
          copy_rows(dst + G::KV_BYTES * 3 / 2, &vmap, row1, bar);
        }
      }
    }
    if (lane < 4) {
      const int row = lane < 2 ? row0 : row1;
      const float* s = ((lane & 1) ? c.v_scales : c.k_scales) + (max(row, 0) >> a.log_block);
      cp_async4(smem_u32(&sm.sc[warp][st][lane]), s, row >= 0);
    }
  };
  // the warp's rows of a run's queries: asked for a run ahead and ahead of tiles (two row groups
  // have no registers for that)
  constexpr int QR = RG / KD_WARPS, QE = HD / 32;  // rows a warp, channels a lane
  float qx[QR][QE];
  auto load_q = [&](const KDSeg& s) {
#pragma unroll
    for (int i = 0; i < QR; ++i) {
      const int r = warp + i * KD_WARPS, f = s.f0 + r;
      const int64_t qb = ((int64_t)s.b * a.tokens + a.t0 + f / a.group) * a.ldq + (int64_t)(s.h * a.group + f % a.group) * HD + lane * QE;
#pragma unroll
      for (int e = 0; e < QE; ++e) qx[i][e] = r < s.nrow ? kv8_load1(a.q, qb + e, a.dtype) : 0.f;
    }
  };
  int rows_now = -1;
  if (sm.seg[0].valid) {
    rows_now = lookup(sm.seg[0], 0);
    if (NB == 1) load_q(sm.seg[0]);
    if (tiles_of(sm.seg[0])) issue(rows_now, 0);
  }
  cp_commit();

  for (int turn = 0;; ++turn) {
    const KDSeg& run = sm.seg[turn % 3];
    const KDSeg& after = sm.seg[(turn + 1) % 3];
    if (!run.valid) break;
    const int b = run.b, h = run.h, f0 = run.f0, nrow = run.nrow, L = run.L, total = run.total, ta = run.ta;
    const int n_tile = lost ? 0 : tiles_of(run);
    int rows_next = lookup(run, 32);
    if (tid == WALKER) next_run(sm.seg[(turn + 1) % 3]);

    // ---- Q: a row per warp at a time, scaled by a power of two, as the B operand ----
    if (NB == 2) load_q(run);
#pragma unroll
    for (int i = 0; i < QR; ++i) {
      const int r = warp + i * KD_WARPS;
      float m = 0.f;
#pragma unroll
      for (int e = 0; e < QE; ++e) m = fmaxf(m, fabsf(qx[i][e]));
      m = warp_max(m);
      // the largest magnitude goes into [2^13, 2^14); rows of zeros or with an infinity stay
      const int ex = (int)((__float_as_uint(m) >> 23) & 255u);
      const bool plain = ex == 0 || ex == 255;
      const int sh = plain ? 0 : min(max(140 - ex, -126), 126);
      const float mul = __uint_as_float((uint32_t)(127 + sh) << 23);
      if (lane == 0) sm.rowmul[r] = a.scale_log2e * __uint_as_float((uint32_t)(127 - sh) << 23);
#pragma unroll
      for (int e = 0; e < QE; ++e) {
        const int dch = lane * QE + e, ks = (dch >> 6) * 4 + ((dch >> 2) & 3), tt = (dch >> 4) & 3, w = dch & 3;
        const float y = qx[i][e] * mul;
        const __half hi = __float2half_rn(y);
        reinterpret_cast<__half*>(&sm.qf[LO ? 0 : r >> 3][ks][(r & 7) * 4 + tt])[w] = hi;
        if (LO)  // an infinite y gives NaN, as it should
          reinterpret_cast<__half*>(&sm.qf[1][ks][(r & 7) * 4 + tt])[w] = __float2half_rn(y - __half2float(hi));
      }
    }
    // what the last run's threads did to shared memory comes before the copies of this one's loop
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    const int rows_after = after.valid ? lookup(after, 0) : -1;
    uint2 qreg[NB == 1 && !LO ? KS : 1];  // one row group's Q stays in registers, two are read as needed
    if (NB == 1 && !LO)
#pragma unroll
      for (int k = 0; k < KS; ++k) qreg[k] = sm.qf[0][k][lane];
    float rm[NB][2];
    int vis[NB][2];  // positions below vis are seen by the row
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = n * 8 + 2 * t4 + e;
        const bool live = r < nrow;
        rm[n][e] = live ? sm.rowmul[r] : 0.f;
        vis[n][e] = live ? (int)min((int64_t)L + (f0 + r) / a.group + 1, (int64_t)cap) : 0;
      }
    const int all_see = (int)min((int64_t)L + f0 / a.group + 1, (int64_t)cap);  // positions every row sees
    const int kg = G::key_of(g), kv0 = G::key_of(2 * t4), kv1 = G::key_of(2 * t4 + 1);
    float* score_row = a.scores ? a.scores + (((int64_t)b * c.n_kv + h) * a.rows + f0) * cap : nullptr;

    float o[NB][MT][4];  // O^T: channels g HD/8 + 2 u, + 1 (c0 c1, c2 c3) of rows 2 t4, 2 t4 + 1
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int k = 0; k < MT; ++k) o[n][k][0] = o[n][k][1] = o[n][k][2] = o[n][k][3] = 0.f;
    float m_ref[NB][2], mo_ref[NB][2], fm[NB][2], l_run[NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) { m_ref[n][e] = mo_ref[n][e] = -INFINITY; fm[n][e] = l_run[n][e] = 0.f; }

    for (int qi = 0; qi < n_tile; ++qi) {
      __syncwarp();  // every lane is done with the buffer that the next copies go to
      if (qi + 1 < n_tile) {
        if (((qi + 1) & 15) == 0) { rows_now = rows_next; rows_next = lookup(run, 2 * (qi + 1) + 32); }
        issue(rows_now, (qi + 1) & 15);
      }
      cp_commit();
      const int st = uses % ST;
      // the same twice: as a value the verdict costs the two-term form registers (64 sequences of 2048 fp32 rows 47.1 us
      // for 45.7, a prompt of 300 541 for 499), as a branch the other form (64 of 16-bit rows 40.7 us for 39.6)
      if (LO) {
        if (!kv8_wait(&sm.full[warp][st], (uses / ST) & 1, KD_WAIT_NS)) { lost = true; break; }
      } else {
        lost = !kv8_wait(&sm.full[warp][st], (uses / ST) & 1, KD_WAIT_NS);
        if (lost) break;
      }
      ++uses;
      cp_wait<ST - 1>();
      __syncwarp();
      const int okm = sm.ok[warp][st];
#pragma unroll
      for (int t0 = 0; t0 < 2; t0 += TT) {
      float y[TT][NB][4];  // base-2 scores: keys key_of(g) (0, 1) and + 8 (2, 3) of rows 2 t4, 2 t4 + 1
      float vsc[TT], lv[TT];
      int p0[TT];
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
        const int half = t0 + tt;
        const bool seen = (okm >> half) & 1;
        p0[tt] = (ta + warp + qi * KD_WARPS) * KD_TILE + half * 16;
        const float ksc = seen ? sm.sc[warp][st][2 * half] : 0.f;
        vsc[tt] = seen ? sm.sc[warp][st][2 * half + 1] : 0.f;
        if (vsc[tt] < KV8_TINY) vsc[tt] = 0.f;
        lv[tt] = lg2(vsc[tt]);
        const uint8_t* kt = sm.ring[warp][st] + half * 16 * HD;
        float s[G::KCH][NB][4];
#pragma unroll
        for (int j = 0; j < G::KCH; ++j) {
#pragma unroll
          for (int n = 0; n < NB; ++n) s[j][n][0] = s[j][n][1] = s[j][n][2] = s[j][n][3] = 0.f;
          const uint4 k0 = *reinterpret_cast<const uint4*>(kt + G::chunk(kg, j * 4 + t4));
          const uint4 k1 = *reinterpret_cast<const uint4*>(kt + 8 * HD + G::chunk(kg, j * 4 + t4));
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t x0 = code_word<CODE>(w0[e]), x1 = code_word<CODE>(w1[e]);
            const uint4 ka = make_uint4(codes2<CODE, 0>(x0), codes2<CODE, 0>(x1), codes2<CODE, 1>(x0), codes2<CODE, 1>(x1));
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              const uint2 q = NB == 1 && !LO ? qreg[NB == 1 && !LO ? j * 4 + e : 0] : sm.qf[n][j * 4 + e][lane];
              mma16816(s[j][n], ka, q.x, q.y);
              if (LO) {
                const uint2 ql = sm.qf[1][j * 4 + e][lane];
                mma16816(s[j][n], ka, ql.x, ql.y);
              }
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float raw = G::KCH == 2 ? s[0][n][e] + s[G::KCH - 1][n][e] : s[0][n][e];
            y[tt][n][e] = raw * (rm[n][e & 1] * ksc);
          }
        if (p0[tt] + 16 > all_see || !seen) {
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (p0[tt] + kg + 8 * (e >> 1) >= vis[n][e & 1] || !seen) y[tt][n][e] = -INFINITY;
        }
        if (score_row && p0[tt] < cap) {
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = n * 8 + 2 * t4 + (e & 1);
              if (r < nrow) score_row[(int64_t)r * cap + p0[tt] + kg + 8 * (e >> 1)] = y[tt][n][e];
            }
        }
      }
      // ---- move the references when a weight would be too large against them ----
      bool move = false;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = -INFINITY, mv = -INFINITY;
#pragma unroll
          for (int tt = 0; tt < TT; ++tt) {
            const float x = fmaxf(y[tt][n][e], y[tt][n][e + 2]);
            mx = fmaxf(mx, x);
            mv = fmaxf(mv, x + lv[tt]);
          }
          move |= mx > m_ref[n][e] + KD_SLACK || mv > mo_ref[n][e] + KV8_P_MOST;
        }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = m_ref[n][e], mv = -INFINITY;
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
              const float x = fmaxf(y[tt][n][e], y[tt][n][e + 2]);
              mx = fmaxf(mx, x);
              mv = fmaxf(mv, x + lv[tt]);
            }
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) {
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
              mv = fmaxf(mv, __shfl_xor_sync(0xffffffffu, mv, k));
            }
            mv = fmaxf(fmaxf(mo_ref[n][e], mx - KV8_REFS_APART), mv - P_NEW);
            if (mx != m_ref[n][e]) {  // from -infinity: the sums are still 0
              l_run[n][e] *= ex2(m_ref[n][e] - mx);
              m_ref[n][e] = mx;
            }
            if (mv != mo_ref[n][e]) {
              const float f = ex2(mo_ref[n][e] - mv);
#pragma unroll
              for (int k = 0; k < MT; ++k) { o[n][k][e] *= f; o[n][k][e + 2] *= f; }
              mo_ref[n][e] = mv;
            }
            fm[n][e] = mv == -INFINITY ? 0.f : ex2(mx - mv);
          }
      }
      // ---- O^T += V^T P^T ----
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
        const uint8_t* vt = sm.ring[warp][st] + G::KV_BYTES + (t0 + tt) * 16 * HD;
        uint32_t pb[NB][2], pl[NB][2];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          float w[4];
          // weight x V scale: V scale x fm leaves fp32's range where a row sees little or nothing of a block whose scale
          // is far above its others'; the weight goes first then
          float f1[2], f2[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float f = vsc[tt] * fm[n][e];
            const bool in_range = f < 0x1p127f;
            f1[e] = in_range ? f : vsc[tt];
            f2[e] = in_range ? 1.f : fm[n][e];
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float m = m_ref[n][e & 1];
            const float pe = ex2(y[tt][n][e] - (m == -INFINITY ? 0.f : m));
            l_run[n][e & 1] += pe;
            w[e] = pe * f1[e & 1] * f2[e & 1];
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t hi = pack_h2(w[2 * i], w[2 * i + 1]);
            pb[n][i] = transpose8(hi);
            if (LO) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
              pl[n][i] = transpose8(pack_h2(w[2 * i] - f.x, w[2 * i + 1] - f.y));
            }
          }
        }
        constexpr int VW = G::VB / 4;  // words a key
        uint32_t v[4][VW];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = (i & 1) ? kv1 : kv0;
          const uint8_t* src = vt + 8 * (i >> 1) * HD + (HD == 128 ? G::chunk(r, g) : G::chunk(r, g >> 1) + (g & 1) * 8);
          if (VW == 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(src);
            v[i][0] = x.x; v[i][1] = x.y; v[i][VW - 2] = x.z; v[i][VW - 1] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(src);
            v[i][0] = x.x; v[i][1] = x.y;
          }
        }
        if (p0[tt] + 16 > total || !((okm >> (t0 + tt)) & 1)) {  // rows never written may hold NaN codes
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (p0[tt] + ((i & 1) ? kv1 : kv0) + 8 * (i >> 1) >= total || !((okm >> (t0 + tt)) & 1))
#pragma unroll
              for (int k = 0; k < VW; ++k) v[i][k] = 0u;
        }
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          const uint32_t v0 = code_word<CODE>(v[0][k]), v1 = code_word<CODE>(v[1][k]);
          const uint32_t v2 = code_word<CODE>(v[2][k]), v3 = code_word<CODE>(v[3][k]);
          const uint32_t a01 = __byte_perm(v0, v1, 0x5140), b01 = __byte_perm(v0, v1, 0x7362);
          const uint32_t a23 = __byte_perm(v2, v3, 0x5140), b23 = __byte_perm(v2, v3, 0x7362);
          const uint4 va = make_uint4(codes2<CODE, 0>(a01), codes2<CODE, 1>(a01), codes2<CODE, 0>(a23), codes2<CODE, 1>(a23));
          const uint4 vb = make_uint4(codes2<CODE, 0>(b01), codes2<CODE, 1>(b01), codes2<CODE, 0>(b23), codes2<CODE, 1>(b23));
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            mma16816(o[n][2 * k], va, pb[n][0], pb[n][1]);
            mma16816(o[n][2 * k + 1], vb, pb[n][0], pb[n][1]);
            if (LO) {
              mma16816(o[n][2 * k], va, pl[n][0], pl[n][1]);
              mma16816(o[n][2 * k + 1], vb, pl[n][0], pl[n][1]);
            }
          }
        }
      }
      }
    }
    if (lost && lane == 0) *a.status = 1;
    __syncwarp();
    // the next run's first tile goes into one buffer, this run's outputs into the other
    rows_now = rows_after;
    if (after.valid) {
      if (NB == 1) load_q(after);
      if (tiles_of(after)) issue(rows_now, 0);
    }
    cp_commit();
    float* const mine = reinterpret_cast<float*>(sm.ring[warp][fills % ST]);  // [row][HD], 16-byte groups spread by row

    // ---- join the warps ----
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) l_run[n][e] += __shfl_xor_sync(0xffffffffu, l_run[n][e], k);
        if (g == 0) {
          const int r = n * 8 + 2 * t4 + e;
          sm.wm[warp][r] = m_ref[n][e];
          sm.wmo[warp][r] = mo_ref[n][e];
          sm.wl[warp][r] = l_run[n][e];
        }
      }
    if (lane == 0) sm.out_at[warp] = fills % ST;
    // 16-byte group q of row r lies at q ^ (r & 7): the lanes of a store meet few banks twice
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < MT; ++k) {
          const int r = n * 8 + 2 * t4 + e, d = g * G::VB + 2 * k;
          *reinterpret_cast<float2*>(mine + r * HD + (((d >> 2) ^ (r & 7)) << 2) + (d & 2)) = make_float2(o[n][k][e], o[n][k][e + 2]);
        }
    __syncthreads();
    const bool whole = ta == 0 && run.te == run.units;
    const int slot = 2 * cta + (ta == 0 ? 1 : 0);
    if (tid < RG) {
      float M = -INFINITY, Mo = -INFINITY, l = 0.f;
#pragma unroll
      for (int k = 0; k < KD_WARPS; ++k) { M = fmaxf(M, sm.wm[k][tid]); Mo = fmaxf(Mo, sm.wmo[k][tid]); }
      const float ms = M == -INFINITY ? 0.f : M, mos = Mo == -INFINITY ? 0.f : Mo;
#pragma unroll
      for (int k = 0; k < KD_WARPS; ++k) {
        l += sm.wl[k][tid] * ex2(sm.wm[k][tid] - ms);
        sm.wmo[k][tid] = ex2(sm.wmo[k][tid] - mos);
      }
      sm.tot[tid][0] = Mo; sm.tot[tid][1] = M; sm.tot[tid][2] = l;
      if (!whole && tid < nrow)
        *reinterpret_cast<float4*>(a.part_ml + ((int64_t)slot * RG + tid) * 4) = make_float4(Mo, M, l, 0.f);
    }
    __syncthreads();
    for (int i = tid; i < nrow * (HD / 4); i += KD_THREADS) {
      const int r = i / (HD / 4), d = i % (HD / 4) * 4;
      float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < KD_WARPS; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm.ring[k][sm.out_at[k]]) + r * HD +
                                                          (((d >> 2) ^ (r & 7)) << 2));
        const float f = sm.wmo[k][r];
        num.x = fmaf(x.x, f, num.x); num.y = fmaf(x.y, f, num.y); num.z = fmaf(x.z, f, num.z); num.w = fmaf(x.w, f, num.w);
      }
      if (whole) kd_answer<HD>(a, b, h, f0 + r, d, num, sm.tot[r][0], sm.tot[r][1], sm.tot[r][2]);
      else *reinterpret_cast<float4*>(a.part + ((int64_t)slot * RG + r) * HD + d) = num;
    }
    if (whole && a.lse && tid < nrow)
      a.lse[((int64_t)b * c.n_kv + h) * a.rows + f0 + tid] =
          sm.tot[tid][2] == 0.f ? INFINITY : sm.tot[tid][1] + log2f(sm.tot[tid][2]);
  }
  cp_wait<0>();
  if (lost)  // copies in flight end before the shared memory they go to is given up
    for (; uses != fills; ++uses) kv8_wait(&sm.full[warp][uses % ST], (uses / ST) & 1, KD_WAIT_NS);
}

// ---------------------------------------------------------------------------
// Finishing: joins the parts of items that several CTAs worked on, and accumulates the softmax weights:
//   w[b, h, p] += sum over the KV head's rows of exp2(score - lse), in row order.
// The first rg / rb blocks of each row group join rb of its rows of (head y, sequence z), with as many of
// the block's 4 warps on a row as rb leaves; blocks behind them take 512 positions each.
// ---------------------------------------------------------------------------
constexpr int KF_THREADS = 128;
constexpr int KF_POSITIONS = 4 * KF_THREADS;

struct KFArgs {
  KDArgs d;
  int rg, rb;
  int splits;  // room for parts of an item, one behind the other (prompts); 0: by the parts table
  const float* w_in; float* w_out;
  int64_t ldw;
};

// An item's parts: row r of part k lies in the first CTA's second slot (k = 0), the others' first.
__device__ __forceinline__ int64_t kf_row(const KFArgs& a, const int2& p, int k, int r) {
  return (a.splits ? (int64_t)(p.x + k) : (int64_t)(2 * (p.x + k) + (k == 0))) * a.rg + r;
}
// A warp's log2 of the softmax sum of row r over the parts (+inf for an empty row).
__device__ __forceinline__ float kf_lse_of(const KFArgs& a, const int2& p, int r) {
  float M = -INFINITY, l = 0.f;
  for (int k = threadIdx.x & 31; k < p.y; k += 32) {
    const float4 ml = reinterpret_cast<const float4*>(a.d.part_ml)[kf_row(a, p, k, r)];
    const float m = fmaxf(M, ml.y), ms = m == -INFINITY ? 0.f : m;
    l = l * ex2(M - ms) + ml.z * ex2(ml.y - ms);
    M = m;
  }
  const float m = warp_max(M), ms = m == -INFINITY ? 0.f : m;
  l = warp_sum(l * ex2(M - ms));
  return l == 0.f ? INFINITY : m + log2f(l);
}

// sums of weight x V against mo, and of weights l against m, of two sets of parts
struct KFSum { float4 num; float mo, m, l; };
__device__ __forceinline__ void kf_add(KFSum& s, const float4& x, float mo, float m, float l) {
  const float o1 = fmaxf(s.mo, mo), os = o1 == -INFINITY ? 0.f : o1, m1 = fmaxf(s.m, m), ms = m1 == -INFINITY ? 0.f : m1;
  const float f = ex2(s.mo - os), g = ex2(mo - os);
  s.num.x = fmaf(x.x, g, s.num.x * f); s.num.y = fmaf(x.y, g, s.num.y * f);
  s.num.z = fmaf(x.z, g, s.num.z * f); s.num.w = fmaf(x.w, g, s.num.w * f);
  s.l = s.l * ex2(s.m - ms) + l * ex2(m - ms);
  s.mo = o1;
  s.m = m1;
}

template <int HD>
__global__ void __launch_bounds__(KF_THREADS) kv8_finish_kernel(const KFArgs a) {
  constexpr int LPP = HD / 4, WARPS = KF_THREADS / 32;  // lanes that a part of a row takes
  extern __shared__ float kf_lse[];
  __shared__ KFSum share[KF_THREADS];
  const KDArgs& d = a.d;
  const N730KV8Cache& c = d.c;
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cap = c.max_pages * c.page_size;
  pdl_wait();
  const int n_new = kd_new(d, b), rows_b = n_new * d.group;
  const int joins = d.nrg * (a.rg / a.rb);
  if ((int)blockIdx.x < joins) {
    const int rg = blockIdx.x / (a.rg / a.rb), first = blockIdx.x % (a.rg / a.rb) * a.rb, f0 = rg * a.rg;
    if (f0 + first >= rows_b) return;
    const int64_t item = ((int64_t)b * c.n_kv + h) * d.nrg + rg;
    int2 p;
    if (a.splits) {  // as many as the prompt kernel used for what the rows see
      const int sees = (int)min((int64_t)kd_len(d, b, cap) + (min(f0 + a.rg, rows_b) - 1) / d.group + 1, (int64_t)cap);
      p = make_int2((int)item * a.splits, kv8_shares_used(sees, a.splits));
    } else {
      p = d.parts[item];
    }
    if (p.y == 1) return;  // its CTA gave the answer
    const int per_row = a.rb >= WARPS ? 1 : WARPS / a.rb;  // warps
    const int shares = per_row * (32 / LPP), mine = warp % per_row * (32 / LPP) + lane / LPP, d4 = lane % LPP;
    for (int i = 0; i < a.rb; i += WARPS / per_row) {
      const int r = first + i + warp / per_row;
      const bool live = f0 + r < rows_b;
      KFSum sum{make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, -INFINITY, 0.f};
      constexpr int CH = 8;  // parts asked for together
      for (int k0 = mine; live && k0 < p.y; k0 += CH * shares) {
        float4 ml[CH], x[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          const int64_t at = kf_row(a, p, min(k0 + j * shares, p.y - 1), r);
          ml[j] = reinterpret_cast<const float4*>(d.part_ml)[at];
          x[j] = reinterpret_cast<const float4*>(d.part + at * HD)[d4];
        }
#pragma unroll
        for (int j = 0; j < CH; ++j)
          if (k0 + j * shares < p.y) kf_add(sum, x[j], ml[j].x, ml[j].y, ml[j].z);
      }
      __syncthreads();
      share[tid] = sum;
      __syncthreads();
      if (live && mine == 0) {  // the shares in order
        for (int k = 1; k < shares; ++k) {
          const KFSum& t = share[tid + k * LPP];
          kf_add(sum, t.num, t.mo, t.m, t.l);
        }
        kd_answer<HD>(d, b, h, f0 + r, d4 * 4, sum.num, sum.mo, sum.m, sum.l);
        if (a.splits && d.lse && d4 == 0)  // for the prompt's weights
          d.lse[((int64_t)b * c.n_kv + h) * d.rows + f0 + r] = sum.l == 0.f ? INFINITY : sum.m + log2f(sum.l);
      }
    }
    return;
  }
  // ---- weights ----
  if (d.t0 && n_new == 0) return;  // a later chunk without rows of this sequence
  const int L = kd_len(d, b, cap), total = (int)min((int64_t)L + n_new, (int64_t)cap);
  const int p0 = ((int)blockIdx.x - joins) * KF_POSITIONS;
  if (p0 >= total) return;
  const int64_t head = (int64_t)b * c.n_kv + h;
  const int at = p0 + 4 * tid;  // cap is a multiple of 16: four positions are there or none
  const float* s = d.scores + head * d.rows * cap + min(at, cap - 4);
  const float* w_in = a.w_in ? a.w_in + head * a.ldw : nullptr;
  constexpr int CH = 8;  // rows asked for together, the first ones before the sums are known
  float4 x[CH];
  auto load = [&](int f) {
#pragma unroll
    for (int j = 0; j < CH; ++j) x[j] = *reinterpret_cast<const float4*>(s + (int64_t)min(f + j, rows_b - 1) * cap);
  };
  float w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = w_in && at + e < min(L, total) ? w_in[at + e] : 0.f;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (rows_b) {
    load(0);
    for (int f = warp; f < rows_b; f += KF_THREADS / 32) {
      const int2 p = d.parts[head * d.nrg + f / a.rg];
      const float lse = p.y == 1 ? d.lse[head * d.rows + f] : kf_lse_of(a, p, f % a.rg);
      if (lane == 0) kf_lse[f] = lse;
    }
    __syncthreads();
    for (int f = 0; f < rows_b; f += CH) {
      if (f) load(f);
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        const float lse = f + j < rows_b ? kf_lse[f + j] : INFINITY;
        sum[0] += ex2(x[j].x - lse); sum[1] += ex2(x[j].y - lse); sum[2] += ex2(x[j].z - lse); sum[3] += ex2(x[j].w - lse);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (at + e < total) a.w_out[head * a.ldw + at + e] = w[e] + sum[e];
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// Rows of an item from which the prompt kernel takes a call: below, its 256-row tiles are mostly empty and
// the split kernel's 16-row groups read K and V few enough times.  28 / 4 heads x 128, split / prompt kernel: one sequence
// behind 2048 positions, 63 rows 18.4 / 29.0 us, 252 rows 26.7 / 35.5; 8 behind 4096, 35 rows 41.7 / 45.0, 63 rows
// 51.2 / 46.5, 252 rows 137 / 55; 32 behind 2048, 35 rows 67.9 / 61.5, 63 rows 86 / 62.
constexpr int KD_ROWS_MAX = 64;

struct KDPlan {
  bool prompt;
  int chunk;  // tokens a launch: fp32 rows keep to the split kernel, which has both their terms
  KV8PromptPlan pp;
  int rg, nrg, n_cta;
  int64_t part, ml, lse, scores, bytes;  // offsets; the status word is at 0, the parts table at 256
};
static KDPlan kd_plan(const N730KV8Cache& c, int batch, int tokens, int heads, int dtype, bool weights) {
  KDPlan p{};
  const int group = heads / c.n_kv;
  const int64_t items = (int64_t)batch * c.n_kv;
  p.prompt = (int64_t)tokens * group > KD_ROWS_MAX && dtype != N730_F32;
  p.chunk = p.prompt || (int64_t)tokens * group <= KD_ROWS_MAX ? tokens : std::max(1, KD_ROWS_MAX / group);
  const int64_t rows = (int64_t)p.chunk * group;
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  int64_t slots;
  if (p.prompt) {
    p.pp = kv8_prompt_plan(c, batch, tokens, heads);
    p.rg = p.pp.rg;
    p.nrg = p.pp.tail;
    p.part = 256;
    slots = items * p.nrg * p.pp.splits;
  } else {
    // fp32 rows take both terms' products, and up to 8 rows need no second group of columns
    p.rg = dtype == N730_F32 || rows <= 8 ? 8 : 16;
    p.nrg = (int)((rows + p.rg - 1) / p.rg);
    p.n_cta = KD_CTAS_PER_SM * num_sms();
    p.part = 256 + up(items * p.nrg * 8);
    slots = 2 * p.n_cta;
  }
  p.ml = p.part + up(slots * p.rg * c.head_dim * 4);
  p.lse = p.ml + up(slots * p.rg * 16);
  p.scores = p.lse + (weights ? up(items * rows * 4) : 0);
  p.bytes = p.scores + (weights && !p.prompt ? items * rows * c.max_pages * c.page_size * 4 : 0);
  return p;
}

int kv8_attention_check(const N730KV8Cache* c, int batch, int tokens, int heads) {
  if (int rc = kv8_check(c, batch, "kv8_attention")) return rc;
  N730_REQUIRE(batch <= KV8_MAX_BATCH, N730_BAD_ARG, "kv8_attention: batch %d", batch);
  N730_REQUIRE(tokens >= 1 && tokens <= (1 << 20), N730_BAD_ARG, "kv8_attention: tokens %d", tokens);
  N730_REQUIRE(heads >= 1 && heads <= 65535 && heads % c->n_kv == 0, N730_BAD_ARG,
               "kv8_attention: %d heads over %d KV heads", heads, c->n_kv);
  // a token's queries of a KV head keep their sums in the finishing kernel's shared memory
  N730_REQUIRE(heads / c->n_kv <= 8192, N730_BAD_ARG, "kv8_attention: %d heads over %d KV heads", heads, c->n_kv);
  // the sequences' tiles are counted in 32 bits on the device
  N730_REQUIRE((int64_t)batch * ((int64_t)c->max_pages * c->page_size / KD_TILE + 1 + KD_ITEM_COST) < (1ll << 31), N730_BAD_ARG,
               "kv8_attention: %d sequences of up to %d pages", batch, c->max_pages);
  // CTAs of one grid axis
  N730_REQUIRE((int64_t)batch * tokens * heads <= (1ll << 36), N730_BAD_ARG, "kv8_attention: %d sequences of %d tokens of %d heads",
               batch, tokens, heads);
  N730_REQUIRE((int64_t)tokens * (heads / c->n_kv) <= (1 << 23), N730_BAD_ARG,
               "kv8_attention: %d tokens of %d heads over %d KV heads", tokens, heads, c->n_kv);
  return N730_OK;
}

int64_t kv8_attention_ws(const N730KV8Cache& c, int batch, int tokens, int heads, bool weights) {
  // fp32 calls take more row groups and keep a prompt's scores, 16-bit calls larger parts
  return std::max(kd_plan(c, batch, tokens, heads, N730_F32, weights).bytes,
                  kd_plan(c, batch, tokens, heads, N730_F16, weights).bytes);
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (no libcuda link).
static PFN_cuTensorMapEncodeTiled_v12000 kv8_encoder() {
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

// A code pool as a 2-D tensor of bytes, one row per position and KV head of a page; a copy takes
// `box` whole rows (x is always 0), swizzled over the row's 128 or 64 bytes.
static int kv8_map(const N730KV8Cache& c, const void* codes, int box, CUtensorMap* out) {
  auto enc = kv8_encoder();
  N730_REQUIRE(enc, N730_CUDA_ERR, "kv8_attention: cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[2] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.n_pages * c.n_kv * c.page_size};
  const cuuint64_t strides[1] = {(cuuint64_t)c.head_dim};
  const cuuint32_t boxes[2] = {(cuuint32_t)c.head_dim, (cuuint32_t)box};
  const cuuint32_t es[2] = {1, 1};
  N730_REQUIRE(enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, boxes, es,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, c.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS,
               N730_CUDA_ERR, "kv8_attention: cuTensorMapEncodeTiled failed");
  return N730_OK;
}

// of every call of up to `tokens` tokens: the need does not grow with them (other kernels, other shares)
int64_t kv8_attention_ws_upto(const N730KV8Cache& c, int batch, int tokens, int heads) {
  int64_t most = 0;
  for (int t = 1; t <= tokens; ++t) most = std::max(most, kv8_attention_ws(c, batch, t, heads, false));
  return most;
}

template <int HD, int CODE, int NB, bool LO>
static int split_launch(const KDArgs& a, const CUtensorMap& km, const CUtensorMap& vm, bool pdl, cudaStream_t st) {
  const size_t fixed = sizeof(KDSmem<HD>) + 1024;
  if (int rc = smem_attr_once<kv8_split_kernel<HD, CODE, NB, LO>>((int)(fixed + KV8_MAX_BATCH * 12))) return rc;
  return kv8_launch(kv8_split_kernel<HD, CODE, NB, LO>, dim3(a.n_cta), dim3(KD_THREADS), fixed + (size_t)a.batch * 12, st,
                    pdl, a, km, vm);
}

static int finish_launch(const KV8AttnCall& k, const KDPlan& p, const KDArgs& a, cudaStream_t st) {
  const float* w_in = a.t0 ? k.w_out : k.w_in;  // a later chunk adds to the ones before
  const bool weights = k.w_out && !p.prompt;
  KFArgs f{};
  f.d = a;
  f.rg = p.rg;
  f.splits = p.prompt ? p.pp.splits : 0;
  f.w_in = w_in; f.w_out = k.w_out; f.ldw = k.ldw;
  const int cap = k.c.max_pages * k.c.page_size;
  // rows of a block: one where that leaves the SMs few blocks, more where most items have one part.  From 8 x SMs on; from
  // 2 x and 32 x: 32 sequences with weights 53.5 (51.5, 53.5) us, 64 of 28 / 4 heads 39.8 (38.9, 42.9), 128 of 64 / 8
  // heads 115.2 (115.2, 119.3)
  const int64_t all_rows = (int64_t)k.batch * k.c.n_kv * p.nrg * p.rg;
  f.rb = 1;
  while (f.rb < p.rg && all_rows / f.rb > 8 * num_sms()) f.rb *= 2;
  const dim3 grid(p.nrg * (p.rg / f.rb) + (weights ? (cap + KF_POSITIONS - 1) / KF_POSITIONS : 0), k.c.n_kv, k.batch);
  const size_t smem = weights ? (size_t)p.nrg * p.rg * 4 : 0;
  if (k.c.head_dim == 128) return kv8_launch(kv8_finish_kernel<128>, grid, dim3(KF_THREADS), smem, st, true, f);
  return kv8_launch(kv8_finish_kernel<64>, grid, dim3(KF_THREADS), smem, st, true, f);
}

int kv8_attention_launch(const KV8AttnCall& k, cudaStream_t st) {
  const N730KV8Cache& c = k.c;
  const bool weights = k.w_out != nullptr;
  const KDPlan p = kd_plan(c, k.batch, k.tokens, k.heads, k.dtype, weights);
  N730_REQUIRE(k.ws_bytes >= p.bytes, N730_BAD_ARG, "kv8_attention: workspace of %lld bytes, %lld needed",
               (long long)k.ws_bytes, (long long)p.bytes);
  uint8_t* ws = reinterpret_cast<uint8_t*>(k.ws);
  KDArgs a{};
  a.c = c;
  a.q = k.q; a.out = k.out; a.ldq = k.ldq; a.ldo = k.ldo; a.dtype = k.dtype; a.odtype = k.out_dtype;
  a.batch = k.batch; a.tokens = k.tokens; a.heads = k.heads; a.group = k.heads / c.n_kv;
  a.rows = p.chunk * a.group; a.nrg = p.nrg;
  a.chunk = p.chunk;
  a.scale_log2e = k.scale * 1.4426950408889634f;
  a.lens = k.lens; a.n_new = k.n_new;
  a.status = k.status ? k.status : reinterpret_cast<int*>(ws);
  a.parts = reinterpret_cast<int2*>(ws + 256);
  a.part = reinterpret_cast<float*>(ws + p.part);
  a.part_ml = reinterpret_cast<float*>(ws + p.ml);
  a.lse = weights ? reinterpret_cast<float*>(ws + p.lse) : nullptr;
  a.scores = weights && !p.prompt ? reinterpret_cast<float*>(ws + p.scores) : nullptr;
  a.n_cta = p.n_cta;
  a.log_block = c.block == 16 ? 4 : c.block == 32 ? 5 : 6;
  a.box = c.page_size % KD_TILE == 0 ? KD_TILE : 16;
  if (p.prompt) {
    if (int rc = kv8_prompt_launch(k, p.pp, a.status, a.part, a.part_ml, a.lse, st)) return rc;
    if (p.pp.splits > 1)
      if (int rc = finish_launch(k, p, a, st)) return rc;
    return weights ? kv8_prompt_weights_launch(k, p.pp, a.status, a.lse, st) : N730_OK;
  }
  CUtensorMap km, vm;
  int rc = kv8_map(c, c.k_codes, a.box, &km);
  if (!rc) rc = kv8_map(c, c.v_codes, a.box, &vm);
  if (rc) return rc;
#define N730_SPLIT(HD, CODE)                                                 \
  (k.dtype == N730_F32 ? split_launch<HD, CODE, 1, true>(a, km, vm, k.pdl, st)       \
   : p.rg == 8         ? split_launch<HD, CODE, 1, false>(a, km, vm, k.pdl, st)      \
                       : split_launch<HD, CODE, 2, false>(a, km, vm, k.pdl, st))
  for (; a.t0 < k.tokens; a.t0 += p.chunk) {
    if (c.head_dim == 128) rc = c.code == N730_KV8_INT8 ? N730_SPLIT(128, N730_KV8_INT8) : N730_SPLIT(128, N730_KV8_E4M3);
    else rc = c.code == N730_KV8_INT8 ? N730_SPLIT(64, N730_KV8_INT8) : N730_SPLIT(64, N730_KV8_E4M3);
    if (!rc) rc = finish_launch(k, p, a, st);
    if (rc) return rc;
  }
#undef N730_SPLIT
  return N730_OK;
}

// One warp waits as the attention's do, on a barrier that nobody (0), a thread beforehand (1) or another warp after half
// the limit (2) arrives at; in the last case one lane's own limit has run out by then.
__global__ void kv8_wait_check_kernel(int arrives, uint64_t limit_ns, int* status) {
  __shared__ uint64_t bar;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    fence_mbar_init();
    if (arrives == 1) mbar_arrive_expect_tx(&bar, 0);
  }
  __syncthreads();
  if (warp == 0) {
    if (!kv8_wait(&bar, 0, arrives == 2 && lane == 7 ? 1 : limit_ns) && lane == 0) *status = DEV_ERR_TIMEOUT;
  } else if (arrives == 2 && lane == 0) {
    auto now = [] { uint64_t t; asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t)); return t; };
    const uint64_t t0 = now();
    while (now() - t0 < limit_ns / 2) {}
    mbar_arrive_expect_tx(&bar, 0);
  }
}

int* gemv_err_word();
int gemv_check_error(bool reset);

}  // namespace n730

using namespace n730;

N730_API int n730_kv8_wait_check(int64_t wait_ns, int arrives, void* stream) {
  N730_REQUIRE(wait_ns > 0 && wait_ns <= 1000000000ll, N730_BAD_ARG, "kv8_wait_check: wait %lld ns", (long long)wait_ns);
  N730_REQUIRE(arrives >= 0 && arrives <= 2, N730_BAD_ARG, "kv8_wait_check: arrives %d", arrives);
  int* err = gemv_err_word();
  if (!err) return N730_OOM;
  cudaStream_t st = (cudaStream_t)stream;
  kv8_wait_check_kernel<<<1, 64, 0, st>>>(arrives, (uint64_t)wait_ns, err);
  N730_CHECK_LAUNCH();
  N730_CUDA(cudaStreamSynchronize(st));
  return gemv_check_error(true);
}

N730_API int64_t n730_kv8_attention_ws(const N730KV8Cache* c, int batch, int tokens, int n_heads, int weights) {
  if (int rc = kv8_attention_check(c, batch, tokens, n_heads)) return rc;
  return kv8_attention_ws(*c, batch, tokens, n_heads, weights != 0);
}

N730_API int64_t n730_kv8_attention_ws_of(const N730KV8Cache* c, int dtype, int batch, int tokens, int n_heads, int weights) {
  if (int rc = kv8_attention_check(c, batch, tokens, n_heads)) return rc;
  N730_REQUIRE(dtype == N730_F32 || dtype == N730_F16 || dtype == N730_BF16, N730_BAD_ARG, "kv8_attention: dtype %d", dtype);
  return kd_plan(*c, batch, tokens, n_heads, dtype, weights != 0).bytes;
}

N730_API int n730_kv8_attention(const N730KV8Cache* c, const void* d_q, int dtype, int64_t ldq, int batch, int tokens,
                                int n_heads, float scale, const int32_t* d_lens, const int32_t* d_new, void* d_out,
                                int64_t ldo, const float* d_w, float* d_w_out, int64_t ldw, void* d_ws,
                                int64_t ws_bytes, void* stream) {
  if (int rc = kv8_attention_check(c, batch, tokens, n_heads)) return rc;
  N730_REQUIRE(dtype == N730_F32 || dtype == N730_F16 || dtype == N730_BF16, N730_BAD_ARG, "kv8_attention: dtype %d", dtype);
  N730_REQUIRE(d_q && d_out && d_lens && d_ws, N730_NULL, "kv8_attention: null pointer");
  N730_REQUIRE(kv8_aligned(kv8_esize(dtype), (const char*)d_q, (const char*)d_out) && kv8_aligned(4, d_lens, d_new) &&
                   kv8_aligned(4, d_w, d_w_out), N730_BAD_ARG, "kv8_attention: pointers must lie on whole elements");
  const int64_t row = (int64_t)n_heads * c->head_dim;
  N730_REQUIRE(ldq >= row && ldo >= row, N730_BAD_ARG, "kv8_attention: row strides %lld, %lld < %d heads x %d",
               (long long)ldq, (long long)ldo, n_heads, c->head_dim);
  N730_REQUIRE(!d_w || d_w_out, N730_BAD_ARG, "kv8_attention: weights in without weights out");
  N730_REQUIRE(!d_w_out || ldw >= (int64_t)c->max_pages * c->page_size, N730_BAD_ARG,
               "kv8_attention: row stride %lld of the weights is below the table's %lld positions", (long long)ldw,
               (long long)c->max_pages * c->page_size);
  N730_REQUIRE(scale == scale && scale - scale == 0.f, N730_BAD_ARG, "kv8_attention: scale %g", scale);
  N730_REQUIRE(((uintptr_t)d_ws & 15) == 0, N730_BAD_ARG, "kv8_attention: the workspace must be 16-byte aligned");
  KV8AttnCall k{};
  k.c = *c;
  k.q = d_q; k.out = d_out; k.dtype = k.out_dtype = dtype; k.ldq = ldq; k.ldo = ldo;
  k.batch = batch; k.tokens = tokens; k.heads = n_heads; k.scale = scale;
  k.lens = d_lens; k.n_new = d_new;
  k.w_in = d_w; k.w_out = d_w_out; k.ldw = ldw;
  k.ws = d_ws; k.ws_bytes = ws_bytes;
  return kv8_attention_launch(k, (cudaStream_t)stream);
}
