// Sampling with settings of each row and given random numbers.
//
// Per row, V logits l, temperature T, top-k k, top-p p, min-p q, number u:
//   T <= 0: the first index of the largest logit.  Otherwise tokens are ordered by logit, ties by index, with weights
//   w = exp((l - max l) / T).  Kept is the shortest of three prefixes of that order: the first k tokens; the shortest
//   whose mass reaches p times the mass of those k; the tokens with w >= q.  The token is the first whose cumulative
//   mass exceeds u times the kept mass.
//
// A cluster of 8 CTAs takes a row: each copies an eighth of the logits into its shared memory, so that HBM is read once
// and whatever follows runs on the chip.  (Short rows, and many of them, take 4, 2 or one CTA.)  The first CTA leads; the others
// serve its commands, and all meet around each.
//   1. largest and smallest logit, and each thread's largest.
//   2. A list: tokens are gathered in the first CTA's shared memory and sorted, the rest is a scan over it with weights in
//      64 bits.  With min-p and no top-p they are those of weight >= q; with a top-k those up to the bin (of RS_BINS
//      linear ones of max - l) that k of the threads' largest reach, 4096 of a long row: the first k tokens all lie up to
//      there, and seldom many more.
//   3. Rows of neither kind, or whose list is too long: a histogram of all tokens and their masses.  A bin's mass is
//      w(edge) * sum of w / w(edge), the sum in fixed point, 43 bits below 21 of count in two words; these bins reach 40
//      temperatures, not further, so each is T / 38 wide or less and w / w(edge) lies within 3 % of 1, where fp32 holds its
//      distance from 1 to 2^-24 of that.  (Bins of 32 logits whatever T: at T = 0.001 a token's mass was rounded against an
//      edge's 10^9 times its own, 7e-4 of a row's mass in all.  One word of 22 bits below 10 was no
//      faster: shared-memory atomics cost 5 cycles a warp's worth, a token's arithmetic twice that.)
//      Each prefix's end is then looked up in its bin: the bin's tokens are gathered and sorted, or, where they are too
//      many (equal logits, coarse types), found by four rounds of 8 bits of the logit, after which the tokens left are
//      equal and go by index.
// One row of 152064 with a top-k is bound by six meetings of the cluster, 1.2 us each (11.6 us).  192 rows of 152064 bf16
// logits without one take 136 us, 0.43 TB/s at 39 % of the issue slots: a token's polynomial and two dependent atomics, behind
// a pass for the largest, and CTAs that wait while the first one looks ends up (barriers are the longest stall).
// Sums are integers, or 64-bit floats in a fixed order: the same inputs give the same token.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "kv8.h"

namespace n730 {
namespace cg = cooperative_groups;

constexpr int RS_CLUSTER = 8;      // most CTAs of a row
// Threads of a CTA: 512 and all of an SM's registers while a row's CTAs find an SM each (one row of 152064 without a cut:
// 20.8 us, 22.3 with 256), 256 beyond that.  Then two CTAs an SM, or three of 16-bit logits, which shared memory has room
// for, where that saves more waves than registers that do not suffice cost (192 rows of 152064
// bf16 logits without a cut: 136 us, 152 with two; 40 rows of 100000, where it does not: 38, and 31 with two).
constexpr int RS_THREADS_FEW = 512, RS_THREADS_MANY = 256;
constexpr int RS_WARPS = RS_THREADS_FEW / 32;  // most warps
constexpr int RS_BINS = 1536;      // as many as leave room for two CTAs of 19008 fp32 logits (a row of 152064) an SM
constexpr int RS_CAP = 1024;       // tokens that are sorted at once
constexpr int RS_COUNT = 160;      // lists up to this long are sorted by counting
constexpr uint32_t RS_ROOM = 4000;  // tokens of a CTA's bin that the sums have room for
constexpr float RS_SPAN = 32.f;    // bins of counts reach this many logits, or temperatures where that is more, below the largest
constexpr float RS_TEMPS = 40.f;   // bins of masses this many temperatures: e^-40 of the largest's weight counts as none
constexpr size_t RS_HALF = 76 * 1024;  // longest slice of which two fit an SM
constexpr size_t RS_STAGE_MAX = 160 * 1024;  // longest slice that is kept in shared memory

struct RSArgs {
  const void* logits;
  int64_t ld;
  int vocab, per;                  // per: logits of a CTA
  bool vec;                        // rows lie on 16 bytes
  const float* temperature; const int* top_k; const float* top_p; const float* min_p; const float* u;
  int* tokens; float* prob; int* kept;
};

// what the bins hold: nothing, threads' largest, all tokens, all tokens and their masses
enum { RS_NONE = 0, RS_LARGEST, RS_COUNTS, RS_MASSES };
enum { RS_DONE = 0, RS_FILL, RS_GATHER, RS_RADIX, RS_OVER, RS_FIND };
struct RSCommand {
  int op, b0, b1;         // bins [b0, b1]
  int last;               // GATHER: nothing follows for the other CTAs
  int sure;               // FILL: tokens of a CTA's bin to have room for
  uint32_t prefix, shift; // RADIX: digits found, where the next one starts
  uint32_t key, skip;     // FIND: the skip-th token of this key
  double z0;              // RADIX: the bin's edge / T
};
struct RSStat { float mx, mn; uint32_t n; };  // n: tokens

// What the first CTA knows of its row between two commands.
struct RSLead {
  int state, mode, purpose, b, round;
  uint32_t cut, kept, before, left, prefix;
  bool cut_k, by_mass, strict;
  double top_p, u, over, mass, target, base, in_mass, unit, each;  // over: place of weight min-p
};
struct RSSmem {
  uint32_t cnt[RS_BINS];             // by bin; also the counts of 256 digits
  uint32_t low[RS_BINS];             // the second word; also the digits' masses, low and high words
  union { unsigned long long list[RS_CAP]; uint32_t bin_cnt[RS_BINS]; };  // list: ~order << 32 | index
  union { double cum[RS_CAP]; double bin_mass[RS_BINS]; unsigned long long mine[RS_CAP]; };
  RSCommand cmd;
  RSLead lead;
  RSStat stats[RS_CLUSTER];
  RSStat wstat[RS_WARPS];
  double wsum[RS_WARPS];
  uint32_t wcnt[RS_WARPS];
  float spread;                      // largest logit less smallest, and a little more
  uint32_t most[RS_CLUSTER], own_most;  // tokens of a share's fullest bin, where it has no room for them
  double sel_base, sel_mass, pick_w;
  uint32_t n_list, n_mine, list_at, over, sel_cnt, sel_in, pick_cnt, occur;
  int bin_k, bin_p, pick, found, first;
};

// a row's CTAs meet
template <int CL>
__device__ __forceinline__ void rs_arrive() {
  if (CL == 1) return;
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
template <int CL>
__device__ __forceinline__ void rs_wait() {
  if (CL == 1) { __syncthreads(); return; }
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <int CL>
__device__ __forceinline__ void rs_sync() { rs_arrive<CL>(); rs_wait<CL>(); }

// the order of logits as unsigned numbers (largest largest); logits here are no NaN and no -0
__device__ __forceinline__ uint32_t rs_order(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float rs_unorder(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ float rs_clean(float x) { return x != x ? -INFINITY : x + 0.f; }
__device__ __forceinline__ float rs_float(float x) { return x; }
__device__ __forceinline__ float rs_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float rs_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// A row's bins: bin = floor((max - l) * sx); edge(b), its upper end, is max - b * width as fp32 rounds it.  max * sx is
// rounded once, which moves all of a row's places by as much as 2^-24 of it, and an edge by 2^-24 of itself: rows whose
// largest logit is 2^21 bins or more from 0 (or a bin of T / 38 or more: places, edges and logits would leave the bins that
// they belong to, the last ones for no bin at all) go by the logits' distances from it, which are exact for all that have a
// weight.  For the others this is 1/8 of a bin each: what a place and an edge say is off by one bin at most.
struct RSGeom {
  float mx, sx, top, width, inv_t;  // top: max * sx
  double t;
  bool far;                         // logits go by their distance from `from`, the largest, RS_LEAST at least
  float from;
};
constexpr float RS_LEAST = -3e38f, RS_FAR = 0x1p21f;  // RS_FAR: bins
constexpr int RS_SLACK = 1;
__device__ __forceinline__ float rs_place(float l, const RSGeom& g) { return fmaf(-l, g.sx, g.top); }
// the row's bins reach `most` logits below the largest, or the whole row where that is less
__device__ __forceinline__ void rs_reach(RSGeom& g, float spread, float most) {
  const float span = fminf(spread, most);
  const bool some = span > 1e-33f;  // below that, 1/700 of the smallest temperature, all logits count as one
  g.sx = some ? (float)RS_BINS / span : 0.f;
  g.top = g.mx * g.sx;
  g.width = some ? span / (float)RS_BINS : 0.f;
}
// NaN and -infinity have no place below RS_BINS
__device__ __forceinline__ int rs_bin(float l, const RSGeom& g) {
  const float x = rs_place(l, g);
  return x < (float)RS_BINS ? max((int)x, 0) : RS_BINS;
}
__device__ __forceinline__ float rs_edge(float b, const RSGeom& g) { return fmaf(-b, g.width, g.mx); }
__device__ __forceinline__ float rs_seen(float l, const RSGeom& g) {
  return !g.far || !(l > -INFINITY) ? l : l == g.from ? 0.f : fmaxf(l - g.from, RS_LEAST);
}
__device__ __forceinline__ double rs_weight(float l, const RSGeom& g) { return l == g.mx ? 1.0 : exp(((double)l - (double)g.mx) / g.t); }

// Exclusive scans over the block in thread order; the totals.
template <int TH>
__device__ __forceinline__ void rs_scan2(uint32_t& k, double& m, RSSmem& s, uint32_t* all_k, double* all_m) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t ik = k;
  double im = m;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t nk = __shfl_up_sync(0xffffffffu, ik, o);
    const double nm = __shfl_up_sync(0xffffffffu, im, o);
    if (lane >= o) { ik += nk; im += nm; }
  }
  __syncthreads();
  if (lane == 31) { s.wcnt[warp] = ik; s.wsum[warp] = im; }
  __syncthreads();
  uint32_t bk = 0, tk = 0;
  double bm = 0, tm = 0;
#pragma unroll
  for (int w = 0; w < (TH / 32); ++w) {
    const uint32_t xk = s.wcnt[w];
    const double xm = s.wsum[w];
    if (w < warp) { bk += xk; bm += xm; }
    tk += xk; tm += xm;
  }
  *all_k = tk; *all_m = tm;
  k = bk + ik - k;
  m = bm + im - m;
}
// Exclusive scan over the block in thread order; *total the sum.
template <int TH, class V>
__device__ V rs_scan(V v, V* warps, V* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = inc;
  __syncthreads();
  V before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < (TH / 32); ++w) {
    const V x = warps[w];
    if (w < warp) before += x;
    all += x;
  }
  *total = all;
  return before + inc - v;
}

template <class T, bool STAGED, int CL, int TH>
struct RSRow {
  static constexpr int RS_PER = RS_BINS / TH, RS_EACH = RS_CAP / TH;
  static constexpr int V = 16 / sizeof(T), SHARE = RS_BINS / CL;
  RSSmem& s;
  T* stage;              // this CTA's logits
  const RSArgs& a;
  const T* row;          // the row's first logit
  int i0, n;             // this CTA's share
  RSGeom g;
  cg::cluster_group cl;
  double min_p;
  uint32_t all_cnt;      // the row's tokens
  int sure;              // tokens of a CTA's bin that two words are to have room for

  __device__ float raw(int i) const { return rs_float(STAGED ? stage[i] : row[i0 + i]); }
  __device__ float get(int i) const { return rs_seen(rs_clean(raw(i)), g); }
  // f(first index, V logits) over this CTA's, V = 16 bytes of them, NaN behind the last.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int i = threadIdx.x * V; i < n; i += TH * V) {
      float l[V];
      if (STAGED) {
        const uint4 x = *reinterpret_cast<const uint4*>(stage + i);
        const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
        for (int j = 0; j < V; ++j) l[j] = rs_float(e[j]);
        if (i + V > n)
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (i + j >= n) l[j] = NAN;
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) l[j] = i + j < n ? rs_float(row[i0 + i + j]) : NAN;
      }
      if (g.far)
#pragma unroll
        for (int j = 0; j < V; ++j) l[j] = rs_seen(l[j], g);
      f(i, l);
    }
  }

  // Units of a weight over its bin edge's: 43 bits have room for `sure` of them.
  __device__ float unit_of() const { return ldexpf(1.f, 31 - (32 - __clz(sure / 4001))); }

  // Counts, and sums of w / w(edge), by bin.
  template <bool MASSES>
  __device__ __forceinline__ void fill() {
    const float unit = unit_of();
    each([&](int, const float (&l)[V]) {
      int b[V], c[V];
      uint32_t old[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float x = fmaxf(rs_place(l[j], g), 0.f), f = __fadd_rd(x, 8388608.f);  // 2^23 + floor(x)
        b[j] = l[j] > -INFINITY && x < (float)RS_BINS ? __float_as_int(f) & 0x7fffff : -1;
        if (!MASSES) continue;
        // y = (l - edge) / T: the two are near, their difference is exact but for what is below 2^-24 of a bin
        const float y = (l[j] - rs_edge(f - 8388608.f, g)) * g.inv_t;
        const float e = y * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 1.f / 120, 1.f / 24), 1.f / 6), 0.5f), 1.f);  // exp(y) - 1
        c[j] = (int)((uint32_t)__float2int_rn(e * unit) + (uint32_t)unit);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (b[j] < 0) continue;
        if (MASSES) old[j] = atomicAdd(&s.low[b[j]], (uint32_t)c[j]);
        else atomicAdd(&s.cnt[b[j]], 1u << 11);
      }
      if (MASSES)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (b[j] >= 0) atomicAdd(&s.cnt[b[j]], (1u << 11) + (old[j] + (uint32_t)c[j] < old[j]));
    });
  }
  // This CTA's share of the bins, added up over the cluster, to the first CTA.  The cluster has filled before.
  __device__ __forceinline__ void reduce(bool masses) {
    const float unit = unit_of();
    auto mass_of = [&](int b, uint32_t k, unsigned long long m) {
      return k && masses ? rs_weight(rs_edge((float)b, g), g) * ((double)m / unit) : 0.0;
    };
    auto tokens = [](uint32_t x) { return x >> 11; };
    auto sum = [](const RSSmem* o, int b, uint32_t x) { return (unsigned long long)(x & 2047u) << 32 | o->low[b]; };
    const uint32_t room = masses ? max((uint32_t)sure, RS_ROOM) : 0xffffffffu;
    if (CL == 1) {
      uint32_t most = 0;
      for (int b = threadIdx.x; b < RS_BINS; b += TH) {
        const uint32_t x = s.cnt[b], k = tokens(x);
        most = max(most, k);
        s.bin_cnt[b] = k;
        s.bin_mass[b] = mass_of(b, k, sum(&s, b, x));
      }
      if (threadIdx.x == 0) s.own_most = 0;
      __syncthreads();
      if (most > room) atomicMax(&s.own_most, most);
      __syncthreads();
      if (threadIdx.x == 0) s.most[0] = s.own_most;
      return;
    }
    const int t = threadIdx.x, rank = (int)cl.block_rank();
    RSSmem* lead = cl.map_shared_rank(&s, 0);
    if (t == 0) s.own_most = 0;
    __syncthreads();
    for (int b = rank * SHARE + t; b < (rank + 1) * SHARE; b += TH) {
      uint32_t k = 0, most = 0;
      unsigned long long m = 0;
#pragma unroll
      for (int r = 0; r < CL; ++r) {
        const RSSmem* o = cl.map_shared_rank(&s, r);
        const uint32_t x = o->cnt[b];
        k += tokens(x);
        most = max(most, tokens(x));
        m += sum(o, b, x);
      }
      if (most > room) atomicMax(&s.own_most, most);
      lead->bin_cnt[b] = k;
      lead->bin_mass[b] = mass_of(b, k, m);
    }
    __syncthreads();
    if (t == 0) lead->most[rank] = s.own_most;
  }
  // The bins of all CTAs' tokens, or of their threads' largest.
  __device__ __forceinline__ void histogram(int mode, float largest) {
    if (mode == RS_MASSES) {
      fill<true>();
    } else if (mode == RS_COUNTS) {
      fill<false>();
    } else if (largest > -INFINITY) {
      const int b = rs_bin(rs_seen(largest, g), g);
      if (b < RS_BINS) atomicAdd(&s.cnt[b], 1u << 11);
    }
    rs_sync<CL>();
    reduce(mode == RS_MASSES);
  }

  // A CTA's share of a command.
  __device__ __forceinline__ void serve(const RSCommand& c, float of_thread) {
    const int tid = threadIdx.x;
    if (c.op == RS_FILL) {
      sure = c.sure;
      rs_reach(g, s.spread, RS_TEMPS * (float)g.t);
      for (int i = tid; i < RS_BINS; i += TH) s.cnt[i] = s.low[i] = 0;
      __syncthreads();
      histogram(RS_MASSES, of_thread);
    } else if (c.op == RS_GATHER) {
      // into this CTA's own shared memory first: a place in the first CTA's list takes a trip there
      const float lo = (float)c.b0, hi = c.b1 == RS_BINS ? INFINITY : (float)(c.b1 + 1);  // -infinity's place is infinity
      // nothing below this is wanted
      const float least = c.b1 == RS_BINS || g.sx == 0.f ? -INFINITY : rs_edge((float)(c.b1 + 1 + RS_SLACK), g);
      const float largest = c.b0 < 2 || g.sx == 0.f ? INFINITY : rs_edge((float)(c.b0 - RS_SLACK), g);  // or above this
      if (tid == 0) s.n_mine = 0;
      __syncthreads();
      each([&](int i, const float (&l)[V]) {
        bool any = false;
#pragma unroll
        for (int j = 0; j < V; ++j) any = any || (l[j] >= least && l[j] <= largest);
        if (!any) return;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (!(l[j] >= least && l[j] <= largest)) continue;
          const float x = rs_place(l[j], g);
          if (!((x >= lo && x < hi) || (lo == 0.f && x < 0.f) || (hi == INFINITY && x == hi && l[j] > -INFINITY))) continue;
          const uint32_t at = atomicAdd(&s.n_mine, 1u);
          if (at < RS_CAP) s.mine[at] = (unsigned long long)~rs_order(l[j] + 0.f) << 32 | (uint32_t)(i0 + i + j);
        }
      });
      __syncthreads();
      RSSmem* lead = cl.map_shared_rank(&s, 0);
      const uint32_t k = s.n_mine;
      if (tid == 0 && k) s.list_at = atomicAdd(&lead->n_list, k);
      __syncthreads();
      for (uint32_t i = tid; i < min(k, (uint32_t)RS_CAP); i += TH)
        if (s.list_at + i < RS_CAP) lead->list[s.list_at + i] = s.mine[i];
    } else if (c.op == RS_RADIX) {
      uint32_t* lo = s.low;
      for (int i = tid; i < 256; i += TH) s.cnt[i] = lo[i] = lo[256 + i] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += TH) {
        const float l = get(i);
        if (l == -INFINITY || rs_bin(l, g) != c.b0) continue;
        const uint32_t o = rs_order(l);
        if (c.shift < 24 && (o >> (c.shift + 8)) != c.prefix) continue;
        const uint32_t d = (o >> c.shift) & 255u;
        atomicAdd(&s.cnt[d], 1u);
        if (c.b0 == RS_BINS) continue;  // no mass behind the last bin
        const double z = l == g.mx ? 0.0 : ((double)l - (double)g.mx) / g.t;
        const unsigned long long w = __double2ull_rn(exp(z + c.z0) * 0x1p40);
        const uint32_t wl = (uint32_t)w, old = atomicAdd(&lo[d], wl);
        const uint32_t wh = (uint32_t)(w >> 32) + (old + wl < old);
        if (wh) atomicAdd(&lo[256 + d], wh);
      }
    } else if (c.op == RS_OVER) {  // tokens of weight >= min-p; bins below b0 are sure to have it
      uint32_t k = 0;
      for (int i = tid; i < n; i += TH) {
        const float l = get(i);
        if (l == -INFINITY) continue;
        const int b = rs_bin(l, g);
        k += b < c.b0 || (b <= c.b1 && rs_weight(l, g) >= min_p);
      }
      uint32_t all;
      rs_scan<TH, uint32_t>(k, s.wcnt, &all);
      if (tid == 0) atomicAdd(&cl.map_shared_rank(&s, 0)->over, all);
    } else if (c.op == RS_FIND) {
      // tokens of the key in this CTA, then its place among the CTAs', then in thread order (contiguous runs)
      const int run = (n + TH - 1) / TH, j0 = min(n, tid * run), j1 = min(n, j0 + run);
      uint32_t k = 0, all;
      for (int i = j0; i < j1; ++i) k += get(i) != -INFINITY && rs_order(get(i)) == c.key;
      const uint32_t before = rs_scan<TH, uint32_t>(k, s.wcnt, &all);
      if (tid == 0) s.occur = all;
      rs_sync<CL>();
      uint32_t first = before;
      for (int r = 0; r < (int)cl.block_rank(); ++r) first += cl.map_shared_rank(&s, r)->occur;
      if (c.skip >= first && c.skip < first + k) {
        uint32_t left = c.skip - first;
        for (int i = j0; i < j1; ++i)
          if (get(i) != -INFINITY && rs_order(get(i)) == c.key && left-- == 0) cl.map_shared_rank(&s, 0)->found = i0 + i;
      }
    }
  }

  // ---- the first CTA's side ----
  uint32_t bin_cnt[RS_PER], cnt_before;   // this thread's bins: tokens, tokens of all bins before
  double bin_mass[RS_PER], mass_before, all_mass;

  __device__ __forceinline__ void post(const RSCommand& c) {  // to every CTA
    __syncthreads();
    if (threadIdx.x < CL) cl.map_shared_rank(&s, threadIdx.x)->cmd = c;
    if (threadIdx.x == 0) { s.n_list = 0; s.over = 0; }
  }
  // the bins that the cluster has put here, scanned
  __device__ void scan_bins() {
    uint32_t kc = 0, all;
    double mc = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < RS_PER; ++e) {
      bin_cnt[e] = s.bin_cnt[threadIdx.x * RS_PER + e];
      bin_mass[e] = s.bin_mass[threadIdx.x * RS_PER + e];
      kc += bin_cnt[e];
      mc += bin_mass[e];
    }
    cnt_before = kc;
    mass_before = mc;
    rs_scan2<TH>(cnt_before, mass_before, s, &all, &all_mass);
  }
  // whether a bin has more tokens than its words have room for
  __device__ bool crowded() const {
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < CL; ++r) m |= s.most[r];
    return m;
  }
  // First bin at which the running count or mass reaches the target (strict: exceeds it); when none does, RS_BINS by
  // count and the last one with a token by mass (a rounding is missing).
  __device__ void cross(bool by_mass, double target, bool strict, int* bin) {
    uint32_t k = cnt_before;
    double m = mass_before;
    int at = RS_BINS, full = 0;
#pragma unroll
    for (int e = 0; e < RS_PER; ++e) {
      k += bin_cnt[e];
      m += bin_mass[e];
      if (!bin_cnt[e]) continue;
      const int b = (int)threadIdx.x * RS_PER + e;
      const double x = by_mass ? m : (double)k;
      full = b;
      if (at == RS_BINS && (strict ? x > target : x >= target)) at = b;
    }
    at = __reduce_min_sync(0xffffffffu, at);
    full = __reduce_max_sync(0xffffffffu, full);
    if ((threadIdx.x & 31) == 0) {
      if (at < RS_BINS) atomicMin(bin, at);
      if (by_mass) atomicMax(&s.pick, full);
    }
  }
  __device__ int cross_one(bool by_mass, double target, bool strict) {
    __syncthreads();
    if (threadIdx.x == 0) { s.bin_k = RS_BINS; s.pick = 0; }
    __syncthreads();
    cross(by_mass, target, strict, &s.bin_k);
    __syncthreads();
    return by_mass && s.bin_k == RS_BINS ? s.pick : s.bin_k;
  }
  // tokens and mass of all bins before b, and of b
  __device__ void at_bin(int b, uint32_t* before, double* mass, uint32_t* in, double* in_mass) {
    if ((int)threadIdx.x == min(b, RS_BINS - 1) / RS_PER) {
      uint32_t k = cnt_before, c = 0;
      double m = mass_before, cm = 0;
#pragma unroll
      for (int e = 0; e < RS_PER; ++e) {
        const int at = (int)threadIdx.x * RS_PER + e;
        if (at < b) { k += bin_cnt[e]; m += bin_mass[e]; }
        if (at == b) { c = bin_cnt[e]; cm = bin_mass[e]; }
      }
      s.sel_cnt = k;
      s.sel_base = m;
      s.sel_in = b >= RS_BINS ? all_cnt - k : c;
      s.sel_mass = cm;
    }
    __syncthreads();
    *before = s.sel_cnt; *mass = s.sel_base; *in = s.sel_in; *in_mass = s.sel_mass;
  }

  // sorts the first n_list of the list
  __device__ void sort(int n_list) {
    const int t = threadIdx.x;
    if (n_list <= RS_COUNT) {  // each token's place is how many come before it
      unsigned long long x = 0;
      int at = 0;
      if (t < n_list) {
        x = s.list[t];
#pragma unroll 8
        for (int i = 0; i < n_list; ++i) at += s.list[i] < x;
      }
      __syncthreads();
      if (t < n_list) s.list[at] = x;
      __syncthreads();
      return;
    }
    // two pairs of neighbours a thread: steps of up to 32 stay in a warp
    int np2 = 256;
    while (np2 < n_list) np2 <<= 1;
    for (int i = n_list + t; i < np2; i += TH) s.list[i] = ~0ull;
    __syncthreads();
    unsigned long long x[2], y[2];
    auto load = [&] {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int q = t + e * TH;
        x[e] = y[e] = ~0ull;
        if (2 * q < np2) { x[e] = s.list[2 * q]; y[e] = s.list[2 * q + 1]; }
      }
    };
    auto store = [&] {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int q = t + e * TH;
        if (2 * q < np2) { s.list[2 * q] = x[e]; s.list[2 * q + 1] = y[e]; }
      }
    };
    load();
    for (int size = 2; size <= np2; size <<= 1) {
      int step = size >> 1;
      if (step > 32) {
        store();
        __syncthreads();
        for (; step > 32; step >>= 1) {
          for (int i = t; i < np2 / 2; i += TH) {
            const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
            const unsigned long long p = s.list[lo], q = s.list[hi];
            if ((p > q) == ((lo & size) == 0)) { s.list[lo] = q; s.list[hi] = p; }
          }
          __syncthreads();
        }
        load();
      }
      for (; step > 1; step >>= 1) {
        const int o = step >> 1;  // threads between the two
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const bool up = ((2 * (t + e * TH)) & size) == 0;
          const unsigned long long px = __shfl_xor_sync(0xffffffffu, x[e], o), py = __shfl_xor_sync(0xffffffffu, y[e], o);
          const bool keep_small = ((t & o) == 0) == up;
          x[e] = (px < x[e]) == keep_small ? px : x[e];
          y[e] = (py < y[e]) == keep_small ? py : y[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool up = ((2 * (t + e * TH)) & size) == 0;
        if ((x[e] > y[e]) == up) { const unsigned long long z = x[e]; x[e] = y[e]; y[e] = z; }
      }
    }
    store();
    __syncthreads();
  }
  __device__ float list_logit(int i) const { return rs_unorder(~(uint32_t)(s.list[i] >> 32)); }
  // s.cum: base and the mass of the sorted list up to and with each token
  template <int EACH>
  __device__ void list_masses_of(int n_list, double base) {
    double w[EACH], loc = 0, total;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int i = threadIdx.x * EACH + e;
      w[e] = i < n_list ? rs_weight(list_logit(i), g) : 0.0;
      loc += w[e];
    }
    double m = base + rs_scan<TH, double>(loc, s.wsum, &total);
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int i = threadIdx.x * EACH + e;
      m += w[e];
      if (i < n_list) s.cum[i] = m;
    }
    __syncthreads();
  }
  __device__ void list_masses(int n_list, double base) {
    if (n_list <= TH) list_masses_of<1>(n_list, base);
    else list_masses_of<RS_EACH>(n_list, base);
  }
  // how many of the list's first n tokens lie before the target: mass below it (strict: not above it)
  __device__ int list_before(int n_list, double target, bool strict) {
    int c = 0;
#pragma unroll
    for (int e = 0; e < RS_EACH; ++e) {
      const int i = threadIdx.x + e * TH;
      if (e && n_list <= e * TH) break;
      c += __syncthreads_count(i < n_list && (strict ? s.cum[i] <= target : s.cum[i] < target));
    }
    return c;
  }

  __device__ void answer(int r, int idx, double prob, uint32_t kept) {
    if (threadIdx.x == 0) {
      a.tokens[r] = idx;
      if (a.prob) a.prob[r] = (float)prob;
      if (a.kept) a.kept[r] = (int)kept;
    }
  }
  // The answer that a sorted list holds which has every kept token; `rest`: mass of the tokens that are not in it.
  __device__ __forceinline__ void settle(int r, int n_list, uint32_t cut, bool cut_k, double top_p, double u, double rest) {
    int kept = (int)min(cut, (uint32_t)n_list);
    if (top_p < 1) {  // the mass it goes by is that of the first k, or of all
      const double target = top_p * (cut_k ? s.cum[kept - 1] : s.cum[n_list - 1] + rest);
      kept = min(kept, list_before(kept, target, false) + 1);
    }
    if (min_p > 0) {
      int ok = 0;
#pragma unroll
      for (int e = 0; e < RS_EACH; ++e) {
        const int i = threadIdx.x + e * TH;
        if (e && n_list <= e * TH) break;
        ok += __syncthreads_count(i < n_list && rs_weight(list_logit(i), g) >= min_p);
      }
      kept = min(kept, max(ok, 1));
    }
    const double mass = s.cum[kept - 1];
    const int i = min(list_before(kept, u * mass, true), kept - 1);
    answer(r, (int)(uint32_t)s.list[i], rs_weight(list_logit(i), g) / mass, (uint32_t)kept);
  }

  // What the first CTA does between two commands, as a machine whose states are what the last command was for: every
  // command is served at one place in the code, which keeps a row's state in registers.  Ends are looked up (LOOK) for
  // a purpose: the first k (mass of), top-p's end, min-p's (mass of), the token, the last kept token.
  enum { START, LISTED, REFILLED, LAST_LIST, LOOKED, DIGIT, FOUND, COUNTED };
  enum { OF_K, OF_P, OF_M, OF_TOKEN, OF_LAST };
  // the next command (DONE: the row is answered); the row's state is in shared memory while a command is served
  __device__ __forceinline__ RSCommand next(int r) {
    RSLead m = s.lead;
    const RSCommand c = step(m, r);
    __syncthreads();
    if (threadIdx.x == 0) s.lead = m;
    return c;
  }
  __device__ __forceinline__ RSCommand step(RSLead& m, int r) {
    RSCommand c{};
    const bool by_p = m.top_p < 1, by_m = min_p > 0;
    if ((m.state == START || m.state == REFILLED) && by_m) m.over = -log(min_p) * g.t * (double)g.sx;
    const int over_bin = m.over < RS_BINS ? (int)fmax(m.over, 0.0) : RS_BINS;
    int idx = 0;          // what a look found
    double w = 0, mass = 0;
    uint32_t cnt = 0;
    const int near = RS_SLACK;
    auto ended = [&](uint32_t cnt, double mass) {  // a prefix's end, and what it leads to
      if (m.purpose != OF_P || cnt < m.kept) { m.kept = m.purpose == OF_M ? m.kept : cnt; m.mass = mass; }
      const int was = m.purpose;
      m.purpose = was == OF_K && by_p ? OF_P : was != OF_M && by_m ? OF_M : OF_TOKEN;
    };
    auto count_over = [&] {
      m.state = COUNTED;
      c.op = RS_OVER; c.b0 = over_bin - near; c.b1 = min(over_bin + near, RS_BINS);
      return c;
    };
    const bool first = m.state == START;
    if (first) {
      c.op = RS_GATHER;
      m.state = m.mode == RS_MASSES ? REFILLED : LISTED;
      if (m.mode == RS_NONE) {
        c.last = all_cnt <= RS_COUNT;
        c.b1 = c.last ? RS_BINS : min(over_bin + near, RS_BINS);
        return c;
      }
    }
    if (first || m.state == REFILLED) scan_bins();
    if (first && m.state == LISTED) {
      c.b1 = cross_one(false, (double)m.cut, false);
      return c;
    }
    if (m.state == LISTED || m.state == LAST_LIST) {
      const int n_list = (int)s.n_list;
      if (n_list <= RS_CAP) {
        sort(n_list);
        list_masses(n_list, 0.0);
        settle(r, n_list, m.cut, m.cut_k, m.top_p, m.u, m.state == LISTED ? 0.0 : all_mass - m.base - m.in_mass);
        return c;
      }
      m.state = REFILLED;
      c.op = RS_FILL; c.sure = (int)RS_ROOM;
      return c;
    }
    if (m.state == REFILLED) {
      if (crowded() && sure < a.per) {
        c.op = RS_FILL; c.sure = a.per;
        return c;
      }
      // the last bin that a kept token can lie in
      __syncthreads();
      if (threadIdx.x == 0) { s.bin_k = s.bin_p = RS_BINS; s.pick = 0; }
      __syncthreads();
      if (m.cut_k) cross(false, (double)m.cut, false, &s.bin_k);
      if (by_p && !m.cut_k) cross(true, m.top_p * all_mass, false, &s.bin_p);
      __syncthreads();
      int last = s.bin_k;
      if (by_m && !(m.cut_k && by_p)) last = min(last, min(over_bin + near, RS_BINS));
      if (by_p && !m.cut_k) last = min(last, s.bin_p == RS_BINS ? s.pick : s.bin_p);
      uint32_t in;
      at_bin(last, &m.before, &m.base, &in, &m.in_mass);
      if (m.before + in <= RS_CAP) {
        m.state = LAST_LIST;
        c.op = RS_GATHER; c.b1 = last; c.last = 1;
        return c;
      }
      // long prefixes: each end by itself
      m.kept = m.cut;
      m.mass = all_mass;
      m.purpose = m.cut_k ? OF_K : by_p ? OF_P : by_m ? OF_M : OF_TOKEN;
      if (m.purpose == OF_M) return count_over();
    } else if (m.state == LOOKED) {
      const int n_list = (int)s.n_list;
      sort(n_list);
      list_masses(n_list, m.base);
      const int i = min(max(m.by_mass ? list_before(n_list, m.target, m.strict) : (int)(m.target - m.before) - 1, 0), n_list - 1);
      idx = (int)(uint32_t)s.list[i];
      w = rs_weight(list_logit(i), g);
      cnt = m.before + i + 1;
      mass = s.cum[i];
    } else if (m.state == DIGIT) {
      // digits in descending order: thread t < 256 has digit 255 - t
      uint32_t k = 0;
      unsigned long long x = 0;
      const int d = 255 - (int)threadIdx.x;
      if (threadIdx.x < 256)
        for (int q = 0; q < CL; ++q) {
          const RSSmem* o = cl.map_shared_rank(&s, q);
          k += o->cnt[d];
          x += (unsigned long long)o->low[256 + d] << 32 | o->low[d];
        }
      uint32_t kb = k, all_k;
      const double of_digit = (double)x * 0x1p-40 * m.unit;
      double mb = of_digit, all_m;
      rs_scan2<TH>(kb, mb, s, &all_k, &all_m);
      if (threadIdx.x == 0) { s.pick = 256; s.pick_cnt = 0; }
      __syncthreads();
      const double at_end = m.by_mass ? m.base + mb + of_digit : (double)(m.before + kb + k);
      if (k) {
        if (m.strict ? at_end > m.target : at_end >= m.target) atomicMin(&s.pick, (int)threadIdx.x);
        atomicMax(&s.pick_cnt, threadIdx.x);  // the last digit that is there, should rounding leave no crossing
      }
      __syncthreads();
      const int at = s.pick < 256 ? s.pick : (int)s.pick_cnt;
      if ((int)threadIdx.x == at) {
        s.sel_cnt = m.before + kb;
        s.sel_base = m.base + mb;
        s.sel_in = k;
        s.pick_w = k ? of_digit / k : 0.0;
      }
      __syncthreads();
      m.before = s.sel_cnt; m.base = s.sel_base; m.left = s.sel_in; m.each = s.pick_w;
      m.prefix = m.prefix << 8 | (uint32_t)(255 - at);
      if (++m.round < 4) {
        c.op = RS_RADIX; c.b0 = m.b; c.prefix = m.prefix; c.shift = 24 - 8 * m.round;
        c.z0 = m.in_mass;
        return c;
      }
      // `left` tokens of the same logit: the j-th of them by index
      double j = 0;
      if (!m.by_mass) j = m.target - m.before - 1;
      else if (m.each > 0) {
        j = floor((m.target - m.base) / m.each);
        if (!m.strict && j * m.each >= m.target - m.base) j -= 1;  // reaching is enough
      }
      m.left = (uint32_t)fmin(fmax(j, 0.0), (double)m.left - 1);
      m.state = FOUND;
      c.op = RS_FIND; c.key = m.prefix; c.skip = m.left;
      return c;
    } else if (m.state == FOUND) {
      idx = s.found;
      w = rs_weight(rs_unorder(m.prefix), g);
      cnt = m.before + m.left + 1;
      mass = m.base + (double)(m.left + 1) * m.each;
    } else {  // COUNTED: tokens of weight >= min-p
      const uint32_t n_over = max(s.over, 1u);
      m.purpose = n_over < m.kept ? OF_M : OF_TOKEN;
      if (m.purpose == OF_M) m.kept = n_over;
    }
    if (m.state == LOOKED || m.state == FOUND) {  // what was found, and what it leads to
      if (m.purpose == OF_TOKEN && cnt > m.kept) {  // the two sums of a bin differ by a rounding
        m.purpose = OF_LAST;
      } else if (m.purpose >= OF_TOKEN) {
        answer(r, idx, w / m.mass, m.kept);
        return c;
      } else {
        ended(cnt, mass);
        if (m.purpose == OF_M) return count_over();
      }
    }
    // LOOK
    uint32_t in;
    double in_mass;
    for (;;) {
      m.by_mass = m.purpose == OF_P || m.purpose == OF_TOKEN;
      m.strict = m.purpose == OF_TOKEN;
      m.target = m.purpose == OF_P ? m.top_p * m.mass : m.purpose == OF_TOKEN ? m.u * m.mass : (double)m.kept;
      m.b = cross_one(m.by_mass, m.target, m.strict);
      at_bin(m.b, &m.before, &m.base, &in, &in_mass);
      if (m.b < RS_BINS || m.purpose >= OF_TOKEN) break;
      ended(m.kept, m.base);  // by count, and behind the bins, where nothing has a mass: which token it is does not matter
      if (m.purpose == OF_M) return count_over();
    }
    if (in <= RS_CAP) {
      m.state = LOOKED;
      c.op = RS_GATHER; c.b0 = c.b1 = m.b;
      c.last = m.purpose == OF_TOKEN && m.kept == all_cnt;  // no prefix ends before the token that is found
      return c;
    }
    // crowded: digit by digit, masses in units of the bin edge's weight
    m.state = DIGIT;
    m.round = 0;
    m.prefix = 0;
    m.in_mass = m.b > 0 && m.b < RS_BINS ? ((double)g.mx - (double)rs_edge((float)m.b, g)) / g.t : 0.0;  // edge / T
    m.unit = m.b < RS_BINS ? exp(-m.in_mass) : 0.0;
    c.op = RS_RADIX; c.b0 = m.b; c.shift = 24; c.z0 = m.in_mass;
    return c;
  }
};

template <class T, bool STAGED, int CL, int TH, int CTAS>
__global__ void __launch_bounds__(TH, CTAS) sample_rows_kernel(const RSArgs a) {
  extern __shared__ __align__(16) uint8_t rs_raw[];
  RSSmem& s = *reinterpret_cast<RSSmem*>(rs_raw);
  T* stage = reinterpret_cast<T*>(rs_raw + (sizeof(RSSmem) + 15) / 16 * 16);
  cg::cluster_group cl = cg::this_cluster();
  rs_arrive<CL>();  // waited for before anything is written to another CTA: it has to be there
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = CL == 1 ? 0 : (int)cl.block_rank();
  const int r = (int)(blockIdx.x / CL);
  const int i0 = min(rank * a.per, a.vocab), n = min(a.per, a.vocab - i0);
  const T* row = reinterpret_cast<const T*>(a.logits) + (int64_t)r * a.ld;
  RSRow<T, STAGED, CL, TH> w{s, stage, a, row, i0, n, RSGeom{}, cl, 0.0, 0u, (int)RS_ROOM};

  // 1. this CTA's logits, the largest and the smallest that is a number.  Copies of 16 bytes and more; the shares are
  // multiples of 8 logits, what is left of a row's end comes by itself.
  constexpr int V = 16 / sizeof(T);
  const int nv = a.vec ? n / V : 0;
  if (STAGED) {
    for (int v = tid; v < nv; v += TH)
      asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" :: "r"(smem_u32(stage + v * V)), "l"(row + i0 + v * V) : "memory");
  }
  const float t = a.temperature ? a.temperature[r] : 1.f;
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f, q = a.min_p ? a.min_p[r] : 0.f, un = a.u[r];
  for (int i = tid; i < RS_BINS; i += TH) s.cnt[i] = s.low[i] = 0;
  RSStat st{-INFINITY, INFINITY, 0};
  auto see = [&](float l) {  // NaN is neither
    st.mx = fmaxf(st.mx, l);
    st.mn = fminf(st.mn, l > -INFINITY ? l : INFINITY);
    st.n += l > -INFINITY;
  };
  if (STAGED) {
    for (int i = nv * V + tid; i < n; i += TH) {
      const T x = row[i0 + i];
      stage[i] = x;
      see(rs_float(x));
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    for (int v = tid; v < nv; v += TH) {  // what this thread has copied
      const uint4 x = *reinterpret_cast<const uint4*>(stage + v * V);
      const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
      for (int j = 0; j < V; ++j) see(rs_float(e[j]));
    }
  } else {
    for (int i = tid; i < n; i += TH) see(rs_float(row[i0 + i]));
  }
  const float largest = st.mx;  // this thread's
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    st.mx = fmaxf(st.mx, __shfl_xor_sync(0xffffffffu, st.mx, o));
    st.mn = fminf(st.mn, __shfl_xor_sync(0xffffffffu, st.mn, o));
    st.n += __shfl_xor_sync(0xffffffffu, st.n, o);
  }
  if (lane == 0) s.wstat[warp] = st;
  if (tid == 0) s.first = 0x7fffffff;
  __syncthreads();
  rs_wait<CL>();
  if (warp == 0) {
    st = s.wstat[lane % (TH / 32)];
#pragma unroll
    for (int o = (TH / 32) / 2; o > 0; o >>= 1) {
      st.mx = fmaxf(st.mx, __shfl_xor_sync(0xffffffffu, st.mx, o));
      st.mn = fminf(st.mn, __shfl_xor_sync(0xffffffffu, st.mn, o));
      st.n += __shfl_xor_sync(0xffffffffu, st.n, o);
    }
    if (lane < CL) cl.map_shared_rank(&s, lane)->stats[rank] = st;
  }
  rs_sync<CL>();
  st = s.stats[0];
#pragma unroll
  for (int c = 1; c < CL; ++c) {
    st.mx = fmaxf(st.mx, s.stats[c].mx);
    st.mn = fminf(st.mn, s.stats[c].mn);
    st.n += s.stats[c].n;
  }
  st.mx += 0.f;
  if (st.mx == -INFINITY || !(t > 0.f)) {  // no token, or greedy: the first of the largest
    int at = 0x7fffffff;
    if (st.mx > -INFINITY)
      for (int i = tid; i < n; i += TH)
        if (w.raw(i) == st.mx) { at = i0 + i; break; }
    at = (int)__reduce_min_sync(0xffffffffu, (unsigned)at);
    if (lane == 0 && at != 0x7fffffff) atomicMin(&cl.map_shared_rank(&s, 0)->first, at);
    rs_sync<CL>();
    if (rank == 0) w.answer(r, st.mx == -INFINITY ? -1 : s.first, st.mx == -INFINITY ? 0.0 : 1.0, st.mx == -INFINITY ? 0u : 1u);
    return;
  }
  // 2. the bins
  RSGeom& g = w.g;
  const float tc = fminf(fmaxf(t, 0x1p-100f), 0x1p100f);
  // a little more than the row's spread: the smallest logit lies in the last bin, not behind it
  const float spread = (st.mx - st.mn) * (1.f + 0x1p-10f);
  if (tid == 0) s.spread = spread;
  g.from = st.mx;
  g.far = fabsf(st.mx) * (float)RS_BINS > RS_FAR * fminf(spread, RS_TEMPS * tc);
  if (g.far) st.mx = 0.f;
  g.mx = st.mx;
  g.t = tc;
  g.inv_t = 1.f / tc;
  w.min_p = q > 0.f ? (double)q : 0.0;
  w.all_cnt = st.n;
  const bool cut_k = k > 0 && (uint32_t)k < st.n, by_p = p < 1.f;
  const int mode = st.n <= RS_COUNT || (q > 0.f && !by_p) ? RS_NONE
                   // the k largest are sure to be few more than k where k is a small part of the threads' largest
                   : cut_k && k <= RS_CAP / 2             ? (k <= a.vocab / (32 / (int)sizeof(T)) / 4 && k <= TH * CL / 8 ? RS_LARGEST : RS_COUNTS)
                                                          : RS_MASSES;
  rs_reach(g, spread, mode == RS_MASSES ? RS_TEMPS * tc : RS_SPAN * fmaxf(tc, 1.f));
  if (mode != RS_NONE) {
    w.histogram(mode, largest);
    rs_sync<CL>();
  }

  // 3. commands of the first CTA, until the row is answered
  if (tid == 0) {
    RSLead m{};
    m.state = RSRow<T, STAGED, CL, TH>::START;
    m.mode = mode;
    m.cut_k = cut_k;
    m.cut = cut_k ? (uint32_t)k : st.n;
    m.top_p = by_p ? (double)p : 1.0;
    m.u = un > 0.f ? (double)fminf(un, 1.f - 0x1p-24f) : 0.0;  // not 1: the last kept token may have no mass
    s.lead = m;
  }
  __syncthreads();
  bool alone = CL == 1;
  for (;;) {
    RSCommand c;
    if (CL == 1 || rank == 0) {
      c = w.next(r);
      if (c.op == RS_DONE && alone) return;
      w.post(c);
    }
    rs_sync<CL>();
    c = s.cmd;
    if (c.op == RS_DONE) return;
    w.serve(c, largest);
    rs_arrive<CL>();
    if (c.last && CL > 1) {
      if (rank) return;  // nobody reads this CTA's memory any more
      alone = true;
    }
    rs_wait<CL>();
  }
}

template <class T, bool STAGED, int CL, int TH, int CTAS>
static int rs_launch_one(const RSArgs& a, int batch, size_t slice, cudaStream_t st) {
  const size_t fixed = (sizeof(RSSmem) + 15) / 16 * 16;
  if (int rc = smem_attr_once<sample_rows_kernel<T, STAGED, CL, TH, CTAS>>((int)(fixed + (STAGED ? RS_STAGE_MAX : 0)))) return rc;
  return kv8_launch_cluster(sample_rows_kernel<T, STAGED, CL, TH, CTAS>, dim3((unsigned)batch * CL), CL, dim3(TH), fixed + slice, st, false, a);
}
template <class T, bool STAGED, int CL>
static int rs_launch_many(const RSArgs& a, int batch, size_t slice, int ctas, cudaStream_t st) {
  if (ctas == 1) return rs_launch_one<T, STAGED, CL, RS_THREADS_FEW, 1>(a, batch, slice, st);
  if (sizeof(T) == 2 && ctas == 3) return rs_launch_one<T, STAGED, CL, RS_THREADS_MANY, sizeof(T) == 2 ? 3 : 2>(a, batch, slice, st);
  return rs_launch_one<T, STAGED, CL, RS_THREADS_MANY, 2>(a, batch, slice, st);
}
// CTAs of a row: what takes the fewest waves of CTAs times a CTA's time, in us: 12 of meetings (6 without other CTAs), and
// the logits' share.  Measured, 1, 2, 4 and 8 CTAs: 256 rows of 32000 fp32 logits 39, 42, 53, 86 us; 8 rows of them without
// a top-k 18 and 11 (1 and 8); 64 rows of 151936 49 and 48 (4 and 8); 8 rows of 1000 with a top-k 8 and 10.
template <class T>
static int rs_launch(RSArgs& a, int batch, cudaStream_t st) {
  auto slice = [&](int cl) { return (size_t)(((a.vocab + cl - 1) / cl + 7) / 8 * 8) * sizeof(T); };
  // CTAs of an SM: one of 512 threads where it takes an SM's shared memory, or half of the SMs are enough (a cluster lies in
  // one group of SMs, which one CTA an SM does not fill evenly)
  auto ctas = [&](int cl) {
    const double n = (double)batch * cl / num_sms();
    if (slice(cl) > RS_HALF || n <= 0.5) return 1;
    return sizeof(T) == 2 && slice(cl) <= RS_HALF / 2 && 1.25 * std::max(1.0, n / 3) < std::max(1.0, n / 2) ? 3 : 2;
  };
  int best = RS_CLUSTER;
  double least = 1e30;
  for (int cl = RS_CLUSTER; cl >= 1; cl /= 2) {
    if (slice(cl) > RS_STAGE_MAX) break;
    const double us = std::max((double)batch * cl / (num_sms() * ctas(cl)), 1.0) * ((cl == 1 ? 6. : 12.) + (double)a.vocab / cl * (ctas(cl) > 1 ? 0.44e-3 : 0.27e-3));
    if (us < least) { least = us; best = cl; }
  }
  a.per = (int)(slice(best) / sizeof(T));
  const int n = ctas(best);
  if (slice(best) > RS_STAGE_MAX) return rs_launch_one<T, false, RS_CLUSTER, RS_THREADS_FEW, 1>(a, batch, 0, st);
  if (best == 1) return rs_launch_many<T, true, 1>(a, batch, slice(1), n, st);
  if (best == 2) return rs_launch_many<T, true, 2>(a, batch, slice(2), n, st);
  if (best == 4) return rs_launch_many<T, true, 4>(a, batch, slice(4), n, st);
  return rs_launch_many<T, true, RS_CLUSTER>(a, batch, slice(RS_CLUSTER), n, st);
}

}  // namespace n730

using namespace n730;

N730_API int n730_sample_rows(const void* d_logits, int dtype, int batch, int vocab, int64_t ld, const float* d_temperature,
                              const int32_t* d_top_k, const float* d_top_p, const float* d_min_p, const float* d_u,
                              int32_t* d_tokens, float* d_prob, int32_t* d_kept, void* stream) {
  const char* what = "sample_rows";
  N730_REQUIRE(d_logits && d_u && d_tokens, N730_NULL, "%s: null pointer", what);
  N730_REQUIRE(dtype == N730_F32 || dtype == N730_F16 || dtype == N730_BF16, N730_BAD_ARG, "%s: dtype %d", what, dtype);
  N730_REQUIRE(batch >= 1 && batch <= (1 << 24) && vocab >= 1 && vocab <= (1 << 23) && ld >= vocab, N730_BAD_ARG,
               "%s: batch %d, vocab %d, row stride %lld", what, batch, vocab, (long long)ld);
  const int es = kv8_esize(dtype);
  N730_REQUIRE(kv8_aligned(es, (const char*)d_logits) &&
                   kv8_aligned(4, d_temperature, d_top_p, d_min_p, d_u, d_prob) && kv8_aligned(4, d_top_k, d_tokens, d_kept),
               N730_BAD_ARG, "%s: pointers must lie on whole elements", what);
  RSArgs a{};
  a.logits = d_logits; a.ld = ld; a.vocab = vocab;
  a.vec = ((uintptr_t)d_logits & 15) == 0 && ld * es % 16 == 0;
  a.temperature = d_temperature; a.top_k = d_top_k; a.top_p = d_top_p; a.min_p = d_min_p; a.u = d_u;
  a.tokens = d_tokens; a.prob = d_prob; a.kept = d_kept;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == N730_F32 ? rs_launch<float>(a, batch, st) : dtype == N730_F16 ? rs_launch<__half>(a, batch, st)
                                                                                : rs_launch<__nv_bfloat16>(a, batch, st);
}
