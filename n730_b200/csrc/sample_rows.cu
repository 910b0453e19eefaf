// Sampling with settings of each row and given random numbers.
//
// Per row, V logits l, temperature T, top-k k, top-p p, min-p q, number u:
//   T <= 0: the first index of the largest logit.  Otherwise tokens are ordered by logit, ties by index, with weights
//   w = exp((l - max l) / T).  Kept is the shortest of three prefixes of that order: the first k tokens; the shortest
//   whose mass reaches p times the mass of those k; the tokens with w >= q.  The token is the first whose cumulative
//   mass exceeds u times the kept mass.
//
// A cluster of 8 CTAs takes a row: each copies an eighth of the logits into its shared memory, so that HBM is read once
// and whatever follows runs on the chip.
//   1. largest and smallest logit;
//   2. a histogram over RS_BINS linear bins of max - l: how many tokens, and, where the mass of all tokens matters (no
//      top-k, or a large one), the sum of w / w(bin's edge) - 1 in fixed point.  Bins are narrow, so that this is small
//      and fp32 holds it to 2^-24 of w or so; a bin's mass is w(edge) * (count + sum), formed in 64 bits.  Both sums are
//      integers: the order of the atomics does not matter.  Each CTA adds up an eighth of the bins over the cluster and
//      puts them where the first CTA scans them;
//   3. where the bins up to the last one that a kept token can lie in hold at most RS_CAP tokens, these are gathered in
//      the first CTA's shared memory and sorted, and the rest is a scan over them with weights in 64 bits; the other
//      CTAs are gone by then.  Where not (flat rows without a top-k), each prefix's end is looked up in its bin by itself:
//      the bin's tokens are gathered and sorted, or, where they are too many (equal logits, coarse types), found by four
//      rounds of 8 bits of the logit, after which the tokens left are equal and go by index.
// All sums are 64-bit floats in a fixed order or integers: the same inputs give the same token.
#include <cooperative_groups.h>

#include <cmath>

#include "kv8.h"

namespace n730 {
namespace cg = cooperative_groups;

constexpr int RS_CLUSTER = 8;      // CTAs of a row, one for rows of up to RS_ALONE logits: no exchange, 15 -> 10 us at 1000
constexpr int RS_ALONE = 16384;
constexpr int RS_THREADS = 512;
constexpr int RS_WARPS = RS_THREADS / 32;
constexpr int RS_BINS = 1536;      // as many as leave room for two CTAs of 19008 fp32 logits (a row of 152064) an SM
constexpr int RS_PER = RS_BINS / RS_THREADS;
constexpr int RS_CAP = 1024;       // tokens that are sorted at once
constexpr int RS_EACH = RS_CAP / RS_THREADS;
constexpr int RS_COUNT = 160;      // lists up to this long are sorted by counting
constexpr int RS_SURE = 2048;      // tokens of a CTA's bin that the fixed point of the bins' masses has room for at first
constexpr float RS_SPAN = 32.f;    // bins reach this many logits, or temperatures where that is more, below the largest
constexpr size_t RS_STAGE_MAX = 160 * 1024;  // longest slice that is kept in shared memory

struct RSArgs {
  const void* logits;
  int64_t ld;
  int vocab, per;                  // per: logits of a CTA
  bool vec;                        // rows lie on 16 bytes
  const float* temperature; const int* top_k; const float* top_p; const float* min_p; const float* u;
  int* tokens; float* prob; int* kept;
};

enum { RS_DONE = 0, RS_MASSES, RS_GATHER, RS_RADIX, RS_OVER, RS_FIND };
struct RSCommand {
  int op, b0, b1;         // bins [b0, b1]
  int last;               // GATHER: nothing follows for the other CTAs
  uint32_t prefix, shift; // RADIX: digits found, where the next one starts
  uint32_t key, skip;     // FIND: the skip-th token of this key
  int sure;               // MASSES: tokens of a CTA's bin to have room for
  double z0;              // RADIX: the bin's edge / T
};
struct RSStat { float mx, mn; };

struct RSSmem {
  uint32_t cnt[RS_BINS];             // by bin; also the counts of 256 digits
  int32_t dev[RS_BINS];              // sums of w / w(edge) - 1; also the digits' masses, low and high words
  uint2 share[2 * RS_BINS / RS_CLUSTER];
  union { unsigned long long list[RS_CAP]; uint32_t bin_cnt[RS_BINS]; };  // list: ~order << 32 | index
  union { double cum[RS_CAP]; double bin_mass[RS_BINS]; };
  RSCommand cmd;
  RSStat stats[RS_CLUSTER];
  RSStat wstat[RS_WARPS];
  double wsum[RS_WARPS];
  uint32_t wcnt[RS_WARPS];
  uint32_t beyond[RS_CLUSTER], most[RS_CLUSTER];  // tokens behind the last bin; of the fullest bin of a share
  uint32_t own_beyond, own_most;
  double sel_base, sel_mass, pick_w;
  uint32_t n_list, over, sel_cnt, sel_in, pick_cnt, occur;
  int bin_k, bin_p, bin_last, pick, found, first;
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

// A row's bins: bin = floor((max - l) * sx); edge(b), its upper end, is max - b * width as fp32 rounds it.
struct RSGeom {
  float mx, sx, width, inv_t;
  double t;
};
__device__ __forceinline__ float rs_place(float l, const RSGeom& g) { return (l == g.mx ? 0.f : g.mx - l) * g.sx; }
// NaN and -infinity have no place below RS_BINS
__device__ __forceinline__ int rs_bin(float l, const RSGeom& g) {
  const float x = rs_place(l, g);
  return x < (float)RS_BINS ? (int)x : RS_BINS;
}
__device__ __forceinline__ float rs_edge(float b, const RSGeom& g) { return fmaf(-b, g.width, g.mx); }
__device__ __forceinline__ double rs_weight(float l, const RSGeom& g) {
  return l == g.mx ? 1.0 : g.mx == INFINITY ? 0.0 : exp(((double)l - (double)g.mx) / g.t);
}

// Exclusive scans over the block in thread order; the totals.
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
  for (int w = 0; w < RS_WARPS; ++w) {
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
template <class V>
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
  for (int w = 0; w < RS_WARPS; ++w) {
    const V x = warps[w];
    if (w < warp) before += x;
    all += x;
  }
  *total = all;
  return before + inc - v;
}

template <class T, bool STAGED, int CL>
struct RSRow {
  static constexpr int V = 16 / sizeof(T), SHARE = RS_BINS / CL;
  RSSmem& s;
  T* stage;              // this CTA's logits
  const RSArgs& a;
  const T* row;          // the row's first logit
  int i0, n;             // this CTA's share
  RSGeom g;
  cg::cluster_group cl;
  double min_p;
  int sure;              // tokens of a CTA's bin that the masses have room for
  bool alone;            // the other CTAs are gone

  __device__ float raw(int i) const { return rs_float(STAGED ? stage[i] : row[i0 + i]); }
  __device__ float get(int i) const { return rs_clean(raw(i)); }
  // f(first index, V logits) over this CTA's, V = 16 bytes of them, NaN behind the last.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int i = threadIdx.x * V; i < n; i += RS_THREADS * V) {
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
      f(i, l);
    }
  }

  // Fixed-point unit of the deviations: a CTA's sum of a bin with up to `sure` tokens stays inside 31 bits.
  __device__ float dev_unit() const {
    const float most = fmaxf(1.f - expf(-g.width * g.inv_t * 1.01f), 0x1p-20f) * (float)sure;
    return ldexpf(1.f, (int)floorf(29.f - log2f(most)));
  }
  // Sums of w / w(edge) - 1 by bin; with `count`, the bins' tokens as well.
  __device__ void fill(bool count, bool masses) {
    const float unit = dev_unit();
    const bool narrow = g.width * g.inv_t < 0x1p-6f;
    uint32_t beyond = 0;
    each([&](int, const float (&l)[V]) {
      int b[V], c[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float x = rs_place(l[j], g), f = __fadd_rd(x, 8388608.f);  // 2^23 + floor(x)
        const bool in = x < (float)RS_BINS;
        beyond += !in && l[j] > -INFINITY;
        b[j] = in ? __float_as_int(f) & 0x7fffff : -1;
        if (masses) {
          // y = (l - edge) / T: the two are near, their difference is exact but for what is below 2^-24 of a bin
          const float y = l[j] == g.mx ? 0.f : (l[j] - rs_edge(f - 8388608.f, g)) * g.inv_t;
          const float e = narrow ? y * fmaf(y, fmaf(y, fmaf(y, 1.f / 24, 1.f / 6), 0.5f), 1.f) : expm1f(y);
          c[j] = __float_as_int(fmaf(e, unit, 12582912.f)) - 0x4b400000;  // to the nearest whole number, below 2^22
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (b[j] >= 0) {
          if (count) atomicAdd(&s.cnt[b[j]], 1u);
          if (masses) atomicAdd(&s.dev[b[j]], c[j]);
        }
    });
    if (count && beyond) atomicAdd(&s.own_beyond, beyond);
  }
  // This CTA's share of the bins, added up over the cluster, to the first CTA.  The cluster has filled before.
  __device__ void reduce(bool masses) {
    const float unit = dev_unit();
    auto mass_of = [&](int b, uint32_t k, int64_t d) {
      return masses && k ? rs_weight(rs_edge((float)b, g), g) * ((double)k + (double)d / unit) : 0.0;
    };
    if (CL == 1) {
      uint32_t most = 0;
      for (int b = threadIdx.x; b < RS_BINS; b += RS_THREADS) {
        const uint32_t k = s.cnt[b];
        most = max(most, k);
        s.bin_cnt[b] = k;
        s.bin_mass[b] = mass_of(b, k, s.dev[b]);
      }
      if (threadIdx.x == 0) s.own_most = 0;
      __syncthreads();
      if (most > RS_SURE) atomicMax(&s.own_most, most);
      __syncthreads();
      if (threadIdx.x == 0) { s.beyond[0] = s.own_beyond; s.most[0] = s.own_most; }
      return;
    }
    const int t = threadIdx.x, rank = (int)cl.block_rank();
    uint32_t k = 0, most = 0;
    int d[CL] = {};
    if (t < 2 * SHARE) {  // two threads a bin, half of the CTAs each
      const int b = rank * SHARE + t % SHARE, r0 = t / SHARE * (CL / 2);
#pragma unroll
      for (int r = 0; r < CL / 2; ++r) {
        const RSSmem* o = cl.map_shared_rank(&s, r0 + r);
        const uint32_t x = o->cnt[b];
        k += x;
        most = max(most, x);
        if (masses) d[r] = o->dev[b];
      }
    }
    int64_t dd = 0;
#pragma unroll
    for (int r = 0; r < CL / 2; ++r) dd += d[r];
    if (t >= SHARE && t < 2 * SHARE) {  // deviations in two words
      s.share[t] = make_uint2((uint32_t)dd, (uint32_t)(dd >> 32));
      s.share[t - SHARE].x = k;
    }
    if (t == 0) s.own_most = 0;
    __syncthreads();
    RSSmem* lead = cl.map_shared_rank(&s, 0);
    if (most > RS_SURE) atomicMax(&s.own_most, most);
    if (t < SHARE) {
      k += s.share[t].x;
      dd += (int64_t)((unsigned long long)s.share[t + SHARE].y << 32 | s.share[t + SHARE].x);
      lead->bin_cnt[rank * SHARE + t] = k;
      lead->bin_mass[rank * SHARE + t] = mass_of(rank * SHARE + t, k, dd);
    }
    __syncthreads();
    if (t == 0) { lead->beyond[rank] = s.own_beyond; lead->most[rank] = s.own_most; }
  }

  // A CTA's share of a command.
  __device__ void serve(const RSCommand& c) {
    const int tid = threadIdx.x;
    if (c.op == RS_MASSES) {
      sure = c.sure;
      for (int i = tid; i < RS_BINS; i += RS_THREADS) s.dev[i] = 0;
      __syncthreads();
      fill(false, true);
      rs_sync<CL>();
      reduce(true);
    } else if (c.op == RS_GATHER) {
      RSSmem* lead = CL == 1 ? &s : cl.map_shared_rank(&s, 0);
      const float lo = (float)c.b0, hi = c.b1 == RS_BINS ? INFINITY : (float)(c.b1 + 1);  // -infinity's place is infinity
      each([&](int i, const float (&l)[V]) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float x = rs_place(l[j], g);
          if (!((x >= lo && x < hi) || (hi == INFINITY && x == hi && l[j] > -INFINITY))) continue;
          const uint32_t at = atomicAdd(&lead->n_list, 1u);
          if (at < RS_CAP) lead->list[at] = (unsigned long long)~rs_order(l[j] + 0.f) << 32 | (uint32_t)(i0 + i + j);
        }
      });
    } else if (c.op == RS_RADIX) {
      uint32_t* lo = reinterpret_cast<uint32_t*>(s.dev);
      for (int i = tid; i < 256; i += RS_THREADS) s.cnt[i] = lo[i] = lo[256 + i] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += RS_THREADS) {
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
      for (int i = tid; i < n; i += RS_THREADS) {
        const float l = get(i);
        if (l == -INFINITY) continue;
        const int b = rs_bin(l, g);
        k += b < c.b0 || (b <= c.b1 && rs_weight(l, g) >= min_p);
      }
      uint32_t all;
      rs_scan<uint32_t>(k, s.wcnt, &all);
      if (tid == 0) atomicAdd(&cl.map_shared_rank(&s, 0)->over, all);
    } else if (c.op == RS_FIND) {
      // tokens of the key in this CTA, then its place among the CTAs', then in thread order (contiguous runs)
      const int run = (n + RS_THREADS - 1) / RS_THREADS, j0 = min(n, tid * run), j1 = min(n, j0 + run);
      uint32_t k = 0, all;
      for (int i = j0; i < j1; ++i) k += get(i) != -INFINITY && rs_order(get(i)) == c.key;
      const uint32_t before = rs_scan<uint32_t>(k, s.wcnt, &all);
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
  uint32_t bin_cnt[RS_PER], cnt_before, all_cnt;   // this thread's bins: tokens, tokens of all bins before; of the row
  double bin_mass[RS_PER], mass_before, all_mass;

  __device__ void post(const RSCommand& c) {  // to every CTA
    if (threadIdx.x < CL) cl.map_shared_rank(&s, threadIdx.x)->cmd = c;
  }
  __device__ void command(const RSCommand& c) {
    __syncthreads();
    post(c);
    if (threadIdx.x == 0) { s.n_list = 0; s.over = 0; }
    rs_sync<CL>();
    serve(c);
    rs_sync<CL>();
    if (c.last || CL == 1) alone = true;
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
    rs_scan2(cnt_before, mass_before, s, &all, &all_mass);
#pragma unroll
    for (int r = 0; r < CL; ++r) all += s.beyond[r];
    all_cnt = all;
  }
  __device__ uint32_t most() const {
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < CL; ++r) m = max(m, s.most[r]);
    return m;
  }
  // the bins' masses once more, or at last
  __device__ void recollect(int room) {
    RSCommand c{};
    c.op = RS_MASSES; c.sure = room;
    command(c);
    scan_bins();
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
    // two neighbours a thread: steps of up to 32 stay in a warp
    int np2 = 256;
    while (np2 < n_list) np2 <<= 1;
    for (int i = n_list + t; i < np2; i += RS_THREADS) s.list[i] = ~0ull;
    __syncthreads();
    unsigned long long x = ~0ull, y = ~0ull;
    const bool mine = 2 * t < np2;
    if (mine) { x = s.list[2 * t]; y = s.list[2 * t + 1]; }
    for (int size = 2; size <= np2; size <<= 1) {
      const bool up = ((2 * t) & size) == 0;
      int step = size >> 1;
      if (step > 32) {
        if (mine) { s.list[2 * t] = x; s.list[2 * t + 1] = y; }
        __syncthreads();
        for (; step > 32; step >>= 1) {
          for (int i = t; i < np2 / 2; i += RS_THREADS) {
            const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
            const unsigned long long p = s.list[lo], q = s.list[hi];
            if ((p > q) == ((lo & size) == 0)) { s.list[lo] = q; s.list[hi] = p; }
          }
          __syncthreads();
        }
        if (mine) { x = s.list[2 * t]; y = s.list[2 * t + 1]; }
      }
      for (; step > 1; step >>= 1) {
        const int o = step >> 1;  // threads between the two
        const unsigned long long px = __shfl_xor_sync(0xffffffffu, x, o), py = __shfl_xor_sync(0xffffffffu, y, o);
        const bool keep_small = ((t & o) == 0) == up;
        x = (px < x) == keep_small ? px : x;
        y = (py < y) == keep_small ? py : y;
      }
      if ((x > y) == up) { const unsigned long long z = x; x = y; y = z; }
    }
    if (mine) { s.list[2 * t] = x; s.list[2 * t + 1] = y; }
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
    double m = base + rs_scan<double>(loc, s.wsum, &total);
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int i = threadIdx.x * EACH + e;
      m += w[e];
      if (i < n_list) s.cum[i] = m;
    }
    __syncthreads();
  }
  __device__ void list_masses(int n_list, double base) {
    if (n_list <= RS_THREADS) list_masses_of<1>(n_list, base);
    else list_masses_of<RS_EACH>(n_list, base);
  }
  // how many of the list's first n tokens lie before the target: mass below it (strict: not above it)
  __device__ int list_before(int n_list, double target, bool strict) {
    int c = 0;
#pragma unroll
    for (int e = 0; e < RS_EACH; ++e) {
      const int i = threadIdx.x + e * RS_THREADS;
      if (e && n_list <= e * RS_THREADS) break;
      c += __syncthreads_count(i < n_list && (strict ? s.cum[i] <= target : s.cum[i] < target));
    }
    return c;
  }

  // The first token in order at which the running count or mass reaches the target (strict: exceeds it): its index, its
  // weight, and the count and mass up to and with it.
  struct Pick { int idx; double w; uint32_t cnt; double mass; };
  __device__ Pick select(bool by_mass, double target, bool strict, bool last) {
    const int b = cross_one(by_mass, target, strict);
    uint32_t before, in;
    double base, in_mass;
    at_bin(b, &before, &base, &in, &in_mass);
    Pick p;
    if (in <= RS_CAP) {
      RSCommand c{};
      c.op = RS_GATHER; c.b0 = c.b1 = b; c.last = last;
      command(c);
      const int n_list = (int)s.n_list;
      sort(n_list);
      list_masses(n_list, base);
      const int i = min(max(by_mass ? list_before(n_list, target, strict) : (int)(target - before) - 1, 0), n_list - 1);
      p.mass = s.cum[i];
      p.idx = (int)(uint32_t)s.list[i];
      p.w = rs_weight(list_logit(i), g);
      p.cnt = before + i + 1;
      __syncthreads();
      return p;
    }
    // crowded: digit by digit, masses in units of the bin edge's weight
    RSCommand c{};
    c.op = RS_RADIX; c.b0 = b;
    c.z0 = b > 0 && b < RS_BINS ? ((double)g.mx - (double)rs_edge((float)b, g)) / g.t : 0.0;
    const double unit = b < RS_BINS ? exp(-c.z0) : 0.0;
    double each = 0;   // of the tokens left: their weight
    uint32_t left = 0;
    for (int round = 0; round < 4; ++round) {
      c.shift = 24 - 8 * round;
      command(c);
      // digits in descending order: thread t < 256 has digit 255 - t
      uint32_t k = 0;
      unsigned long long m = 0;
      const int d = 255 - (int)threadIdx.x;
      if (threadIdx.x < 256)
        for (int r = 0; r < CL; ++r) {
          const RSSmem* o = cl.map_shared_rank(&s, r);
          const uint32_t* lo = reinterpret_cast<const uint32_t*>(o->dev);
          k += o->cnt[d];
          m += (unsigned long long)lo[256 + d] << 32 | lo[d];
        }
      uint32_t all_k;
      double all_m;
      const double mass = (double)m * 0x1p-40 * unit;
      const uint32_t kb = rs_scan<uint32_t>(k, s.wcnt, &all_k);
      const double mb = rs_scan<double>(mass, s.wsum, &all_m);
      if (threadIdx.x == 0) { s.pick = 256; s.pick_cnt = 0; }
      __syncthreads();
      const double x = by_mass ? base + mb + mass : (double)(before + kb + k);
      if (k) {
        if (strict ? x > target : x >= target) atomicMin(&s.pick, (int)threadIdx.x);
        atomicMax(&s.pick_cnt, threadIdx.x);  // the last digit that is there, should rounding leave no crossing
      }
      __syncthreads();
      const int at = s.pick < 256 ? s.pick : (int)s.pick_cnt;
      if ((int)threadIdx.x == at) { s.sel_cnt = before + kb; s.sel_base = base + mb; s.sel_in = k; s.pick_w = k ? mass / k : 0.0; }
      __syncthreads();
      before = s.sel_cnt; base = s.sel_base; left = s.sel_in; each = s.pick_w;
      c.prefix = c.prefix << 8 | (uint32_t)(255 - at);
      __syncthreads();
    }
    // `left` tokens of the same logit: the j-th of them by index
    double j = 0;
    if (!by_mass) j = target - before - 1;
    else if (each > 0) {
      j = floor((target - base) / each);
      if (!strict && j * each >= target - base) j -= 1;  // reaching is enough
    }
    const uint32_t skip = (uint32_t)min(max(j, 0.0), (double)left - 1);
    c.op = RS_FIND; c.key = c.prefix; c.skip = skip;
    command(c);
    p.idx = s.found;
    p.w = rs_weight(rs_unorder(c.prefix), g);
    p.cnt = before + skip + 1;
    p.mass = base + (double)(skip + 1) * each;
    __syncthreads();
    return p;
  }

  __device__ void answer(int r, int idx, double prob, uint32_t kept) {
    if (threadIdx.x == 0) {
      a.tokens[r] = idx;
      if (a.prob) a.prob[r] = (float)prob;
      if (a.kept) a.kept[r] = (int)kept;
    }
  }

  __device__ void lead(int r, int k, double top_p, double u, bool masses) {
    scan_bins();
    if (masses && most()) recollect((int)most());
    const uint32_t all = all_cnt;
    const bool cut_k = k > 0 && (uint32_t)k < all;
    const uint32_t cut = cut_k ? (uint32_t)k : all;
    const bool by_p = top_p < 1, by_m = min_p > 0;
    const bool listed = cut_k || !masses;  // the mass that top-p goes by is that of tokens that are all in the list
    // the last bin that a kept token can lie in
    const double over = by_m ? -log(min_p) * g.t * (double)g.sx : 0.0;
    __syncthreads();
    if (threadIdx.x == 0) { s.bin_k = s.bin_p = RS_BINS; s.pick = 0; }
    __syncthreads();
    if (cut_k) cross(false, (double)k, false, &s.bin_k);
    if (by_p && !listed) cross(true, top_p * all_mass, false, &s.bin_p);
    __syncthreads();
    int last = s.bin_k;
    if (by_m && !(listed && by_p)) last = min(last, over < RS_BINS ? (int)fmax(over, 0.0) + 1 : RS_BINS);
    if (by_p && !listed) last = min(last, s.bin_p == RS_BINS ? s.pick : s.bin_p);
    uint32_t before, in;
    double base, in_mass;
    at_bin(last, &before, &base, &in, &in_mass);
    if (before + in <= RS_CAP) {
      RSCommand c{};
      c.op = RS_GATHER; c.b1 = last; c.last = 1;
      command(c);
      const int n_list = (int)s.n_list;
      sort(n_list);
      list_masses(n_list, 0.0);
      int kept = (int)min(cut, (uint32_t)n_list);
      if (by_p) {
        // mass of the cut: of the list's first k, or of the list and the bins behind it
        const double mass = listed ? s.cum[kept - 1] : s.cum[n_list - 1] + (all_mass - base - in_mass);
        kept = min(kept, list_before(kept, top_p * mass, false) + 1);
      }
      if (by_m) {
        int ok = 0;
#pragma unroll
        for (int e = 0; e < RS_EACH; ++e) {
          const int i = threadIdx.x + e * RS_THREADS;
          if (e && n_list <= e * RS_THREADS) break;
          ok += __syncthreads_count(i < n_list && rs_weight(list_logit(i), g) >= min_p);
        }
        kept = min(kept, max(ok, 1));
      }
      const double mass = s.cum[kept - 1];
      const int i = min(list_before(kept, u * mass, true), kept - 1);
      answer(r, (int)(uint32_t)s.list[i], rs_weight(list_logit(i), g) / mass, (uint32_t)kept);
      return;
    }
    // long prefixes: each end by itself
    if (!masses) recollect((int)max(most(), (uint32_t)RS_SURE));  // the k-th token's bin is crowded
    uint32_t kept = cut;
    double mass = all_mass;
    if (cut_k) mass = select(false, (double)k, false, false).mass;
    if (by_p) {
      const Pick p = select(true, top_p * mass, false, false);
      if (p.cnt < kept) { kept = p.cnt; mass = p.mass; }
    }
    if (by_m) {
      const int b = over < RS_BINS ? (int)fmax(over, 0.0) : RS_BINS;
      RSCommand c{};
      c.op = RS_OVER; c.b0 = b - 1; c.b1 = min(b + 1, RS_BINS);
      command(c);
      const uint32_t n_over = max(s.over, 1u);
      __syncthreads();
      if (n_over < kept) { kept = n_over; mass = select(false, (double)n_over, false, false).mass; }
    }
    Pick p = select(true, u * mass, true, !cut_k && !by_p && !by_m);
    if (p.cnt > kept) p = select(false, (double)kept, false, true);  // the two sums of a bin differ by a rounding
    answer(r, p.idx, p.w / mass, kept);
  }
};

template <class T, bool STAGED, int CL>
__global__ void __launch_bounds__(RS_THREADS, 2) sample_rows_kernel(const RSArgs a) {
  extern __shared__ __align__(16) uint8_t rs_raw[];
  RSSmem& s = *reinterpret_cast<RSSmem*>(rs_raw);
  T* stage = reinterpret_cast<T*>(rs_raw + (sizeof(RSSmem) + 15) / 16 * 16);
  cg::cluster_group cl = cg::this_cluster();
  rs_arrive<CL>();  // waited for before anything is written to another CTA: it has to be there
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = CL == 1 ? 0 : (int)cl.block_rank();
  const int r = (int)(blockIdx.x / CL);
  const int i0 = min(rank * a.per, a.vocab), n = min(a.per, a.vocab - i0);
  const T* row = reinterpret_cast<const T*>(a.logits) + (int64_t)r * a.ld;
  RSRow<T, STAGED, CL> w{s, stage, a, row, i0, n, RSGeom{}, cl, 0.0, RS_SURE, false};

  // 1. this CTA's logits, the largest and the smallest that is a number.  Copies of 16 bytes and more; the shares are
  // multiples of 8 logits, what is left of a row's end comes by itself.
  constexpr int V = 16 / sizeof(T);
  const int nv = a.vec ? n / V : 0;
  if (STAGED) {
    for (int v = tid; v < nv; v += RS_THREADS)
      asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" :: "r"(smem_u32(stage + v * V)), "l"(row + i0 + v * V) : "memory");
  }
  const float t = a.temperature ? a.temperature[r] : 1.f;
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f, q = a.min_p ? a.min_p[r] : 0.f, un = a.u[r];
  for (int i = tid; i < RS_BINS; i += RS_THREADS) { s.cnt[i] = 0; s.dev[i] = 0; }
  if (tid == 0) s.own_beyond = 0;
  RSStat st{-INFINITY, INFINITY};
  auto see = [&](float l) {  // NaN is neither
    st.mx = fmaxf(st.mx, l);
    st.mn = fminf(st.mn, l > -INFINITY ? l : INFINITY);
  };
  if (STAGED) {
    for (int i = nv * V + tid; i < n; i += RS_THREADS) {
      const T x = row[i0 + i];
      stage[i] = x;
      see(rs_float(x));
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    for (int v = tid; v < nv; v += RS_THREADS) {  // what this thread has copied
      const uint4 x = *reinterpret_cast<const uint4*>(stage + v * V);
      const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
      for (int j = 0; j < V; ++j) see(rs_float(e[j]));
    }
  } else {
    for (int i = tid; i < n; i += RS_THREADS) see(rs_float(row[i0 + i]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    st.mx = fmaxf(st.mx, __shfl_xor_sync(0xffffffffu, st.mx, o));
    st.mn = fminf(st.mn, __shfl_xor_sync(0xffffffffu, st.mn, o));
  }
  if (lane == 0) s.wstat[warp] = st;
  if (tid == 0) s.first = 0x7fffffff;
  __syncthreads();
  rs_wait<CL>();
  if (warp == 0) {
    st = s.wstat[lane % RS_WARPS];
#pragma unroll
    for (int o = RS_WARPS / 2; o > 0; o >>= 1) {
      st.mx = fmaxf(st.mx, __shfl_xor_sync(0xffffffffu, st.mx, o));
      st.mn = fminf(st.mn, __shfl_xor_sync(0xffffffffu, st.mn, o));
    }
    if (lane < CL) cl.map_shared_rank(&s, lane)->stats[rank] = st;
  }
  rs_sync<CL>();
  st = s.stats[0];
#pragma unroll
  for (int c = 1; c < CL; ++c) { st.mx = fmaxf(st.mx, s.stats[c].mx); st.mn = fminf(st.mn, s.stats[c].mn); }
  st.mx += 0.f;
  if (st.mx == -INFINITY || !(t > 0.f)) {  // no token, or greedy: the first of the largest
    int at = 0x7fffffff;
    if (st.mx > -INFINITY)
      for (int i = tid; i < n; i += RS_THREADS)
        if (w.raw(i) == st.mx) { at = i0 + i; break; }
    at = (int)__reduce_min_sync(0xffffffffu, (unsigned)at);
    if (lane == 0 && at != 0x7fffffff) atomicMin(&cl.map_shared_rank(&s, 0)->first, at);
    rs_sync<CL>();
    if (rank == 0) w.answer(r, st.mx == -INFINITY ? -1 : s.first, st.mx == -INFINITY ? 0.0 : 1.0, st.mx == -INFINITY ? 0u : 1u);
    return;
  }
  const bool masses = !(k > 0 && k <= RS_CAP / 2);

  // 2. the bins
  RSGeom& g = w.g;
  g.mx = st.mx;
  const float tc = fminf(fmaxf(t, 0x1p-100f), 0x1p100f);
  g.t = tc;
  g.inv_t = 1.f / tc;
  // a little more than the row's spread: the smallest logit lies in the last bin, not behind it
  const float span = fminf((st.mx - st.mn) * (1.f + 0x1p-20f), RS_SPAN * fmaxf(tc, 1.f));
  g.sx = span > 1e-30f ? (float)RS_BINS / span : 0.f;
  g.width = span > 1e-30f ? span / (float)RS_BINS : 0.f;
  w.min_p = q > 0.f ? (double)q : 0.0;
  w.fill(true, masses);
  rs_sync<CL>();
  w.reduce(masses);
  rs_sync<CL>();

  // 3. ends of the prefixes and the token
  if (CL == 1 || rank == 0) {
    const double up = un > 0.f ? fmin((double)un, 1.0) : 0.0;
    w.lead(r, k, p < 1.f ? (double)p : 1.0, up, masses);
    if (!w.alone) {
      __syncthreads();
      RSCommand c{};
      w.post(c);
      rs_sync<CL>();
    }
    return;
  }
  for (;;) {
    rs_sync<CL>();
    const RSCommand c = s.cmd;
    if (c.op == RS_DONE) return;
    w.serve(c);
    rs_arrive<CL>();
    if (c.last) return;  // nobody reads this CTA's memory any more
    rs_wait<CL>();
  }
}

template <class T, bool STAGED, int CL>
static int rs_launch_one(const RSArgs& a, int batch, size_t slice, cudaStream_t st) {
  const size_t fixed = (sizeof(RSSmem) + 15) / 16 * 16;
  if (int rc = smem_attr_once<sample_rows_kernel<T, STAGED, CL>>((int)(fixed + (STAGED ? RS_STAGE_MAX : 0)))) return rc;
  return kv8_launch_cluster(sample_rows_kernel<T, STAGED, CL>, dim3((unsigned)batch * CL), CL, dim3(RS_THREADS), fixed + slice, st,
                            false, a);
}
template <class T>
static int rs_launch(RSArgs& a, int batch, cudaStream_t st) {
  const int cl = a.vocab <= RS_ALONE ? 1 : RS_CLUSTER;
  a.per = ((a.vocab + cl - 1) / cl + 7) / 8 * 8;
  const size_t slice = (size_t)a.per * sizeof(T);
  if (cl == 1) return rs_launch_one<T, true, 1>(a, batch, slice, st);
  if (slice <= RS_STAGE_MAX) return rs_launch_one<T, true, RS_CLUSTER>(a, batch, slice, st);
  return rs_launch_one<T, false, RS_CLUSTER>(a, batch, 0, st);
}

}  // namespace n730

using namespace n730;

N730_API int n730_sample_rows(const void* d_logits, int dtype, int batch, int vocab, int64_t ld, const float* d_temperature,
                              const int32_t* d_top_k, const float* d_top_p, const float* d_min_p, const float* d_u,
                              int32_t* d_tokens, float* d_prob, int32_t* d_kept, void* stream) {
  const char* what = "sample_rows";
  N730_REQUIRE(d_logits && d_u && d_tokens, N730_NULL, "%s: null pointer", what);
  N730_REQUIRE(dtype == N730_F32 || dtype == N730_F16 || dtype == N730_BF16, N730_BAD_ARG, "%s: dtype %d", what, dtype);
  N730_REQUIRE(batch >= 1 && batch <= (1 << 24) && vocab >= 1 && vocab <= (1 << 24) && ld >= vocab, N730_BAD_ARG,
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
