// Sampling with settings of each row and given random numbers.
//
// Per row, V logits l, temperature T, top-k k, top-p p, min-p q, number u:
//   T <= 0: the first index of the largest logit.  Otherwise tokens are ordered by logit, ties by index, with weights
//   w = exp((l - max l) / T).  Kept is the shortest of three prefixes of that order: the first k tokens; the shortest
//   whose mass reaches p times the mass of those k; the tokens with w >= q.  The token is the first whose cumulative
//   mass exceeds u times the kept mass.
//
// A cluster of 8 CTAs takes a row: each keeps an eighth of the logits in shared memory, so that HBM is read once and
// whatever follows runs on the chip.
//   1. largest and smallest logit;
//   2. a histogram over RS_BINS linear bins of max - l: how many tokens, and, where the mass of all tokens matters (no
//      top-k, or a large one), the sum of w / w(bin's edge) - 1 in fixed point.  Bins are narrow, so that this is small
//      and fp32 holds it to 2^-24 of w or so; a bin's mass is w(edge) * (count + sum), formed in 64 bits.  Both sums are
//      integers: the order of the atomics does not matter;
//   3. the first CTA scans the bins.  Where the bins up to the last one that a kept token can lie in hold at most
//      RS_CAP tokens, these are gathered in its shared memory and sorted, and the rest is a scan over them with weights
//      in 64 bits.  Where not (flat rows without a top-k), each prefix's end is looked up in its bin by itself: the
//      bin's tokens are gathered and sorted, or, where they are too many (equal logits, coarse types), found by four
//      rounds of 8 bits of the logit, after which the tokens left are equal and go by index.
// All sums are 64-bit floats in a fixed order or integers: the same inputs give the same token.
#include <cooperative_groups.h>

#include <cmath>

#include "kv8.h"

namespace n730 {
namespace cg = cooperative_groups;

constexpr int RS_CLUSTER = 8;
constexpr int RS_THREADS = 512;
constexpr int RS_WARPS = RS_THREADS / 32;
constexpr int RS_BINS = 2048;      // and one more for what lies behind the last
constexpr int RS_PER = RS_BINS / RS_THREADS;
constexpr int RS_CAP = 2048;       // tokens that are sorted at once
constexpr int RS_EACH = RS_CAP / RS_THREADS;
constexpr int RS_SURE = 2048;      // tokens of a CTA's bin that the fixed point of the bins' masses has room for at first
constexpr float RS_SPAN = 32.f;    // bins reach this many logits, or temperatures where that is more, below the largest
constexpr size_t RS_STAGE_MAX = 160 * 1024;  // longest slice that is kept in shared memory

struct RSArgs {
  const void* logits;
  int64_t ld;
  int vocab, dtype, per;           // per: logits of a CTA
  bool vec;                        // rows lie on 16 bytes
  const float* temperature; const int* top_k; const float* top_p; const float* min_p; const float* u;
  int* tokens; float* prob; int* kept;
};

enum { RS_DONE = 0, RS_MASSES, RS_GATHER, RS_RADIX, RS_OVER, RS_FIND };
struct RSCommand {
  int op, b0, b1;         // bins [b0, b1]
  uint32_t prefix, shift; // RADIX: digits found, where the next one starts
  uint32_t key, skip;     // FIND: the skip-th token of this key
  int sure;               // MASSES: tokens of a CTA's bin to have room for
  double z0;              // RADIX: the bin's edge / T
};
struct RSStat { float mx, mn; int idx, pad; };

struct RSSmem {
  uint32_t cnt[RS_BINS + 4];       // by bin; also the counts of 256 digits
  int32_t dev[RS_BINS + 4];        // sums of w / w(edge) - 1; also the digits' masses, low and high words
  unsigned long long list[RS_CAP]; // (order of the logit, largest first) << 32 | index
  RSCommand cmd;
  RSStat stat;
  RSStat wstat[RS_WARPS];
  double wsum[RS_WARPS];
  uint32_t wcnt[RS_WARPS];
  double all_mass, pick_mass, pick_w, sel_base;
  uint32_t all_cnt, most_cnt, n_list, over, sel_cnt, sel_bin_cnt, pick_cnt;
  int sel_bin, pick, found;
  uint32_t occur;
};

// the order of logits as unsigned numbers (largest largest); logits here are no NaN and no -0
__device__ __forceinline__ uint32_t rs_order(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float rs_unorder(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ float rs_clean(float x) { return x != x ? -INFINITY : x + 0.f; }

// A row's bins: bin = floor((max - l) * sx), edge(b) = b * width below the largest.
struct RSGeom {
  float mx, sx, width, inv_t;
  double t;
};
__device__ __forceinline__ float rs_below(float l, const RSGeom& g) { return l == g.mx ? 0.f : g.mx - l; }
__device__ __forceinline__ int rs_bin(float l, const RSGeom& g) {
  const float x = rs_below(l, g) * g.sx;
  return x < (float)RS_BINS ? (int)x : RS_BINS;
}
__device__ __forceinline__ double rs_weight(float l, const RSGeom& g) {
  return l == g.mx ? 1.0 : g.mx == INFINITY ? 0.0 : exp(((double)l - (double)g.mx) / g.t);
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

template <bool STAGED>
struct RSRow {
  RSSmem& s;
  float* stage;          // this CTA's logits
  const RSArgs& a;
  int64_t base;          // the row's first logit
  int i0, n;             // this CTA's share
  RSGeom g;
  cg::cluster_group cl;
  double zmin;           // log of min-p
  int sure;              // tokens of a CTA's bin that the masses have room for

  __device__ float get(int i) const {
    return STAGED ? stage[i] : rs_clean(kv8_load1(a.logits, base + i0 + i, a.dtype));
  }

  // Sums of w / w(edge) - 1 by bin; with `count`, the bins' tokens as well.
  __device__ void fill(bool count, bool masses) {
    const float unit = dev_unit();
    const bool narrow = g.width * g.inv_t < 0x1p-6f;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += RS_THREADS) {
      const float l = get(i);
      if (l == -INFINITY) continue;
      const int b = rs_bin(l, g);
      if (count) atomicAdd(&s.cnt[b], 1u);
      if (masses && b < RS_BINS) {
        // y = (l - max + edge) / T, with the rounding of max - l put back
        const float d = rs_below(l, g), bb = d - g.mx, err = l == g.mx ? 0.f : (g.mx - (d - bb)) - (l + bb);
        const float y = -(fmaf(-(float)b, g.width, d) + err) * g.inv_t;
        const float c = narrow ? y * fmaf(y, fmaf(y, fmaf(y, 1.f / 24, 1.f / 6), 0.5f), 1.f) : expm1f(y);
        atomicAdd(&s.dev[b], __float2int_rn(c * unit));
      }
    }
  }

  // A CTA's share of a command.
  __device__ void serve(const RSCommand& c) {
    const int tid = threadIdx.x;
    if (c.op == RS_MASSES) {
      sure = c.sure;
      for (int i = tid; i < RS_BINS; i += RS_THREADS) s.dev[i] = 0;
      __syncthreads();
      fill(false, true);
    } else if (c.op == RS_GATHER) {
      RSSmem* lead = cl.map_shared_rank(&s, 0);
      for (int i = tid; i < n; i += RS_THREADS) {
        const float l = get(i);
        if (l == -INFINITY) continue;
        const int b = rs_bin(l, g);
        if (b < c.b0 || b > c.b1) continue;
        const uint32_t at = atomicAdd(&lead->n_list, 1u);
        if (at < RS_CAP) lead->list[at] = (unsigned long long)~rs_order(l) << 32 | (uint32_t)(i0 + i);
      }
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
      const double q = exp(zmin);
      for (int i = tid; i < n; i += RS_THREADS) {
        const float l = get(i);
        if (l == -INFINITY) continue;
        const int b = rs_bin(l, g);
        k += b < c.b0 || (b <= c.b1 && rs_weight(l, g) >= q);
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
      cl.sync();
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
  double bin_mass[RS_PER], mass_before;

  __device__ void command(const RSCommand& c) {
    __syncthreads();
    if (threadIdx.x == 0) { s.cmd = c; s.n_list = 0; s.over = 0; }
    cl.sync();
    serve(c);
    cl.sync();
  }

  // the histogram of all CTAs, scanned
  __device__ void collect(bool masses) {
    const int b = threadIdx.x * RS_PER;
    uint32_t k[RS_PER] = {}, beyond = 0, most = 0;
    if (threadIdx.x == 0) s.most_cnt = 0;
    __syncthreads();
    int64_t d[RS_PER] = {};
    for (int r = 0; r < RS_CLUSTER; ++r) {
      const RSSmem* o = cl.map_shared_rank(&s, r);
      const uint4 x = *reinterpret_cast<const uint4*>(&o->cnt[b]);
      k[0] += x.x; k[1] += x.y; k[2] += x.z; k[3] += x.w;
      most = max(most, max(max(x.x, x.y), max(x.z, x.w)));
      if (masses) {
        const int4 y = *reinterpret_cast<const int4*>(&o->dev[b]);
        d[0] += y.x; d[1] += y.y; d[2] += y.z; d[3] += y.w;
      }
      if (threadIdx.x == 0) beyond += o->cnt[RS_BINS];
    }
    if (most > RS_SURE) atomicMax(&s.most_cnt, most);
    uint32_t kc = 0;
    double mc = 0;
#pragma unroll
    for (int e = 0; e < RS_PER; ++e) {
      bin_cnt[e] = k[e];
      bin_mass[e] = k[e] && masses ? exp(-(double)(b + e) * (double)g.width / g.t) * ((double)k[e] + (double)d[e] / dev_unit()) : 0.0;
      kc += bin_cnt[e];
      mc += bin_mass[e];
    }
    uint32_t all;
    double mass;
    cnt_before = rs_scan<uint32_t>(kc, s.wcnt, &all);
    mass_before = rs_scan<double>(mc, s.wsum, &mass);
    if (threadIdx.x == 0) { s.all_cnt = all + beyond; s.all_mass = mass; }
    __syncthreads();
  }
  // Fixed-point unit of the deviations: a CTA's sum of a bin with up to `sure` tokens stays inside 31 bits.
  __device__ float dev_unit() const {
    const float most = fmaxf(1.f - expf(-g.width * g.inv_t * 1.01f), 0x1p-20f) * (float)sure;
    return ldexpf(1.f, (int)floorf(29.f - log2f(most)));
  }

  // First bin at which the running count or mass reaches the target (strict: exceeds it); when none does, RS_BINS by
  // count and the last one with a token by mass (a rounding is missing).
  __device__ int cross(bool by_mass, double target, bool strict) {
    if (threadIdx.x == 0) { s.sel_bin = RS_BINS; s.pick = 0; }
    __syncthreads();
    uint32_t k = cnt_before;
    double m = mass_before;
#pragma unroll
    for (int e = 0; e < RS_PER; ++e) {
      k += bin_cnt[e];
      m += bin_mass[e];
      const double x = by_mass ? m : (double)k;
      if (!bin_cnt[e]) continue;
      atomicMax(&s.pick, (int)threadIdx.x * RS_PER + e);
      if (strict ? x > target : x >= target) { atomicMin(&s.sel_bin, (int)threadIdx.x * RS_PER + e); break; }
    }
    __syncthreads();
    const int b = by_mass && s.sel_bin == RS_BINS ? s.pick : s.sel_bin;
    __syncthreads();
    return b;
  }
  // tokens and mass of all bins before b, and of b
  __device__ void at_bin(int b, uint32_t* before, double* mass, uint32_t* in) {
    if ((int)threadIdx.x == min(b, RS_BINS - 1) / RS_PER) {
      uint32_t k = cnt_before;
      double m = mass_before;
#pragma unroll
      for (int e = 0; e < RS_PER; ++e)
        if ((int)threadIdx.x * RS_PER + e < b) { k += bin_cnt[e]; m += bin_mass[e]; }
      s.sel_cnt = k;
      s.sel_base = m;
      uint32_t c = 0;
#pragma unroll
      for (int e = 0; e < RS_PER; ++e)
        if ((int)threadIdx.x * RS_PER + e == b) c = bin_cnt[e];
      s.sel_bin_cnt = b >= RS_BINS ? s.all_cnt - k : c;
    }
    __syncthreads();
    *before = s.sel_cnt; *mass = s.sel_base; *in = s.sel_bin_cnt;
    __syncthreads();
  }

  // sorts the n first of the list
  __device__ void sort(int n_list) {
    int np2 = 2;
    while (np2 < n_list) np2 <<= 1;
    for (int i = n_list + threadIdx.x; i < np2; i += RS_THREADS) s.list[i] = ~0ull;
    __syncthreads();
    for (int size = 2; size <= np2; size <<= 1) {
      for (int step = size >> 1; step > 0; step >>= 1) {
        for (int i = threadIdx.x; i < np2 / 2; i += RS_THREADS) {
          const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
          const unsigned long long x = s.list[lo], y = s.list[hi];
          if ((x > y) == ((lo & size) == 0)) { s.list[lo] = y; s.list[hi] = x; }
        }
        __syncthreads();
      }
    }
  }
  __device__ float list_logit(int i) const { return rs_unorder(~(uint32_t)(s.list[i] >> 32)); }
  // weights of this thread's share of the sorted list and the mass before them
  __device__ double list_masses(int n_list, double (&w)[RS_EACH], double* total) {
    double loc = 0;
#pragma unroll
    for (int e = 0; e < RS_EACH; ++e) {
      const int i = threadIdx.x * RS_EACH + e;
      w[e] = i < n_list ? rs_weight(list_logit(i), g) : 0.0;
      loc += w[e];
    }
    return rs_scan<double>(loc, s.wsum, total);
  }
  // First of the list's first n tokens at which base + mass reaches the target (strict: exceeds it); n - 1 when none does.
  __device__ int list_cross(int n_list, const double (&w)[RS_EACH], double before, double target, bool strict) {
    if (threadIdx.x == 0) s.pick = n_list - 1;
    __syncthreads();
    double m = before;
#pragma unroll
    for (int e = 0; e < RS_EACH; ++e) {
      m += w[e];
      const int i = threadIdx.x * RS_EACH + e;
      if (i < n_list && (strict ? m > target : m >= target)) { atomicMin(&s.pick, i); break; }
    }
    __syncthreads();
    const int p = s.pick;
    __syncthreads();
    return p;
  }
  // mass of the list's tokens up to and with i
  __device__ double list_mass_at(int i, const double (&w)[RS_EACH], double before) {
    if ((int)threadIdx.x == i / RS_EACH) {
      double m = before;
#pragma unroll
      for (int e = 0; e < RS_EACH; ++e)
        if ((int)threadIdx.x * RS_EACH + e <= i) m += w[e];
      s.pick_mass = m;
    }
    __syncthreads();
    const double m = s.pick_mass;
    __syncthreads();
    return m;
  }

  // The first token in order at which the running count or mass reaches the target (strict: exceeds it): its index, its
  // weight, and the count and mass up to and with it.
  struct Pick { int idx; double w; uint32_t cnt; double mass; };
  __device__ Pick select(bool by_mass, double target, bool strict) {
    const int b = cross(by_mass, target, strict);
    uint32_t before, in;
    double base;
    at_bin(b, &before, &base, &in);
    Pick p;
    if (in <= RS_CAP) {
      RSCommand c{};
      c.op = RS_GATHER; c.b0 = c.b1 = b;
      command(c);
      const int n_list = (int)s.n_list;
      sort(n_list);
      double w[RS_EACH], total;
      const double m0 = list_masses(n_list, w, &total);
      const int i = by_mass ? list_cross(n_list, w, base + m0, target, strict)
                            : min(max((int)(target - before) - 1, 0), n_list - 1);
      p.mass = list_mass_at(i, w, base + m0);
      p.idx = (int)(uint32_t)s.list[i];
      p.w = rs_weight(list_logit(i), g);
      p.cnt = before + i + 1;
      __syncthreads();
      return p;
    }
    // crowded: digit by digit, masses in units of the bin edge's weight
    RSCommand c{};
    c.op = RS_RADIX; c.b0 = b;
    c.z0 = b < RS_BINS ? (double)b * (double)g.width / g.t : 0.0;
    const double unit = b < RS_BINS ? exp(-c.z0) : 0.0;
    double each = 0;   // of the tokens left: their weight / unit
    uint32_t left = 0;
    for (int round = 0; round < 4; ++round) {
      c.shift = 24 - 8 * round;
      command(c);
      // digits in descending order: thread t < 256 has digit 255 - t
      uint32_t k = 0;
      unsigned long long m = 0;
      const int d = 255 - (int)threadIdx.x;
      if (threadIdx.x < 256)
        for (int r = 0; r < RS_CLUSTER; ++r) {
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
      __syncthreads();
      if ((int)threadIdx.x == at) { s.sel_cnt = before + kb; s.sel_base = base + mb; s.sel_bin_cnt = k; s.pick_w = k ? mass / k : 0.0; }
      __syncthreads();
      before = s.sel_cnt; base = s.sel_base; left = s.sel_bin_cnt; each = s.pick_w;
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

  __device__ void answer(int row, int idx, double prob, uint32_t kept) {
    if (threadIdx.x == 0) {
      a.tokens[row] = idx;
      if (a.prob) a.prob[row] = (float)prob;
      if (a.kept) a.kept[row] = (int)kept;
    }
  }

  // the bins' masses once more, or at last
  __device__ void recollect(int room) {
    RSCommand c{};
    c.op = RS_MASSES; c.sure = room;
    command(c);
    collect(true);
  }

  __device__ void lead(int row, int k, double top_p, double min_p, double u, bool masses) {
    collect(masses);
    if (masses && s.most_cnt) recollect((int)s.most_cnt);
    const uint32_t all = s.all_cnt;
    const bool cut_k = k > 0 && (uint32_t)k < all;
    const uint32_t cut = cut_k ? (uint32_t)k : all;
    const bool by_p = top_p < 1, by_m = min_p > 0;
    const bool listed = cut_k || !masses;  // the mass that top-p goes by is that of tokens that are all in the list
    // the last bin that a kept token can lie in
    int last = RS_BINS;
    if (cut_k) last = cross(false, (double)k, false);
    if (by_m && !(listed && by_p)) {
      const double x = -log(min_p) * g.t * (double)g.sx;
      last = min(last, x < RS_BINS ? (int)fmax(x, 0.0) + 1 : RS_BINS);
    }
    if (by_p && !listed) last = min(last, cross(true, top_p * s.all_mass, false));
    uint32_t before, in;
    double base;
    at_bin(last, &before, &base, &in);
    if (before + in <= RS_CAP) {
      RSCommand c{};
      c.op = RS_GATHER; c.b1 = last;
      command(c);
      const int n_list = (int)s.n_list;
      sort(n_list);
      double w[RS_EACH], total;
      const double m0 = list_masses(n_list, w, &total);
      int kept = (int)min(cut, (uint32_t)n_list);
      if (by_p) {
        // mass of the cut: of the list's first k, or of the list and the bins behind it
        const double mass = listed ? list_mass_at(kept - 1, w, m0) : total + (s.all_mass - base - bin_mass_of(last));
        kept = min(kept, list_cross(kept, w, m0, top_p * mass, false) + 1);
      }
      if (by_m) {
        uint32_t ok = 0, all_ok;
#pragma unroll
        for (int e = 0; e < RS_EACH; ++e) ok += (int)threadIdx.x * RS_EACH + e < n_list && w[e] >= min_p;
        rs_scan<uint32_t>(ok, s.wcnt, &all_ok);
        kept = min(kept, max((int)all_ok, 1));
      }
      const double mass = list_mass_at(kept - 1, w, m0);
      const int i = list_cross(kept, w, m0, u * mass, true);
      answer(row, (int)(uint32_t)s.list[i], rs_weight(list_logit(i), g) / mass, (uint32_t)kept);
      return;
    }
    // long prefixes: each end by itself
    if (!masses) {  // the k-th token's bin is crowded
      recollect((int)max(s.most_cnt, (uint32_t)RS_SURE));
    }
    uint32_t kept = cut;
    double mass = s.all_mass;
    if (cut_k) mass = select(false, (double)k, false).mass;
    if (by_p) {
      const Pick p = select(true, top_p * mass, false);
      if (p.cnt < kept) { kept = p.cnt; mass = p.mass; }
    }
    if (by_m) {
      const double x = -log(min_p) * g.t * (double)g.sx;
      const int b = x < RS_BINS ? (int)fmax(x, 0.0) : RS_BINS;
      RSCommand c{};
      c.op = RS_OVER; c.b0 = b - 1; c.b1 = min(b + 1, RS_BINS);
      command(c);
      const uint32_t over = max(s.over, 1u);
      __syncthreads();
      if (over < kept) { kept = over; mass = select(false, (double)over, false).mass; }
    }
    Pick p = select(true, u * mass, true);
    if (p.cnt > kept) p = select(false, (double)kept, false);  // the two sums of a bin differ by a rounding
    answer(row, p.idx, p.w / mass, kept);
  }
  __device__ double bin_mass_of(int b) {
    if (threadIdx.x == 0) s.pick_mass = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < RS_PER; ++e)
      if ((int)threadIdx.x * RS_PER + e == b) s.pick_mass = bin_mass[e];
    __syncthreads();
    const double m = s.pick_mass;
    __syncthreads();
    return m;
  }
};

template <bool STAGED>
__global__ void __launch_bounds__(RS_THREADS, 2) sample_rows_kernel(const RSArgs a) {
  extern __shared__ __align__(16) uint8_t rs_raw[];
  RSSmem& s = *reinterpret_cast<RSSmem*>(rs_raw);
  float* stage = reinterpret_cast<float*>(rs_raw + sizeof(RSSmem));
  cg::cluster_group cl = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cl.block_rank();
  const int row = (int)(blockIdx.x / RS_CLUSTER);
  const int i0 = min(rank * a.per, a.vocab), n = min(a.per, a.vocab - i0);
  RSRow<STAGED> r{s, stage, a, (int64_t)row * a.ld, i0, n, RSGeom{}, cl, 0.0, RS_SURE};

  // 1. this CTA's logits, the largest with its index, the smallest that is a number
  RSStat st{-INFINITY, INFINITY, 0x7fffffff, 0};
  auto see = [&](int i, float l) {
    if (l > st.mx) { st.mx = l; st.idx = i0 + i; }
    if (l > -INFINITY) st.mn = fminf(st.mn, l);
    if (STAGED) stage[i] = l;
  };
  if (a.vec) {  // 16 bytes a lane; the shares are multiples of 8 logits
    const int v = a.dtype == N730_F32 ? 4 : 8, nv = n / v;
    const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.logits) +
                                                    (r.base + i0) * (a.dtype == N730_F32 ? 4 : 2));
    constexpr int U = 4;
    for (int j = tid; j < nv; j += U * RS_THREADS) {
      uint4 x[U];
#pragma unroll
      for (int e = 0; e < U; ++e)
        if (j + e * RS_THREADS < nv) x[e] = ld_stream_v4(p + j + e * RS_THREADS);
#pragma unroll
      for (int e = 0; e < U; ++e) {
        const int i = (j + e * RS_THREADS) * v;
        if (j + e * RS_THREADS >= nv) break;
        const uint32_t y[4] = {x[e].x, x[e].y, x[e].z, x[e].w};
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          if (a.dtype == N730_F32) {
            see(i + h, rs_clean(__uint_as_float(y[h])));
          } else {
            const float2 f = a.dtype == N730_F16 ? __half22float2(*reinterpret_cast<const __half2*>(&y[h]))
                                                 : make_float2(__uint_as_float(y[h] << 16), __uint_as_float(y[h] & 0xffff0000u));
            see(i + 2 * h, rs_clean(f.x));
            see(i + 2 * h + 1, rs_clean(f.y));
          }
        }
      }
    }
    for (int i = nv * v + tid; i < n; i += RS_THREADS) see(i, rs_clean(kv8_load1(a.logits, r.base + i0 + i, a.dtype)));
  } else {
    for (int i = tid; i < n; i += RS_THREADS) see(i, rs_clean(kv8_load1(a.logits, r.base + i0 + i, a.dtype)));
  }
  auto join = [](RSStat& x, const RSStat& y) {
    if (y.mx > x.mx || (y.mx == x.mx && y.idx < x.idx)) { x.mx = y.mx; x.idx = y.idx; }
    x.mn = fminf(x.mn, y.mn);
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    RSStat y;
    y.mx = __shfl_xor_sync(0xffffffffu, st.mx, o);
    y.mn = __shfl_xor_sync(0xffffffffu, st.mn, o);
    y.idx = __shfl_xor_sync(0xffffffffu, st.idx, o);
    join(st, y);
  }
  if (lane == 0) s.wstat[warp] = st;
  for (int i = tid; i < RS_BINS + 4; i += RS_THREADS) { s.cnt[i] = 0; s.dev[i] = 0; }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < RS_WARPS; ++w) join(st, s.wstat[w]);
    s.stat = st;
  }
  cl.sync();
  st = cl.map_shared_rank(&s, 0)->stat;
  for (int k = 1; k < RS_CLUSTER; ++k) join(st, cl.map_shared_rank(&s, k)->stat);
  const float t = a.temperature ? a.temperature[row] : 1.f;
  if (st.mx == -INFINITY || !(t > 0.f)) {  // no token, or greedy
    if (rank == 0) r.answer(row, st.mx == -INFINITY ? -1 : st.idx, st.mx == -INFINITY ? 0.0 : 1.0, st.mx == -INFINITY ? 0u : 1u);
    cl.sync();  // the others may still read this CTA's statistics
    return;
  }
  const int k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 1.f, q = a.min_p ? a.min_p[row] : 0.f, un = a.u[row];
  const bool masses = !(k > 0 && k <= RS_CAP / 2);

  // 2. the bins
  RSGeom& g = r.g;
  g.mx = st.mx;
  const float tc = fminf(fmaxf(t, 0x1p-100f), 0x1p100f);
  g.t = tc;
  g.inv_t = 1.f / tc;
  // a little more than the row's spread: the smallest logit lies in the last bin, not behind it
  const float span = fminf((st.mx - st.mn) * (1.f + 0x1p-20f), RS_SPAN * fmaxf(tc, 1.f));
  g.sx = span > 1e-30f ? (float)RS_BINS / span : 0.f;
  g.width = span > 1e-30f ? span / (float)RS_BINS : 0.f;
  r.zmin = q > 0.f ? log((double)q) : -INFINITY;
  r.fill(true, masses);
  cl.sync();

  // 3. ends of the prefixes and the token
  if (rank == 0) {
    const double up = un > 0.f ? fmin((double)un, 1.0) : 0.0;
    r.lead(row, k, p < 1.f ? (double)p : 1.0, q > 0.f ? (double)q : 0.0, up, masses);
    __syncthreads();
    if (tid == 0) s.cmd.op = RS_DONE;
    cl.sync();
  } else {
    for (;;) {
      cl.sync();
      const RSCommand c = cl.map_shared_rank(&s, 0)->cmd;
      if (c.op == RS_DONE) break;
      r.serve(c);
      cl.sync();
    }
  }
  cl.sync();  // no CTA leaves while another reads its shared memory
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
  a.logits = d_logits; a.ld = ld; a.vocab = vocab; a.dtype = dtype;
  a.per = ((vocab + RS_CLUSTER - 1) / RS_CLUSTER + 7) / 8 * 8;
  a.vec = ((uintptr_t)d_logits & 15) == 0 && ld * es % 16 == 0;
  a.temperature = d_temperature; a.top_k = d_top_k; a.top_p = d_top_p; a.min_p = d_min_p; a.u = d_u;
  a.tokens = d_tokens; a.prob = d_prob; a.kept = d_kept;
  const size_t slice = (size_t)a.per * 4;
  const bool staged = slice <= RS_STAGE_MAX;
  const dim3 grid((unsigned)batch * RS_CLUSTER), block(RS_THREADS);
  if (staged) {
    if (int rc = smem_attr_once<sample_rows_kernel<true>>((int)(sizeof(RSSmem) + RS_STAGE_MAX))) return rc;
    return kv8_launch_cluster(sample_rows_kernel<true>, grid, RS_CLUSTER, block, sizeof(RSSmem) + slice, (cudaStream_t)stream, false, a);
  }
  return kv8_launch_cluster(sample_rows_kernel<false>, grid, RS_CLUSTER, block, sizeof(RSSmem), (cudaStream_t)stream, false, a);
}
