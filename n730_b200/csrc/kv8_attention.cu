// Attention over the 8-bit paged key/value cache.
//
//   out[b, t, head] = softmax_p(scale q . k_p) v_p,  positions p <= lens[b] + t of KV head head / G
//
// Split kernel (single tokens and few rows).  The rows of an item (sequence, KV head) are its
// tokens x G query heads, up to RG = 16 at a time (8 for fp32 queries).  All items' 16-position
// tiles form one line that the CTAs cut into equal runs, so ragged lengths and few sequences load
// every SM alike; a run that covers part of an item leaves its (max, sum, output) in the workspace,
// and the last CTA to finish an item joins the parts in run order (the result does not depend on
// which CTA that is).  Within a CTA each warp takes every fourth tile.
//
// A lane copies into shared memory, with cp.async, exactly the bytes that it later feeds to the
// tensor cores, so tiles need no CTA barrier and no transposition through shared memory:
//   K: S = Q K^T by mma.m16n8k16.  The order of the channels in the sum is free, so lane (g, t)
//      reads 16 contiguous bytes of row g's key and each 4 of them are one k-step's slots.
//   V: the order of the keys is free too.  Lane (g, t) owns keys 4t..4t+3 in both products: P
//      passes from the accumulators of the first to the operand of the second in registers, and V
//      needs 16 contiguous channels of those four keys, interleaved by byte permutes.
// int8 codes become fp16 exactly (1024 + 128 + q by a byte permute, then one subtraction), e4m3
// codes by a conversion; K's scale multiplies the scores, V's scale goes into the exponent.
//
// Numerics.  Queries are scaled by a power of two per row so that a 16-bit query is exact in fp16;
// an fp32 query is split into two fp16 terms that fill rows 0-7 and 8-15 of the same product, and
// so is P: fp32 calls lose about 2^-22.  For 16-bit calls P is rounded to fp16 (2^-11 of each weight,
// below the rounding of the output).  Maxima, sums and outputs are fp32.
#include <algorithm>

#include "kv8.h"

namespace n730 {

constexpr int KD_WARPS = 4;
constexpr int KD_THREADS = KD_WARPS * 32;
constexpr int KD_STAGES = 4;
constexpr int KD_TILE = 16;
constexpr int KD_CTAS_PER_SM = 3;
constexpr int KD_MIN_UNITS = 8;  // tiles of a run: fewer would leave warps idle and joins to do
constexpr int KD_MAX_BATCH = 4096;

struct KDArgs {
  N730KV8Cache c;
  const void* q; void* out;
  int64_t ldq, ldo;
  int dtype, batch, tokens, heads, group, rows, nrg;  // rows = tokens * group; nrg row groups of RG
  float scale_log2e;
  const int* lens; const int* n_new;
  unsigned* cnt;       // [batch][n_kv][nrg] arrivals, zero between calls
  float* part;         // [2 * n_cta][RG][HD]
  float* part_ml;      // [2 * n_cta][RG][4]: reference of the output, max, sum
  float* lse;          // [batch][n_kv][rows] log2 of the softmax sum, +inf for an empty row (weights only)
  float* scores;       // [batch][n_kv][rows][cap] base-2 scores (weights only)
  int n_cta, log_block;
};

template <int HD>
struct KDGeom {
  static constexpr int KCH = HD / 64;                 // 16-byte K chunks per lane and 8 keys
  static constexpr int VB = HD / 8;                   // V bytes per lane and key
  static constexpr int K_BYTES = 2 * KCH * 512;       // per tile
  static constexpr int TILE_BYTES = K_BYTES + 4 * VB * 32;
  static constexpr int OSTRIDE = HD + 8;              // padded output row (bank spread)
};

template <int HD>
struct KDSmem {
  uint8_t ring[KD_WARPS][KD_STAGES][KDGeom<HD>::TILE_BYTES];
  uint4 qf[HD / 16][32];           // Q as the A operand, by k-step and lane
  float sc[KD_WARPS][KD_STAGES][2];
  int ok[KD_WARPS][KD_STAGES];
  float rowmul[16];
  float wm[KD_WARPS][16], wmo[KD_WARPS][16], wl[KD_WARPS][16];
  float tot[16][4];
  int flag;
  int pre[1];                      // [batch + 1] prefix sums of the sequences' tiles
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) { return h2_bits(__floats2half2_rn(lo, hi)); }
__device__ __forceinline__ void mma16816(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool pred) {
  if (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(pred ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" :: "r"(dst), "l"(src), "n"(BYTES), "r"(pred ? BYTES : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

// two codes (the bytes of x selected by SEL: low or high pair) as fp16
template <int CODE, int HIGH>
__device__ __forceinline__ uint32_t codes2(uint32_t x) {
  if (CODE == N730_KV8_INT8) {  // x has its sign bits flipped: bytes 128 + q
    const uint32_t y = __byte_perm(x, 0x64646464u, HIGH ? 0x4342 : 0x4140);
    return h2_bits(__hsub2(*reinterpret_cast<const __half2*>(&y), __float2half2_rn(1152.f)));
  }
  uint32_t y;
  asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, %2;\n}"
      : "=r"(y) : "r"(x), "h"((uint16_t)(HIGH ? x >> 16 : x)));
  return y;
}
template <int CODE>
__device__ __forceinline__ uint32_t code_word(uint32_t x) { return CODE == N730_KV8_INT8 ? x ^ 0x80808080u : x; }

// tiles of sequence b: at least one when it has new rows (they need an answer)
__device__ __forceinline__ int kd_units(const KDArgs& a, int b, int cap) {
  const int n = kv8_new(a.n_new, b, a.tokens);
  if (n == 0) return 0;
  const int tot = (int)min((int64_t)kv8_len(a.lens, b, cap) + n, (int64_t)cap);
  return (tot + KD_TILE - 1) / KD_TILE;
}

// HL: fp32 queries, 8 rows as high and low fp16 halves; else 16 rows.
template <int HD, int CODE, bool HL>
__global__ void __launch_bounds__(KD_THREADS, KD_CTAS_PER_SM) kv8_split_kernel(const KDArgs a) {
  using G = KDGeom<HD>;
  constexpr int RG = HL ? 8 : 16, NT = HD / 8, ST = KD_STAGES;
  extern __shared__ __align__(128) uint8_t kd_raw[];
  KDSmem<HD>& sm = *reinterpret_cast<KDSmem<HD>*>(kd_raw);
  static_assert(sizeof(float) * KD_WARPS * RG * G::OSTRIDE <= sizeof(sm.ring), "per-warp outputs fit the ring");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const N730KV8Cache& c = a.c;
  const int cap = c.max_pages * c.page_size;
  pdl_wait();

  // ---- prefix sums of the sequences' tiles ----
  if (warp == 0) {
    int run = 0;
    if (lane == 0) sm.pre[0] = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      int v = b0 + lane < a.batch ? kd_units(a, b0 + lane, cap) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
      }
      if (b0 + lane < a.batch) sm.pre[b0 + lane + 1] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  const int items = c.n_kv * a.nrg;  // per sequence
  const int64_t U = (int64_t)sm.pre[a.batch] * items;
  const int64_t N = min((int64_t)a.n_cta, (U + KD_MIN_UNITS - 1) / KD_MIN_UNITS);
  const int cta = blockIdx.x;
  if (cta >= N) return;
  int64_t u = U * cta / N;
  const int64_t u1 = U * (cta + 1) / N;
  int b = 0;
  {
    int lo = 0, hi = a.batch - 1;  // the last b with pre[b] * items <= u
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((int64_t)sm.pre[mid] * items <= u) lo = mid; else hi = mid - 1;
    }
    b = lo;
  }

  while (u < u1) {
    while ((int64_t)sm.pre[b + 1] * items <= u) ++b;  // past sequences without tiles
    const int units = sm.pre[b + 1] - sm.pre[b];
    const int64_t ub = u - (int64_t)sm.pre[b] * items;
    const int item = (int)(ub / units), ta = (int)(ub % units), te = (int)min((int64_t)units, ta + (u1 - u));
    u += te - ta;
    const int h = item / a.nrg, rg = item % a.nrg;
    const int L = kv8_len(a.lens, b, cap), n_new = kv8_new(a.n_new, b, a.tokens);
    const int rows_b = n_new * a.group, f0 = rg * RG;
    if (f0 >= rows_b) continue;  // a row group behind this sequence's new rows
    const int nrow = min(RG, rows_b - f0);
    const int total = (int)min((int64_t)L + n_new, (int64_t)cap);  // positions cached with the new rows

    __syncthreads();  // shared memory of the previous run is free
    // ---- the warp's tiles ----
    const int n_tile = te - ta > warp ? (te - ta - warp + KD_WARPS - 1) / KD_WARPS : 0;
    const int* bt = c.block_table + (int64_t)b * c.max_pages;
    // pool row of tile q0 + lane of this warp (-1: no page), looked up 32 tiles at a time
    auto lookup = [&](int q0) {
      const int qi = q0 + lane;
      if (qi >= n_tile) return -1;
      const int p = (ta + warp + qi * KD_WARPS) * KD_TILE;
      const int page = bt[p / c.page_size];
      return (unsigned)page < (unsigned)c.n_pages ? (page * c.n_kv + h) * c.page_size + p % c.page_size : -1;
    };
    int rows_now = lookup(0), rows_next = lookup(32);
    const uint32_t ring = smem_u32(sm.ring[warp]);
    auto issue = [&](int qi) {
      const int st = qi % ST;
      if (qi && (qi & 31) == 0) { rows_now = rows_next; rows_next = lookup(qi + 32); }
      const int row = __shfl_sync(0xffffffffu, rows_now, qi & 31);
      const bool ok = row >= 0;
      const int64_t r0 = ok ? row : 0;
      const uint32_t dst = ring + st * G::TILE_BYTES + lane * 16;
      const uint8_t* kc = reinterpret_cast<const uint8_t*>(c.k_codes) + r0 * HD;
      const uint8_t* vc = reinterpret_cast<const uint8_t*>(c.v_codes) + r0 * HD;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < G::KCH; ++j)
          cp_async<16>(dst + (i * G::KCH + j) * 512, kc + (4 * (g >> 1) + 2 * i + (g & 1)) * HD + j * 64 + t4 * 16, ok);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        cp_async<G::VB>(ring + st * G::TILE_BYTES + G::K_BYTES + i * 32 * G::VB + lane * G::VB,
                        vc + (4 * t4 + i) * HD + g * G::VB, ok);
      if (lane < 2) {
        const float* s = (lane ? c.v_scales : c.k_scales) + (r0 >> a.log_block);
        cp_async<4>(smem_u32(&sm.sc[warp][st][lane]), s, ok);
      }
      if (lane == 0) sm.ok[warp][st] = ok;
    };
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) {
      if (s < n_tile) issue(s);
      cp_commit();
    }

    // ---- Q: a row per warp at a time, scaled by a power of two, as the A operand ----
    for (int r = warp; r < RG; r += KD_WARPS) {
      constexpr int E = HD / 32;  // channels a lane
      float x[E];
      float m = 0.f;
      const int f = f0 + r;
      const int64_t qb = r < nrow ? ((int64_t)b * a.tokens + f / a.group) * a.ldq + (int64_t)(h * a.group + f % a.group) * HD : 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[e] = r < nrow ? kv8_load1(a.q, qb + lane * E + e, a.dtype) : 0.f;
        m = fmaxf(m, fabsf(x[e]));
      }
      m = warp_max(m);
      // the largest magnitude goes into [2^13, 2^14); rows of zeros or with an infinity stay
      const int ex = (int)((__float_as_uint(m) >> 23) & 255u);
      const bool plain = ex == 0 || ex == 255;
      const int sh = plain ? 0 : min(max(140 - ex, -126), 126);
      const float mul = __uint_as_float((uint32_t)(127 + sh) << 23);
      if (lane == 0) sm.rowmul[r] = a.scale_log2e * __uint_as_float((uint32_t)(127 - sh) << 23);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int dch = lane * E + e, ks = (dch >> 6) * 4 + ((dch >> 2) & 3), tt = (dch >> 4) & 3, w = dch & 3;
        __half* slot = reinterpret_cast<__half*>(&sm.qf[ks][(r & 7) * 4 + tt]);  // a0, a1, a2, a3 as 8 halves
        const float y = x[e] * mul;
        const __half hi = __float2half_rn(y);
        const int at = (w >> 1) * 4 + (w & 1);  // a0 or a2
        if (HL) {
          slot[at] = hi;
          slot[at + 2] = __float2half_rn(y - __half2float(hi));  // an infinite y gives NaN, as it should
        } else {
          slot[at + (r >> 3) * 2] = hi;
        }
      }
    }
    __syncthreads();
    float rm[2];
    int vis[2];  // positions below vis are seen by the row
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = g + 8 * i;
      const bool live = r < nrow;  // HL: row 1 of the lane is the low half of row 0
      rm[i] = live ? sm.rowmul[HL ? g : r] : 0.f;
      vis[i] = live ? (int)min((int64_t)L + (f0 + r) / a.group + 1, (int64_t)cap) : 0;
    }
    const int all_see = (int)min((int64_t)L + f0 / a.group + 1, (int64_t)cap);  // positions every row sees

    float o[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    constexpr int NR = HL ? 1 : 2;  // rows a lane answers for
    float m_run[NR], mo_run[NR], l_run[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) { m_run[i] = mo_run[i] = -INFINITY; l_run[i] = 0.f; }

    for (int qi = 0; qi < n_tile; ++qi) {
      cp_wait<ST - 2>();
      __syncwarp();
      const int st = qi % ST;
      const uint8_t* kt = sm.ring[warp][st];
      const uint8_t* vt = kt + G::K_BYTES;
      const float ksc = sm.sc[warp][st][0], vsc = sm.sc[warp][st][1];
      const bool tile_ok = sm.ok[warp][st];
      const int p0 = (ta + warp + qi * KD_WARPS) * KD_TILE;

      // ---- S = Q K^T ----
      float s[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
      for (int j = 0; j < G::KCH; ++j) {
        const uint4 k0 = *reinterpret_cast<const uint4*>(kt + j * 512 + lane * 16);
        const uint4 k1 = *reinterpret_cast<const uint4*>(kt + (G::KCH + j) * 512 + lane * 16);
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint4 qa = sm.qf[j * 4 + e][lane];
          const uint32_t x0 = code_word<CODE>(w0[e]), x1 = code_word<CODE>(w1[e]);
          mma16816(s[0], qa, codes2<CODE, 0>(x0), codes2<CODE, 1>(x0));
          mma16816(s[1], qa, codes2<CODE, 0>(x1), codes2<CODE, 1>(x1));
        }
      }
      // ---- base-2 scores x of keys p0 + 4 t4 + 0..3 ----
      float x[NR][4];
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const float f = rm[i] * ksc;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float raw = HL ? s[e >> 1][e & 1] + s[e >> 1][2 + (e & 1)] : s[e >> 1][2 * i + (e & 1)];
          x[i][e] = raw * f;
        }
      }
      if (p0 + KD_TILE > all_see || !tile_ok) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (p0 + 4 * t4 + e >= vis[i] || !tile_ok) x[i][e] = -INFINITY;
      }
      if (a.scores) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
          if (g + 8 * i < nrow)
            *reinterpret_cast<float4*>(a.scores + (((int64_t)b * c.n_kv + h) * a.rows + f0 + g + 8 * i) * cap + p0 + 4 * t4) =
                make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
      }
      // ---- online softmax: sums against m_run, weights times V's scale against mo_run ----
      const float lv = lg2(vsc);
      float w[NR][4];
      bool grew = false;
      float al[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        float mt = fmaxf(fmaxf(x[i][0], x[i][1]), fmaxf(x[i][2], x[i][3]));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
        const float mn = fmaxf(m_run[i], mt), ms = mn == -INFINITY ? 0.f : mn;
        float ps = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) ps += ex2(x[i][e] - ms);
        l_run[i] = l_run[i] * ex2(m_run[i] - ms) + ps;
        m_run[i] = mn;
        const float mo = fmaxf(mo_run[i], mt + lv), mos = mo == -INFINITY ? 0.f : mo;
        al[i] = ex2(mo_run[i] - mos);
        grew |= mo > mo_run[i];
        mo_run[i] = mo;
        const float off = lv - mos;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[i][e] = ex2(x[i][e] + off);
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          o[n][0] *= al[0]; o[n][1] *= al[0];
          o[n][2] *= al[NR - 1]; o[n][3] *= al[NR - 1];
        }
      }
      uint4 pa;  // a0, a1: keys 4 t4, 4 t4 + 1 of rows g, g + 8; a2, a3: keys 4 t4 + 2, + 3
      if (HL) {
        pa.x = pack_h2(w[0][0], w[0][1]);
        pa.z = pack_h2(w[0][2], w[0][3]);
        const float2 f0h = __half22float2(*reinterpret_cast<__half2*>(&pa.x)), f1h = __half22float2(*reinterpret_cast<__half2*>(&pa.z));
        pa.y = pack_h2(w[0][0] - f0h.x, w[0][1] - f0h.y);
        pa.w = pack_h2(w[0][2] - f1h.x, w[0][3] - f1h.y);
      } else {
        pa.x = pack_h2(w[0][0], w[0][1]); pa.y = pack_h2(w[NR - 1][0], w[NR - 1][1]);
        pa.z = pack_h2(w[0][2], w[0][3]); pa.w = pack_h2(w[NR - 1][2], w[NR - 1][3]);
      }
      // ---- O += P V ----
      constexpr int VW = G::VB / 4;  // words a key
      uint32_t v[4][VW];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* src = vt + i * 32 * G::VB + lane * G::VB;
        if (VW == 4) {
          const uint4 y = *reinterpret_cast<const uint4*>(src);
          v[i][0] = y.x; v[i][1] = y.y; v[i][VW - 2] = y.z; v[i][VW - 1] = y.w;
        } else {
          const uint2 y = *reinterpret_cast<const uint2*>(src);
          v[i][0] = y.x; v[i][1] = y.y;
        }
        if (p0 + KD_TILE > total && p0 + 4 * t4 + i >= total) {  // rows never written may hold NaN codes
#pragma unroll
          for (int k = 0; k < VW; ++k) v[i][k] = 0u;
        }
      }
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        const uint32_t v0 = code_word<CODE>(v[0][k]), v1 = code_word<CODE>(v[1][k]);
        const uint32_t v2 = code_word<CODE>(v[2][k]), v3 = code_word<CODE>(v[3][k]);
        const uint32_t a01 = __byte_perm(v0, v1, 0x5140), b01 = __byte_perm(v0, v1, 0x7362);
        const uint32_t a23 = __byte_perm(v2, v3, 0x5140), b23 = __byte_perm(v2, v3, 0x7362);
        mma16816(o[4 * k + 0], pa, codes2<CODE, 0>(a01), codes2<CODE, 0>(a23));
        mma16816(o[4 * k + 1], pa, codes2<CODE, 1>(a01), codes2<CODE, 1>(a23));
        mma16816(o[4 * k + 2], pa, codes2<CODE, 0>(b01), codes2<CODE, 0>(b23));
        mma16816(o[4 * k + 3], pa, codes2<CODE, 1>(b01), codes2<CODE, 1>(b23));
      }
      __syncwarp();  // every lane is done with the buffer that the next copies go to
      if (qi + ST - 1 < n_tile) issue(qi + ST - 1);
      cp_commit();
    }
    cp_wait<0>();

    // ---- join the warps ----
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 1);
      l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 2);
      if (t4 == 0) {
        sm.wm[warp][g + 8 * i] = m_run[i];
        sm.wmo[warp][g + 8 * i] = mo_run[i];
        sm.wl[warp][g + 8 * i] = l_run[i];
      }
    }
    __syncthreads();  // all tiles are read: the ring takes the outputs
    float* wo = reinterpret_cast<float*>(&sm.ring[0][0][0]);  // [warp][row][OSTRIDE], channel n VB + u at u * 8 + n
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float* d0 = wo + (warp * RG + g) * G::OSTRIDE + n * 8 + 2 * t4;
      if (HL) {
        *reinterpret_cast<float2*>(d0) = make_float2(o[n][0] + o[n][2], o[n][1] + o[n][3]);
      } else {
        *reinterpret_cast<float2*>(d0) = make_float2(o[n][0], o[n][1]);
        *reinterpret_cast<float2*>(d0 + 8 * G::OSTRIDE) = make_float2(o[n][2], o[n][3]);
      }
    }
    __syncthreads();
    const bool whole = ta == 0 && te == units;
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
      if (!whole && tid < nrow) {
        float* ml = a.part_ml + ((int64_t)slot * RG + tid) * 4;
        ml[0] = Mo; ml[1] = M; ml[2] = l;
      }
    }
    __syncthreads();
    const int64_t ob = (int64_t)b * a.tokens;
    auto finish = [&](int r, int d, float num) {  // the answer of row r, channel d
      const float Mo = sm.tot[r][0], M = sm.tot[r][1], l = sm.tot[r][2];
      const float y = l == 0.f ? 0.f : num * (Mo == -INFINITY ? 0.f : ex2(Mo - M)) / l;  // a NaN query: NaN
      const int f = f0 + r;
      kv8_store1(a.out, (ob + f / a.group) * a.ldo + (int64_t)(h * a.group + f % a.group) * HD + d, a.dtype, y);
    };
    auto store_lse = [&]() {
      if (a.lse && tid < nrow)
        a.lse[((int64_t)b * c.n_kv + h) * a.rows + f0 + tid] =
            sm.tot[tid][2] == 0.f ? INFINITY : sm.tot[tid][1] + lg2(sm.tot[tid][2]);
    };
    for (int i = tid; i < nrow * HD; i += KD_THREADS) {
      const int r = i / HD, d = i % HD, at = (d % G::VB) * 8 + d / G::VB;
      float num = 0.f;
#pragma unroll
      for (int k = 0; k < KD_WARPS; ++k) num = fmaf(wo[(k * RG + r) * G::OSTRIDE + at], sm.wmo[k][r], num);
      if (whole) finish(r, d, num);
      else a.part[((int64_t)slot * RG + r) * HD + d] = num;
    }
    if (whole) {
      store_lse();
      continue;
    }
    // ---- parts: the last CTA of the item joins them ----
    const int64_t i0 = (int64_t)sm.pre[b] * items + (int64_t)item * units;  // the item's first tile on the line
    const int c0 = (int)(((i0 + 1) * N - 1) / U), c1 = (int)(((i0 + units) * N - 1) / U), parts = c1 - c0 + 1;
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      unsigned* cnt = a.cnt + ((int64_t)b * c.n_kv + h) * a.nrg + rg;
      sm.flag = atomicInc(cnt, (unsigned)(parts - 1)) == (unsigned)(parts - 1);  // wraps to 0: ready for the next call
    }
    __syncthreads();
    if (!sm.flag) continue;
    __threadfence();
    float* wts = wo;  // [row][part]
    for (int r = warp; r < nrow; r += KD_WARPS) {
      auto ml = [&](int k, int j) { return __ldcg(a.part_ml + ((int64_t)(2 * (c0 + k) + (k == 0)) * RG + r) * 4 + j); };
      float M = -INFINITY, Mo = -INFINITY, l = 0.f;
      for (int k = lane; k < parts; k += 32) { Mo = fmaxf(Mo, ml(k, 0)); M = fmaxf(M, ml(k, 1)); }
      M = warp_max(M);
      Mo = warp_max(Mo);
      const float ms = M == -INFINITY ? 0.f : M, mos = Mo == -INFINITY ? 0.f : Mo;
      for (int k = lane; k < parts; k += 32) {
        l += ml(k, 2) * ex2(ml(k, 1) - ms);
        wts[r * parts + k] = ex2(ml(k, 0) - mos);
      }
      l = warp_sum(l);
      if (lane == 0) { sm.tot[r][0] = Mo; sm.tot[r][1] = M; sm.tot[r][2] = l; }
    }
    __syncthreads();
    for (int i = tid; i < nrow * HD; i += KD_THREADS) {
      const int r = i / HD, d = i % HD;
      float num = 0.f;
#pragma unroll 8
      for (int k = 0; k < parts; ++k)
        num = fmaf(__ldcg(a.part + ((int64_t)(2 * (c0 + k) + (k == 0)) * RG + r) * HD + d), wts[r * parts + k], num);
      finish(r, d, num);
    }
    store_lse();
  }
}

// ---------------------------------------------------------------------------
// accumulated weights: w[b, h, p] += sum over the KV head's rows of exp2(score - lse)
// ---------------------------------------------------------------------------
struct KWArgs {
  N730KV8Cache c;
  int batch, tokens, group, rows;
  const int* lens; const int* n_new;
  const float* scores; const float* lse;
  const float* w_in; float* w_out;
  int64_t ldw;
};

// A thread sums one position over the rows in row order.
__global__ void __launch_bounds__(128) kv8_weights_kernel(const KWArgs a) {
  pdl_wait();
  const N730KV8Cache& c = a.c;
  const int b = blockIdx.z, h = blockIdx.y;
  const int cap = c.max_pages * c.page_size;
  const int L = kv8_len(a.lens, b, cap), n = kv8_new(a.n_new, b, a.tokens);
  const int total = (int)min((int64_t)L + n, (int64_t)cap);
  const int p = blockIdx.x * 128 + threadIdx.x;
  if (p >= total) return;
  const int64_t head = (int64_t)b * c.n_kv + h;
  const float* s = a.scores + head * a.rows * cap + p;
  const float* lse = a.lse + head * a.rows;
  float sum = 0.f;
  for (int f = 0; f < n * a.group; ++f) sum += ex2(s[(int64_t)f * cap] - lse[f]);
  a.w_out[head * a.ldw + p] = (a.w_in && p < L ? a.w_in[head * a.ldw + p] : 0.f) + sum;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
struct KDPlan {
  int rg, nrg, n_cta;
  int64_t cnt, part, ml, lse, scores, bytes;  // offsets
};
static KDPlan kd_plan(const N730KV8Cache& c, int batch, int tokens, int heads, int dtype, bool weights) {
  KDPlan p{};
  const int64_t rows = (int64_t)tokens * (heads / c.n_kv);
  p.rg = dtype == N730_F32 ? 8 : 16;
  p.nrg = (int)((rows + p.rg - 1) / p.rg);
  p.n_cta = KD_CTAS_PER_SM * num_sms();
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  p.part = up((int64_t)batch * c.n_kv * p.nrg * 4);
  p.ml = p.part + up((int64_t)2 * p.n_cta * p.rg * c.head_dim * 4);
  p.lse = p.ml + up((int64_t)2 * p.n_cta * p.rg * 16);
  p.scores = p.lse + (weights ? up((int64_t)batch * c.n_kv * rows * 4) : 0);
  p.bytes = p.scores + (weights ? (int64_t)batch * c.n_kv * rows * c.max_pages * c.page_size * 4 : 0);
  return p;
}

static int kv8_attention_check(const N730KV8Cache* c, int batch, int tokens, int heads) {
  if (int rc = kv8_check(c, batch, "kv8_attention")) return rc;
  N730_REQUIRE(batch <= KD_MAX_BATCH, N730_BAD_ARG, "kv8_attention: batch %d", batch);
  N730_REQUIRE(tokens >= 1 && tokens <= (1 << 20), N730_BAD_ARG, "kv8_attention: tokens %d", tokens);
  N730_REQUIRE(heads >= 1 && heads <= 65535 && heads % c->n_kv == 0, N730_BAD_ARG,
               "kv8_attention: %d heads over %d KV heads", heads, c->n_kv);
  N730_REQUIRE((int64_t)tokens * (heads / c->n_kv) <= (1 << 23), N730_BAD_ARG,
               "kv8_attention: %d tokens of %d heads over %d KV heads", tokens, heads, c->n_kv);
  return N730_OK;
}

int64_t kv8_attention_ws(const N730KV8Cache& c, int batch, int tokens, int heads, bool weights) {
  // fp32 calls take more row groups, 16-bit calls larger parts
  return std::max(kd_plan(c, batch, tokens, heads, N730_F32, weights).bytes,
                  kd_plan(c, batch, tokens, heads, N730_F16, weights).bytes);
}

template <int HD, int CODE, bool HL>
static int split_launch(const KDArgs& a, bool pdl, cudaStream_t st) {
  const size_t smem = sizeof(KDSmem<HD>) + (size_t)a.batch * 4;
  if (int rc = smem_attr_once<kv8_split_kernel<HD, CODE, HL>>((int)(sizeof(KDSmem<HD>) + KD_MAX_BATCH * 4))) return rc;
  return kv8_launch(kv8_split_kernel<HD, CODE, HL>, dim3(a.n_cta), dim3(KD_THREADS), smem, st, pdl, a);
}

int kv8_attention_launch(const KV8AttnCall& k, cudaStream_t st) {
  const N730KV8Cache& c = k.c;
  const bool weights = k.w_out != nullptr;
  const KDPlan p = kd_plan(c, k.batch, k.tokens, k.heads, k.dtype, weights);
  uint8_t* ws = reinterpret_cast<uint8_t*>(k.ws);
  KDArgs a{};
  a.c = c;
  a.q = k.q; a.out = k.out; a.ldq = k.ldq; a.ldo = k.ldo; a.dtype = k.dtype;
  a.batch = k.batch; a.tokens = k.tokens; a.heads = k.heads; a.group = k.heads / c.n_kv;
  a.rows = k.tokens * a.group; a.nrg = p.nrg;
  a.scale_log2e = k.scale * 1.4426950408889634f;
  a.lens = k.lens; a.n_new = k.n_new;
  a.cnt = reinterpret_cast<unsigned*>(ws);
  a.part = reinterpret_cast<float*>(ws + p.part);
  a.part_ml = reinterpret_cast<float*>(ws + p.ml);
  a.lse = weights ? reinterpret_cast<float*>(ws + p.lse) : nullptr;
  a.scores = weights ? reinterpret_cast<float*>(ws + p.scores) : nullptr;
  a.n_cta = p.n_cta;
  a.log_block = c.block == 16 ? 4 : c.block == 32 ? 5 : 6;
  const bool hl = k.dtype == N730_F32;
  int rc;
#define N730_SPLIT(HD, CODE) (hl ? split_launch<HD, CODE, true>(a, k.pdl, st) : split_launch<HD, CODE, false>(a, k.pdl, st))
  if (c.head_dim == 128) rc = c.code == N730_KV8_INT8 ? N730_SPLIT(128, N730_KV8_INT8) : N730_SPLIT(128, N730_KV8_E4M3);
  else rc = c.code == N730_KV8_INT8 ? N730_SPLIT(64, N730_KV8_INT8) : N730_SPLIT(64, N730_KV8_E4M3);
#undef N730_SPLIT
  if (rc || !weights) return rc;
  KWArgs w{};
  w.c = c;
  w.batch = k.batch; w.tokens = k.tokens; w.group = a.group; w.rows = a.rows;
  w.lens = k.lens; w.n_new = k.n_new;
  w.scores = a.scores; w.lse = a.lse;
  w.w_in = k.w_in; w.w_out = k.w_out; w.ldw = k.ldw;
  const int cap = c.max_pages * c.page_size;
  return kv8_launch(kv8_weights_kernel, dim3((cap + 127) / 128, c.n_kv, k.batch), dim3(128), 0, st, true, w);
}

}  // namespace n730

using namespace n730;

N730_API int64_t n730_kv8_attention_ws(const N730KV8Cache* c, int batch, int tokens, int n_heads, int weights) {
  if (int rc = kv8_attention_check(c, batch, tokens, n_heads)) return rc;
  return kv8_attention_ws(*c, batch, tokens, n_heads, weights != 0);
}

N730_API int n730_kv8_attention(const N730KV8Cache* c, const void* d_q, int dtype, int64_t ldq, int batch, int tokens,
                                int n_heads, float scale, const int32_t* d_lens, const int32_t* d_new, void* d_out,
                                int64_t ldo, const float* d_w, float* d_w_out, int64_t ldw, void* d_ws,
                                int64_t ws_bytes, void* stream) {
  if (int rc = kv8_attention_check(c, batch, tokens, n_heads)) return rc;
  N730_REQUIRE(dtype == N730_F32 || dtype == N730_F16 || dtype == N730_BF16, N730_BAD_ARG, "kv8_attention: dtype %d", dtype);
  N730_REQUIRE(d_q && d_out && d_lens && d_ws, N730_NULL, "kv8_attention: null pointer");
  const int64_t row = (int64_t)n_heads * c->head_dim;
  N730_REQUIRE(ldq >= row && ldo >= row, N730_BAD_ARG, "kv8_attention: row strides %lld, %lld < %d heads x %d",
               (long long)ldq, (long long)ldo, n_heads, c->head_dim);
  N730_REQUIRE(!d_w || d_w_out, N730_BAD_ARG, "kv8_attention: weights in without weights out");
  N730_REQUIRE(!d_w_out || ldw >= (int64_t)c->max_pages * c->page_size, N730_BAD_ARG,
               "kv8_attention: row stride %lld of the weights is below the table's %lld positions", (long long)ldw,
               (long long)c->max_pages * c->page_size);
  N730_REQUIRE(scale == scale && scale - scale == 0.f, N730_BAD_ARG, "kv8_attention: scale %g", scale);
  N730_REQUIRE(ws_bytes >= kv8_attention_ws(*c, batch, tokens, n_heads, d_w_out != nullptr) && ((uintptr_t)d_ws & 15) == 0,
               N730_BAD_ARG, "kv8_attention: workspace of %lld bytes", (long long)ws_bytes);
  KV8AttnCall k{};
  k.c = *c;
  k.q = d_q; k.out = d_out; k.dtype = dtype; k.ldq = ldq; k.ldo = ldo;
  k.batch = batch; k.tokens = tokens; k.heads = n_heads; k.scale = scale;
  k.lens = d_lens; k.n_new = d_new;
  k.w_in = d_w; k.w_out = d_w_out; k.ldw = ldw;
  k.ws = d_ws; k.ws_bytes = ws_bytes;
  return kv8_attention_launch(k, (cudaStream_t)stream);
}
