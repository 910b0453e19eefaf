// Rotary positions, and rows written into the 16-bit paged key/value cache.
//
// A pair (x0, x1) of a head at position p becomes  f (x0 cos a - x1 sin a, x1 cos a + x0 sin a),  a = p * freq[i];
// pairs are (i, i + n/2) of the first n channels (half) or (2 i, 2 i + 1) (interleaved); the other channels stay.
// Scaling for long contexts is in the frequencies (n730_rotary_frequencies) and in f.
//
// Angles reach 2^31 radians, where fp32 knows nothing of the fraction of a turn: p * freq / 2 pi is formed in 64
// bits, whole turns are taken off there, and the rest, at most half a turn, goes to sincospif in 32.
//
// Bound by bytes: every element is read and written once.  A thread has one unit of a row (8 channels, or both runs of
// 8 that a half layout pairs) in up to 16 rows, so that what the unit is costs nothing a row; angles are computed once a
// row and pair, not once a head, in shared memory.  2048 rows of 28 fp32 heads x 128 take 11.5 us (5.1 TB/s), a
// prompt of 4133 rows of 36 fp16 heads x 128 18 us (4.2 TB/s), both partly from L2; the prompt from memory 23.
#include <cmath>

#include "kv16.h"

namespace n730 {

int kv16_check(const N730KV16Cache* c, int batch, const char* what) {
  N730_REQUIRE(c, N730_NULL, "%s: null cache", what);
  N730_REQUIRE(c->k && c->v && c->block_table, N730_NULL, "%s: null cache pointer", what);
  N730_REQUIRE(c->dtype == N730_F16 || c->dtype == N730_BF16, N730_BAD_ARG, "%s: cache of dtype %d", what, c->dtype);
  N730_REQUIRE(c->head_dim == 64 || c->head_dim == 128, N730_UNSUPPORTED, "%s: head_dim %d", what, c->head_dim);
  N730_REQUIRE(c->page_size > 0 && c->page_size % 16 == 0, N730_BAD_ARG, "%s: page_size %d is not a multiple of 16", what,
               c->page_size);
  N730_REQUIRE(c->n_kv >= 1 && c->n_kv <= 65535 && c->n_pages >= 1 && c->max_pages >= 1 && c->prefix_pages >= 0, N730_BAD_ARG,
               "%s: n_kv %d, n_pages %d, max_pages %d, prefix_pages %d", what, c->n_kv, c->n_pages, c->max_pages,
               c->prefix_pages);
  N730_REQUIRE(c->prefix_pages == 0 || (c->prefix_table && c->prefix_len), N730_NULL, "%s: null prefix", what);
  N730_REQUIRE((int64_t)c->n_pages * c->n_kv <= ((1ll << 31) - 1) / c->page_size, N730_BAD_ARG,
               "%s: the pool holds 2^31 or more rows", what);
  N730_REQUIRE((int64_t)c->max_pages * c->page_size <= (1ll << 29) && (int64_t)c->prefix_pages * c->page_size <= (1ll << 29),
               N730_BAD_ARG, "%s: a table's pages hold more than 2^29 positions", what);
  N730_REQUIRE((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0, N730_BAD_ARG, "%s: pools must be 16-byte aligned", what);
  N730_REQUIRE(kv8_aligned(4, c->block_table, c->prefix_table, c->prefix_len), N730_BAD_ARG,
               "%s: tables must lie on whole elements", what);
  N730_REQUIRE(batch >= 1 && batch <= 65535, N730_BAD_ARG, "%s: batch %d", what, batch);
  return N730_OK;
}

constexpr int RO_THREADS = 320;  // most threads of a CTA
constexpr int RO_ROWS = 16;      // most rows of a CTA
constexpr int RO_V = 8;          // channels of a vector unit
constexpr int64_t RO_TABLE = 40 * 1024;  // bytes of a CTA's cosines and sines

// One group of heads of a row: where it is read, and where it goes.
struct RotaryPart {
  const void* x; void* y;  // y null: into the cache's pool
  int64_t ldx, ldy;
  int heads;               // 0: none
  int pool;                // 0: k, 1: v
};
struct RotaryArgs {
  RotaryPart part[3];      // queries (or plain rows), keys, values
  const double* freq;
  const int* pos;
  float factor;
  int head_dim, rd;        // rd: rotated channels (0: none)
  int interleaved, dtype;
  int units_head, units_copy;  // units of a rotated head, of one that is copied
  int units, chunk;        // units of a row; those that a CTA takes
  int at_once, rows_cta;   // rows that a CTA works on side by side, and in all
  int rows, tokens, has_cache;
  FastDiv by_chunk, by_last, by_head, by_copy, by_tokens, by_page, by_pairs;  // by_last: units of the last chunk
  N730KV16Cache c;
  const int* lens; const int* n_new;
};

// A run of N consecutive elements as it lies in memory.
template <int N, int ES> struct RoRun { uint4 w[N * ES / 16]; };
template <> struct RoRun<1, 2> { uint16_t w; };
template <> struct RoRun<1, 4> { uint32_t w; };
template <int N, int ES>
__device__ __forceinline__ RoRun<N, ES> ro_load(const void* p, int64_t i) {
  return *reinterpret_cast<const RoRun<N, ES>*>(reinterpret_cast<const uint8_t*>(p) + i * ES);
}
__device__ __forceinline__ float2 ro_wide(uint32_t w, bool f16) {
  return f16 ? __half22float2(*reinterpret_cast<const __half2*>(&w)) : make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t ro_pack(float a, float b, bool f16) {
  if (f16) return h2_bits(__floats2half2_rn(a, b));
  const __nv_bfloat162 y = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&y);
}
template <int N, int ES>
__device__ __forceinline__ void ro_widen(const RoRun<N, ES>& r, bool f16, float* x) {
  if constexpr (N == 1) {
    x[0] = ES == 4 ? __uint_as_float(r.w) : ro_wide(r.w, f16).x;
  } else if constexpr (ES == 4) {
#pragma unroll
    for (int e = 0; e < N / 4; ++e) {
      x[4 * e] = __uint_as_float(r.w[e].x); x[4 * e + 1] = __uint_as_float(r.w[e].y);
      x[4 * e + 2] = __uint_as_float(r.w[e].z); x[4 * e + 3] = __uint_as_float(r.w[e].w);
    }
  } else {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = ro_wide(w[e], f16);
      x[2 * e] = f.x; x[2 * e + 1] = f.y;
    }
  }
}
template <int N>
__device__ __forceinline__ void ro_store(void* p, int64_t i, int dtype, const float* x) {
  if (N == 1) {
    kv8_store1(p, i, dtype, x[0]);
  } else if (dtype == N730_F32) {
    float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
    d[0] = make_float4(x[0], x[1], x[2], x[3]);
    d[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = ro_pack(x[2 * e], x[2 * e + 1], dtype == N730_F16);
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// A unit: N consecutive channels (a half layout's rotated ones: two runs of N, rd / 2 apart; N = 1 interleaved: the
// pair), N = 8 where every run starts on a 16-byte boundary, 1 otherwise.  A thread has one unit of a row, the same in
// each of its rows: what it is and where it lies is found out once.
template <int N, int ES>
__global__ void __launch_bounds__(RO_THREADS, 3) rotary_kernel(const RotaryArgs a) {
  extern __shared__ __align__(16) float2 ro_cs[];  // [row of the CTA][pair]
  __shared__ int row_pos[RO_ROWS * 32], row_slot[RO_ROWS * 32];  // position; row of the pool, -1: dropped, -2: no row at all
  constexpr int BATCH = N == 1 || ES == 4 ? 1 : 2;            // rows asked for at a time
  const int tid = threadIdx.x, np = a.rd / 2;
  const int r0 = (int)blockIdx.x * a.rows_cta, nr = min(a.rows_cta, a.rows - r0);
  const int u0 = blockIdx.y * a.chunk, uc = min(a.chunk, a.units - u0);
  const int prefix = a.has_cache ? kv16_prefix(a.c) : 0, cap = a.has_cache ? a.c.max_pages * a.c.page_size : 0;

  // this thread's unit
  const int first = (int)(uc == a.chunk ? a.by_chunk : a.by_last).div(tid);  // its first row of the CTA
  int u = u0 + tid - first * uc, which = 0, per = a.units_head;
  if (u >= a.part[0].heads * per) {
    u -= a.part[0].heads * per;
    which = 1;
    if (u >= a.part[1].heads * per) { u -= a.part[1].heads * per; which = 2; per = a.units_copy; }
  }
  const int head = (int)(which == 2 ? a.by_copy : a.by_head).div(u), w = u - head * per;
  int ch, rot = -1, gap = 0;  // its first channel, its first pair (-1: it stays), elements to its second run
  if (which == 2 || a.rd == 0) {
    ch = w * N;
  } else if (a.interleaved) {
    const int nu = N == 1 ? np : a.rd / N;
    if (w < nu) { ch = N == 1 ? 2 * w : w * N; rot = ch / 2; gap = N == 1 ? 1 : 0; }
    else ch = a.rd + (w - nu) * N;
  } else {
    const int nu = np / N;
    if (w < nu) { ch = rot = w * N; gap = np; }
    else ch = a.rd + (w - nu) * N;
  }
  const RotaryPart& p = a.part[which];
  const int col = head * a.head_dim + ch;
  const bool to_pool = p.y == nullptr, f16 = a.dtype == N730_F16, mine = first < a.at_once;

  RoRun<N, ES> x[BATCH], x2[BATCH];
  auto load = [&](int k, int r) {
    const int64_t at = (int64_t)(r0 + r) * p.ldx + col;
    x[k] = ro_load<N, ES>(p.x, at);
    if (gap) x2[k] = ro_load<N, ES>(p.x, at + gap);
  };
  // rows that are surely there are asked for before what follows is known
  const bool early = mine && first < nr && (!a.has_cache || a.tokens == 1);
  if (early) load(0, first);

  for (int r = tid; r < nr; r += blockDim.x) {
    const int row = r0 + r;
    int pos = 0, slot = 0;
    if (a.has_cache) {
      const int b = (int)a.by_tokens.div(row), t = row - b * a.tokens, len = kv8_len(a.lens, b, cap);
      pos = prefix + len + t;
      slot = -1;
      if (t >= kv8_new(a.n_new, b, a.tokens)) {
        slot = -2;
      } else if (len + t < cap) {
        const int pi = (int)a.by_page.div(len + t), page = a.c.block_table[(int64_t)b * a.c.max_pages + pi];
        if ((unsigned)page < (unsigned)a.c.n_pages) slot = page * a.c.n_kv * a.c.page_size + len + t - pi * a.c.page_size;
      }
    }
    if (a.pos) pos = a.pos[row];
    row_pos[r] = pos;
    row_slot[r] = slot;
  }
  __syncthreads();
  if (np) {
    for (int i = tid; i < nr * np; i += blockDim.x) {
      const int r = (int)a.by_pairs.div(i);
      double turns = (double)row_pos[r] * a.freq[i - r * np] * 0.15915494309189533577;  // 1 / 2 pi
      turns -= rint(turns);
      float sn, cs;
      sincospif(2.f * (float)turns, &sn, &cs);
      ro_cs[i] = make_float2(cs * a.factor, sn * a.factor);
    }
    __syncthreads();
  }
  if (!mine) return;

  for (int rb = first; rb < nr; rb += BATCH * a.at_once) {
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int r = rb + k * a.at_once;
      if (r < nr && row_slot[r] != -2 && !(early && r == first)) load(k, r);
    }
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int r = rb + k * a.at_once;
      if (r >= nr) break;
      const int slot = row_slot[r];
      if (slot == -2 || (to_pool && slot < 0)) continue;
      float y[2 * N];
      ro_widen<N, ES>(x[k], f16, y);
      if (gap) ro_widen<N, ES>(x2[k], f16, y + N);
      if (rot >= 0) {
        const float2* cs = ro_cs + r * np + rot;  // on 16 bytes where units are vectors
        float4 c4;
        if (gap) {
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float2 t = N == 1 ? cs[0] : e % 2 ? make_float2(c4.z, c4.w) : (c4 = reinterpret_cast<const float4*>(cs)[e / 2], make_float2(c4.x, c4.y));
            const float y0 = y[e], y1 = y[N + e];
            y[e] = y0 * t.x - y1 * t.y;
            y[N + e] = y1 * t.x + y0 * t.y;
          }
        } else {
#pragma unroll
          for (int e = 0; e < N / 2; ++e) {
            const float2 t = e % 2 ? make_float2(c4.z, c4.w) : (c4 = reinterpret_cast<const float4*>(cs)[e / 2], make_float2(c4.x, c4.y));
            const float y0 = y[2 * e], y1 = y[2 * e + 1];
            y[2 * e] = y0 * t.x - y1 * t.y;
            y[2 * e + 1] = y1 * t.x + y0 * t.y;
          }
        }
      }
      void* dst = to_pool ? (p.pool ? a.c.v : a.c.k) : p.y;
      const int type = to_pool ? a.c.dtype : a.dtype;
      const int64_t at = to_pool ? (int64_t)(slot + head * a.c.page_size) * a.head_dim + ch : (int64_t)(r0 + r) * p.ldy + col;
      ro_store<N>(dst, at, type, y);
      if (gap) ro_store<N>(dst, at + gap, type, y + N);
    }
  }
}

static int rotary_check(const N730Rotary* r, int head_dim, const char* what) {
  N730_REQUIRE(r->d_freq, N730_NULL, "%s: null frequencies", what);
  N730_REQUIRE(((uintptr_t)r->d_freq & 7) == 0, N730_BAD_ARG, "%s: frequencies must lie on whole elements", what);
  N730_REQUIRE(r->rotary_dim >= 2 && r->rotary_dim % 2 == 0 && r->rotary_dim <= head_dim, N730_BAD_ARG,
               "%s: rotary_dim %d of heads of %d", what, r->rotary_dim, head_dim);
  N730_REQUIRE(r->layout == N730_ROTARY_HALF || r->layout == N730_ROTARY_INTERLEAVED, N730_BAD_ARG, "%s: layout %d", what,
               r->layout);
  N730_REQUIRE(std::isfinite(r->factor), N730_BAD_ARG, "%s: factor %g", what, r->factor);
  return N730_OK;
}

static int rotary_launch(RotaryArgs& a, const N730Rotary* r, const char* what, cudaStream_t st) {
  a.rd = r ? r->rotary_dim : 0;
  a.freq = r ? r->d_freq : nullptr;
  a.factor = r ? r->factor : 1.f;
  a.interleaved = r && r->layout == N730_ROTARY_INTERLEAVED;
  // vectors of 8 channels where every run of them starts on 16 bytes
  const int run = a.interleaved ? a.rd : a.rd / 2, es = kv8_esize(a.dtype);
  bool vec = run % RO_V == 0 && a.head_dim % RO_V == 0;
  for (const RotaryPart& p : a.part)
    if (p.heads) vec = vec && (((uintptr_t)p.x | (uintptr_t)p.y) & 15) == 0 && p.ldx * es % 16 == 0 && (!p.y || p.ldy * es % 16 == 0);
  const int n = vec ? RO_V : 1;
  a.units_copy = a.head_dim / n;
  a.units_head = a.rd == 0 ? a.units_copy : a.interleaved && vec ? a.units_copy : a.rd / 2 / n + (a.head_dim - a.rd) / n;
  const int64_t units = (int64_t)(a.part[0].heads + a.part[1].heads) * a.units_head + (int64_t)a.part[2].heads * a.units_copy;
  N730_REQUIRE(units <= (int64_t)RO_THREADS * 65535, N730_BAD_ARG, "%s: rows of %lld channels", what,
               (long long)(a.part[0].heads + a.part[1].heads + a.part[2].heads) * a.head_dim);
  a.units = (int)units;
  const int most = (a.units + RO_THREADS - 1) / RO_THREADS;
  a.chunk = (a.units + most - 1) / most;  // even shares
  const int chunks = (a.units + a.chunk - 1) / a.chunk;
  // short rows go side by side; a CTA takes as many of its up to 16 rows as fill whole waves of three CTAs an SM (4133 rows
  // in two chunks: 10 of them, 23 us; 16, a wave and a sixth, 29)
  a.at_once = std::min(std::max(RO_THREADS / a.chunk, 1), 32);
  const int64_t turns = ((int64_t)a.rows + a.at_once - 1) / a.at_once * chunks, slots = 3 * num_sms();
  const int64_t waves = (turns + slots * RO_ROWS - 1) / (slots * RO_ROWS);
  a.rows_cta = a.at_once * (int)((turns + slots * waves - 1) / (slots * waves));
  const int threads = (a.chunk * a.at_once + 31) / 32 * 32;
  a.by_chunk = FastDiv(a.chunk);
  a.by_last = FastDiv(a.units - (chunks - 1) * a.chunk);
  a.by_head = FastDiv(a.units_head);
  a.by_copy = FastDiv(a.units_copy);
  a.by_tokens = FastDiv(a.tokens);
  a.by_page = FastDiv(a.has_cache ? a.c.page_size : 1);
  a.by_pairs = FastDiv(std::max(a.rd / 2, 1));
  while ((int64_t)a.rows_cta * (a.rd / 2) * sizeof(float2) > RO_TABLE) a.rows_cta -= a.at_once;
  const dim3 g((unsigned)(((int64_t)a.rows + a.rows_cta - 1) / a.rows_cta), chunks);
  const size_t smem = (size_t)a.rows_cta * (a.rd / 2) * sizeof(float2);
  if (vec) {
    if (es == 4) rotary_kernel<RO_V, 4><<<g, threads, smem, st>>>(a);
    else rotary_kernel<RO_V, 2><<<g, threads, smem, st>>>(a);
  } else {
    if (es == 4) rotary_kernel<1, 4><<<g, threads, smem, st>>>(a);
    else rotary_kernel<1, 2><<<g, threads, smem, st>>>(a);
  }
  N730_CHECK_LAUNCH();
  return N730_OK;
}

static bool dtype_ok(int d) { return d == N730_F32 || d == N730_F16 || d == N730_BF16; }

}  // namespace n730

using namespace n730;

N730_API int n730_rotary_frequencies(int rotary_dim, double theta, int scaling, double factor, double low, double high,
                                     int trained, double* freq, float* out_factor) {
  const char* what = "rotary_frequencies";
  N730_REQUIRE(freq && out_factor, N730_NULL, "%s: null pointer", what);
  N730_REQUIRE(rotary_dim >= 2 && rotary_dim % 2 == 0, N730_BAD_ARG, "%s: rotary_dim %d", what, rotary_dim);
  N730_REQUIRE(std::isfinite(theta) && theta > 1, N730_BAD_ARG, "%s: theta %g", what, theta);
  N730_REQUIRE(scaling >= N730_ROTARY_PLAIN && scaling <= N730_ROTARY_BANDS, N730_BAD_ARG, "%s: scaling %d", what, scaling);
  N730_REQUIRE(scaling == N730_ROTARY_PLAIN || (std::isfinite(factor) && factor >= 1), N730_BAD_ARG, "%s: factor %g", what, factor);
  const int n = rotary_dim / 2;
  const double pi = 3.14159265358979323846, d = rotary_dim;
  if (scaling == N730_ROTARY_RAMP || scaling == N730_ROTARY_BANDS)
    N730_REQUIRE(trained >= 1 && std::isfinite(low) && std::isfinite(high) && low > 0 && high > low, N730_BAD_ARG,
                 "%s: %d trained positions, bounds %g and %g", what, trained, low, high);
  if (scaling == N730_ROTARY_BASE) {
    N730_REQUIRE(rotary_dim > 2, N730_BAD_ARG, "%s: rotary_dim 2 has no other base", what);
    theta *= std::pow(factor, d / (d - 2));
  }
  *out_factor = 1.f;
  double lo = 0, hi = 0;
  if (scaling == N730_ROTARY_RAMP) {  // pairs (as numbers) that make `high` and `low` turns over the trained positions
    lo = std::max(std::floor(d * std::log(trained / (high * 2 * pi)) / (2 * std::log(theta))), 0.0);
    hi = std::min(std::ceil(d * std::log(trained / (low * 2 * pi)) / (2 * std::log(theta))), d - 1);
    *out_factor = (float)(0.1 * std::log(factor) + 1);
  }
  for (int i = 0; i < n; ++i) {
    const double f = std::pow(theta, -2.0 * i / d);
    double keep = 1;  // how much of the pair's own frequency stays, the rest is slowed by `factor`
    if (scaling == N730_ROTARY_LINEAR) keep = 0;
    if (scaling == N730_ROTARY_RAMP) keep = 1 - std::min(std::max((i - lo) / std::max(hi - lo, 0.001), 0.0), 1.0);
    if (scaling == N730_ROTARY_BANDS) keep = std::min(std::max((trained * f / (2 * pi) - low) / (high - low), 0.0), 1.0);
    freq[i] = keep == 1 ? f : f / factor * (1 - keep) + f * keep;
  }
  return N730_OK;
}

N730_API int n730_rotary(const N730Rotary* r, const void* d_x, int64_t ldx, void* d_y, int64_t ldy, int dtype, int64_t rows,
                         int n_heads, int head_dim, const int32_t* d_pos, void* stream) {
  const char* what = "rotary";
  N730_REQUIRE(r && d_x && d_y && d_pos, N730_NULL, "%s: null pointer", what);
  N730_REQUIRE(dtype_ok(dtype), N730_BAD_ARG, "%s: dtype %d", what, dtype);
  N730_REQUIRE(head_dim >= 2 && head_dim <= 512 && n_heads >= 1 && n_heads <= 65535, N730_BAD_ARG, "%s: %d heads of %d", what,
               n_heads, head_dim);
  if (int rc = rotary_check(r, head_dim, what)) return rc;
  N730_REQUIRE(rows >= 1 && rows < (1ll << 31), N730_BAD_ARG, "%s: %lld rows", what, (long long)rows);
  const int64_t row = (int64_t)n_heads * head_dim;
  N730_REQUIRE(ldx >= row && ldy >= row, N730_BAD_ARG, "%s: row strides %lld, %lld < %d heads x %d", what, (long long)ldx,
               (long long)ldy, n_heads, head_dim);
  N730_REQUIRE(d_x != d_y || ldx == ldy, N730_BAD_ARG, "%s: rows in place have one stride", what);
  N730_REQUIRE(kv8_aligned(kv8_esize(dtype), (const char*)d_x, (const char*)d_y) && kv8_aligned(4, d_pos), N730_BAD_ARG,
               "%s: pointers must lie on whole elements", what);
  RotaryArgs a{};
  a.part[0] = RotaryPart{d_x, d_y, ldx, ldy, n_heads, 0};
  a.head_dim = head_dim; a.dtype = dtype; a.rows = (int)rows; a.tokens = 1;
  a.pos = d_pos;
  return rotary_launch(a, r, what, (cudaStream_t)stream);
}

N730_API int n730_kv16_append(const N730KV16Cache* c, const N730Rotary* r, const void* d_q, int64_t ldq, void* d_q_out,
                              int64_t ldqo, int n_heads, const void* d_k, const void* d_v, int64_t ld, int dtype, int batch,
                              int tokens, const int32_t* d_lens, const int32_t* d_new, const int32_t* d_pos, void* stream) {
  const char* what = "kv16_append";
  if (int rc = kv16_check(c, batch, what)) return rc;
  N730_REQUIRE(d_k && d_v && d_lens, N730_NULL, "%s: null pointer", what);
  N730_REQUIRE(dtype_ok(dtype), N730_BAD_ARG, "%s: dtype %d", what, dtype);
  N730_REQUIRE(tokens >= 1 && tokens <= (1 << 24), N730_BAD_ARG, "%s: tokens %d", what, tokens);
  if (r)
    if (int rc = rotary_check(r, c->head_dim, what)) return rc;
  N730_REQUIRE(ld >= (int64_t)c->n_kv * c->head_dim, N730_BAD_ARG, "%s: row stride %lld < %d heads x %d", what, (long long)ld,
               c->n_kv, c->head_dim);
  N730_REQUIRE(kv8_aligned(kv8_esize(dtype), (const char*)d_k, (const char*)d_v, (const char*)d_q, (const char*)d_q_out) &&
                   kv8_aligned(4, d_lens, d_new, d_pos), N730_BAD_ARG, "%s: pointers must lie on whole elements", what);
  RotaryArgs a{};
  if (d_q || d_q_out) {
    N730_REQUIRE(d_q && d_q_out, N730_NULL, "%s: queries without a place, or a place without queries", what);
    N730_REQUIRE(r, N730_BAD_ARG, "%s: queries without a rotary", what);
    N730_REQUIRE(n_heads >= 1 && n_heads <= 65535, N730_BAD_ARG, "%s: %d query heads", what, n_heads);
    const int64_t row = (int64_t)n_heads * c->head_dim;
    N730_REQUIRE(ldq >= row && ldqo >= row, N730_BAD_ARG, "%s: row strides %lld, %lld < %d heads x %d", what, (long long)ldq,
                 (long long)ldqo, n_heads, c->head_dim);
    N730_REQUIRE(d_q != d_q_out || ldq == ldqo, N730_BAD_ARG, "%s: rows in place have one stride", what);
    a.part[0] = RotaryPart{d_q, d_q_out, ldq, ldqo, n_heads, 0};
  }
  a.part[1] = RotaryPart{d_k, nullptr, ld, 0, c->n_kv, 0};
  a.part[2] = RotaryPart{d_v, nullptr, ld, 0, c->n_kv, 1};
  N730_REQUIRE((int64_t)batch * tokens < (1ll << 31), N730_BAD_ARG, "%s: %d x %d rows", what, batch, tokens);
  a.head_dim = c->head_dim; a.dtype = dtype; a.rows = batch * tokens; a.tokens = tokens;
  a.pos = d_pos;
  a.has_cache = 1;
  a.c = *c;
  a.lens = d_lens; a.n_new = d_new;
  return rotary_launch(a, r, what, (cudaStream_t)stream);
}
