// 8-bit paged key/value cache: appending rows, reading them back, eviction by
// accumulated attention weight.
//
// Quantisation.  A block of 16, 32 or 64 positions of one KV head has one fp32
// scale s; with top = 127 (int8) or 448 (e4m3)
//   new block          s' = amax / top                 (amax over the new rows)
//   block with rows    s' = max(s, amax / top), older codes q' = round(q * (s / s'))
//   codes              q  = round(x / s'), ties to even, saturated to +-top
// with every quotient and product rounded to fp32.  amax runs over finite
// values; a NaN becomes 0 and an infinity saturates, so one bad value cannot
// blank a block.  s' = 0 (a block of zeros) has codes 0.
//
// Every output block is written by one CTA from inputs that no other CTA of
// the call writes, with no atomics: results do not depend on the order of CTAs.
#include "kv8.h"

namespace n730 {

constexpr int KV8_THREADS = 128;

int kv8_check(const N730KV8Cache* c, int batch, const char* what) {
  N730_REQUIRE(c, N730_NULL, "%s: null cache", what);
  N730_REQUIRE(c->k_codes && c->v_codes && c->k_scales && c->v_scales && c->block_table, N730_NULL,
               "%s: null cache pointer", what);
  N730_REQUIRE(c->code == N730_KV8_INT8 || c->code == N730_KV8_E4M3, N730_BAD_ARG, "%s: code type %d", what, c->code);
  N730_REQUIRE(c->head_dim == 64 || c->head_dim == 128, N730_UNSUPPORTED, "%s: head_dim %d", what, c->head_dim);
  N730_REQUIRE(c->block == 16 || c->block == 32 || c->block == 64, N730_BAD_ARG, "%s: block %d (16, 32 or 64)", what,
               c->block);
  N730_REQUIRE(c->page_size > 0 && c->page_size % c->block == 0, N730_BAD_ARG,
               "%s: page_size %d is not a multiple of the block %d", what, c->page_size, c->block);
  N730_REQUIRE(c->n_kv >= 1 && c->n_kv <= 65535 && c->n_pages >= 1 && c->max_pages >= 1, N730_BAD_ARG,
               "%s: n_kv %d, n_pages %d, max_pages %d", what, c->n_kv, c->n_pages, c->max_pages);
  N730_REQUIRE((int64_t)c->n_pages * c->n_kv * c->page_size < (1ll << 31), N730_BAD_ARG,
               "%s: the pool holds 2^31 or more rows", what);
  N730_REQUIRE((int64_t)c->max_pages * c->page_size <= (1ll << 30), N730_BAD_ARG,
               "%s: a sequence's pages hold more than 2^30 positions", what);
  N730_REQUIRE((((uintptr_t)c->k_codes | (uintptr_t)c->v_codes) & 15) == 0, N730_BAD_ARG,
               "%s: code pools must be 16-byte aligned", what);
  N730_REQUIRE(kv8_aligned(4, c->k_scales, c->v_scales, c->block_table), N730_BAD_ARG,
               "%s: scales and block table must lie on whole elements", what);
  N730_REQUIRE(batch >= 1 && batch <= 65535, N730_BAD_ARG, "%s: batch %d", what, batch);
  return N730_OK;
}

static int kv8_check_dtype(int dtype, const char* what) {
  N730_REQUIRE(dtype == N730_F32 || dtype == N730_F16 || dtype == N730_BF16, N730_BAD_ARG, "%s: dtype %d", what, dtype);
  return N730_OK;
}

// 16 consecutive elements as fp32; `vec`: the rows are 16-byte aligned.
__device__ __forceinline__ void kv8_load16(const void* p, int64_t i, int dtype, bool vec, float (&x)[16]) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = kv8_load1(p, i + e, dtype);
  } else if (dtype == N730_F32) {
    const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 v = s[e];
      x[4 * e] = v.x; x[4 * e + 1] = v.y; x[4 * e + 2] = v.z; x[4 * e + 3] = v.w;
    }
  } else {
    const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
    const uint4 a = s[0], b = s[1];
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (dtype == N730_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
        x[2 * e] = f.x; x[2 * e + 1] = f.y;
      } else {  // a bf16 is the upper half of the fp32 with the same value
        x[2 * e] = __uint_as_float(w[e] << 16);
        x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      }
    }
  }
}

__device__ __forceinline__ void kv8_store16(void* p, int64_t i, int dtype, bool vec, const float (&x)[16]) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < 16; ++e) kv8_store1(p, i + e, dtype, x[e]);
  } else if (dtype == N730_F32) {
    float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
  } else {
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (dtype == N730_F16) {
        const __half2 h = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    uint4* d = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i);
    d[0] = make_uint4(w[0], w[1], w[2], w[3]);
    d[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// ---- codes of 16 values in one 16-byte word group ----
__device__ __forceinline__ uint32_t pack4_e4m3(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// Of values that round to -127 .. 127.  + 1.5 * 2^23 rounds to an integer, ties to even, and leaves it in the low byte:
// conversions to and from integers run at a quarter of this rate and bounded the eviction.
__device__ __forceinline__ uint32_t pack4_int8(float a, float b, float c, float d) {
  const float2 x = add2(make_float2(a, b), both(12582912.f)), y = add2(make_float2(c, d), both(12582912.f));
  return __byte_perm(__byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x0040),
                     __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x0040), 0x5410);
}
template <int CODE>
__device__ __forceinline__ uint4 kv8_pack(const float (&y)[16]) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] = CODE == N730_KV8_INT8 ? pack4_int8(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3])
                                 : pack4_e4m3(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int CODE>
__device__ __forceinline__ void kv8_unpack(const uint4& c, float (&y)[16]) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (CODE == N730_KV8_INT8) {
      // 128 + q in the low byte of 2^23 is 2^23 + 128 + q
      const uint32_t u = w[e] ^ 0x80808080u;
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        const float2 f = add2(make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + k)),
                                          __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441 + k))), both(-8388736.f));
        y[4 * e + k] = f.x; y[4 * e + k + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[e] >> (16 * k)), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        y[4 * e + 2 * k] = f.x; y[4 * e + 2 * k + 1] = f.y;
      }
    }
  }
}
// Quotients by one scale: with r the rounded reciprocal and y = x r rounded, y + (x - y s) r, each by one FMA, is the
// rounded quotient unless s's significand is all ones (P. Markstein, "Computation of elementary functions on the
// IBM RISC System/6000 processor", 1990, theorem on correctly rounded quotients).  It needs the remainder to be
// exact, so the scale is asked to lie in [2^-60, 2^60]: quotients of rows too small for that are codes of 0.  Other
// scales take the division (which cost more than the row's memory traffic: 4096 rows of 8 heads 13.9 us).
template <int CODE>
__device__ __forceinline__ uint4 kv8_encode(const float (&x)[16], float s) {
  constexpr float top = CODE == N730_KV8_INT8 ? 127.f : 448.f;
  float y[16];
  if (s >= 0x1p-60f && s <= 0x1p60f && (__float_as_uint(s) & 0x7fffffu) != 0x7fffffu) {
    const float r = __frcp_rn(s), most = top * s;  // its quotient rounds to top, as those past it do
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      float2 v;
      v.x = x[e] == x[e] ? fminf(fmaxf(x[e], -most), most) : 0.f;
      v.y = x[e + 1] == x[e + 1] ? fminf(fmaxf(x[e + 1], -most), most) : 0.f;
      // the remainder negated: that way -0 stays -0
      const float2 q = mul2(v, both(r)), z = fma2(fma2(q, both(s), make_float2(-v.x, -v.y)), both(-r), q);
      y[e] = z.x; y[e + 1] = z.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float v = x[e] == x[e] ? x[e] : 0.f;
      y[e] = s > 0.f ? fminf(fmaxf(__fdiv_rn(v, s), -top), top) : 0.f;
    }
  }
  return kv8_pack<CODE>(y);
}
// the code values of a scale `from` on a scale `to`, which is not smaller
template <int CODE>
__device__ __forceinline__ uint4 kv8_recode(const uint4& c, float from, float to) {
  const float r = __fdiv_rn(from, to > 0.f ? to : 1.f);
  float y[16];
  kv8_unpack<CODE>(c, y);
#pragma unroll
  for (int e = 0; e < 16; ++e) y[e] = __fmul_rn(y[e], r);  // a packed product is fused with the addition that rounds it
  return kv8_pack<CODE>(y);
}
__device__ __forceinline__ float kv8_amax(const float (&x)[16]) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float a = fabsf(x[e]);
    m = a < INFINITY ? fmaxf(m, a) : m;  // false for NaN too
  }
  return m;
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct KV8AppendArgs {
  N730KV8Cache c;
  const void* x[2];  // K rows, V rows
  int dtype, tokens;
  int64_t ld;
  bool vec;
  const int* lens; const int* n_new;
};

// One CTA per (touched block of positions, K or V, KV head, sequence): the block's rows stay in
// registers between the maximum and the codes, so new rows are read once.  A thread holds NP
// chunks of 16 channels.  Bound by HBM for prompts, by one launch and three dependent round
// trips (length, page, rows) for a single token.
template <int HD, int CODE, int NP>
__global__ void __launch_bounds__(KV8_THREADS) kv8_append_kernel(const KV8AppendArgs a) {
  constexpr int CPR = HD / 16, RPP = KV8_THREADS / CPR;  // chunks a row, rows a pass
  __shared__ float red[32];
  pdl_wait();
  const N730KV8Cache& c = a.c;
  const int b = blockIdx.z, h = blockIdx.y, which = blockIdx.x & 1, j = blockIdx.x >> 1;
  const int tid = threadIdx.x;
  const int cap = c.max_pages * c.page_size;
  const int L = kv8_len(a.lens, b, cap);
  const int end = min(L + kv8_new(a.n_new, b, a.tokens), cap);
  const int p0 = (L / c.block + j) * c.block;
  if (p0 >= end || L >= end) return;
  const int page = c.block_table[(int64_t)b * c.max_pages + p0 / c.page_size];
  const void* x = which ? a.x[1] : a.x[0];
  const int chunk = tid % CPR, r0 = tid / CPR;
  const bool had = p0 < L;
  float v[NP][16];
#pragma unroll
  for (int i = 0; i < NP; ++i) {  // the rows do not wait for the page
    const int r = r0 + i * RPP, p = p0 + r;
    if (r < c.block && p >= L && p < end)
      kv8_load16(x, ((int64_t)b * a.tokens + (p - L)) * a.ld + (int64_t)h * HD + chunk * 16, a.dtype, a.vec, v[i]);
    else
#pragma unroll
      for (int e = 0; e < 16; ++e) v[i][e] = 0.f;
  }
  if ((unsigned)page >= (unsigned)c.n_pages) return;  // no page: its rows are dropped
  const int64_t row0 = ((int64_t)page * c.n_kv + h) * c.page_size + p0 % c.page_size;
  uint8_t* codes = reinterpret_cast<uint8_t*>(which ? c.v_codes : c.k_codes) + row0 * HD;
  float* scale = (which ? c.v_scales : c.k_scales) + row0 / c.block;
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < NP; ++i) m = fmaxf(m, kv8_amax(v[i]));
  const float s0 = had ? *scale : 0.f;
  m = warp_max(m);
  if ((tid & 31) == 0) red[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < KV8_THREADS / 32; ++w) m = fmaxf(m, red[w]);
  const float need = __fdiv_rn(m, CODE == N730_KV8_INT8 ? 127.f : 448.f);
  const float s = had ? fmaxf(s0, need) : need;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = r0 + i * RPP, p = p0 + r;
    if (r >= c.block) continue;
    uint4* dst = reinterpret_cast<uint4*>(codes + (int64_t)r * HD + chunk * 16);
    if (p >= L && p < end) *dst = kv8_encode<CODE>(v[i], s);
    else if (p < L && s != s0) *dst = kv8_recode<CODE>(*dst, s0, s);
  }
  if (tid == 0) *scale = s;  // every thread has read s0 before the barrier
}

int kv8_append_launch(const N730KV8Cache& c, const void* k, const void* v, int dtype, int64_t ld, int batch,
                      int tokens, const int* lens, const int* n_new, bool pdl, cudaStream_t st) {
  KV8AppendArgs a{};
  a.c = c;
  a.x[0] = k; a.x[1] = v;
  a.dtype = dtype; a.tokens = tokens; a.ld = ld;
  a.vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && ld * kv8_esize(dtype) % 16 == 0;
  a.lens = lens; a.n_new = n_new;
  // blocks that `tokens` rows can touch, whatever the length they follow
  const int64_t nblk = ((int64_t)tokens + c.block - 2) / c.block + 1;
  const dim3 grid((unsigned)(2 * nblk), c.n_kv, batch);
  const int np = (c.block * (c.head_dim / 16) + KV8_THREADS - 1) / KV8_THREADS;
#define N730_APPEND(HD, CODE, NP) kv8_launch(kv8_append_kernel<HD, CODE, NP>, grid, dim3(KV8_THREADS), 0, st, pdl, a)
#define N730_APPEND_CODE(CODE)                                                     \
  if (c.head_dim == 128)                                                           \
    return np == 1 ? N730_APPEND(128, CODE, 1) : np == 2 ? N730_APPEND(128, CODE, 2) : N730_APPEND(128, CODE, 4); \
  return np == 1 ? N730_APPEND(64, CODE, 1) : N730_APPEND(64, CODE, 2);
  if (c.code == N730_KV8_INT8) { N730_APPEND_CODE(N730_KV8_INT8) }
  N730_APPEND_CODE(N730_KV8_E4M3)
#undef N730_APPEND_CODE
#undef N730_APPEND
}

// ---------------------------------------------------------------------------
// read
// ---------------------------------------------------------------------------
struct KV8ReadArgs {
  N730KV8Cache c;
  void* y[2];
  int dtype, tokens, log_block;
  int64_t ld;
  bool vec;
  const int* first; const int* lens;
};

// A thread takes 16 channels of RD_ROWS positions, a warp's lanes whole rows one behind the other (contiguous in a
// page); its loads do not wait for one another.  Bound by HBM: 1 byte read, 2 or 4 written a value.  With one
// position a thread 8192 positions of 8 sequences and heads took 67 us, too few bytes in flight; with four 63 us
// (5.45 TB/s).
constexpr int RD_ROWS = 4;

template <int HD, int CODE>
__global__ void __launch_bounds__(KV8_THREADS) kv8_read_kernel(const KV8ReadArgs a) {
  constexpr int CPR = HD / 16, RPP = KV8_THREADS / CPR;  // chunks a row, rows a pass
  const N730KV8Cache& c = a.c;
  const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1;
  const int chunk = threadIdx.x % CPR;
  const int64_t t0 = (int64_t)blockIdx.x * (RPP * RD_ROWS) + threadIdx.x / CPR;
  const int cap = c.max_pages * c.page_size;
  const int L = kv8_len(a.lens, b, cap);
  const int64_t p0 = (a.first ? a.first[b] : 0) + t0;
  const uint8_t* codes = reinterpret_cast<const uint8_t*>(which ? c.v_codes : c.k_codes);
  const float* scales = which ? c.v_scales : c.k_scales;
  int64_t row[RD_ROWS];
#pragma unroll
  for (int i = 0; i < RD_ROWS; ++i) {
    const int64_t p = p0 + i * RPP;
    row[i] = -1;
    if (p >= 0 && p < L && t0 + i * RPP < a.tokens) {
      const int page = c.block_table[(int64_t)b * c.max_pages + (int)p / c.page_size];
      if ((unsigned)page < (unsigned)c.n_pages) row[i] = ((int64_t)page * c.n_kv + h) * c.page_size + (int)p % c.page_size;
    }
  }
  uint4 q[RD_ROWS];
  float s[RD_ROWS];
#pragma unroll
  for (int i = 0; i < RD_ROWS; ++i) {
    q[i] = make_uint4(0, 0, 0, 0);
    s[i] = 0.f;
    if (row[i] >= 0) {
      q[i] = __ldcs(reinterpret_cast<const uint4*>(codes + row[i] * HD + chunk * 16));
      s[i] = scales[row[i] >> a.log_block];
    }
  }
#pragma unroll
  for (int i = 0; i < RD_ROWS; ++i) {
    const int64_t t = t0 + i * RPP;
    if (t >= a.tokens) break;
    float y[16];
    kv8_unpack<CODE>(q[i], y);
#pragma unroll
    for (int e = 0; e < 16; ++e) y[e] = row[i] >= 0 ? y[e] * s[i] : 0.f;  // 0 x 0 is slower: 65.3 us for 63.0
    kv8_store16(which ? a.y[1] : a.y[0], ((int64_t)b * a.tokens + t) * a.ld + (int64_t)h * HD + chunk * 16, a.dtype, a.vec, y);
  }
}

// ---------------------------------------------------------------------------
// evict
// ---------------------------------------------------------------------------
// Per (sequence, KV head) with more than `keep` cached slots, `keep` of them stay: the protected
// ones (position < first, or among the last `recent` seen), then the largest weights, ties to the
// lowest slot.  Kept slots at or behind `keep` move into the holes before it, the j-th into the
// j-th; all others stay where they are with the codes they have.  A cache in order would have to
// move, and requantise, nearly every row at every call; attention does not ask for order.
//
// Two kernels: the selection (one CTA per sequence and head) writes src[slot], the pool row whose
// codes belong at `slot` (-1 without a page, -2 in the first entry when nothing is to move); the move
// rewrites the blocks that take rows in.  Rows read from behind `keep` (a multiple of the block) are
// written by nobody.
//
// Selection: the keys are read once into shared memory (up to EV_KEYS of them; longer contexts read
// them again), the keep-th largest is found 11 bits at a time, and ranks of ties, holes and movers come
// from ballots: a warp owns a run of slots, one scan over the warps' counts a pass.
// 2304 slots of 4 heads take 14 us, all latency; 256 rows of up to 8192 32 us in one wave, two CTAs an SM (32 registers):
// the issue slots are 58 % busy, and warps wait for global memory first, for barriers next.  Table widths count too: from
// EV_KEYS positions on keys are read again, and the outputs' rows are written to their ends (one sequence of 2304 slots,
// whole call, 20.5 us in a table of 8192 positions, 24.6 in 32768, 30.4 in 65536).  The move is bound by the arithmetic on
// codes (80 % of the issue slots): 32 x 8 heads cut from up to 8192 slots to 2048, about 43 us; 55 with conversions to and
// from integers.
struct KV8EvictArgs {
  N730KV8Cache c;
  int keep, first, recent, log_block;
  int64_t ldw;
  const int* seen; const int* lens_in; int* lens_out;
  const float* w_in; float* w_out;
  const int* pos_in; int* pos_out;
  int* src;  // [batch][n_kv][keep] pool rows, then as many slots
  int keys;   // of a row held in shared memory: all that the table can hold, or none
  int lists;  // whether the lists of slots are held there too
};

constexpr int EV_THREADS = 1024;
constexpr int EV_BINS = 2048;   // 11 bits a pass, three passes over the 32-bit key
constexpr int EV_KEYS = 50000;  // 200 KB

// Order of the kept: protected slots first, then by weight (NaN as the smallest, -0 as 0).
__device__ __forceinline__ uint32_t ev_key(float w, int pos, int first, int last) {
  if (pos < first || pos >= last) return 0xffffffffu;
  if (isnan(w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Sum over the warps before the caller's of one count a warp (the same in its lanes).  One barrier: every warp adds up
// the counts by itself; `buf` is not used by the call before.
__device__ __forceinline__ long long ev_before(long long n, long long* buf) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) buf[warp] = n;
  __syncthreads();
  long long v = lane < warp ? buf[lane] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__global__ void __launch_bounds__(EV_THREADS) kv8_evict_select_kernel(const KV8EvictArgs a) {
  extern __shared__ uint32_t ev_keys[];
  __shared__ int hist[EV_BINS];
  __shared__ long long sums[2][EV_THREADS / 32];
  __shared__ int pick_bin, pick_above;
  const N730KV8Cache& c = a.c;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int cap = c.max_pages * c.page_size;
  const int L = kv8_len(a.lens_in, b, cap);
  const int64_t head = (int64_t)b * c.n_kv + h;
  const float* w_in = a.w_in + head * a.ldw;
  float* w_out = a.w_out + head * a.ldw;
  const int* pos_in = a.pos_in + head * a.ldw;
  int* pos_out = a.pos_out + head * a.ldw;
  int* src = a.src + head * a.keep;
  if (L <= a.keep) {
    if (tid == 0) src[0] = -2;
    for (int64_t i = tid; i < a.ldw; i += EV_THREADS) {
      w_out[i] = i < L ? w_in[i] : 0.f;
      pos_out[i] = pos_in[i];
    }
    return;
  }
  const int seen = a.seen[b], last = seen - a.recent;
  const int lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < EV_BINS; i += EV_THREADS) hist[i] = 0;
#pragma unroll 4
  for (int i = tid; i < min(L, a.keys); i += EV_THREADS) ev_keys[i] = ev_key(w_in[i], pos_in[i], a.first, last);
  __syncthreads();
  auto key = [&](int i) { return a.keys ? ev_keys[i] : ev_key(w_in[i], pos_in[i], a.first, last); };
  // the keep-th largest key, 11 + 11 + 10 bits at a time
  uint32_t prefix = 0;
  int want = a.keep;  // of the slots whose key has the chosen prefix
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < L; i += EV_THREADS) {
      const uint32_t k = key(i);
      if (pass == 0 || (k >> (shift + bits)) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1);
    }
    __syncthreads();
    // bins from the top: thread t holds bins 2047 - 2t and 2046 - 2t
    const int hi = hist[EV_BINS - 1 - 2 * tid], lo = hist[EV_BINS - 2 - 2 * tid];
    hist[EV_BINS - 1 - 2 * tid] = hist[EV_BINS - 2 - 2 * tid] = 0;  // for the next pass
    int inc = hi + lo;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += n;
    }
    const int above = (int)ev_before(__shfl_sync(0xffffffffu, inc, 31), sums[pass & 1]) + inc - hi - lo;
    if (above < want && above + hi >= want) { pick_bin = EV_BINS - 1 - 2 * tid; pick_above = above; }
    else if (above + hi < want && above + hi + lo >= want) { pick_bin = EV_BINS - 2 - 2 * tid; pick_above = above + hi; }
    __syncthreads();
    prefix = (prefix << bits) | (uint32_t)pick_bin;
    want -= pick_above;
  }
  const uint32_t cut = prefix;  // slots above it stay, and the first `want` equal to it
  // each warp a run of slots, 32 at a time; counts(flag) is how many of the warps before have it
  const int run = ((L + EV_THREADS - 1) / EV_THREADS) * 32, i0 = min(L, warp * run), i1 = min(L, i0 + run);
  const uint32_t before = (1u << lane) - 1u;
  int ties = 0;
  for (int i = i0; i < i1; i += 32) ties += __popc(__ballot_sync(0xffffffffu, i + lane < i1 && key(i + lane) == cut));
  const int tie0 = (int)ev_before(ties, sums[1]);
  // stays(i): called for i = i0 + lane, + 32, ... with the ties so far in t
  auto stays = [&](int i, int& t) {
    const uint32_t k = i < i1 ? key(i) : 0u;
    const uint32_t tie = __ballot_sync(0xffffffffu, i < i1 && k == cut);
    const bool yes = i < i1 && (k > cut || (k == cut && t + __popc(tie & before) < want));
    t += __popc(tie);
    return yes;
  };
  int holes = 0, movers = 0, t = tie0;
  for (int i = i0 + lane; i - lane < i1; i += 32) {
    const bool yes = stays(i, t);
    holes += __popc(__ballot_sync(0xffffffffu, i < i1 && !yes && i < a.keep));
    movers += __popc(__ballot_sync(0xffffffffu, yes && i >= a.keep));
  }
  const long long ranks = ev_before(((long long)holes << 32) | (unsigned)movers, sums[0]);
  const int hole0 = (int)(ranks >> 32), mover0 = (int)(ranks & 0xffffffff);
  // slots before the budget: their own, or (holes, listed by rank) a mover's
  // from: the slot that comes to a slot; list: the holes by rank (in global memory until the rows go there)
  int* from = a.lists ? reinterpret_cast<int*>(ev_keys + a.keys) : a.src + (int64_t)gridDim.y * c.n_kv * a.keep + head * a.keep;
  int* list = a.lists ? from + a.keep : src;
  t = tie0;
  int hr = hole0;
  for (int i = i0 + lane; i - lane < i1; i += 32) {
    const bool yes = stays(i, t), hole = i < i1 && !yes && i < a.keep;
    const uint32_t m = __ballot_sync(0xffffffffu, hole);
    if (yes && i < a.keep) from[i] = i;
    if (hole) list[hr + __popc(m & before)] = i;
    hr += __popc(m);
  }
  __syncthreads();
  t = tie0;
  int mr = mover0;
  for (int i = i0 + lane; i - lane < i1; i += 32) {
    const bool mover = stays(i, t) && i >= a.keep;
    const uint32_t m = __ballot_sync(0xffffffffu, mover);
    if (mover) from[list[mr + __popc(m & before)]] = i;
    mr += __popc(m);
  }
  __syncthreads();
  // weights and positions; in and out may be the same arrays: sources are never slots written before
  const int* bt = c.block_table + (int64_t)b * c.max_pages;
#pragma unroll 2
  for (int i = tid; i < a.keep; i += EV_THREADS) {
    const int s = from[i], page = bt[s / c.page_size];
    w_out[i] = w_in[s];
    pos_out[i] = pos_in[s];
    src[i] = (unsigned)page < (unsigned)c.n_pages ? (page * c.n_kv + h) * c.page_size + s % c.page_size : -1;
  }
  __syncthreads();
  for (int64_t i = a.keep + tid; i < a.ldw; i += EV_THREADS) {
    w_out[i] = 0.f;
    pos_out[i] = (int)(seen + (i - a.keep));
  }
}

// One CTA per (block of the kept slots, KV head, sequence): K and V rows whose block takes rows in.
template <int HD, int CODE, int NP>
__global__ void __launch_bounds__(KV8_THREADS) kv8_evict_move_kernel(const KV8EvictArgs a) {
  constexpr int CPR = HD / 16, RPP = KV8_THREADS / CPR;
  const N730KV8Cache& c = a.c;
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  pdl_wait();
  if (blockIdx.x == 0 && h == 0 && tid == 0)
    a.lens_out[b] = min(kv8_len(a.lens_in, b, c.max_pages * c.page_size), a.keep);
  const int64_t head = (int64_t)b * c.n_kv + h;
  const int* src = a.src + head * a.keep;
  const int p0 = blockIdx.x * c.block;
  const int chunk = tid % CPR, r0 = tid / CPR, lane = tid & 31;
  // the block's own rows, and those that belong there
  const int page = c.block_table[(int64_t)b * c.max_pages + p0 / c.page_size];
  int row[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) row[i] = r0 + i * RPP < c.block ? src[p0 + r0 + i * RPP] : -1;
  const int lr0 = lane < c.block ? src[p0 + lane] : -1, lr1 = lane + 32 < c.block ? src[p0 + 32 + lane] : -1;
  if (src[0] == -2) return;
  const int row0 = (unsigned)page < (unsigned)c.n_pages ? (page * c.n_kv + h) * c.page_size + p0 % c.page_size : -1;
  // does any come from elsewhere, and the largest scale among them: every warp on its own
  bool any = lane < c.block && lr0 != row0 + lane;
  any |= lane + 32 < c.block && lr1 != row0 + 32 + lane;
  float sk = 0.f, sv = 0.f;
  if (lr0 >= 0) { sk = c.k_scales[lr0 >> a.log_block]; sv = c.v_scales[lr0 >> a.log_block]; }
  if (lr1 >= 0) { sk = fmaxf(sk, c.k_scales[lr1 >> a.log_block]); sv = fmaxf(sv, c.v_scales[lr1 >> a.log_block]); }
  any = __any_sync(0xffffffffu, any);
  if (!any || row0 < 0) return;  // the same in every warp
  float sf[NP][2];
  uint4 q[NP][2];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    q[i][0] = q[i][1] = make_uint4(0, 0, 0, 0);
    sf[i][0] = sf[i][1] = -1.f;
    if (row[i] < 0) continue;  // a row without a page reads as zeros
    sf[i][0] = c.k_scales[row[i] >> a.log_block];
    sf[i][1] = c.v_scales[row[i] >> a.log_block];
    q[i][0] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(c.k_codes) + (int64_t)row[i] * HD + chunk * 16);
    q[i][1] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(c.v_codes) + (int64_t)row[i] * HD + chunk * 16);
  }
  sk = warp_max(sk);
  sv = warp_max(sv);
  __syncthreads();  // every thread has read the block's old scales
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = r0 + i * RPP;
    if (r >= c.block) continue;
    const int64_t at = ((int64_t)row0 + r) * HD + chunk * 16;
    const bool stays = row[i] == row0 + r;  // rows in place are written only where the scale grows
    if (!stays || sf[i][0] != sk)
      *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(c.k_codes) + at) =
          sf[i][0] == sk || row[i] < 0 ? q[i][0] : kv8_recode<CODE>(q[i][0], sf[i][0], sk);
    if (!stays || sf[i][1] != sv)
      *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(c.v_codes) + at) =
          sf[i][1] == sv || row[i] < 0 ? q[i][1] : kv8_recode<CODE>(q[i][1], sf[i][1], sv);
  }
  if (tid == 0) {
    c.k_scales[row0 >> a.log_block] = sk;
    c.v_scales[row0 >> a.log_block] = sv;
  }
}

// ---------------------------------------------------------------------------
// the model's own steps around the cache
// ---------------------------------------------------------------------------
__global__ void kv8_rope_kernel(float* qkv, int64_t ld, int heads, int n_kv, int head_dim, const float* cos_t,
                                const float* sin_t, const int* pos, int per_row, __half* q16) {
  pdl_wait();
  const int r = blockIdx.x, h2 = head_dim / 2;
  const int p = per_row ? pos[r] : pos[0] + r;
  float* row = qkv + (int64_t)r * ld;
  const float* cs = cos_t + (int64_t)p * h2;
  const float* sn = sin_t + (int64_t)p * h2;
  for (int i = threadIdx.x; i < (heads + n_kv) * h2; i += blockDim.x) {
    const int h = i / h2, j = i % h2;
    float* x = row + (int64_t)h * head_dim;
    const float x0 = x[j], x1 = x[j + h2], y0 = x0 * cs[j] - x1 * sn[j], y1 = x1 * cs[j] + x0 * sn[j];
    if (q16 && h < heads) {
      __half* q = q16 + ((int64_t)r * heads + h) * head_dim;
      q[j] = __float2half_rn(y0);
      q[j + h2] = __float2half_rn(y1);
    } else {
      x[j] = y0;
      x[j + h2] = y1;
    }
  }
}

int kv8_rope_launch(float* qkv, int64_t ld, int rows, int heads, int n_kv, int head_dim, const float* cos_t,
                    const float* sin_t, const int* pos, bool per_row, __half* q16, bool pdl, cudaStream_t st) {
  return kv8_launch(kv8_rope_kernel, dim3(rows), dim3(256), 0, st, pdl, qkv, ld, heads, n_kv, head_dim, cos_t, sin_t, pos,
                    (int)per_row, q16);
}

}  // namespace n730

using namespace n730;

N730_API int n730_kv8_append(const N730KV8Cache* c, const void* d_k, const void* d_v, int dtype, int64_t ld, int batch,
                             int tokens, const int32_t* d_lens, const int32_t* d_new, void* stream) {
  if (int rc = kv8_check(c, batch, "kv8_append")) return rc;
  if (int rc = kv8_check_dtype(dtype, "kv8_append")) return rc;
  N730_REQUIRE(d_k && d_v && d_lens, N730_NULL, "kv8_append: null pointer");
  N730_REQUIRE(kv8_aligned(kv8_esize(dtype), d_k, d_v) && kv8_aligned(4, d_lens, d_new), N730_BAD_ARG,
               "kv8_append: pointers must lie on whole elements");
  N730_REQUIRE(tokens >= 1 && tokens <= (1 << 24), N730_BAD_ARG, "kv8_append: tokens %d", tokens);
  N730_REQUIRE(ld >= (int64_t)c->n_kv * c->head_dim, N730_BAD_ARG, "kv8_append: row stride %lld < %d heads x %d",
               (long long)ld, c->n_kv, c->head_dim);
  return kv8_append_launch(*c, d_k, d_v, dtype, ld, batch, tokens, d_lens, d_new, false, (cudaStream_t)stream);
}

N730_API int n730_kv8_read(const N730KV8Cache* c, void* d_k, void* d_v, int dtype, int64_t ld, int batch, int tokens,
                           const int32_t* d_first, const int32_t* d_lens, void* stream) {
  if (int rc = kv8_check(c, batch, "kv8_read")) return rc;
  if (int rc = kv8_check_dtype(dtype, "kv8_read")) return rc;
  N730_REQUIRE(d_k && d_v && d_lens, N730_NULL, "kv8_read: null pointer");
  N730_REQUIRE(kv8_aligned(kv8_esize(dtype), d_k, d_v) && kv8_aligned(4, d_lens, d_first), N730_BAD_ARG,
               "kv8_read: pointers must lie on whole elements");
  N730_REQUIRE(tokens >= 1 && tokens <= (1 << 30), N730_BAD_ARG, "kv8_read: tokens %d", tokens);
  N730_REQUIRE(c->n_kv <= 32767, N730_BAD_ARG, "kv8_read: n_kv %d", c->n_kv);
  N730_REQUIRE(ld >= (int64_t)c->n_kv * c->head_dim, N730_BAD_ARG, "kv8_read: row stride %lld < %d heads x %d",
               (long long)ld, c->n_kv, c->head_dim);
  KV8ReadArgs a{};
  a.c = *c;
  a.y[0] = d_k; a.y[1] = d_v;
  a.dtype = dtype; a.tokens = tokens; a.ld = ld;
  a.vec = (((uintptr_t)d_k | (uintptr_t)d_v) & 15) == 0 && ld * kv8_esize(dtype) % 16 == 0;
  a.first = d_first; a.lens = d_lens;
  a.log_block = c->block == 16 ? 4 : c->block == 32 ? 5 : 6;
  const int rows = KV8_THREADS / (c->head_dim / 16) * RD_ROWS;
  const dim3 grid((unsigned)(((int64_t)tokens + rows - 1) / rows), 2 * c->n_kv, batch);
  cudaStream_t st = (cudaStream_t)stream;
  if (c->head_dim == 128) {
    if (c->code == N730_KV8_INT8) return kv8_launch(kv8_read_kernel<128, N730_KV8_INT8>, grid, dim3(KV8_THREADS), 0, st, false, a);
    return kv8_launch(kv8_read_kernel<128, N730_KV8_E4M3>, grid, dim3(KV8_THREADS), 0, st, false, a);
  }
  if (c->code == N730_KV8_INT8) return kv8_launch(kv8_read_kernel<64, N730_KV8_INT8>, grid, dim3(KV8_THREADS), 0, st, false, a);
  return kv8_launch(kv8_read_kernel<64, N730_KV8_E4M3>, grid, dim3(KV8_THREADS), 0, st, false, a);
}

static int evict_check(const N730KV8Cache* c, int batch, int keep) {
  if (int rc = kv8_check(c, batch, "kv8_evict")) return rc;
  N730_REQUIRE(keep >= c->block && keep % c->block == 0 && (int64_t)keep <= (int64_t)c->max_pages * c->page_size,
               N730_BAD_ARG, "kv8_evict: keep %d must be a multiple of the block %d within the table's %d pages", keep,
               c->block, c->max_pages);
  return N730_OK;
}

N730_API int64_t n730_kv8_evict_ws(const N730KV8Cache* c, int batch, int keep) {
  if (int rc = evict_check(c, batch, keep)) return rc;
  return (int64_t)batch * c->n_kv * keep * 2 * sizeof(int);
}

N730_API int n730_kv8_evict(const N730KV8Cache* c, int batch, int keep, int first, int recent, const int32_t* d_seen,
                            const int32_t* d_lens, int32_t* d_lens_out, const float* d_w, float* d_w_out,
                            const int32_t* d_pos, int32_t* d_pos_out, int64_t ldw, void* d_ws, int64_t ws_bytes,
                            void* stream) {
  if (int rc = evict_check(c, batch, keep)) return rc;
  N730_REQUIRE(d_seen && d_lens && d_lens_out && d_w && d_w_out && d_pos && d_pos_out && d_ws, N730_NULL,
               "kv8_evict: null pointer");
  N730_REQUIRE(kv8_aligned(4, d_seen, d_lens, d_lens_out) && kv8_aligned(4, d_w, d_w_out, d_pos, d_pos_out), N730_BAD_ARG,
               "kv8_evict: pointers must lie on whole elements");
  N730_REQUIRE(first >= 0 && recent >= 0 && (int64_t)first + recent <= keep, N730_BAD_ARG,
               "kv8_evict: first %d + recent %d exceed keep %d", first, recent, keep);
  N730_REQUIRE(ldw >= (int64_t)c->max_pages * c->page_size, N730_BAD_ARG,
               "kv8_evict: row stride %lld of the weights is below the table's %lld positions", (long long)ldw,
               (long long)c->max_pages * c->page_size);
  N730_REQUIRE(ws_bytes >= n730_kv8_evict_ws(c, batch, keep) && ((uintptr_t)d_ws & 3) == 0, N730_BAD_ARG,
               "kv8_evict: workspace of %lld bytes", (long long)ws_bytes);
  KV8EvictArgs a{};
  a.c = *c;
  a.keep = keep; a.first = first; a.recent = recent; a.ldw = ldw;
  a.seen = d_seen; a.lens_in = d_lens; a.lens_out = d_lens_out;
  a.w_in = d_w; a.w_out = d_w_out; a.pos_in = d_pos; a.pos_out = d_pos_out;
  a.src = reinterpret_cast<int*>(d_ws);
  a.log_block = c->block == 16 ? 4 : c->block == 32 ? 5 : 6;
  const int cap = c->max_pages * c->page_size;
  a.keys = cap <= EV_KEYS ? cap : 0;
  a.lists = (int64_t)a.keys + 2 * (int64_t)keep <= EV_KEYS;
  const size_t smem = ((size_t)a.keys + (a.lists ? 2 * (size_t)keep : 0)) * 4;
  cudaStream_t st = (cudaStream_t)stream;
  if (int rc = smem_attr_once<kv8_evict_select_kernel>(EV_KEYS * 4)) return rc;
  if (int rc = kv8_launch(kv8_evict_select_kernel, dim3(c->n_kv, batch), dim3(EV_THREADS), smem, st, false, a))
    return rc;
  const dim3 grid(keep / c->block, c->n_kv, batch);
  const int np = (c->block * (c->head_dim / 16) + KV8_THREADS - 1) / KV8_THREADS;
#define N730_MOVE(HD, CODE, NP) kv8_launch(kv8_evict_move_kernel<HD, CODE, NP>, grid, dim3(KV8_THREADS), 0, st, true, a)
#define N730_MOVE_CODE(CODE)                                                     \
  if (c->head_dim == 128)                                                        \
    return np == 1 ? N730_MOVE(128, CODE, 1) : np == 2 ? N730_MOVE(128, CODE, 2) : N730_MOVE(128, CODE, 4); \
  return np == 1 ? N730_MOVE(64, CODE, 1) : N730_MOVE(64, CODE, 2);
  if (c->code == N730_KV8_INT8) { N730_MOVE_CODE(N730_KV8_INT8) }
  N730_MOVE_CODE(N730_KV8_E4M3)
#undef N730_MOVE_CODE
#undef N730_MOVE
}
