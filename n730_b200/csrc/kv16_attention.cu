// Attention over the 16-bit paged cache behind a prefix that the batch shares.
//
//   out[b, t, head] = softmax_p(scale q . k_p) v_p,  p over the prefix and own positions <= lens[b] + t
#include <cmath>

#include "kv16.h"

namespace n730 {

struct KSArgs {
  N730KV16Cache c;
  const void* q; void* out;
  int64_t ldq, ldo;
  int batch, tokens, heads;
  float scale;
  const int* lens; const int* n_new;
};

constexpr int KS_THREADS = 128;

// A CTA takes one query row: scores of 128 positions, a thread each, then outputs, a thread a channel.
__global__ void __launch_bounds__(KS_THREADS) kv16_simple_kernel(const KSArgs a) {
  __shared__ float q[128], p[KS_THREADS], red[32];
  __shared__ int64_t row[KS_THREADS];
  const N730KV16Cache& c = a.c;
  const int tid = threadIdx.x, D = c.head_dim, b = blockIdx.x / a.tokens, t = blockIdx.x % a.tokens, head = blockIdx.y;
  if (t >= kv8_new(a.n_new, b, a.tokens)) return;
  const int h = head / (a.heads / c.n_kv), cap = c.max_pages * c.page_size;
  const int prefix = kv16_prefix(c), own = min(kv8_len(a.lens, b, cap) + t + 1, cap), n = prefix + own;
  if (tid < D) q[tid] = kv8_load1(a.q, (int64_t)blockIdx.x * a.ldq + (int64_t)head * D + tid, c.dtype) * a.scale;
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int j0 = 0; j0 < n; j0 += KS_THREADS) {
    __syncthreads();
    const int j = j0 + tid;
    int page = -1, off = 0;
    if (j < prefix) { page = c.prefix_table[j / c.page_size]; off = j % c.page_size; }
    else if (j < n) { page = c.block_table[(int64_t)b * c.max_pages + (j - prefix) / c.page_size]; off = (j - prefix) % c.page_size; }
    const bool here = (unsigned)page < (unsigned)c.n_pages;
    row[tid] = here ? (((int64_t)page * c.n_kv + h) * c.page_size + off) * D : -1;
    float x = -INFINITY;
    if (here) {
      x = 0.f;
      for (int d = 0; d < D; ++d) x = fmaf(q[d], kv8_load1(c.k, row[tid] + d, c.dtype), x);
    }
    float mx = warp_max(x);
    if ((tid & 31) == 0) red[tid >> 5] = mx;
    __syncthreads();
    mx = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float ms = mx == -INFINITY ? 0.f : mx, f = expf(m - ms), e = here ? expf(x - ms) : 0.f;
    p[tid] = e;
    m = mx;
    l = l * f + block_sum(e, red);
    acc *= f;
    if (tid < D)
      for (int k = 0; k < KS_THREADS; ++k)
        if (row[k] >= 0) acc = fmaf(p[k], kv8_load1(c.v, row[k] + tid, c.dtype), acc);
  }
  if (tid < D) kv8_store1(a.out, (int64_t)blockIdx.x * a.ldo + (int64_t)head * D + tid, c.dtype, l == 0.f ? 0.f : acc / l);
}

static int kv16_attention_check(const N730KV16Cache* c, int batch, int tokens, int heads) {
  const char* what = "kv16_attention";
  if (int rc = kv16_check(c, batch, what)) return rc;
  N730_REQUIRE(batch <= KV8_MAX_BATCH && tokens >= 1 && tokens <= (1 << 20), N730_BAD_ARG, "%s: batch %d, tokens %d", what, batch, tokens);
  N730_REQUIRE(heads >= c->n_kv && heads % c->n_kv == 0 && heads <= 65535, N730_BAD_ARG, "%s: %d heads over %d KV heads", what,
               heads, c->n_kv);
  return N730_OK;
}

}  // namespace n730

using namespace n730;

N730_API int64_t n730_kv16_attention_ws(const N730KV16Cache* c, int batch, int tokens, int n_heads) {
  if (int rc = kv16_attention_check(c, batch, tokens, n_heads)) return rc;
  return 256;
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
  N730_REQUIRE(std::isfinite(scale), N730_BAD_ARG, "%s: scale %g", what, scale);
  N730_REQUIRE(((uintptr_t)d_ws & 15) == 0, N730_BAD_ARG, "%s: the workspace must be 16-byte aligned", what);
  const int64_t need = n730_kv16_attention_ws(c, batch, tokens, n_heads);
  N730_REQUIRE(ws_bytes >= need, N730_BAD_ARG, "%s: workspace of %lld bytes, %lld needed", what, (long long)ws_bytes, (long long)need);
  KSArgs a{*c, d_q, d_out, ldq, ldo, batch, tokens, n_heads, scale, d_lens, d_new};
  kv16_simple_kernel<<<dim3((unsigned)(batch * tokens), n_heads), KS_THREADS, 0, (cudaStream_t)stream>>>(a);
  N730_CHECK_LAUNCH();
  return N730_OK;
}
