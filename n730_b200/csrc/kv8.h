// Paged key/value cache in 8 bits: shared definitions of its kernels.
//
// Codes lie as [pages][n_kv][page_size][head_dim] bytes, int8 or e4m3; `block` consecutive
// positions of a page and KV head share one fp32 scale, [pages][n_kv][page_size / block]; a
// value is code * scale.  Position p of sequence b lies in page block_table[b * max_pages +
// p / page_size]; an id outside [0, n_pages) is no page.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "n730_cuda.h"

namespace n730 {

int kv8_check(const N730KV8Cache* c, int batch, const char* what);
int kv8_append_launch(const N730KV8Cache& c, const void* k, const void* v, int dtype, int64_t ld, int batch,
                      int tokens, const int* lens, const int* n_new, bool pdl, cudaStream_t st);

// RoPE of q and k (rotate_half, in place) in rows [heads | n_kv | ...] of fp32 qkv; row r is at position
// *pos + r (one sequence) or pos[r] (a row per sequence).  q16 (may be null): q rounded to fp16 instead.
int kv8_rope_launch(float* qkv, int64_t ld, int rows, int heads, int n_kv, int head_dim, const float* cos_t,
                    const float* sin_t, const int* pos, bool per_row, __half* q16, bool pdl, cudaStream_t st);

struct KV8AttnCall {
  N730KV8Cache c;
  const void* q; void* out;
  int dtype, out_dtype;  // of q; of out
  int64_t ldq, ldo;
  int batch, tokens, heads;
  float scale;
  const int* lens; const int* n_new;
  const float* w_in; float* w_out;
  int64_t ldw;
  void* ws; int64_t ws_bytes;
  int* status;  // where a wait that ran out leaves its mark (null: the workspace's first word)
  bool pdl;
};
constexpr int KV8_MAX_BATCH = 4096;
// what n730_kv8_attention refuses of the cache and the sizes
int kv8_attention_check(const N730KV8Cache* c, int batch, int tokens, int heads);
int64_t kv8_attention_ws(const N730KV8Cache& c, int batch, int tokens, int heads, bool weights);
int64_t kv8_attention_ws_upto(const N730KV8Cache& c, int batch, int tokens, int heads);
int kv8_attention_launch(const KV8AttnCall& a, cudaStream_t st);

// The tensor-memory kernel for prompts (kv8_prompt.cu): 256 rows of an item a CTA; the positions of the first `tail`
// tiles are cut into `splits` shares whose parts lie as [item][tail tile][split][rg rows].
constexpr int KV8_PROMPT_TILE = 128;  // positions of a tile
// How many of the planned shares a row tile uses whose rows see `sees` positions: each gets four tiles of them at least.
// The plan knows the table's width alone.
__device__ __forceinline__ int kv8_shares_used(int sees, int splits) {
  return min(splits, max(1, (sees + KV8_PROMPT_TILE - 1) / KV8_PROMPT_TILE / 4));
}
struct KV8PromptPlan { int rows, tiles, tail, splits, rg, shares; };  // shares: of the rows, for the weights
KV8PromptPlan kv8_prompt_plan(const N730KV8Cache& c, int batch, int tokens, int heads);
int kv8_prompt_launch(const KV8AttnCall& k, const KV8PromptPlan& p, int* status, float* part, float* part_ml, float* lse,
                      cudaStream_t st);
int kv8_prompt_weights_launch(const KV8AttnCall& k, const KV8PromptPlan& p, int* status, float* lse, cudaStream_t st);

// The first 1024-byte boundary of dynamic shared memory.  Formed by an offset, not by rounding the pointer: the
// compiler would lose sight of the address space and fall back to generic loads and stores.
__device__ __forceinline__ uint8_t* aligned_smem(uint8_t* raw) { return raw + ((0u - smem_u32(raw)) & 1023u); }

// a * b + c, a + b and a * b of two fp32 pairs
__device__ __forceinline__ float2 fma2(const float2& a, const float2& b, const float2& c) {
  float2 d;
  asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 w, x, y, z;\n mov.b64 {%0, %1}, w;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(const float2& a, const float2& b) {
  float2 d;
  asm("{\n .reg .b64 x, y, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 w, x, y;\n"
      " mov.b64 {%0, %1}, w;\n}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(const float2& a, const float2& b) {
  float2 d;
  asm("{\n .reg .b64 x, y, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 w, x, y;\n"
      " mov.b64 {%0, %1}, w;\n}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// one element of a row in the caller's type, widened to fp32
__device__ __forceinline__ float kv8_load1(const void* p, int64_t i, int dtype) {
  if (dtype == N730_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == N730_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void kv8_store1(void* p, int64_t i, int dtype, float x) {
  if (dtype == N730_F32) reinterpret_cast<float*>(p)[i] = x;
  else if (dtype == N730_F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(x);
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}
// Softmax weight x V scale (P) is fp16 against a reference: log2 of where a new reference puts the largest P, and of how
// large P may grow before the reference moves (fp16 ends at 2^16).  What lies below goes down to fp16's smallest normal,
// 2^-14, at full accuracy: 2^-21 of the largest.
constexpr float KV8_P_NEW = 7.f, KV8_P_MOST = 15.f;
// log2 of how far P's reference may lie below the weights': V scales reach 100 and KV8_P_MOST below, scores of blocks
// whose scale is 0 put the weights' reference anywhere above, and 2^distance has to stay in fp32's range
constexpr float KV8_REFS_APART = 120.f;
// V scales below this count as 0: quotients by them would leave fp32's range
constexpr float KV8_TINY = 0x1p-100f;
// whether pointers lie on whole elements of `size` bytes (null ones do)
template <class... P>
inline bool kv8_aligned(int size, const P*... p) { return ((0 | ... | reinterpret_cast<uintptr_t>(p)) & (uintptr_t)(size - 1)) == 0; }
inline int kv8_esize(int dtype) { return dtype == N730_F32 ? 4 : 2; }

// cached positions of a sequence before a call's new rows, within the table's capacity
__device__ __forceinline__ int kv8_len(const int* lens, int b, int cap) { return min(max(lens[b], 0), cap); }
// new rows of a sequence (all `tokens` without a count array)
__device__ __forceinline__ int kv8_new(const int* n_new, int b, int tokens) {
  return n_new ? min(max(n_new[b], 0), tokens) : tokens;
}

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

// Wait of a whole warp for the phase of `bar`, at most `limit_ns` long; false in every lane when one of them gave up:
// what that lane reads next may not be there yet.
__device__ __forceinline__ bool kv8_wait(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
  bool ok = mbar_try_wait(bar, parity);
  if (!ok) {
    auto now = [] { uint64_t t; asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t)); return t; };
    const uint64_t t0 = now();
    while (!(ok = mbar_try_wait(bar, parity)))
      if (now() - t0 > limit_ns) break;
  }
  ok = __all_sync(0xffffffffu, ok);
  __syncwarp();
  return ok;
}

// Launch with or without programmatic dependent launch.
template <class... KArgs, class... Args>
int kv8_launch_cluster(void (*k)(KArgs...), dim3 grid, int cluster, dim3 block, size_t smem, cudaStream_t st, bool pdl, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (pdl) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  N730_CUDA(cudaLaunchKernelEx(&cfg, k, args...));
  return N730_OK;
}
template <class... KArgs, class... Args>
int kv8_launch(void (*k)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool pdl, Args... args) {
  return kv8_launch_cluster(k, grid, 1, block, smem, st, pdl, args...);
}

}  // namespace n730
