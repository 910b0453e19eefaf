// Prompt attention over the 8-bit paged key/value cache on the 5th-generation tensor cores.
//
//   out[b, t, head] = softmax_p(scale q . k_p) v_p,  positions p <= lens[b] + t of KV head head / G
//
// The rows of an item (sequence, KV head) are its tokens x G query heads, row = token * G + head, so
// every row of a tile reads the same K and V.  One CTA takes 256 rows (two 128-row tiles, A and B) and
// walks over the positions in tiles of 128:
//   warps 8-10  load the tile's codes (16 bytes a lane, whole 128-byte rows), turn them into fp16
//               exactly and store them swizzled: K as [64-channel block][position][128 B], the K-major
//               operand of S = Q K^T; V in the same layout, which is the MN-major operand of O += P V.
//               Each conversion serves 256 rows;
//   warp 11     issues S = Q K^T (both operands in shared memory) and O += P V (P in tensor memory) of
//               A and B in turn, so that one's products run while the other's softmax does;
//   warps 0-3   softmax of A, warps 4-7 of B: a thread owns a row (TMEM lane).  P, fp16, overwrites the
//               tile's scores in place.
// Tensor memory: scores of A and B, 128 columns each, outputs of A and B, head_dim columns each.
//
// Softmax.  The weight x V scale of a position is formed by one FMA and one exp2: its exponent is
// score * (row, block factor) + lv - reference with lv the approximate log2(V scale), and the sum of
// weights gets each block's sum times 2^(reference - maximum - lv).  Both references follow the largest values lazily (P
// grows from 2^KV8_P_NEW to 2^KV8_P_MOST meanwhile), so outputs in tensor memory are rescaled only when a row's maximum
// has grown by that much.
//
// Bounds: per tile of 128 positions and head_dim 128, 2 x 512 cycles of tensor work against 1024 of exp2 and about as many
// of issue slots on the 4 schedulers, for each of A and B.  Measured: 2048 tokens behind 6144 positions, 64 / 8 heads x
// 128, 578 us, 832 TFLOP/s (0.50 of a large bf16 product): about 2.75k cycles of softmax in a period of 4.6k a tile, 2.2
// times what the tensor cores or exp2 would need: latency.
//
// Numerics: 16-bit queries are exact in fp16 after a power-of-two scaling of their row; the softmax
// weights are rounded to fp16 (2^-11 of each, below the rounding of a 16-bit output, down to 2^-21 of the largest weight
// x V scale; 2^-32 of that largest below).  Sums and outputs are fp32.  fp32 queries do not come here.
// Every wait is bounded; one that runs out sets the workspace's status word, ends the CTA's work and
// still frees the tensor memory.
#include "kv8.h"
#include "tcgen05.cuh"

namespace n730 {

constexpr int KP_ROWS = 256;      // query rows of a CTA
constexpr int KP_KEYS = KV8_PROMPT_TILE;  // positions of a tile
// Twelve warps leave 168 registers a thread: the softmax holds a row's 128 scores (reading tensor memory twice
// cost as much as the arithmetic).
constexpr int KP_THREADS = 12 * 32;
constexpr int KP_CODE_WARPS = 3, KP_MMA_WARP = 11;
constexpr int KW_ROW_WARPS = 8, KW_MMA_WARP = 8 + KW_ROW_WARPS, KW_THREADS = (KW_MMA_WARP + 1) * 32;
constexpr int KW_SHARES = 8;      // most CTAs of a cluster
constexpr int KP_RING = 4;        // tiles whose scales are kept: two more than tiles of codes
constexpr float KP_SUM_SLACK = 64.f;  // log2 of how far a weight in the sum (fp32) may exceed its reference
// V scales and references this close leave weight x V scale and the way back to the weight inside fp32's range
constexpr float KP_NEAR_MIN = 0x1p-24f, KP_NEAR_MAX = 0x1p24f, KP_NEAR_REFS = 40.f, KP_NEAR_BACK = 0x1p64f;

template <int HD>
struct KPCfg {
  static constexpr int NB = HD / 64;                           // 64-channel blocks
  static constexpr int QB = KP_ROWS * 128, KB = KP_KEYS * 128;  // bytes of a block of Q, of K or V
  static constexpr int KV = NB * KB;                           // bytes of a tile of K or V
  static constexpr uint32_t TMEM = 512;
  static constexpr uint32_t S0 = 0, O0 = 2 * KP_KEYS;           // columns: scores of A, B; outputs of A, B
  // kind::f16: D fp32, A = B = fp16, M = 128
  static constexpr uint32_t IDESC_S = (1u << 4) | ((uint32_t)(KP_KEYS >> 3) << 17) | (8u << 24);
  static constexpr uint32_t IDESC_O = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | (8u << 24);  // B is MN-major
};

template <int HD>
struct KPSmem {
  uint8_t q[KPCfg<HD>::NB * KPCfg<HD>::QB];
  uint8_t k[2][KPCfg<HD>::KV];
  uint8_t v[2][KPCfg<HD>::KV];
  float sc[KP_RING][3][8];   // by block of 16 positions: K's scale (-infinity: no page), lv = log2 of V's scale, 2^-lv
  int odd[KP_RING][4];       // by warp of the codes: some block has no page, or a V scale of 0 or far from 1
  float rowmul[KP_ROWS];
  uint64_t kfull[2], vfull[2], kfree[2], vfree[2], sfull[2], pready[2], odone[2], drain;
  uint32_t tmem;
  int abort;
};

// Bounded wait of one lane that also gives up when another role raised the CTA's abort flag, and raises it
// itself after 2 s.  The clock is read once in 64 polls: reading it takes longer than most of these waits.
__device__ __forceinline__ bool kp_wait(uint64_t* bar, uint32_t parity, volatile int* abortf) {
  uint64_t t0 = 0;
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*abortf) return false;
    if (!t0) t0 = gtimer();
    else if (gtimer() - t0 > 2000000000ull) { *abortf = 1; return false; }
  }
}
// The same by a whole warp, which goes on together: with one lane waiting for the others the compiler kept that lane
// apart, and what followed ran twice.
__device__ __forceinline__ bool kp_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abortf) {
  const bool ok = __all_sync(0xffffffffu, kp_wait(bar, parity, abortf));
  __syncwarp();
  return ok;
}
// MN-major operand, 128-byte swizzle: atoms of 64 elements x 8 k; the next 64 elements lie `lead` bytes on,
// the next 8 k 1024 bytes on.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t saddr, uint32_t lead) {
  uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)(lead >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// One lane of a warp that runs together.  Products are issued under this, with descriptors that are the same in
// every lane: from code that one lane runs by itself an instruction took 180 cycles to issue instead of the 64 that a
// 128x128x16 product lasts.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
// D[tmem_d] (+)= A . B with both operands in shared memory
template <uint32_t IDESC>
__device__ __forceinline__ void tc_mma_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
               :: "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(IDESC), "r"(accumulate) : "memory");
}

// After the barrier behind all roles' work, when a wait of the CTA ran out, whichever role's: leaves the mark, and the warp
// that issued the products waits for those in flight, so that tensor and shared memory can be given up.
__device__ __forceinline__ void kp_give_up(uint64_t* drain, bool issuer, int* status) {
  if (threadIdx.x == 0) *status = 1;
  if (!issuer) return;
  if (elect_one()) tc_commit(drain);
  __syncwarp();
  kv8_wait(drain, 0, 2000000000ull);
}

// Rows of a warp's share of the 16-bit queries: a lane holds 8 channels of U rows, RPI rows an instruction.  `at(r)`
// gives row r's first element, negative for rows that are not there.
template <int HD>
struct KPRows { static constexpr int LPR = HD / 8, RPI = 32 / LPR; };
template <int HD, int U, class At>
__device__ __forceinline__ void kp_load_rows(const void* q, bool vec, int first, At at, uint4 (&x)[U]) {
  const int lane = threadIdx.x & 31, sub = lane / KPRows<HD>::LPR, ch = lane % KPRows<HD>::LPR;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = at(first + u * KPRows<HD>::RPI + sub);
    x[u] = make_uint4(0, 0, 0, 0);
    if (i < 0) continue;
    const uint16_t* p = reinterpret_cast<const uint16_t*>(q) + i + ch * 8;
    if (vec) x[u] = *reinterpret_cast<const uint4*>(p);
    else x[u] = make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16, p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16);
  }
}
// Writes them as rows of a K-major, swizzled operand with `block` bytes between 64-channel blocks, each scaled by a
// power of two, so that its largest magnitude lies in [2^13, 2^14) (rows of zeros or with an infinity stay);
// `put(r, mul)` is called by one lane a row with what scores of it are to be multiplied by.
template <int HD, int U, class Put>
__device__ __forceinline__ void kp_put_rows(const uint4 (&raw)[U], int dtype, float sign, float scale, uint8_t* dst, int block,
                                            int first, Put put) {
  constexpr int LPR = KPRows<HD>::LPR;
  const int lane = threadIdx.x & 31, sub = lane / LPR, ch = lane % LPR;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t y[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
    float x[8], m = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = dtype == N730_F16 ? __half22float2(u2h(y[e]))
                                         : make_float2(__uint_as_float(y[e] << 16), __uint_as_float(y[e] & 0xffff0000u));
      x[2 * e] = f.x; x[2 * e + 1] = f.y;
      m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y)));
    }
#pragma unroll
    for (int k = 1; k < LPR; k <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
    const int ex = (int)((__float_as_uint(m) >> 23) & 255u);
    const int sh = ex == 0 || ex == 255 ? 0 : min(max(140 - ex, -126), 126);
    const float mul = __uint_as_float((uint32_t)(127 + sh) << 23) * sign;
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = h2u(__floats2half2_rn(x[2 * e] * mul, x[2 * e + 1] * mul));
    const int r = first + u * KPRows<HD>::RPI + sub;
    *reinterpret_cast<uint4*>(dst + (ch >> 3) * block + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
    if (ch == 0) put(r, scale * __uint_as_float((uint32_t)(127 - sh) << 23));
  }
}
// 16 codes as fp16 into a row of a swizzled operand, at the row's 128 bytes in the 64-channel block of `chunk`;
// r7: the row's number mod 8.
template <int CODE>
__device__ __forceinline__ void kp_put_codes(const uint4& x, uint8_t* rowp, int r7, int chunk) {
  const uint32_t wd[4] = {x.x, x.y, x.z, x.w};
  uint32_t y[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t z = code_word<CODE>(wd[e]);
    y[2 * e] = codes2<CODE, 0>(z);
    y[2 * e + 1] = codes2<CODE, 1>(z);
  }
  // the two halves lie in neighbouring 16 bytes; lanes of the second 64-channel block store them in the other
  // order, or they would meet the banks of the first block's
  const bool swap = chunk >= 4;
  const int at = (((chunk & 3) * 2 + swap) ^ r7) << 4;
  *reinterpret_cast<uint4*>(rowp + at) = swap ? make_uint4(y[4], y[5], y[6], y[7]) : make_uint4(y[0], y[1], y[2], y[3]);
  *reinterpret_cast<uint4*>(rowp + (at ^ 16)) = swap ? make_uint4(y[0], y[1], y[2], y[3]) : make_uint4(y[4], y[5], y[6], y[7]);
}

// 8 consecutive columns of this thread's TMEM lane multiplied by f
__device__ __forceinline__ void tc_scale8(uint32_t taddr, float f) {
  float v[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n tcgen05.wait::ld.sync.aligned;"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(taddr) : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= f;
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n tcgen05.wait::st.sync.aligned;"
               :: "r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
// 64 consecutive columns of this thread's TMEM lane
__device__ __forceinline__ void tc_ld64(uint32_t taddr, float* v) {
  uint32_t r[64];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
               "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
               "%24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, "
               "%46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63"
               "}, [%64];\n tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), 
                 "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), 
                 "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), 
                 "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), 
                 "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), 
                 "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), 
                 "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), 
                 "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
               : "r"(taddr) : "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}

// Moves a row's references to the largest score mx of a tile, and to where its largest score + log2(V scale) mv becomes
// a P of 2^KV8_P_NEW, where those are larger; sums and, when there are any, outputs (at to) are rescaled.  A warp at a time.
template <int HD>
__device__ __forceinline__ void kp_move(uint32_t to, bool outputs, float mx, float mv, float& m_ref, float& mo_ref, float& l) {
  const float mn = fmaxf(m_ref, mx), mon = fmaxf(fmaxf(mo_ref, mn - KV8_REFS_APART), mv - KV8_P_NEW);
  if (mn != m_ref) l *= ex2(m_ref - mn);
  const float f = mon != mo_ref ? ex2(mo_ref - mon) : 1.f;
  m_ref = mn;
  mo_ref = mon;
  if (!outputs) return;
#pragma unroll 1
  for (int cc = 0; cc < HD; cc += 8) tc_scale8(to + cc, f);  // few registers: a row's scores are held meanwhile
}

// One tile of a row: moves the references when a weight would be too large against them, then writes the weights
// (fp16) over the scores at ts and adds their sum to l.  This is the short way: every row sees all of the tile, every
// block has a page and a V scale.
template <int HD>
__device__ __forceinline__ void kp_softmax(uint32_t ts, uint32_t to, const float* ksc, const float* lvs, float rm,
                                           bool outputs, float& m_ref, float& mo_ref, float& l) {
  float v[KP_KEYS];
  tc_ld64(ts, v);
  tc_ld64(ts + 64, v + 64);
  float mx = -INFINITY, mv = -INFINITY;
#pragma unroll
  for (int blk = 0; blk < KP_KEYS / 16; ++blk) {
    float m = v[16 * blk];
#pragma unroll
    for (int i = 16 * blk + 1; i < 16 * blk + 16; ++i) m = fmaxf(m, v[i]);
    const float y = m * (rm * ksc[blk]);
    mx = fmaxf(mx, y);
    mv = fmaxf(mv, y + lvs[blk]);
  }
  if (__any_sync(0xffffffffu, mx > m_ref + KP_SUM_SLACK || mv > mo_ref + KV8_P_MOST))
    kp_move<HD>(to, outputs, mx, mv, m_ref, mo_ref, l);
  const float mos = mo_ref == -INFINITY ? 0.f : mo_ref, ms = m_ref == -INFINITY ? 0.f : m_ref, back0 = ex2(mos - ms);
#pragma unroll
  for (int half = 0; half < 2; ++half) {  // 64 positions: 32 columns of P
    uint32_t w[32];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int blk = half * 4 + k;
      const float fk = rm * ksc[blk], off = lvs[blk] - mos;
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float2 y = fma2(make_float2(v[16 * blk + i], v[16 * blk + i + 1]), make_float2(fk, fk), make_float2(off, off));
        const float2 p = make_float2(ex2(y.x), ex2(y.y));
        sum = add2(sum, p);
        w[8 * k + i / 2] = h2u(__floats2half2_rn(p.x, p.y));
      }
      l = fmaf(sum.x + sum.y, back0 * lvs[8 + blk], l);
    }
    tc_st32(ts + half * 32, w);
  }
}

// The same for any tile: the first `sees` positions are seen, blocks may have no page or any V scale.
template <int HD>
__device__ __forceinline__ void kp_softmax_any(uint32_t ts, uint32_t to, const float* ksc, const float* lvs, float rm, int sees,
                                               bool outputs, float& m_ref, float& mo_ref, float& l) {
  float mx = -INFINITY, mv = -INFINITY;
#pragma unroll 1
  for (int cc = 0; cc < 4; ++cc) {
    float v[32];
    tc_ld32(ts + cc * 32, v);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) m = fmaxf(m, cc * 32 + 16 * e + i < sees ? v[16 * e + i] : -INFINITY);
      const float ks = ksc[2 * cc + e];
      const float y = m == -INFINITY || ks == -INFINITY ? -INFINITY : m * (rm * ks);
      mx = fmaxf(mx, y);
      mv = fmaxf(mv, y + lvs[2 * cc + e]);
    }
  }
  if (__any_sync(0xffffffffu, mx > m_ref + KP_SUM_SLACK || mv > mo_ref + KV8_P_MOST))
    kp_move<HD>(to, outputs, mx, mv, m_ref, mo_ref, l);
  const float mos = mo_ref == -INFINITY ? 0.f : mo_ref, ms = m_ref == -INFINITY ? 0.f : m_ref, back0 = ex2(mos - ms);
#pragma unroll 1
  for (int c2 = 0; c2 < 2; ++c2) {  // 64 positions: 32 columns of P over scores that have been read
    uint32_t w[32];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      float v[32];
      tc_ld32(ts + c2 * 64 + hh * 32, v);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int blk = c2 * 4 + hh * 2 + e;
        const float ks = ksc[blk], lv = lvs[blk];
        // zero V: the weights count in the sum, their product with V is zero
        const bool none = ks == -INFINITY, zero = lv == -INFINITY;  // the same for all rows
        float back = zero ? 1.f : back0 * lvs[8 + blk];
        const bool apart = back > KP_NEAR_BACK;  // the row's sum takes its own exp2
        const float fk = rm * ks, off = zero ? -ms : lv - mos;
        const int n = none ? 0 : sees - blk * 16;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float p0 = i < n ? ex2(fmaf(v[16 * e + i], fk, off)) : 0.f;
          const float p1 = i + 1 < n ? ex2(fmaf(v[16 * e + i + 1], fk, off)) : 0.f;
          sum += p0 + p1;
          w[hh * 16 + e * 8 + i / 2] = zero ? 0u : h2u(__floats2half2_rn(p0, p1));
        }
        if (__any_sync(0xffffffffu, apart)) {
          float own = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) own += i < n ? ex2(fmaf(v[16 * e + i], fk, -ms)) : 0.f;
          if (apart) { sum = own; back = 1.f; }
        }
        l = fmaf(sum, back, l);
      }
    }
    tc_st32(ts + c2 * 32, w);
  }
}

struct KPArgs {
  N730KV8Cache c;
  const void* q; void* out;
  int64_t ldq, ldo;
  int dtype, odtype, tokens, group, rows, tiles;  // rows = tokens * group; tiles of KP_ROWS rows
  int log_block;
  int batch, tail, splits;                // the first `tail` tiles' positions are cut into shares, each a CTA
  int shares;                             // of the rows, for the weights
  bool vec, qvec;                         // out rows, query rows are 16-byte aligned
  float scale_log2e;                      // its absolute value; the sign goes with the queries
  float sign;
  const int* lens; const int* n_new;
  int* status;
  float* part; float* part_ml;            // [item][tail tile][split][KP_ROWS] rows, as the split kernel's
  float* lse;                             // [batch][n_kv][rows] (may be null)
};

template <int HD, int CODE>
__global__ void __launch_bounds__(KP_THREADS, 1) kv8_prompt_kernel(const KPArgs a) {
  using Cfg = KPCfg<HD>;
  extern __shared__ __align__(1024) uint8_t kp_raw[];
  KPSmem<HD>& sm = *reinterpret_cast<KPSmem<HD>*>(aligned_smem(kp_raw));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const N730KV8Cache& c = a.c;
  // all items' last tiles first, which see most, the tail's shares at the end
  const int items = a.batch * c.n_kv, unit = (int)blockIdx.x / items, item = (int)blockIdx.x % items, whole = a.tiles - a.tail;
  const int b = item / c.n_kv, h = item % c.n_kv;
  const bool tail = unit >= whole;
  const int split = tail ? (unit - whole) % a.splits : 0;
  const int tile = tail ? a.tail - 1 - (unit - whole) / a.splits : a.tiles - 1 - unit;
  const int cap = c.max_pages * c.page_size;
  pdl_wait();
  const int L = kv8_len(a.lens, b, cap), n_new = kv8_new(a.n_new, b, a.tokens);
  const int f0 = tile * KP_ROWS, nrow = min(KP_ROWS, n_new * a.group - f0);
  if (nrow <= 0) return;
  // positions [p_lo, p_hi) of this share: what the tile's last row sees, cut into whole tiles
  const int sees_last = (int)min((int64_t)L + (f0 + nrow - 1) / a.group + 1, (int64_t)cap);
  const int sees_all = (int)min((int64_t)L + f0 / a.group + 1, (int64_t)cap);
  const int all_tiles = (sees_last + KP_KEYS - 1) / KP_KEYS, used = tail ? kv8_shares_used(sees_last, a.splits) : 1;
  if (split >= used) return;
  const bool part = used > 1;
  const int j0 = (int)((int64_t)all_tiles * split / used), nt = (int)((int64_t)all_tiles * (split + 1) / used) - j0;
  const int64_t head = (int64_t)b * c.n_kv + h;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.kfull[i], KP_CODE_WARPS);
      mbar_init(&sm.vfull[i], KP_CODE_WARPS);
      mbar_init(&sm.kfree[i], 1);
      mbar_init(&sm.vfree[i], 1);
      mbar_init(&sm.sfull[i], 1);
      mbar_init(&sm.pready[i], 4);
      mbar_init(&sm.odone[i], 1);
    }
    mbar_init(&sm.drain, 1);
    fence_mbar_init();
    sm.abort = 0;
  }
  if (warp == KP_MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_u32(&sm.tmem)), "r"(Cfg::TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp < 8) {  // Q, 32 rows each, K-major and swizzled
    constexpr int U = 4;
#pragma unroll 1
    for (int r0 = warp * 32; r0 < warp * 32 + 32; r0 += U * KPRows<HD>::RPI) {
      uint4 x[U];
      kp_load_rows<HD, U>(a.q, a.qvec, r0, [&](int r) -> int64_t {
        const int f = f0 + r;
        return r < nrow ? ((int64_t)b * a.tokens + f / a.group) * a.ldq + (int64_t)(h * a.group + f % a.group) * HD : -1;
      }, x);
      kp_put_rows<HD, U>(x, a.dtype, a.sign, a.scale_log2e, sm.q, Cfg::QB, r0, [&](int r, float mul) { sm.rowmul[r] = mul; });
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  const uint32_t tmem = sm.tmem;
  volatile int* abortf = &sm.abort;

  if (warp >= 8 && warp < 8 + KP_CODE_WARPS) {
    // ---------------- codes to fp16 ----------------
    // A warp takes every third block of 16 positions (each in a page), a lane 16 bytes of every RPI-th row.
    constexpr int LPR = HD / 16, RPI = 32 / LPR, NI = 16 / RPI;  // lanes a row, rows an instruction, instructions a block
    constexpr int BLOCKS = KP_KEYS / 16, MINE = (BLOCKS + KP_CODE_WARPS - 1) / KP_CODE_WARPS;
    const int w = warp - 8, lrow = lane / LPR, chunk = lane % LPR;
    const int* bt = c.block_table + (int64_t)b * c.max_pages;
    auto block = [&](int i) { return w + KP_CODE_WARPS * i; };
    // Walks over the warp's blocks, tile by tile: the page (-1 behind the last position) is looked up a tile before
    // its row is needed, page and offset advance without divisions.
    struct Walk { int p, idx, off, page; };
    const int step_idx = KP_KEYS / c.page_size, step_off = KP_KEYS % c.page_size;
    const int p_end = min(sees_last, (j0 + nt) * KP_KEYS);
    Walk walk[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int p = j0 * KP_KEYS + block(i) * 16;
      walk[i] = {p, p / c.page_size, p % c.page_size, block(i) < BLOCKS && p < p_end ? bt[p / c.page_size] : -1};
    }
    auto next_rows = [&](int (&row)[MINE]) {  // the rows of the pages looked up last; then the next ones' pages
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        Walk& k = walk[i];
        row[i] = (unsigned)k.page < (unsigned)c.n_pages ? (k.page * c.n_kv + h) * c.page_size + k.off : -1;
        k.p += KP_KEYS;
        k.idx += step_idx;
        k.off += step_off;
        if (k.off >= c.page_size) { k.off -= c.page_size; ++k.idx; }
        k.page = block(i) < BLOCKS && k.p < p_end ? bt[k.idx] : -1;
      }
    };
    uint4 x[MINE][NI];  // the next fill's codes, asked for when the last one's have been stored
    auto load = [&](const void* pool, const int (&row)[MINE]) {
#pragma unroll
      for (int k = 0; k < MINE; ++k) {
        if (block(k) >= BLOCKS) break;
        const uint8_t* src = reinterpret_cast<const uint8_t*>(pool) + ((int64_t)max(row[k], 0) + lrow) * HD + chunk * 16;
#pragma unroll
        for (int i = 0; i < NI; ++i) x[k][i] = *reinterpret_cast<const uint4*>(src + i * RPI * HD);
      }
    };
    // lanes 2 i, 2 i + 1: K's and V's scale of block i; its row
    auto lane_row = [&](const int (&row)[MINE]) {
      int r = -1;
#pragma unroll
      for (int i = 0; i < MINE; ++i)
        if (lane >> 1 == i) r = row[i];
      return r;
    };
    auto load_scale = [&](const int (&row)[MINE]) {
      const int r = lane_row(row);
      return r >= 0 ? ((lane & 1) ? c.v_scales : c.k_scales)[r >> a.log_block] : -1.f;
    };
    const int at0 = lrow * 128 + (chunk >> 2) * Cfg::KB;
    auto store = [&](uint8_t* dst, int j, const int (&row)[MINE]) {
#pragma unroll
      for (int k = 0; k < MINE; ++k) {
        if (block(k) >= BLOCKS) break;
        const int seen = sees_last - (j0 + j) * KP_KEYS - block(k) * 16;  // rows behind may hold anything, as may those without a page
        if (seen < 16 || row[k] < 0)
#pragma unroll
          for (int i = 0; i < NI; ++i)
            if (lrow + i * RPI >= seen || row[k] < 0) x[k][i] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < NI; ++i) kp_put_codes<CODE>(x[k][i], dst + at0 + (block(k) * 16 + i * RPI) * 128, (lrow + i * RPI) & 7, chunk);
      }
    };
    auto ready = [&](uint64_t* bar) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive1(bar);
    };
    // fills in the order K0 K1 V0 K2 V1 ...: the next tile's scores go ahead of this one's outputs
    int row_v[MINE], row_k[MINE];
    next_rows(row_k);
    float scale = load_scale(row_k);
    load(c.k_codes, row_k);
#pragma unroll 1
    for (int f = 0; f < 2 * nt; ++f) {
      // (K?, tile) of a fill
      auto is_key = [&](int i) { return i == 0 || ((i & 1) && i < 2 * nt - 1); };
      auto tile_of = [&](int i) { return is_key(i) ? (i + 1) >> 1 : i == 2 * nt - 1 ? nt - 1 : (i >> 1) - 1; };
      const bool is_k = is_key(f);
      const int j = tile_of(f), s = j & 1;
      if (j >= 2 && !kp_wait_warp(is_k ? &sm.kfree[s] : &sm.vfree[s], (uint32_t)((j / 2 - 1) & 1), abortf)) break;
      int row[MINE];
#pragma unroll
      for (int i = 0; i < MINE; ++i) row[i] = is_k ? row_k[i] : row_v[i];
      store(is_k ? sm.k[s] : sm.v[s], j, row);
      if (is_k) {
        const bool mine = lane < 2 * MINE && block(lane >> 1) < BLOCKS, none = lane_row(row) < 0;
        if (mine) {
          float* at = &sm.sc[j % KP_RING][lane & 1][block(lane >> 1)];
          if ((lane & 1) && scale < KV8_TINY) scale = 0.f;
          const float lv = lg2(scale);
          at[0] = none ? -INFINITY : lane & 1 ? lv : scale;
          if (lane & 1) at[8] = none || scale == 0.f ? 0.f : ex2(-lv);  // undoes what lv does, not the scale itself
        }
        // whether every block has a page and a V scale that is not far from 1
        const bool odd = __any_sync(0xffffffffu, mine && (none || ((lane & 1) && !(scale > KP_NEAR_MIN && scale < KP_NEAR_MAX))));
        if (lane == 0) sm.odd[j % KP_RING][w] = odd;
      }
      ready(is_k ? &sm.kfull[s] : &sm.vfull[s]);
      if (f + 1 == 2 * nt) break;
      const bool next_k = is_key(f + 1);
      if (next_k || tile_of(f + 1) == nt - 1) {  // V follows a tile behind
#pragma unroll
        for (int i = 0; i < MINE; ++i) row_v[i] = row_k[i];
      }
      if (next_k) {
        next_rows(row_k);
        scale = load_scale(row_k);
        load(c.k_codes, row_k);
      } else {
        load(c.v_codes, row_v);
      }
    }
  } else if (warp == KP_MMA_WARP) {
    // ---------------- products ----------------
    // descriptors advance by constants from each tile's first (addresses are in units of 16 bytes)
    const uint64_t qd = umma_desc_sw128(smem_u32(sm.q)), kd = umma_desc_sw128(smem_u32(sm.k[0]));
    const uint64_t vd = umma_desc_mn_sw128(smem_u32(sm.v[0]), Cfg::KB);
    auto scores = [&](int x, int s) {  // S = Q K^T
      const uint64_t q0 = qd + (uint64_t)(x * (KP_ROWS / 2) * 128 / 16), k0 = kd + (uint64_t)(s * Cfg::KV / 16);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          tc_mma_ss<Cfg::IDESC_S>(tmem + Cfg::S0 + x * KP_KEYS, q0 + (uint64_t)(((k >> 2) * Cfg::QB + (k & 3) * 32) / 16),
                                  k0 + (uint64_t)(((k >> 2) * Cfg::KB + (k & 3) * 32) / 16), k > 0);
        tc_commit(&sm.sfull[x]);
        if (x == 1) tc_commit(&sm.kfree[s]);
      }
      __syncwarp();
    };
    auto outputs = [&](int x, int s, bool first) {  // O += P V
      const uint64_t v0 = vd + (uint64_t)(s * Cfg::KV / 16);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < KP_KEYS / 16; ++k)
          tc_mma_ts<Cfg::IDESC_O>(tmem + Cfg::O0 + x * HD, tmem + Cfg::S0 + x * KP_KEYS + k * 8, v0 + (uint64_t)(k * 2048 / 16),
                                  !(first && k == 0));
        if (x == 1) tc_commit(&sm.vfree[s]);
      }
      __syncwarp();
    };
    bool go = nt > 0 && kp_wait_warp(&sm.kfull[0], 0, abortf);
    if (go) {
      tc_fence_after();
      scores(0, 0);
      scores(1, 0);
    }
#pragma unroll 1
    for (int j = 0; go && j < nt; ++j) {
      const int s = j & 1, s1 = s ^ 1;
      const uint32_t ph = (uint32_t)((j / 2) & 1), ph1 = (uint32_t)(((j + 1) / 2) & 1);
      go = kp_wait_warp(&sm.vfull[s], ph, abortf);
#pragma unroll 1
      for (int x = 0; go && x < 2; ++x) {
        go = kp_wait_warp(&sm.pready[x], (uint32_t)(j & 1), abortf);
        if (!go) break;
        tc_fence_after();
        outputs(x, s, j == 0);
        if (j + 1 < nt) {
          if (x == 0) go = kp_wait_warp(&sm.kfull[s1], ph1, abortf);
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
    // ---------------- softmax: warps 0-3 of A, 4-7 of B, a thread a row ----------------
    const int x = warp >> 2, q = warp & 3, r = x * (KP_ROWS / 2) + q * 32 + lane, f = f0 + r;
    const bool live = r < nrow;
    const int vis = live ? (int)min((int64_t)L + f / a.group + 1, (int64_t)cap) : 0;
    const float rm = sm.rowmul[r];
    const uint32_t ts = tmem + ((uint32_t)(q * 32) << 16) + Cfg::S0 + x * KP_KEYS;
    const uint32_t to = tmem + ((uint32_t)(q * 32) << 16) + Cfg::O0 + x * HD;
    float m_ref = -INFINITY, mo_ref = -INFINITY, l = 0.f;
    bool go = true, far = false;
    for (int j = 0; j < nt; ++j) {
      if (!kp_wait_warp(&sm.sfull[x], (uint32_t)(j & 1), abortf)) { go = false; break; }
      tc_fence_after();
      const float* ksc = sm.sc[j % KP_RING][0];
      const float* lvs = sm.sc[j % KP_RING][1];
      const int p0 = (j0 + j) * KP_KEYS;
      const bool masked = p0 + KP_KEYS > sees_all;  // some row of the CTA does not see all of the tile
      const int4 odd4 = *reinterpret_cast<const int4*>(sm.odd[j % KP_RING]);
      if (!masked && !far && !(odd4.x | odd4.y | odd4.z)) {
        kp_softmax<HD>(ts, to, ksc, lvs, rm, j > 0, m_ref, mo_ref, l);
      } else {
        kp_softmax_any<HD>(ts, to, ksc, lvs, rm, masked ? vis - p0 : KP_KEYS, j > 0, m_ref, mo_ref, l);
        far = __any_sync(0xffffffffu, fabsf(mo_ref - m_ref) > KP_NEAR_REFS);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive1(&sm.pready[x]);
    }
    if (go && nt > 0) {
      go = kp_wait_warp(&sm.odone[x], 0, abortf);
      tc_fence_after();
    }
    if (go) {
      // by two factors, whose product may leave fp32's normal range when the answer does not; a NaN query: NaN
      const float s = l == 0.f ? 0.f : 1.f / l, f2 = l == 0.f || mo_ref == -INFINITY ? 0.f : ex2(mo_ref - m_ref);
      const int64_t at = ((int64_t)b * a.tokens + f / a.group) * a.ldo + (int64_t)(h * a.group + f % a.group) * HD;
      const int64_t slot = ((head * a.tail + tile) * a.splits + split) * KP_ROWS + r;
#pragma unroll 1
      for (int cc = 0; cc < HD / 32; ++cc) {
        float v[32];
        if (nt > 0) {
          tc_ld32(to + cc * 32, v);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0.f;
        }
        if (!live) continue;
        if (part) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(a.part + slot * HD + cc * 32 + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else if (a.vec && a.odtype == N730_F32) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + at + cc * 32 + i) =
                make_float4(v[i] * s * f2, v[i + 1] * s * f2, v[i + 2] * s * f2, v[i + 3] * s * f2);
        } else if (a.vec) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y0 = v[i + 2 * e] * s * f2, y1 = v[i + 2 * e + 1] * s * f2;
              if (a.odtype == N730_F16) {
                w[e] = h2u(__floats2half2_rn(y0, y1));
              } else {
                const __nv_bfloat162 y = __floats2bfloat162_rn(y0, y1);
                w[e] = *reinterpret_cast<const uint32_t*>(&y);
              }
            }
            *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + at + cc * 32 + i) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) kv8_store1(a.out, at + cc * 32 + i, a.odtype, v[i] * s * f2);
        }
      }
      if (live && part) reinterpret_cast<float4*>(a.part_ml)[slot] = make_float4(mo_ref, m_ref, l, 0.f);
      if (live && a.lse && !part) a.lse[head * a.rows + f] = l == 0.f ? INFINITY : m_ref + log2f(l);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (*abortf) kp_give_up(&sm.drain, warp == KP_MMA_WARP, a.status);
  if (warp == KP_MMA_WARP)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(Cfg::TMEM) : "memory");
}

// ---------------------------------------------------------------------------
// accumulated weights of a prompt: w[b, h, p] += sum over the KV head's rows of exp2(score - lse)
// ---------------------------------------------------------------------------
// A CTA walks over the rows that see its 128 positions of a KV head, 128 at a time, and forms
// S^T = K Q^T, so that a position is a TMEM lane and its sum over the rows stays in one thread: warps 8-15
// bring the rows' queries into shared memory, warp 16 issues the products, warps 0-3 sum the even row
// tiles, 4-7 the odd ones.  Where the positions give the SMs too few CTAs, a cluster of them shares the rows and
// the first adds up the sums, always in the same order.  Bound by latency: a tile's rows pass a loader, the products
// and the sums one behind the other.  4 prompts of 300 tokens, 14 / 2 heads x 64, 6 tiles of positions: 62 us with one
// CTA for all rows and four warps that bring them, 20 us with three CTAs and eight.
template <int HD>
struct KWSmem {
  uint8_t k[KPCfg<HD>::KV];
  uint8_t q[2][KPCfg<HD>::KV];
  float2 row[2][KP_KEYS];    // multiplier, lse
  float sum[KP_KEYS];
  uint64_t qfull[2], qfree[2], sfull[2], sread[2], drain;
  uint32_t tmem;
  int abort;
};

template <int HD, int CODE>
__global__ void __launch_bounds__(KW_THREADS, 1)
kv8_prompt_weights_kernel(const KPArgs a, const float* w_in, float* w_out, int64_t ldw) {
  using Cfg = KPCfg<HD>;
  constexpr int RT = KP_KEYS;               // rows of a tile
  constexpr uint32_t COLS = 2 * RT;         // tensor memory: two score tiles
  extern __shared__ __align__(1024) uint8_t kp_raw[];
  KWSmem<HD>& sm = *reinterpret_cast<KWSmem<HD>*>(aligned_smem(kp_raw));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const N730KV8Cache& c = a.c;
  const int b = blockIdx.z, h = blockIdx.y, rank = blockIdx.x % a.shares, p0 = blockIdx.x / a.shares * KP_KEYS;
  const int cap = c.max_pages * c.page_size;
  // all but lse was there before the attention's grid, which lets this one start when all of it holds its tensor memory
  const int L = kv8_len(a.lens, b, cap), n_new = kv8_new(a.n_new, b, a.tokens), rows = n_new * a.group;
  const int total = (int)min((int64_t)L + n_new, (int64_t)cap);
  if (p0 >= total) {  // the whole cluster
    pdl_wait();
    return;
  }
  const int64_t head = (int64_t)b * c.n_kv + h;
  // row tiles from the first whose last row sees position p0; this CTA's are [i0, i0 + n)
  const int t0 = max(0, p0 - L) * a.group / RT, nt = (rows + RT - 1) / RT - t0;
  const int i0 = t0 + nt * rank / a.shares, n = t0 + nt * (rank + 1) / a.shares - i0;
  const int* bt = c.block_table + (int64_t)b * c.max_pages;
  auto row_of = [&](int p) -> int64_t {
    if (p >= total) return -1;
    const int page = bt[p / c.page_size];
    return (unsigned)page < (unsigned)c.n_pages ? ((int64_t)page * c.n_kv + h) * c.page_size + p % c.page_size : -1;
  };
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.qfull[i], KW_ROW_WARPS);
      mbar_init(&sm.qfree[i], 1);
      mbar_init(&sm.sfull[i], 1);
      mbar_init(&sm.sread[i], 4);
    }
    mbar_init(&sm.drain, 1);
    fence_mbar_init();
    sm.abort = 0;
  }
  if (warp == KW_MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_u32(&sm.tmem)), "r"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  for (int i = tid; i < KP_KEYS * (HD / 16); i += KW_THREADS) {
    const int r = i / (HD / 16), chunk = i % (HD / 16);
    const int64_t row = row_of(p0 + r);
    kp_put_codes<CODE>(row >= 0 ? *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(c.k_codes) + row * HD + chunk * 16)
                                : make_uint4(0, 0, 0, 0), sm.k + (chunk >> 2) * Cfg::KB + r * 128, r & 7, chunk);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  volatile int* abortf = &sm.abort;
  float sum = 0.f;

  pdl_wait();
  if (warp >= 8 && warp < KW_MMA_WARP) {
    // a warp's rows at once: the next tile's are on their way during this one's products
    constexpr int WR = RT / KW_ROW_WARPS, U = WR / KPRows<HD>::RPI;
    const int w0 = (warp - 8) * WR;
    uint4 x[U];
    float lse;
    auto load = [&](int i) {
      const int first = (i0 + i) * RT;
      kp_load_rows<HD, U>(a.q, a.qvec, w0, [&](int r) -> int64_t {
        const int f = first + r;
        return f < rows ? ((int64_t)b * a.tokens + f / a.group) * a.ldq + (int64_t)(h * a.group + f % a.group) * HD : -1;
      }, x);
      const int f = first + w0 + lane;
      lse = lane < WR && f < rows ? a.lse[head * a.rows + f] : INFINITY;
    };
    if (n > 0) load(0);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int s = i & 1;
      // the products of the tile before are done, and its factors read
      if (i >= 2 && !(kp_wait_warp(&sm.qfree[s], (uint32_t)((i / 2 - 1) & 1), abortf) &&
                      kp_wait_warp(&sm.sread[s], (uint32_t)((i / 2 - 1) & 1), abortf)))
        break;
      kp_put_rows<HD, U>(x, a.dtype, a.sign, a.scale_log2e, sm.q[s], Cfg::KB, w0, [&](int r, float mul) { sm.row[s][r].x = mul; });
      if (lane < WR) sm.row[s][w0 + lane].y = lse;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive1(&sm.qfull[s]);
      if (i + 1 < n) load(i + 1);
    }
  } else if (warp == KW_MMA_WARP) {
    const uint64_t kd = umma_desc_sw128(smem_u32(sm.k)), qd = umma_desc_sw128(smem_u32(sm.q[0]));
    bool go = true;
#pragma unroll 1
    for (int i = 0; go && i < n; ++i) {
      const int s = i & 1;
      go = kp_wait_warp(&sm.qfull[s], (uint32_t)((i / 2) & 1), abortf);  // implies that the scores before in this buffer are read
      if (!go) break;
      tc_fence_after();
      const uint64_t q0 = qd + (uint64_t)(s * Cfg::KV / 16);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint64_t at = (uint64_t)(((k >> 2) * Cfg::KB + (k & 3) * 32) / 16);
          tc_mma_ss<Cfg::IDESC_S>(tmem + s * RT, kd + at, q0 + at, k > 0);
        }
        tc_commit(&sm.qfree[s]);
        tc_commit(&sm.sfull[s]);
      }
      __syncwarp();
    }
  } else {
    const int x = warp >> 2, q = warp & 3, p = p0 + q * 32 + lane;
    const int64_t row = row_of(p);
    const float ks = row >= 0 ? c.k_scales[row / c.block] : 0.f;
    const uint32_t ts = tmem + ((uint32_t)(q * 32) << 16) + x * RT;
    for (int i = x; i < n; i += 2) {
      if (!kp_wait_warp(&sm.sfull[x], (uint32_t)((i / 2) & 1), abortf)) break;
      tc_fence_after();
      const int f0 = (i0 + i) * RT;
      const int first_seen = p0 + KP_KEYS - 1 <= L + f0 / a.group ? 0 : max(0, p - L) * a.group - f0;  // rows before it do not see p
#pragma unroll 1
      for (int cc = 0; cc < RT / 32; ++cc) {
        float v[32];
        tc_ld32(ts + cc * 32, v);
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float2 m = sm.row[x][cc * 32 + e];
          const float y = ex2(fmaf(v[e] * ks, m.x, -m.y));
          sum += cc * 32 + e < first_seen ? 0.f : y;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive1(&sm.sread[x]);
    }
    if (row < 0) sum = 0.f;
    if (x == 1) sm.sum[q * 32 + lane] = sum;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (*abortf) kp_give_up(&sm.drain, warp == KW_MMA_WARP, a.status);
  if (tid < KP_KEYS) sm.sum[tid] += sum;
  if (a.shares > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank == 0 && tid < KP_KEYS && p0 + tid < total) {
    const int p = p0 + tid;
    float all = sm.sum[tid];
    for (int k = 1; k < a.shares; ++k) {
      uint32_t at;
      float other;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&sm.sum[tid])), "r"(k));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other) : "r"(at) : "memory");
      all += other;
    }
    w_out[head * ldw + p] = (w_in && p < L ? w_in[head * ldw + p] : 0.f) + all;
  }
  __syncwarp();
  // the others' shared memory stays until it is read
  if (a.shares > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp == KW_MMA_WARP)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(COLS) : "memory");
}

KV8PromptPlan kv8_prompt_plan(const N730KV8Cache& c, int batch, int tokens, int heads) {
  KV8PromptPlan p{};
  p.rows = tokens * (heads / c.n_kv);
  p.tiles = (p.rows + KP_ROWS - 1) / KP_ROWS;
  p.rg = KP_ROWS;
  const int64_t items = (int64_t)batch * c.n_kv;
  const int64_t key_tiles = ((int64_t)c.max_pages * c.page_size + KP_KEYS - 1) / KP_KEYS;
  // CTAs of a cluster that share the rows of 128 positions' weights, two row tiles each at least, and no more than the
  // table's positions leave SMs for: in a wide table one (4 prompts of 300 tokens, 14 / 2 heads x 64, whole call, 42.4 us in
  // a table of 704 positions, 66.9 in 8192, 78 in 65536, where the grid's CTAs behind the last position count as well)
  const int64_t idle = num_sms() / (items * key_tiles);
  p.shares = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(KW_SHARES, idle), p.rows / (2 * KP_KEYS)));
  // The last, partial wave of CTAs (or the only one) leaves SMs idle: its tiles' positions are cut into as many shares
  // as there are SMs, of four tiles at least (of the table's here, of those that a row tile sees on the device).  2048
  // tokens behind 6144 positions, 64 / 8 heads, 3.46 waves: 614 us without, 578 with; shares of three tiles (4 prompts of
  // 300 tokens, 700 positions) 49.8 us for 42.3 without.
  p.splits = 1;
  const int64_t tail = (items * p.tiles % num_sms() + items - 1) / items;
  while (tail && tail * items * (p.splits + 1) <= num_sms() && key_tiles / (p.splits + 1) >= 4) ++p.splits;
  p.tail = p.splits > 1 ? (int)tail : 0;
  return p;
}

static KPArgs kp_args(const KV8AttnCall& k, const KV8PromptPlan& p, int* status, float* part, float* part_ml, float* lse) {
  KPArgs a{};
  a.c = k.c;
  a.q = k.q; a.out = k.out; a.ldq = k.ldq; a.ldo = k.ldo; a.dtype = k.dtype; a.odtype = k.out_dtype;
  a.tokens = k.tokens; a.group = k.heads / k.c.n_kv; a.rows = p.rows; a.tiles = p.tiles; a.splits = p.splits; a.tail = p.tail; a.batch = k.batch; a.shares = p.shares;
  a.vec = ((uintptr_t)k.out & 15) == 0 && k.ldo * kv8_esize(k.out_dtype) % 16 == 0;
  a.qvec = ((uintptr_t)k.q & 15) == 0 && k.ldq * kv8_esize(k.dtype) % 16 == 0;
  a.scale_log2e = fabsf(k.scale) * 1.4426950408889634f;
  a.sign = k.scale < 0.f ? -1.f : 1.f;
  a.lens = k.lens; a.n_new = k.n_new;
  a.log_block = k.c.block == 16 ? 4 : k.c.block == 32 ? 5 : 6;
  a.status = status; a.part = part; a.part_ml = part_ml; a.lse = lse;
  return a;
}

template <int HD, int CODE>
static int prompt_launch(const KPArgs& a, bool pdl, cudaStream_t st) {
  const size_t smem = sizeof(KPSmem<HD>) + 1024;
  if (int rc = smem_attr_once<kv8_prompt_kernel<HD, CODE>>((int)smem)) return rc;
  return kv8_launch(kv8_prompt_kernel<HD, CODE>, dim3((a.tiles + a.tail * (a.splits - 1)) * a.batch * a.c.n_kv), dim3(KP_THREADS), smem, st, pdl, a);
}
template <int HD, int CODE>
static int prompt_weights_launch(const KPArgs& a, const KV8AttnCall& k, cudaStream_t st) {
  const size_t smem = sizeof(KWSmem<HD>) + 1024;
  if (int rc = smem_attr_once<kv8_prompt_weights_kernel<HD, CODE>>((int)smem)) return rc;
  const int cap = a.c.max_pages * a.c.page_size;
  return kv8_launch_cluster(kv8_prompt_weights_kernel<HD, CODE>, dim3((cap + KP_KEYS - 1) / KP_KEYS * a.shares, a.c.n_kv, k.batch),
                            a.shares, dim3(KW_THREADS), smem, st, a.splits == 1, a, k.w_in, k.w_out, k.ldw);
}

int kv8_prompt_launch(const KV8AttnCall& k, const KV8PromptPlan& p, int* status, float* part, float* part_ml, float* lse,
                      cudaStream_t st) {
  const KPArgs a = kp_args(k, p, status, part, part_ml, lse);
  const bool i8 = k.c.code == N730_KV8_INT8;
  if (k.c.head_dim == 128)
    return i8 ? prompt_launch<128, N730_KV8_INT8>(a, k.pdl, st) : prompt_launch<128, N730_KV8_E4M3>(a, k.pdl, st);
  return i8 ? prompt_launch<64, N730_KV8_INT8>(a, k.pdl, st) : prompt_launch<64, N730_KV8_E4M3>(a, k.pdl, st);
}

int kv8_prompt_weights_launch(const KV8AttnCall& k, const KV8PromptPlan& p, int* status, float* lse, cudaStream_t st) {
  const KPArgs a = kp_args(k, p, status, nullptr, nullptr, lse);
  const bool i8 = k.c.code == N730_KV8_INT8;
  if (k.c.head_dim == 128)
    return i8 ? prompt_weights_launch<128, N730_KV8_INT8>(a, k, st) : prompt_weights_launch<128, N730_KV8_E4M3>(a, k, st);
  return i8 ? prompt_weights_launch<64, N730_KV8_INT8>(a, k, st) : prompt_weights_launch<64, N730_KV8_E4M3>(a, k, st);
}

}  // namespace n730
