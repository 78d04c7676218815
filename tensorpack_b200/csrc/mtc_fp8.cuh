// Device helpers of the 8-bit (e4m3) kernels: the quantization of one group
// of 128 values, tcgen05 kind::f8f6f4 with fp32 accumulators in TMEM, TMEM
// loads that are waited for separately, and the token tiles ("slots") that
// dense and grouped products share.
//
// Format.  A weight matrix of K inputs and N outputs is stored as N rows of
// K codes (one row per output feature) with one fp32 scale per 128 x 128
// block; activations are rows of K codes with one fp32 scale per row and 128
// inputs.  A product is a sum over blocks of 128 inputs,
//   Y[m][n] = sum_b sx[m][b] sw[n / 128][b] sum_{k in block b} qx[m][k] qw[n][k],
// whose inner sum the tensor cores leave in TMEM; CUDA cores multiply it by
// the two scales and add it up in fp32 registers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "mtc_common.cuh"
#include "mtc_tc.cuh"

namespace mtc {
namespace fp8 {

constexpr int kBlock = 128;                   // inputs (and outputs) per scale
constexpr float kMax = 448.0f;                // largest e4m3 value
constexpr uint32_t kFloorBits = 27u << 23;    // 2^-100: amax below this is raised to it
constexpr uint32_t kInfBits = 0x7f800000u;

// The scale of a group and the factor its values are multiplied by, from the
// bits of its largest |x| (unsigned order of the bits is the order of the
// values, with infinity and NaN above every number).  amax / 448 and
// 448 / amax are both rounded once; a group holding an infinity or a NaN gets
// a NaN scale and zero codes, so that its row of every product is NaN.
struct GroupScale {
  float scale, mul;
};
__device__ __forceinline__ GroupScale group_scale(uint32_t amax_bits) {
  GroupScale g;
  if (amax_bits >= kInfBits) {
    g.scale = __uint_as_float(0x7fffffffu);
    g.mul = 0.0f;
  } else {
    const float a = __uint_as_float(amax_bits < kFloorBits ? kFloorBits : amax_bits);
    g.scale = __fdiv_rn(a, kMax);
    g.mul = __fdiv_rn(kMax, a);
  }
  return g;
}

// Two codes e4m3(a * mul), e4m3(b * mul): round to nearest even, saturating
// at 448 (a * mul can exceed it by one rounding).  mul = 0 marks a group that
// is not finite.
__device__ __forceinline__ uint32_t codes2(float a, float b, float mul) {
  return __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(a, mul), __fmul_rn(b, mul)), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float mul) {
  if (mul == 0.0f) return make_uint2(0u, 0u);
  uint2 r;
  r.x = codes2(v[0], v[1], mul) | codes2(v[2], v[3], mul) << 16;
  r.y = codes2(v[4], v[5], mul) | codes2(v[6], v[7], mul) << 16;
  return r;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t amax8(const float (&v)[8]) {
  uint32_t m = abs_bits(v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max(m, abs_bits(v[i]));
  return m;
}
// Largest over the 16 lanes of a half warp.
__device__ __forceinline__ uint32_t half_warp_max(uint32_t m) {
#pragma unroll
  for (int d = 8; d; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  return m;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

// Starts bringing `bytes` (a multiple of 16) at the 16-byte aligned p into L2.
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
  if (bytes) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// 16 bytes at p, or zeros: one predicated load, so that several are in flight.
__device__ __forceinline__ uint4 load16_if(const uint4* p, bool on) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.u32 q, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@q ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"((uint32_t)on));
  return v;
}
// Eight values from one (16-bit types) or two (fp32) such vectors.
template <typename T, int NV>
__device__ __forceinline__ void unpack8(const uint4 (&raw)[NV], float (&v)[8]) {
  static_assert(NV * 16 == 8 * sizeof(T), "eight values");
  const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[NV - 1].x, raw[NV - 1].y, raw[NV - 1].z,
                         raw[NV - 1].w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      T lo, hi;
      *reinterpret_cast<uint16_t*>(&lo) = (uint16_t)(w[i] & 0xffffu);
      *reinterpret_cast<uint16_t*>(&hi) = (uint16_t)(w[i] >> 16);
      v[2 * i] = to_f32(lo);
      v[2 * i + 1] = to_f32(hi);
    }
  }
}

// Bits of the largest |value| among those, as fp32.  (The order of 16-bit
// values without their sign is that of their bits, too: two at a time.)
template <typename T, int NV>
__device__ __forceinline__ uint32_t amax_raw(const uint4 (&raw)[NV]) {
  if constexpr (sizeof(T) == 4) {
    float v[8];
    unpack8<T>(raw, v);
    return amax8(v);
  } else {
    const uint4 r = raw[0];
    const uint32_t m = __vmaxu2(__vmaxu2(r.x & 0x7fff7fffu, r.y & 0x7fff7fffu), __vmaxu2(r.z & 0x7fff7fffu, r.w & 0x7fff7fffu));
    const uint16_t top = (uint16_t)max(m & 0xffffu, m >> 16);
    T x;
    *reinterpret_cast<uint16_t*>(&x) = top;
    return __float_as_uint(to_f32(x));
  }
}

// Eight consecutive values at p as fp32; `n` of them exist (the others read
// as zero).  One at a time: for rows that start or end off a vector.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.0f;
}

// One output value in the output's type (fp32, or rounded once to nearest).
__device__ __forceinline__ void store1(void* y, int dt, long long i, float v) {
  if (dt == MTC_F32) reinterpret_cast<float*>(y)[i] = v;
  else if (dt == MTC_BF16) reinterpret_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(y)[i] = __float2half_rn(v);
}
__device__ __forceinline__ uint32_t pack2(int dt, float a, float b) {
  if (dt == MTC_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 2^x and 1 / x by the special function unit (2^-22 relative, 1 ulp);
// denormal results are zero, which saves their handling and, next to the 1
// below, changes nothing.
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The larger of a and |b|, NaN if one of them is.
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

// Activations in a few instructions, to be unrolled over a thread's sums: the
// many-row kernel's epilogue.  (The relative error of the exponential grows
// with |x|, but the result is then next to 0 or x.)  SiLU is x / (1 +
// 2^(-x log2 e)); GELU (tanh form) x / (1 + exp(-2 u)) with u = sqrt(2 / pi)
// (x + 0.044715 x^3), since (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)).
template <int ACT>
__device__ __forceinline__ float act_fast(float x) {
  constexpr float kLog2e = 1.4426950408889634f, kTwoRoot = 1.5957691216057308f;  // log2 e, 2 sqrt(2 / pi)
  if constexpr (ACT == MTC_ACT_RELU) return x < 0.0f ? 0.0f : x;
  else if constexpr (ACT == MTC_ACT_SILU) return x * rcp_fast(1.0f + exp2_fast(-kLog2e * x));
  else if constexpr (ACT == MTC_ACT_GELU_TANH)
    return x * rcp_fast(1.0f + exp2_fast(-x * fmaf(kLog2e * kTwoRoot * 0.044715f, x * x, kLog2e * kTwoRoot)));
  else return x;
}

// ---------------------------------------------------------------------------
// tcgen05, 8-bit operands
// ---------------------------------------------------------------------------
// Instruction descriptor for kind::f8f6f4: e4m3 A and B, fp32 D, both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// D (TMEM) = or += A B^T for 32 inputs; operands by shared-memory descriptor.
__device__ __forceinline__ void mma_e4m3_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 lanes x 16 consecutive fp32 columns, not waited for: thread i gets lane
// (base + i).  tmem_wait16 completes it and ties the registers to the wait.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait16(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]),
                 "+r"(v[15])
               :
               : "memory");
}

// 4-byte asynchronous copy global -> shared memory, and this thread's arrival
// (counted like any other) on `bar` once all its earlier ones have landed.
__device__ __forceinline__ void copy4_async(float* dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Registers per thread of a warpgroup, after the launch.
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Two fp32 values in a register pair: acc += v * s with one instruction for
// both.  Accumulators are kept as pairs throughout, so that no moves are
// needed to form them.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ f32x2 pair(uint32_t lo, uint32_t hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ void unpair(f32x2 x, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
}
__device__ __forceinline__ void fma2(f32x2& acc, f32x2 v, f32x2 s) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(v), "l"(s));
}

// ---------------------------------------------------------------------------
// Token tiles
// ---------------------------------------------------------------------------
// Slots of a grouped product: a list written by the plan kernel (word 0 is
// their number, slot i is {expert, first row, end row of the expert, 0} at
// words 4 + 4 i), or, for a single token (ids, experts > 0), one slot per row
// with the row's expert, or none of its rows if that is no expert.  (Read
// from L2: a product may read them before its predecessor in the stream has
// ended.)  A dense product has neither: slot i covers rows from i * size of
// the single matrix.
struct Slot {
  int e, row0, end;
};
__device__ __forceinline__ int slot_count(const int32_t* slots, int experts, int M, int size) {
  return experts ? M : slots ? __ldcg(slots) : (M + size - 1) / size;
}
__device__ __forceinline__ Slot slot_at(const int32_t* slots, int experts, int M, int size, int i) {
  Slot s;
  if (experts) {
    const int e = __ldcg(slots + i);
    const bool ok = (unsigned)e < (unsigned)experts;
    s.e = ok ? e : 0;
    s.row0 = i;
    s.end = ok ? i + 1 : i;
  } else if (slots) {
    const int4 v = __ldcg(reinterpret_cast<const int4*>(slots + 4 + 4 * i));
    s.e = v.x;
    s.row0 = v.y;
    s.end = v.z;
  } else {
    s.e = 0;
    s.row0 = i * size;
    s.end = M;
  }
  return s;
}

}  // namespace fp8
}  // namespace mtc
