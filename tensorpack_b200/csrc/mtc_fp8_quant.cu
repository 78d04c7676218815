// Activations and weights to e4m3 codes, weights back to fp32, and the dense
// product entry point.
#include "mtc_fp8.cuh"
#include "mtc_fp8_internal.h"

namespace mtc {
namespace fp8 {
namespace {

struct QuantParams {
  const void* X;
  int M, K, Kb;
  long long ldx;
  const int32_t* pos;
  int copies;
  uint8_t* q;
  long long ldq;
  float* s;
  long long lds;
};

// Eight codes of a row of which `left` values exist (VEC: all or none).
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* q, const uint2& c, int left) {
  if (left >= 8) {
    *reinterpret_cast<uint2*>(q) = c;
  } else if (!VEC) {
    for (int i = 0; i < left; ++i) q[i] = (uint8_t)((i < 4 ? c.x >> (8 * i) : c.y >> (8 * i - 32)) & 0xffu);
  }
}

// One half warp per group of 128 inputs, 8 values per lane, U groups at a
// time: their loads are in flight together, their maxima reduced together, and
// lane u of the half warp divides for group u alone.  Bound by memory:
// 4096 x 14336 fp32 takes 49.9 us (5.9 TB/s; 64.3 us one group at a time with
// every lane dividing); bf16 39.3 us, bound by instruction issue (43.0 with
// the maxima of 16-bit values one at a time).  U = 1 when a half warp has one group at most:
// 333 x 4864 fp16 and the product after it take 17.0 us, 19.2 with U = 4.
template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(256) quantize_kernel(const QuantParams p) {
  constexpr int kVec = sizeof(T) == 4 ? 2 : 1;
  const int half = threadIdx.x >> 4, l = threadIdx.x & 15;
  griddep_wait();
  griddep_launch_dependents();
  const long long groups = (long long)p.M * p.Kb;
  const long long step = (long long)gridDim.x * 16;
  const long long last = (groups + 15) & ~15ll;  // whole warps take part in the shuffles
  const int step_m = (int)(step / p.Kb), step_b = (int)(step - (long long)step_m * p.Kb);
  long long g = (long long)blockIdx.x * 16 + half;
  int m = (int)(g / p.Kb), b = (int)(g - (long long)m * p.Kb);
  while (g < last) {
    int mm[U], bb[U];
    float v[U][8];
    uint4 raw[U][kVec];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mm[u] = g < groups ? m : -1;
      bb[u] = b;
      const int k = b * kBlock + 8 * l;
      const T* x = reinterpret_cast<const T*>(p.X) + m * p.ldx + k;
      const int n = mm[u] >= 0 ? p.K - k : 0;
      if (VEC) {
        // (rows of whole groups of 8: a lane has all of its values or none)
#pragma unroll
        for (int q = 0; q < kVec; ++q) raw[u][q] = load16_if(reinterpret_cast<const uint4*>(x) + q, n > 0);
      } else {
        load8(x, n, v[u]);
      }
      g += step;
      m += step_m;
      b += step_b;
      if (b >= p.Kb) {
        b -= p.Kb;
        ++m;
      }
    }
    uint32_t am[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (VEC && U > 1) {
        am[u] = amax_raw<T>(raw[u]);
      } else {
        if (VEC) unpack8<T>(raw[u], v[u]);
        am[u] = amax8(v[u]);
      }
    }
#pragma unroll
    for (int d = 8; d; d >>= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) am[u] = max(am[u], __shfl_xor_sync(0xffffffffu, am[u], d));
    uint32_t mine = am[0];
#pragma unroll
    for (int u = 1; u < U; ++u) mine = (l & (U - 1)) == u ? am[u] : mine;
    const GroupScale gs = group_scale(mine);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (VEC && U > 1) unpack8<T>(raw[u], v[u]);
      const uint2 c = codes8(v[u], __shfl_sync(0xffffffffu, gs.mul, u, 16));
      if (mm[u] < 0) continue;
      const int k = bb[u] * kBlock + 8 * l;
      if (p.pos) {
        for (int j = 0; j < p.copies; ++j) {
          const int r = p.pos[(long long)mm[u] * p.copies + j];
          if (r < 0) continue;
          store_codes<VEC>(p.q + (long long)r * p.ldq + k, c, p.K - k);
          if (l == u) p.s[(long long)bb[u] * p.lds + r] = gs.scale;
        }
      } else {
        store_codes<VEC>(p.q + (long long)mm[u] * p.ldq + k, c, p.K - k);
        if (l == u) p.s[(long long)bb[u] * p.lds + mm[u]] = gs.scale;
      }
    }
  }
}

// One 128 x 128 block of W (K x N fp32, row-major) to codes (N rows of K) and its scale.
__global__ void __launch_bounds__(256) pack_kernel(const float* __restrict__ W, int K, int N, long long ldw,
                                                   uint8_t* __restrict__ codes, long long ldk,
                                                   float* __restrict__ scales, int Kb) {
  __shared__ uint32_t red[8];
  __shared__ uint8_t tile[128][132];
  const int k0 = blockIdx.x * 128, n0 = blockIdx.y * 128;
  const int tn = threadIdx.x & 127, tk = threadIdx.x >> 7;
  uint32_t m = 0;
  for (int k = tk; k < 128; k += 2)
    if (k0 + k < K && n0 + tn < N) m = max(m, abs_bits(W[(long long)(k0 + k) * ldw + n0 + tn]));
  for (int d = 16; d; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int i = 0; i < 8; ++i) m = max(m, red[i]);
  const GroupScale g = group_scale(m);
  if (threadIdx.x == 0) scales[(long long)blockIdx.y * Kb + blockIdx.x] = g.scale;
  for (int k = tk; k < 128; k += 2) {
    float v = 0.0f;
    if (k0 + k < K && n0 + tn < N) v = W[(long long)(k0 + k) * ldw + n0 + tn];
    tile[tn][k] = g.mul == 0.0f ? 0 : (uint8_t)(codes2(v, 0.0f, g.mul) & 0xffu);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 128 * 128; i += 256) {
    const int n = i >> 7, k = i & 127;
    if (n0 + n < N && k0 + k < ldk) codes[(long long)(n0 + n) * ldk + k0 + k] = tile[n][k];
  }
}

// out[k][n] = code * scale, fp32 (one rounding).
__global__ void __launch_bounds__(256) unpack_kernel(const uint8_t* __restrict__ codes, long long ldk,
                                                     const float* __restrict__ scales, int K, int N, int Kb,
                                                     float* __restrict__ out, long long ldo) {
  __shared__ uint8_t tile[128][132];
  const int k0 = blockIdx.x * 128, n0 = blockIdx.y * 128;
  for (int i = threadIdx.x; i < 128 * 128; i += 256) {
    const int n = i >> 7, k = i & 127;
    tile[n][k] = (n0 + n < N && k0 + k < K) ? codes[(long long)(n0 + n) * ldk + k0 + k] : 0;
  }
  __syncthreads();
  const float s = scales[(long long)blockIdx.y * Kb + blockIdx.x];
  for (int i = threadIdx.x; i < 128 * 128; i += 256) {
    const int k = i >> 7, n = i & 127;
    if (n0 + n < N && k0 + k < K) {
      __nv_fp8_e4m3 c;
      c.__x = tile[n][k];
      out[(long long)(k0 + k) * ldo + n0 + n] = __fmul_rn((float)c, s);
    }
  }
}

}  // namespace

int launch_quantize(const QuantRows& a, cudaStream_t st, const char* who) {
  if (a.M == 0) return MTC_OK;
  QuantParams p = {};
  p.X = a.X;
  p.M = a.M;
  p.K = a.K;
  p.Kb = (a.K + kBlock - 1) / kBlock;
  p.ldx = a.ldx;
  p.pos = a.pos;
  p.copies = a.copies;
  p.q = a.q;
  p.ldq = a.ldq;
  p.s = a.s;
  p.lds = a.lds;
  // whole vectors: rows that start on 16 bytes and hold a multiple of 8 values
  const bool vec = (reinterpret_cast<uintptr_t>(a.X) & 15) == 0 && a.ldx % (a.dt == MTC_F32 ? 4 : 8) == 0 && a.K % 8 == 0;
  const int sms = sm_count();
  MTC_REQUIRE(sms > 0, "%s: no CUDA device", who);
  // 8 CTAs of 256 threads per SM hold all that fits; more groups than their
  // half warps are taken several at a time
  const long long blocks = ((long long)a.M * p.Kb + 15) / 16;
  const bool many = blocks > 8ll * sms;
  const int grid = (int)(many ? 8ll * sms : blocks);
  void (*kernel)(QuantParams);
#define MTC_PICK(T, U) \
  (vec ? (many ? quantize_kernel<T, true, U> : quantize_kernel<T, true, 1>) \
       : (many ? quantize_kernel<T, false, U> : quantize_kernel<T, false, 1>))
  if (a.dt == MTC_F32) kernel = MTC_PICK(float, 2);
  else if (a.dt == MTC_BF16) kernel = MTC_PICK(__nv_bfloat16, 4);
  else kernel = MTC_PICK(__half, 4);
#undef MTC_PICK
  MTC_CHECK_CUDA(launch_chained(kernel, dim3(grid), dim3(256), 0, st, 1, p), who);
  return MTC_OK;
}

namespace {
// How a dense product runs.  Times on the device, weights from memory.
//  * Up to 8 rows the product quantizes the activations itself: 13.7 us at
//    8 x 4096 x 14336 against 15.1 with the quantizer before it (its codes
//    are loaded like the weights); 17.8 against 15.6 with 10 rows.
//  * The kernel for few rows takes them in tiles that waste at most half of
//    the MMA.  From 65 rows on the 128 x 256 tiles take over where the few
//    kernel could not split its inputs any more, that is, where its 128 x 128
//    tiles fill more than half of the SMs: 25 against 48 us at
//    129 x 4096 x 14336, 17.2 / 18.7 at 256 x 2048 x 8192 (128 tiles), but
//    23.0 / 18.5 at 200 x 4096 x 4096 (64), 16.6 / 14.9 at 128 x 2048 x 8192
//    (64), 12.3 / 12.6 at 700 x 1024 x 1536 (72) and 27 / 14.1 at
//    333 x 4864 x 901 (24).
struct DensePlan {
  int tile;
  bool many, raw;
  long long ldq, lds;
  size_t q_bytes, bytes;
};
DensePlan dense_plan(int M, int K, int N, int sms) {
  DensePlan d;
  d.many = M > 64 && 2ll * ((M + 127) / 128) * ((N + 127) / 128) > sms;
  d.tile = M > 64 ? 128 : M > 32 ? 64 : M > 16 ? 32 : 16;
  d.raw = M <= 8;
  d.ldq = (K + 15) & ~15ll;
  d.lds = (M + 3) & ~3ll;
  d.q_bytes = d.raw ? 0 : (((size_t)M * d.ldq + 255) & ~(size_t)255);
  d.bytes = d.raw ? 0 : d.q_bytes + (size_t)((K + 127) / 128) * d.lds * 4;
  return d;
}
}  // namespace

}  // namespace fp8
}  // namespace mtc

using namespace mtc;
using namespace mtc::fp8;

extern "C" int mtc_fp8_pack(const float* W, int32_t K, int32_t N, int64_t ldw, uint8_t* codes, int64_t ldk,
                            float* scales, void* stream) {
  clear_error();
  MTC_REQUIRE(W && codes && scales, "mtc_fp8_pack: null pointer");
  MTC_REQUIRE(aligned(W) && aligned(scales), "mtc_fp8_pack: pointer not aligned to its elements");
  MTC_REQUIRE(K >= 1 && N >= 1 && ldw >= N && ldk >= K && (ldk & 15) == 0, "mtc_fp8_pack: bad shape or strides");
  const dim3 grid((K + 127) / 128, (N + 127) / 128);
  MTC_REQUIRE(grid.y <= 65535, "mtc_fp8_pack: N=%d too large", N);
  pack_kernel<<<grid, 256, 0, as_stream(stream)>>>(W, K, N, ldw, codes, ldk, scales, grid.x);
  MTC_CHECK_LAUNCH("mtc_fp8_pack");
  return MTC_OK;
}

extern "C" int mtc_fp8_unpack(const mtc_fp8_matrix* w, int32_t e, float* out, int64_t ldo, void* stream) {
  clear_error();
  const int rc = check_matrix(w, "mtc_fp8_unpack");
  if (rc != MTC_OK) return rc;
  MTC_REQUIRE(out && ldo >= w->N && e >= 0 && e < w->E, "mtc_fp8_unpack: bad argument");
  MTC_REQUIRE(aligned(out), "mtc_fp8_unpack: pointer not aligned to its elements");
  const dim3 grid((w->K + 127) / 128, (w->N + 127) / 128);
  MTC_REQUIRE(grid.y <= 65535, "mtc_fp8_unpack: N=%d too large", w->N);
  unpack_kernel<<<grid, 256, 0, as_stream(stream)>>>(w->codes + (long long)e * w->N * w->ldk, w->ldk,
                                                     w->scales + (long long)e * grid.x * grid.y, w->K, w->N, grid.x,
                                                     out, ldo);
  MTC_CHECK_LAUNCH("mtc_fp8_unpack");
  return MTC_OK;
}

extern "C" int mtc_fp8_quantize(const void* X, int32_t x_type, int32_t M, int32_t K, int64_t ldx, uint8_t* codes,
                                int64_t ldq, float* scales, int64_t lds, void* stream) {
  clear_error();
  MTC_REQUIRE(X && codes && scales, "mtc_fp8_quantize: null pointer");
  MTC_REQUIRE(type_ok(x_type), "mtc_fp8_quantize: unknown element type %d", x_type);
  MTC_REQUIRE(aligned(X, x_type) && aligned(scales), "mtc_fp8_quantize: pointer not aligned to its elements");
  MTC_REQUIRE(M >= 0 && M <= kMaxRows && K >= 1 && K <= kMaxRows && ldx >= K, "mtc_fp8_quantize: bad shape (M=%d, K=%d, ldx=%lld)", M, K,
              (long long)ldx);
  MTC_REQUIRE(ldq >= K && (ldq & 15) == 0 && (reinterpret_cast<uintptr_t>(codes) & 15) == 0 && lds >= M,
              "mtc_fp8_quantize: codes need rows of a multiple of 16 bytes >= K and 16-byte alignment");
  QuantRows a;
  a.X = X;
  a.dt = x_type;
  a.M = M;
  a.K = K;
  a.ldx = ldx;
  a.q = codes;
  a.ldq = ldq;
  a.s = scales;
  a.lds = lds;
  return launch_quantize(a, as_stream(stream), "mtc_fp8_quantize");
}

extern "C" size_t mtc_fp8_gemm_workspace_bytes(const mtc_fp8_matrix* w, int32_t M) {
  if (!w || M < 1 || M > kMaxRows || w->K < 1) return 0;
  return dense_plan(M, w->K, w->N, 1).bytes;  // (the number of SMs does not enter it)
}

extern "C" int mtc_fp8_gemm(const mtc_fp8_matrix* w, const void* X, int32_t x_type, int32_t M, int64_t ldx, void* Y,
                            int32_t y_type, int64_t ldy, void* ws, size_t ws_bytes, uint32_t* status,
                            const mtc_epilogue* ep, void* stream) {
  clear_error();
  int rc = check_matrix(w, "mtc_fp8_gemm");
  if (rc != MTC_OK) return rc;
  MTC_REQUIRE(w->E == 1, "mtc_fp8_gemm: %d stacked matrices", w->E);
  MTC_REQUIRE(X && Y, "mtc_fp8_gemm: null pointer");
  MTC_REQUIRE(type_ok(x_type) && type_ok(y_type), "mtc_fp8_gemm: unknown element type");
  MTC_REQUIRE(aligned(X, x_type) && aligned(Y, y_type) && aligned(status), "mtc_fp8_gemm: pointer not aligned to its elements");
  MTC_REQUIRE(M >= 1 && M <= kMaxRows && ldx >= w->K && ldy >= w->N, "mtc_fp8_gemm: bad shape (M=%d, ldx=%lld, ldy=%lld)", M,
              (long long)ldx, (long long)ldy);
  EpiArg epa;
  rc = read_epilogue(ep, &epa, "mtc_fp8_gemm");
  if (rc != MTC_OK) return rc;
  const int sms = sm_count();
  MTC_REQUIRE(sms > 0, "mtc_fp8_gemm: no CUDA device");
  const DensePlan d = dense_plan(M, w->K, w->N, sms);
  if (ws_bytes < d.bytes || (d.bytes && (!ws || (reinterpret_cast<uintptr_t>(ws) & 255)))) {
    set_error("mtc_fp8_gemm: workspace of %zu bytes (256-byte aligned) needed, %zu given", d.bytes, ws_bytes);
    return MTC_ERR_WORKSPACE;
  }
  const cudaStream_t st = as_stream(stream);
  Product a;
  a.w[0] = w;
  a.rows = M;
  a.tile = d.tile;
  a.many = d.many;
  a.slot_bound = (M + d.tile - 1) / d.tile;
  a.Y = Y;
  a.ydt = y_type;
  a.ldy = ldy;
  a.bias = epa.bias;
  a.act = epa.act;
  a.status = status;
  if (d.raw) {
    a.X = X;
    a.xdt = x_type;
    a.ldx = ldx;
  } else {
    QuantRows q;
    q.X = X;
    q.dt = x_type;
    q.M = M;
    q.K = w->K;
    q.ldx = ldx;
    q.q = reinterpret_cast<uint8_t*>(ws);
    q.ldq = d.ldq;
    q.s = reinterpret_cast<float*>(q.q + d.q_bytes);
    q.lds = d.lds;
    rc = launch_quantize(q, st, "mtc_fp8_gemm");
    if (rc != MTC_OK) return rc;
    a.xq = q.q;
    a.ldq = q.ldq;
    a.sx = q.s;
    a.lds = q.lds;
    a.early = true;
  }
  return launch_product(a, st, "mtc_fp8_gemm");
}
