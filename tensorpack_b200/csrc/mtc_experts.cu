// Mixture-of-experts operators: routing (scores, group limit, top-k), the
// plan that sorts token rows by expert, the weighted sum of the experts'
// outputs, and the gated feed-forward that runs them with the 8-bit products.
#include "mtc_fp8.cuh"
#include "mtc_fp8_internal.h"

namespace mtc {
namespace fp8 {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 32;
constexpr int kMaxGroups = 32;

// ---------------------------------------------------------------------------
// Routing: one warp per token
// ---------------------------------------------------------------------------
struct RouteParams {
  const void* logits;
  long long ld;
  int T, E, k, sigmoid;
  const float* bias;
  int groups, gsize, top_groups, renorm;
  uint32_t by_group;     // e / gsize = e * by_group >> 20 for e < 1024
  int lanes;             // lanes that look at a group (a power of two)
  double scale;
  int32_t* ids;
  float* weights;
};

// Unsigned order of the key = order of the value; key 1 is a masked (-inf or
// NaN) expert, key 0 one that may not be chosen.
__device__ __forceinline__ unsigned long long order_key(double c) {
  if (!(c > -INFINITY)) return 1ull;  // -inf, NaN
  const long long b = __double_as_longlong(c + 0.0);  // (-0 is 0)
  return (unsigned long long)b ^ (b < 0 ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ uint32_t order_key(float c) {
  if (!(c > -INFINITY)) return 1u;
  const uint32_t b = __float_as_uint(c + 0.0f);
  return b ^ ((int)b < 0 ? ~0u : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((int)k < 0 ? 0x80000000u : ~0u));
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int d = 16; d; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
  return x;
}

// Score of a logit: exp(z - max) (to be divided by the total), or
// 1 / (1 + exp(-z)); a masked one has score 0.
template <typename F>
__device__ __forceinline__ F raw_score(float z, float zmax, bool sigmoid) {
  if (z == -INFINITY) return (F)0;
  if (sizeof(F) == 8) return sigmoid ? 1.0 / (1.0 + exp(-(double)z)) : exp((double)z - (double)zmax);
  return sigmoid ? __fdividef(1.0f, 1.0f + __expf(-z)) : __expf(z - zmax);
}

// Bits of the experts' groups that are kept, one per group at bit g * lanes,
// and how far the worst kept group is ahead of the best dropped one.  `cs`:
// the choices in shared memory.  `lanes` lanes (a power of two) find a
// group's two best.
template <typename F>
__device__ __forceinline__ uint32_t keep_groups(const RouteParams& p, const F* cs, int lane, int lanes, F* gap) {
  const int g = lane / lanes, sub = lane & (lanes - 1);
  F g1 = -INFINITY, g2 = -INFINITY;
  if (g < p.groups)
    for (int i = sub; i < p.gsize; i += lanes) {
      const F x = cs[g * p.gsize + i];
      if (x > g1) {
        g2 = g1;
        g1 = x;
      } else if (x > g2) {
        g2 = x;
      }
    }
  for (int d = 1; d < lanes; d <<= 1) {
    const F o1 = __shfl_xor_sync(0xffffffffu, g1, d), o2 = __shfl_xor_sync(0xffffffffu, g2, d);
    if (o1 > g1) {
      g2 = g1 > o2 ? g1 : o2;
      g1 = o1;
    } else {
      g2 = g2 > o1 ? g2 : o1;
    }
  }
  // (a masked expert, -inf here, adds nothing: a group's only free choice
  // counts alone, and -inf is a group without any)
  const F gv = g2 > -INFINITY ? g1 + g2 : g1;
  int rank = 0;
  for (int o = 0; o < p.groups; ++o) {
    const F v = __shfl_sync(0xffffffffu, gv, o * lanes);
    rank += v > gv || (v == gv && o < g);
  }
  const bool real = g < p.groups, kept = real && rank < p.top_groups;
  // the two groups on either side of the border
  const uint32_t last = __ballot_sync(0xffffffffu, real && sub == 0 && rank == p.top_groups - 1);
  const uint32_t first = __ballot_sync(0xffffffffu, real && sub == 0 && rank == p.top_groups);
  const F in = __shfl_sync(0xffffffffu, gv, __ffs(last) - 1), out = __shfl_sync(0xffffffffu, gv, __ffs(first) - 1);
  *gap = in > out ? in - out : (F)0;
  if (in == -INFINITY || out == -INFINITY) *gap = in == out ? (F)INFINITY : *gap;  // masked groups: by index
  return __ballot_sync(0xffffffffu, kept && sub == 0);
}

// Descending order by a network of compare-exchanges (Batcher's odd-even
// merge sort).
template <int N>
__device__ __forceinline__ void sort_descending(uint32_t (&k)[N]) {
#pragma unroll
  for (int p = 1; p < N; p <<= 1)
#pragma unroll
    for (int q = p; q >= 1; q >>= 1)
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t a = k[i + j], b = k[i + j + q];
            k[i + j] = max(a, b);
            k[i + j + q] = min(a, b);
          }
}

// A warp per token.  The choice is made in 64 bits as defined (without bias
// and groups by the logits), but reached in 32 where that is certain: the
// fp32 choices are taken when every decision (between neighbours of the k + 1
// best, at the groups' border) has a margin above twice the error of a choice,
// and made again in 64 bits when one has not (one token in 600 of normal
// logits, 256 experts in 8 groups).
//
// Error of an fp32 choice c = s + b, in units u = 2^-24 (a rounding is 1, an
// ulp 2): |c| for the rounding of the sum, and that of s.  CUDA documents
// 2 + 1.173 |x| ulp for __expf(x), 2 ulp for __fdividef.
//  * Sigmoid 1 / (1 + exp(-z)): s (1 - s) (4 + 2.35 |z|) for the exponential,
//    5 s for the sum and the division.  (1 - s) |z| is below 0.28 for z > 0,
//    and with t = -z > 0 s t falls from t = 1.28 on, so that s t of any expert
//    is at most that of the largest score, or 1.28 times the largest score:
//    smax (9.7 + 2.35 max(t, 1.28)), t that of the largest logit.
//  * Softmax, d the distance to the largest logit, smax = 1 / total: the
//    difference and its exponential s (4 + 3.35 d), where s d < 0.37 smax; the
//    total as much on average (s d adds up to log E < 7 at most) and
//    NPL + 4 additions; division and product 5 s: smax (41.5 + NPL).
// What is flushed to zero is below 2^-126.
//
// 8192 x 256 with groups and bias: 22 us, bound by instruction issue.  (2 to
// 3 us more in 64 bits for all, which also has twice the registers, or without
// the limit on registers that lets 48 warps share an SM.)
template <typename T, int NPL>
__global__ void __launch_bounds__(256, NPL <= 8 ? 6 : 1) route_kernel(const RouteParams p) {
  extern __shared__ double route_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * (blockDim.x >> 5) + warp;
  griddep_wait();
  griddep_launch_dependents();
  if (t >= p.T) return;
  const T* z = reinterpret_cast<const T*>(p.logits) + t * p.ld;
  float v[NPL];
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    const int e = 32 * i + lane;
    v[i] = e < p.E ? to_f32(z[e]) : -INFINITY;
  }
  float zmax = -INFINITY;
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    if (v[i] != v[i]) v[i] = -INFINITY;
    v[i] = fminf(v[i], 3.402823466e38f);
    zmax = fmaxf(zmax, v[i]);
  }
  if (!p.sigmoid) zmax = warp_max(zmax);
  const bool by_logit = !p.bias && p.groups == 1;
  const int lanes = p.lanes;

  // Keys in 32 bits whose last bits hold the lane's index of the expert, so
  // that a lane sorts values and indices at once.  What these bits hide goes
  // into the margin.
  constexpr uint32_t kLow = NPL - 1;
  uint32_t key[NPL];
  float margin;
  bool sure = true;
  {
    // (the hidden bits: below NPL ulp of each)
    float c[NPL], most = 0.0f, error;
    if (by_logit) {
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        c[i] = v[i];
        if (v[i] != -INFINITY) most = fmaxf(most, fabsf(v[i]));
      }
      error = 2.0f * NPL * most;
    } else {
      float sum = 0.0f, smax = 0.0f;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        c[i] = raw_score<float>(v[i], zmax, p.sigmoid);
        sum += c[i];
      }
      float inv = 1.0f;
      if (!p.sigmoid) {
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        inv = __fdividef(1.0f, sum);
      }
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const int e = 32 * i + lane;
        const float sc = c[i] * inv;
        c[i] = p.bias && e < p.E ? sc + p.bias[e] : sc;
        if (v[i] == -INFINITY) c[i] = -INFINITY;
        else most = fmaxf(most, fabsf(c[i]));
        smax = fmaxf(smax, sc);
      }
      // (sigmoid: zmax and smax are the lane's, which bounds its own errors)
      error = (1.0f + 2.0f * NPL) * most +
              (p.sigmoid ? smax * (10.0f + 2.4f * fminf(fmaxf(-zmax, 1.3f), 128.0f)) : inv * (42.0f + NPL));
    }
    margin = warp_max(error) * 1.1920928955078125e-7f + 4.70197740328915e-38f;  // 2 u, 2^-124
    uint32_t keep = ~0u;
    if (p.groups > 1) {
      float* cs = reinterpret_cast<float*>(route_smem + warp * p.E);
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (32 * i + lane < p.E) cs[32 * i + lane] = c[i];
      __syncwarp();
      float gap;
      keep = keep_groups<float>(p, cs, lane, lanes, &gap);
      sure = gap > 2.0f * margin;  // a group's value is the sum of two choices
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const int e = 32 * i + lane;
      const uint32_t o = (order_key(c[i]) & ~kLow) | (kLow - i);  // a tie goes to the lowest index
      key[i] = e < p.E && (p.groups == 1 || (keep >> ((e * p.by_group >> 20) * lanes) & 1u)) ? o : 0u;
    }
  }
  sort_descending(key);
  // k + 1 rounds (the last for the margin of the last place): the best of the
  // lanes' first keys; its lane moves its others up
  int my_id = 0;
  uint32_t before = 0u;
#pragma unroll 1
  for (int j = 0; j <= p.k; ++j) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, key[0]);
    if (j > 0 && top > 2 * kLow + 1 && !(key_value(before & ~kLow) - key_value(top & ~kLow) > margin)) sure = false;
    if (j < p.k && top <= 2 * kLow + 1) sure = false;  // only masked experts are left: by index
    if (!sure || j == p.k) break;
    before = top;
    const int owner = __ffs(__ballot_sync(0xffffffffu, key[0] == top)) - 1;
    if (lane == j) my_id = (int)(32 * (kLow - (top & kLow))) + owner;
    if (lane == owner) {
#pragma unroll
      for (int i = 0; i + 1 < NPL; ++i) key[i] = key[i + 1];
      key[NPL - 1] = 0u;
    }
  }
  if (!sure) {
    // all of it in 64 bits, in registers (a warp that comes here is the one
    // the others' end waits for)
    unsigned long long wide[NPL];
    double c[NPL], sum = 0.0;
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      c[i] = by_logit ? (double)v[i] : raw_score<double>(v[i], zmax, p.sigmoid);
      sum += c[i];
    }
    if (!by_logit) {
      if (!p.sigmoid) {
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      }
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        if (!p.sigmoid) c[i] = c[i] / sum;
        if (p.bias && 32 * i + lane < p.E) c[i] += (double)p.bias[32 * i + lane];
        if (v[i] == -INFINITY) c[i] = -INFINITY;
      }
    }
    uint32_t keep = ~0u;
    if (p.groups > 1) {
      double* cs = route_smem + warp * p.E;
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (32 * i + lane < p.E) cs[32 * i + lane] = c[i];
      __syncwarp();
      double gap;
      keep = keep_groups<double>(p, cs, lane, lanes, &gap);
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const int e = 32 * i + lane;
      wide[i] = e < p.E && (p.groups == 1 || (keep >> ((e * p.by_group >> 20) * lanes) & 1u)) ? order_key(c[i]) : 0ull;
    }
#pragma unroll 1
    for (int j = 0; j < p.k; ++j) {
      unsigned long long best = 0ull;
      int at = 0;
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (wide[i] > best) {
          best = wide[i];
          at = i;
        }
      const uint32_t hi = (uint32_t)(best >> 32), mh = __reduce_max_sync(0xffffffffu, hi);
      const uint32_t lo = hi == mh ? (uint32_t)best : 0u, ml = __reduce_max_sync(0xffffffffu, lo);
      const uint32_t mine = (hi == mh && lo == ml) ? (uint32_t)(32 * at + lane) : ~0u;
      const uint32_t id = __reduce_min_sync(0xffffffffu, mine);
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (mine == id && i == at) wide[i] = 0ull;
      if (lane == j) my_id = (int)id;
    }
  }
  // the weights, from the scores of the chosen in 64 bits
  double w = 0.0;
  if (lane < p.k) {
    float x = to_f32(z[my_id]);
    if (x != x) x = -INFINITY;
    w = raw_score<double>(fminf(x, 3.402823466e38f), zmax, p.sigmoid);
  }
  double div = 1.0;
  if (p.renorm) {
    div = w;
    for (int d = 16; d; d >>= 1) div += __shfl_xor_sync(0xffffffffu, div, d);
  } else if (!p.sigmoid) {
    div = 0.0;
#pragma unroll
    for (int i = 0; i < NPL; ++i) div += raw_score<double>(v[i], zmax, false);
    for (int d = 16; d; d >>= 1) div += __shfl_xor_sync(0xffffffffu, div, d);
  }
  if (lane < p.k) {
    p.ids[(long long)t * p.k + lane] = my_id;
    p.weights[(long long)t * p.k + lane] = (float)(div > 0.0 ? w / div * p.scale : 0.0);
  }
}

// ---------------------------------------------------------------------------
// Plan: rows (t, j) sorted by expert, stable, a CTA per 1024 rows
// ---------------------------------------------------------------------------
struct PlanParams {
  const int32_t* ids;
  int R, E, size;        // rows T * k, experts, rows per slot
  int32_t* order;        // [R] row (t * k + j) at each sorted place
  int32_t* pos;          // [R] sorted place of each row, -1 for an id outside 0..E-1
  int32_t* slots;        // slot list
  int32_t* counts;       // [CTAs][E] rows per expert of each CTA (more than one CTA)
};

constexpr int kPlanThreads = 1024;

// Exclusive scan of one value per thread over the CTA.
__device__ __forceinline__ int block_scan(int x, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = x;
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += o;
  }
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  if (warp == 0) {
    int v = warp_sums[lane], q = v;
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, q, d);
      if (lane >= d) q += o;
    }
    warp_sums[lane] = q - v;
    if (lane == 31) warp_sums[32] = q;
  }
  __syncthreads();
  const int r = warp_sums[warp] + s - x;
  *total = warp_sums[32];
  __syncthreads();
  return r;
}

// Rows per expert of every CTA's 1024 rows.
__global__ void __launch_bounds__(kPlanThreads) plan_count_kernel(const PlanParams p) {
  extern __shared__ int32_t hist[];
  for (int i = threadIdx.x; i < p.E; i += kPlanThreads) hist[i] = 0;
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();
  const long long r = (long long)blockIdx.x * kPlanThreads + threadIdx.x;
  const int e = r < p.R ? p.ids[r] : -1;
  if ((unsigned)e < (unsigned)p.E) atomicAdd(&hist[e], 1);
  __syncthreads();
  for (int i = threadIdx.x; i < p.E; i += kPlanThreads) p.counts[(long long)blockIdx.x * p.E + i] = hist[i];
}

// Each warp owns 32 rows: it counts its experts, the counts of all warps and
// CTAs become places (experts in order, inside an expert the rows in order),
// and the rows take them.  The first CTA writes the slot list.  Every CTA reads
// the counts of all, so the time grows with the square of the rows: 6 us for
// 32768 rows, 0.02 ms for 2^18, 0.2 ms for 2^20 (of some 1 ms for all kernels
// at 128 x 128), but 10 ms for 2^23 with 64 or 256 experts, 18 ms with 1024.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p) {
  extern __shared__ int32_t hist[];  // [32][E]
  __shared__ int warp_sums[33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < 32 * p.E; i += kPlanThreads) hist[i] = 0;
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();
  const long long r = (long long)blockIdx.x * kPlanThreads + threadIdx.x;
  const int id = r < p.R ? p.ids[r] : -1;
  const bool ok = (unsigned)id < (unsigned)p.E;
  const uint32_t same = __match_any_sync(0xffffffffu, ok ? id : -1);
  const int rank = __popc(same & ((1u << lane) - 1u));
  int32_t* mine = hist + warp * p.E;
  if (ok && rank == 0) mine[id] = __popc(same);
  __syncthreads();
  // thread e: rows of expert e by warp, in the CTAs before this one, in all
  const int e = threadIdx.x;
  int rows[32], before = 0, count = 0;
  if (e < p.E) {
#pragma unroll
    for (int w = 0; w < 32; ++w) rows[w] = hist[w * p.E + e];
    if (gridDim.x == 1) {
#pragma unroll
      for (int w = 0; w < 32; ++w) count += rows[w];
    } else {
#pragma unroll 16
      for (int b = 0; b < (int)gridDim.x; ++b) {
        const int c = p.counts[(long long)b * p.E + e];
        count += c;
        before += b < (int)blockIdx.x ? c : 0;
      }
    }
  }
  int total, n_slots;
  const int off = block_scan(count, warp_sums, &total);
  if (blockIdx.x == 0) {
    const int ns = (count + p.size - 1) / p.size;
    const int sl = block_scan(ns, warp_sums, &n_slots);
    for (int i = 0; i < ns; ++i)
      *reinterpret_cast<int4*>(p.slots + 4 + 4 * (sl + i)) = make_int4(e, off + i * p.size, off + count, 0);
    if (threadIdx.x == 0) p.slots[0] = n_slots;
  }
  if (e < p.E) {
    int at = off + before;
#pragma unroll
    for (int w = 0; w < 32; ++w) {
      hist[w * p.E + e] = at;
      at += rows[w];
    }
  }
  __syncthreads();
  if (r < p.R) {
    const int at = ok ? mine[id] + rank : -1;
    p.pos[r] = at;
    if (ok) p.order[at] = (int)r;
  }
}

// ---------------------------------------------------------------------------
// Y[t] = sum_j weights[t][j] * rows[pos[t][j]], j in order
// ---------------------------------------------------------------------------
// Rows and sum are fp32, rounded once to Y's type.  Bound by memory: 32768
// rows of 2048 take 45 us (6.3 TB/s).
struct CombineParams {
  const float* rows;
  long long ldr;
  const int32_t* pos;    // or null: row j, for the ids of one token
  const int32_t* ids;
  int E;
  const float* weights;
  int T, k, D;
  void* Y;
  long long ldy;
  int ydt, vec;
};

__global__ void __launch_bounds__(256) combine_kernel(const CombineParams p) {
  const int parts = (p.D + 2047) >> 11, t = blockIdx.x / parts;
  __shared__ int at[kMaxTopK];
  __shared__ float w[kMaxTopK];
  griddep_wait();
  griddep_launch_dependents();
  if (threadIdx.x < kMaxTopK) {
    const int j = threadIdx.x;
    int a = -1;
    if (j < p.k) {
      a = p.pos ? p.pos[(long long)t * p.k + j] : (unsigned)p.ids[j] < (unsigned)p.E ? j : -1;
      w[j] = p.weights[(long long)t * p.k + j];
    }
    at[j] = a;
  }
  __syncthreads();
  const int d = 8 * ((blockIdx.x - t * parts) * 256 + threadIdx.x);
  if (d >= p.D) return;
  float a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = 0.0f;
  // (rows are padded to 8 values, so the last vector may be read whole)
  constexpr int kMore = 4;
  for (int j0 = 0; j0 < p.k; j0 += kMore) {
    uint4 raw[kMore][2];
#pragma unroll
    for (int j = 0; j < kMore; ++j) {
      const int r = j0 + j < kMaxTopK ? at[j0 + j] : -1;
      const float* row = p.rows + r * p.ldr + d;
#pragma unroll
      for (int q = 0; q < 2; ++q) raw[j][q] = load16_if(reinterpret_cast<const uint4*>(row) + q, r >= 0);
    }
#pragma unroll
    for (int j = 0; j < kMore; ++j)
      if (j0 + j < p.k && at[j0 + j] >= 0) {
        float v[8];
        unpack8<float>(raw[j], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = fmaf(w[j0 + j], v[i], a[i]);
      }
  }
  const long long y = t * p.ldy + d;
  if (p.vec && d + 8 <= p.D) {
    if (p.ydt == MTC_F32) {
      float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.Y) + y);
      o[0] = make_float4(a[0], a[1], a[2], a[3]);
      o[1] = make_float4(a[4], a[5], a[6], a[7]);
    } else {
      *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.Y) + y) =
          make_uint4(pack2(p.ydt, a[0], a[1]), pack2(p.ydt, a[2], a[3]), pack2(p.ydt, a[4], a[5]),
                     pack2(p.ydt, a[6], a[7]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d + i < p.D) store1(p.Y, p.ydt, y + i, a[i]);
  }
}

size_t round256(size_t x) { return (x + 255) & ~(size_t)255; }

// How the experts' products run, from the mean number of rows of an expert:
// up to 12, 16-row tiles whose tokens the first product quantizes itself;
// above, the 128-token kernel on quantized rows.  Device times of the two at a
// mean of m rows:
//    64 experts, 2048 x 1024:   m = 10   91 /  96 us   m = 12   93 /  99   m = 14  103 / 100   m = 24  143 / 104
//   128 experts, 2048 x 768:    m = 8   125 / 133      m = 12  135 / 139   m = 14  144 / 141   m = 16  162 / 138
//     8 experts, 4096 x 14336:  m = 8   268 / 258      m = 12  267 / 275   m = 14  264 / 258   m = 16  358 / 280
//   256 experts, 1024 x 512:    m = 8    99 / 144      m = 10  103 / 110   m = 12  113 /  98   m = 24  184 / 105
//     6 experts, 272 x 264:     m = 14   18 /  20
// (Tiles of 32 rows, between the two, were ahead of neither: 102, 111 and 126
// us at m = 12, 16 and 24 of the first.)
// A single token needs no plan: every row is a slot (20.9 us a call with 8 of
// 64 experts, some 5 more with a plan).
// (R / E counts every id, also those of no expert here: with few of them the
// 128-token kernel runs for less than 13 rows of an expert.  The host cannot
// know.)
struct ExpertsPlan {
  int R, tile, slot_bound;
  bool direct, raw;
  long long ldx, ldh, lds, ldo;
  int plan_ctas;
  size_t order, pos, slots, counts, xq, xs, hq, hs, out, bytes;
};
bool experts_plan(int T, int k, int E, int D, int I, ExpertsPlan* pl) {
  const long long R = (long long)T * k;
  if (R > kMaxRows || (long long)T * ((D + 2047) / 2048) > kMaxRows) return false;
  pl->R = (int)R;
  const double mean = (double)R / E;
  pl->direct = T == 1;
  pl->raw = pl->direct || mean <= 12.0;
  pl->tile = pl->raw ? 16 : 128;
  const long long used = R < E ? R : E;
  long long bound = R / pl->tile + used;
  if (bound > R || pl->direct) bound = R;
  pl->slot_bound = (int)bound;
  pl->ldx = (D + 15) & ~15ll;
  pl->ldh = (I + 31) & ~31ll;
  pl->lds = (R + 3) & ~3ll;
  pl->ldo = (D + 15) & ~15ll;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t here = at;
    at += round256(n);
    return here;
  };
  pl->order = take(4 * (size_t)R);
  pl->pos = take(4 * (size_t)R);
  pl->slots = take(16 * (size_t)(pl->slot_bound + 1));
  pl->plan_ctas = (int)((R + kPlanThreads - 1) / kPlanThreads);
  pl->counts = take(pl->plan_ctas > 1 ? 4 * (size_t)pl->plan_ctas * E : 4);
  pl->xq = pl->xs = 0;
  if (!pl->raw) {
    pl->xq = take((size_t)R * pl->ldx);
    pl->xs = take((size_t)((D + 127) / 128) * pl->lds * 4);
  }
  pl->hq = take((size_t)R * pl->ldh);
  pl->hs = take((size_t)((I + 127) / 128) * pl->lds * 4);
  pl->out = take((size_t)R * pl->ldo * 4);
  pl->bytes = at;
  return true;
}

template <typename T>
int launch_route(const RouteParams& p, cudaStream_t st) {
  const int warps = p.E > 512 ? 4 : 8;
  const size_t smem = (size_t)warps * p.E * 8;  // the choices, where groups compare them: 32 KB at most
  auto go = [&](auto kernel) -> int {
    MTC_CHECK_CUDA(launch_chained(kernel, dim3((p.T + warps - 1) / warps), dim3(32 * warps), smem, st, 1, p),
                   "mtc_route_experts");
    return MTC_OK;
  };
  if (p.E <= 32) return go(route_kernel<T, 1>);
  if (p.E <= 64) return go(route_kernel<T, 2>);
  if (p.E <= 128) return go(route_kernel<T, 4>);
  if (p.E <= 256) return go(route_kernel<T, 8>);
  if (p.E <= 512) return go(route_kernel<T, 16>);
  return go(route_kernel<T, 32>);
}

}  // namespace
}  // namespace fp8
}  // namespace mtc

using namespace mtc;
using namespace mtc::fp8;

extern "C" int mtc_route_experts(const void* logits, int32_t type, int32_t T, int32_t E, int64_t ld, int32_t k,
                                 int32_t score, const float* bias, int32_t groups, int32_t top_groups,
                                 int32_t renormalize, float scale, int32_t* ids, float* weights, void* stream) {
  clear_error();
  MTC_REQUIRE(logits && ids && weights, "mtc_route_experts: null pointer");
  MTC_REQUIRE(type_ok(type), "mtc_route_experts: unknown element type %d", type);
  MTC_REQUIRE(aligned(logits, type) && aligned(bias) && aligned(ids) && aligned(weights),
              "mtc_route_experts: pointer not aligned to its elements");
  MTC_REQUIRE(score == MTC_SCORE_SOFTMAX || score == MTC_SCORE_SIGMOID, "mtc_route_experts: unknown score %d", score);
  MTC_REQUIRE(T >= 0 && T <= kMaxRows && E >= 1 && E <= kMaxExperts && ld >= E, "mtc_route_experts: bad shape (T=%d, E=%d, ld=%lld)", T,
              E, (long long)ld);
  MTC_REQUIRE(groups >= 1 && groups <= kMaxGroups && E % groups == 0 && top_groups >= 1 && top_groups <= groups,
              "mtc_route_experts: %d experts in %d groups, %d of them kept", E, groups, top_groups);
  MTC_REQUIRE(k >= 1 && k <= kMaxTopK && k <= top_groups * (E / groups),
              "mtc_route_experts: k=%d outside 1..%d", k, top_groups * (E / groups) < kMaxTopK ? top_groups * (E / groups) : kMaxTopK);
  if (T == 0) return MTC_OK;
  RouteParams p = {};
  p.logits = logits;
  p.ld = ld;
  p.T = T;
  p.E = E;
  p.k = k;
  p.sigmoid = score == MTC_SCORE_SIGMOID;
  p.bias = bias;
  p.groups = groups == top_groups ? 1 : groups;  // every group kept: no limit
  p.gsize = E / groups;
  p.by_group = ((1u << 20) + p.gsize - 1) / p.gsize;
  p.lanes = 1;
  while (2 * p.lanes * groups <= 32) p.lanes *= 2;
  p.top_groups = top_groups;
  p.renorm = renormalize != 0;
  p.scale = (double)scale;
  p.ids = ids;
  p.weights = weights;
  if (type == MTC_F32) return launch_route<float>(p, as_stream(stream));
  if (type == MTC_BF16) return launch_route<__nv_bfloat16>(p, as_stream(stream));
  return launch_route<__half>(p, as_stream(stream));
}

extern "C" size_t mtc_experts_workspace_bytes(const mtc_fp8_matrix* gate, int32_t T, int32_t k, int32_t) {
  ExpertsPlan pl;
  if (!gate || T < 1 || k < 1 || !experts_plan(T, k, gate->E, gate->K, gate->N, &pl)) return 0;
  return pl.bytes;
}

extern "C" int mtc_experts_forward(const mtc_fp8_matrix* gate, const mtc_fp8_matrix* up, const mtc_fp8_matrix* down,
                                   const void* X, int32_t x_type, int32_t T, int64_t ldx, const int32_t* ids,
                                   const float* weights, int32_t k, int32_t act, void* Y, int32_t y_type, int64_t ldy,
                                   void* ws, size_t ws_bytes, uint32_t* status, void* stream) {
  const char* who = "mtc_experts_forward";
  clear_error();
  int rc = check_matrix(gate, who);
  if (rc == MTC_OK) rc = check_matrix(up, who);
  if (rc == MTC_OK) rc = check_matrix(down, who);
  if (rc != MTC_OK) return rc;
  MTC_REQUIRE(up->E == gate->E && up->K == gate->K && up->N == gate->N, "%s: gate and up differ in shape", who);
  MTC_REQUIRE(down->E == gate->E && down->K == gate->N && down->N == gate->K, "%s: down is not the transpose shape of gate",
              who);
  MTC_REQUIRE(gate->E <= kMaxExperts, "%s: %d experts, at most %d", who, gate->E, kMaxExperts);
  MTC_REQUIRE(X && ids && weights && Y, "%s: null pointer", who);
  MTC_REQUIRE(type_ok(x_type) && type_ok(y_type), "%s: unknown element type", who);
  MTC_REQUIRE(aligned(X, x_type) && aligned(ids) && aligned(weights) && aligned(Y, y_type) && aligned(status),
              "%s: pointer not aligned to its elements", who);
  MTC_REQUIRE(act >= MTC_ACT_NONE && act <= MTC_ACT_GELU_TANH, "%s: unknown activation %d", who, act);
  MTC_REQUIRE(T >= 1 && k >= 1 && k <= kMaxTopK && ldx >= gate->K && ldy >= gate->K,
              "%s: bad shape (T=%d, k=%d, ldx=%lld, ldy=%lld)", who, T, k, (long long)ldx, (long long)ldy);
  const int E = gate->E, D = gate->K, I = gate->N;
  ExpertsPlan pl;
  MTC_REQUIRE(experts_plan(T, k, E, D, I, &pl), "%s: too many rows (%d x %d)", who, T, k);
  if (ws_bytes < pl.bytes || !ws || (reinterpret_cast<uintptr_t>(ws) & 255)) {
    set_error("%s: workspace of %zu bytes (256-byte aligned) needed, %zu given", who, pl.bytes, ws_bytes);
    return MTC_ERR_WORKSPACE;
  }
  const cudaStream_t st = as_stream(stream);
  uint8_t* base = reinterpret_cast<uint8_t*>(ws);
  int32_t* order = reinterpret_cast<int32_t*>(base + pl.order);
  int32_t* pos = reinterpret_cast<int32_t*>(base + pl.pos);
  int32_t* slots = reinterpret_cast<int32_t*>(base + pl.slots);
  if (!pl.direct) {
    const PlanParams p = {ids, pl.R, E, pl.tile, order, pos, slots, reinterpret_cast<int32_t*>(base + pl.counts)};
    const size_t smem = (size_t)32 * E * 4;
    static std::atomic<uint64_t> ready{0};
    MTC_CHECK_CUDA(allow_smem(plan_kernel, (size_t)32 * kMaxExperts * 4, ready), who);
    if (pl.plan_ctas > 1)
      MTC_CHECK_CUDA(launch_chained(plan_count_kernel, dim3(pl.plan_ctas), dim3(kPlanThreads), (size_t)E * 4, st, 1, p),
                     who);
    MTC_CHECK_CUDA(launch_chained(plan_kernel, dim3(pl.plan_ctas), dim3(kPlanThreads), smem, st, 1, p), who);
  }
  Product a;
  a.w[0] = gate;
  a.w[1] = up;
  a.slots = pl.direct ? ids : slots;
  a.experts = pl.direct ? E : 0;
  a.slot_bound = pl.slot_bound;
  a.rows = pl.R;
  a.tile = pl.tile;
  a.many = !pl.raw;
  a.gate_act = act;
  a.status = status;
  Product b = a;
  b.w[0] = down;
  b.w[1] = nullptr;
  b.early = true;  // the plan (or whatever wrote the ids) ran before the first product
  if (!pl.raw) {
    QuantRows q;
    q.X = X;
    q.dt = x_type;
    q.M = T;
    q.K = D;
    q.ldx = ldx;
    q.pos = pos;
    q.copies = k;
    q.q = base + pl.xq;
    q.ldq = pl.ldx;
    q.s = reinterpret_cast<float*>(base + pl.xs);
    q.lds = pl.lds;
    rc = launch_quantize(q, st, who);
    if (rc != MTC_OK) return rc;
    a.xq = q.q;
    a.ldq = q.ldq;
    a.sx = q.s;
    a.lds = q.lds;
  } else {
    a.X = X;
    a.xdt = x_type;
    a.ldx = ldx;
    a.order = pl.direct ? nullptr : order;
    a.kdiv = k;
    if (pl.direct) a.ldx = 0;  // every row is the one token
  }
  a.hq = base + pl.hq;
  a.ldh = pl.ldh;
  a.hs = reinterpret_cast<float*>(base + pl.hs);
  a.hs_ld = pl.lds;
  rc = launch_product(a, st, who);
  if (rc != MTC_OK) return rc;
  b.xq = a.hq;
  b.ldq = a.ldh;
  b.sx = a.hs;
  b.lds = a.hs_ld;
  b.Y = base + pl.out;
  b.ydt = MTC_F32;  // the terms of a sum
  b.ldy = pl.ldo;
  rc = launch_product(b, st, who);
  if (rc != MTC_OK) return rc;
  CombineParams c = {};
  c.rows = reinterpret_cast<const float*>(base + pl.out);
  c.ldr = pl.ldo;
  c.pos = pl.direct ? nullptr : pos;
  c.ids = ids;
  c.E = E;
  c.weights = weights;
  c.T = T;
  c.k = k;
  c.D = D;
  c.Y = Y;
  c.ldy = ldy;
  c.ydt = y_type;
  c.vec = (reinterpret_cast<uintptr_t>(Y) & 15) == 0 && ldy % (y_type == MTC_F32 ? 4 : 8) == 0;
  MTC_CHECK_CUDA(launch_chained(combine_kernel, dim3((unsigned)((D + 2047) / 2048) * (unsigned)T), dim3(256), 0, st, 1, c), who);
  return MTC_OK;
}
