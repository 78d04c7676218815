// Products with 8-bit (e4m3) weights and activations, dense and grouped by
// expert: Y[m][n] = act(sum_b sx[m][b] sw[n/128][b] (qx[m] . qw[n])_b + bias[n])
// with the sums of 128 inputs on the tensor cores and the scaled sums in fp32
// registers (mtc_fp8.cuh).
//
// Two kernels, by the number of rows that share a weight tile:
//
//  * few_kernel<BN, SRC, PAIR>: 128 output features x BN <= 128 tokens.  The
//    features are the M side of the MMA (TMEM lane = feature), so one token
//    costs 16 columns instead of 128 rows, and a warp's stores are
//    consecutive features.  Bound by the weight bytes: a persistent CTA per
//    SM streams its features' codes once through a TMA ring (1 x 4096 x 14336
//    13.9 us, 4.2 TB/s with some 3 us of start-up; 16 x 14336 x 4096 17.5 us
//    with the quantizer).  When there are few tiles a cluster of up to 8 CTAs
//    splits the inputs and adds its partial sums through distributed shared
//    memory in rank order: no workspace, no atomics, the same result every
//    time.  PAIR: the gate and up matrices of a gated product side by side;
//    the output is act(gate) * up, quantized.
//  * many_kernel<MODE>: 128 tokens x 256 features (TMEM lane = token), one
//    persistent CTA per SM, two 256-column accumulators that alternate
//    between the MMA and eight warps that scale and add.  4096 x 4096 x 14336
//    takes 246 us with the quantizer, 1.96 PFLOP/s: 208 us with the scaling
//    taken out, 176 us with the MMAs taken out, 150 us with both (loads and
//    stores alone), so each of them waits for another.  After some 50 ms the
//    power limit lowers the clock (1965 to 1540 MHz) and it takes 289 us.
//    kGated: the 256 features are 128 of the gate matrix and the same 128 of
//    the up matrix; the output is act(gate) * up, quantized.
#include <string.h>

#include <type_traits>

#include "mtc_fp8.cuh"
#include "mtc_internal.h"
#include "mtc_fp8_internal.h"

namespace mtc {
namespace fp8 {
namespace {

constexpr uint32_t kATile = 128 * 128;  // bytes of one 128-row x 128-input tile of codes

__device__ __forceinline__ void flag(uint32_t* st, uint32_t bits) {
  if (st) atomicOr(st, bits);
}

// ---------------------------------------------------------------------------
// few_kernel
// ---------------------------------------------------------------------------
// Where the tokens come from: codes and scales in memory, or activations that
// six more warps of the kernel quantize on the way (at most 16 rows per tile).
enum { SRC_CODES = 0, SRC_F32 = 1, SRC_BF16 = 2, SRC_F16 = 3 };

// Warps 0..3 scale, 4 issues TMA, the next 4 issue MMAs (for one accumulator
// each: a thread needs some 0.3 us to wait for and issue the four MMAs of a
// block and their commits, longer than the block's bytes take to arrive; 2
// for wide tiles, whose sums want the registers), and 6 more quantize when
// the kernel takes activations as they are.
constexpr int kAccs = 4, kQuantWarps = 6;

template <int BN, bool PAIR>
struct FewCfg {
  static constexpr int kMats = PAIR ? 2 : 1;
  static constexpr uint32_t kBTile = BN * 128;
  static constexpr uint32_t kStage = kMats * kATile + kBTile;
  static constexpr int kCols = kMats * BN;              // TMEM columns of one accumulator
  static constexpr int kAcc = kAccs;                    // TMEM accumulators
  static constexpr int kIssue = kCols >= 128 ? 2 : 4;   // issuing warps
  static constexpr int kThreads = 32 * (5 + kIssue);    // without the quantizing warps
  static constexpr uint32_t kRed = 16 * 128 * 4 * kMats;  // staged sums of 16 tokens
  static constexpr uint32_t kMul = 4 * 2 * kCols * 4;   // per scaling warp, two buffers of scales
  static constexpr uint32_t kRoom = 227 * 1024 - 1024 - 512 - 1024 - kRed - kMul;
  // As many stages as fit; 6 of 18 KB for 16 tokens (13.7 us at 1 x 4096 x
  // 14336, 14.4 with 11, 13.8 with 5, 15.3 with 4).
  static constexpr int kStages = BN == 16 ? 6 : kRoom / kStage < 12 ? kRoom / kStage : 12;
  static constexpr int kRing = kStages + kAcc;          // slots of in-kernel token scales
  static constexpr uint32_t kBars = kStages * kStage;
  static constexpr uint32_t kRedAt = kBars + 512;
  static constexpr uint32_t kMulAt = kRedAt + kRed;
  static constexpr uint32_t kScaleAt = kMulAt + kMul;
  static constexpr size_t kSmem = 1024 + kScaleAt + (BN == 16 ? kRing * BN * 4 : 0);
  static_assert(kCols * kAcc <= 512 && kSmem <= 227 * 1024, "TMEM and shared memory of one CTA");
  static_assert(kMats * BN * 128 * 4 <= kStages * kStage, "a cluster's partial sums fit the stages");
};
struct FewParams {
  int K, nkb, N, Nb;                  // Nb: 128-feature tiles
  const float* sw[2];                 // scales of the matrix (or of gate and up)
  const int32_t* slots;               // slot list, or ids of one token's rows (experts > 0)
  int experts;
  int M;
  const float* sx;                    // SRC_CODES: token scales [nkb][lds]
  long long lds;
  const void* X;                      // else: activations
  int vec;
  long long ldx;
  const int32_t* order;               // grouped: row r is token order[r] / kdiv
  int kdiv;
  void* Y;
  int ydt;
  long long ldy;
  const float* bias;
  int act;                            // PAIR: of the gate
  uint8_t* hq;                        // PAIR: codes [row][ldh] and scales [n / 128][hs_ld] of act(gate) * up
  long long ldh;
  float* hs;
  long long hs_ld;
  int split;                          // CTAs of a cluster
  int early;                          // slots and weights may be read before the predecessor ends
  uint32_t* status;
  unsigned long long timeout_ns;
  uint32_t withhold;                  // diagnostic: the first stage of a CTA never becomes full
};

template <int SRC>
struct SrcType {
  typedef float T;
};
template <>
struct SrcType<SRC_BF16> {
  typedef __nv_bfloat16 T;
};
template <>
struct SrcType<SRC_F16> {
  typedef __half T;
};

// Barrier of the four scaling warps; the second form tells all whether any
// of them passed true.
__device__ __forceinline__ void few_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool few_sync_or(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)x)
      : "memory");
  return r != 0;
}

// Four floats of the object at this offset in CTA `rank` of the cluster (the
// loads of several ranks may be in flight together: not volatile, ordered by
// the cluster barrier before them).
__device__ __forceinline__ float4 load_cluster4(const float* p, int rank) {
  float4 v;
  asm("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(tc::mapa(p, rank))
      : "memory");
  return v;
}
__device__ __forceinline__ uint32_t load_cluster1(const volatile uint32_t* p, int rank) {
  uint32_t v;
  asm("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(tc::mapa(const_cast<const uint32_t*>(p), rank)) : "memory");
  return v;
}

// Staged values [i][128 features] of the tokens j0 + i * step, i < count, to
// codes and scales: one half warp per token.  Called by the four scaling warps.
__device__ __forceinline__ void quantize_staged(const FewParams& p, const float* h, int row0, int j0, int step,
                                                int count, int f0, int warp, int lane) {
  const int l = lane & 15;
#pragma unroll 1
  for (int i = 2 * warp + (lane >> 4); i < ((count + 7) & ~7); i += 8) {
    float v[8];
    const float4 a = *reinterpret_cast<const float4*>(h + i * 128 + 8 * l);
    const float4 b = *reinterpret_cast<const float4*>(h + i * 128 + 8 * l + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    const GroupScale g = group_scale(half_warp_max(amax8(v)));
    const uint2 c = codes8(v, g.mul);
    if (i < count) {
      const long long row = row0 + j0 + i * step;
      if (f0 + 8 * l < p.ldh) *reinterpret_cast<uint2*>(p.hq + row * p.ldh + f0 + 8 * l) = c;
      if (l == 0) p.hs[(long long)(f0 >> 7) * p.hs_ld + row] = g.scale;
    }
  }
}

// Persistent: CTAs (or clusters, which then have one work item each) take the
// items slot + n_slots * feature tile in turn, so that neighbours in time
// share weights, and the TMA warp runs ahead over their boundaries.
template <int BN, int SRC, bool PAIR>
__global__ void __launch_bounds__(FewCfg<BN, PAIR>::kThreads + (SRC == SRC_CODES ? 0 : 32 * kQuantWarps), 1)
    few_kernel(const __grid_constant__ CUtensorMap tw0, const __grid_constant__ CUtensorMap tw1,
               const __grid_constant__ CUtensorMap tx, const FewParams p) {
  using C = FewCfg<BN, PAIR>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBars);
  uint64_t* empty = full + C::kStages;
  uint64_t* acc_full = empty + C::kStages;
  uint64_t* acc_empty = acc_full + C::kAcc;
  uint64_t* drain = acc_empty + C::kAcc;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(drain + C::kAcc);
  uint32_t* tmem_slot = const_cast<uint32_t*>(abort_flag) + 1;
  float* red = reinterpret_cast<float*>(smem + C::kRedAt);
  float* sring = reinterpret_cast<float*>(smem + C::kScaleAt);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = p.split, rank = split > 1 ? (int)tc::cluster_rank() : 0;
  const int cid = blockIdx.x / split, n_cid = gridDim.x / split;
  const int kb0 = (int)((long long)rank * p.nkb / split), kb1 = (int)((long long)(rank + 1) * p.nkb / split);
  const int n_it = kb1 - kb0;

  if (tid == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      // (one arrival too many under mtc_debug_withhold_bytes only: in the
      // first stage, of one CTA of a cluster)
      mbar_init(&full[i], (SRC == SRC_CODES ? 1 : 2) + (i == 0 && rank == 0 && p.withhold ? 1 : 0));
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < C::kAcc; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4);
      mbar_init(&drain[i], 1);
    }
    abort_flag[0] = 0;
    fence_barrier_init();
  }
  if (warp == 5) tc::tmem_alloc(tmem_slot, C::kAcc * C::kCols);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  if (!p.early) griddep_wait();
  const int n_slots = slot_count(p.slots, p.experts, p.M, BN), n_items = n_slots * p.Nb;
  auto load_weights = [&](int s, const Slot& slot, int f0, int kb) {
    mbar_expect_tx(&full[s], SRC == SRC_CODES ? C::kStage : C::kStage - C::kBTile);
    tc::tma_load_2d(smem + s * C::kStage, &tw0, kb * 128, slot.e * p.N + f0, &full[s]);
    if constexpr (PAIR) tc::tma_load_2d(smem + s * C::kStage + kATile, &tw1, kb * 128, slot.e * p.N + f0, &full[s]);
  };
  if (p.early) {
    if (tid == 128 && cid < n_items) {
      const Slot slot = slot_at(p.slots, p.experts, p.M, BN, cid % n_slots);
      for (int i = 0; i < min(n_it, C::kStages); ++i) load_weights(i, slot, cid / n_slots * 128, kb0 + i);
    }
    griddep_wait();
  }
  griddep_launch_dependents();

  f32x2 acc[C::kCols / 2];  // sums of two tokens each
  uint32_t issued = 0;      // thread 128: stages it has loaded
  if (warp == 4) {
    // ------------------------------------------------------------ weights (and codes of the tokens) by TMA
    if (lane == 0) {
      uint32_t it = 0;
      Slot next = {};
      if (cid < n_items) next = slot_at(p.slots, p.experts, p.M, BN, cid % n_slots);  // one item ahead
      for (int w = cid; w < n_items && !abort_flag[0]; w += n_cid) {
        const Slot slot = next;
        if (w + n_cid < n_items) next = slot_at(p.slots, p.experts, p.M, BN, (w + n_cid) % n_slots);
        const int f0 = w / n_slots * 128;
        for (int i = 0; i < n_it; ++i, ++it) {
          const int s = it % C::kStages;
          if (it >= C::kStages && !mbar_wait(&empty[s], ((it / C::kStages) & 1) ^ 1, p.timeout_ns)) {
            abort_flag[0] = 1;
            break;
          }
          if (!p.early || it >= C::kStages || w != cid) load_weights(s, slot, f0, kb0 + i);
          if constexpr (SRC == SRC_CODES)
            tc::tma_load_2d(smem + s * C::kStage + C::kMats * kATile, &tx, (kb0 + i) * 128, slot.row0, &full[s]);
        }
      }
      issued = p.early && cid < n_items ? max(it, (uint32_t)min(n_it, C::kStages)) : it;
    }
  } else if (warp >= 5 && warp < 5 + C::kIssue) {
    // ------------------------------------------------------------ MMA: warp 5 + q issues the iterations q, q + kIssue, ...
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_e4m3_f32(128, BN);
      const int q = warp - 5;
      const int mine = cid < n_items ? (n_items - 1 - cid) / n_cid + 1 : 0;  // items of this CTA
      const uint32_t total = (uint32_t)mine * n_it;
      for (uint32_t it = q; it < total && !abort_flag[0]; it += C::kIssue) {
        const int s = it % C::kStages, b = it % C::kAcc;
        // The accumulator first: once it is free the sums up to it - kAcc
        // have been read, so the stage's previous phase is over and the
        // parity below means this one.
        if ((it >= C::kAcc && !mbar_wait(&acc_empty[b], ((it / C::kAcc) & 1) ^ 1, p.timeout_ns)) ||
            !mbar_wait(&full[s], (it / C::kStages) & 1, p.timeout_ns)) {
          abort_flag[0] = 1;
          break;
        }
        tc::fence_after();
        const uint32_t a0 = smem_u32(smem + s * C::kStage), b0 = a0 + C::kMats * kATile;
#pragma unroll
        for (int m = 0; m < C::kMats; ++m)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_e4m3_ss(tmem + b * C::kCols + m * BN, tc::smem_desc_k_sw128(a0 + m * kATile + 32 * j),
                        tc::smem_desc_k_sw128(b0 + 32 * j), idesc, j > 0);
        tc::commit(&acc_full[b]);
        tc::commit(&empty[s]);
      }
    }
  } else if (warp < 4) {
    // ------------------------------------------------------------ scale and add
    constexpr int kLanes = (BN + 31) / 32;  // tokens per lane
    const int feat = 32 * warp + lane;
    float* mul = reinterpret_cast<float*>(smem + C::kMulAt) + warp * 2 * C::kCols;
    uint32_t it = 0;
    for (int w = cid; w < n_items; w += n_cid) {
      const Slot slot = slot_at(p.slots, p.experts, p.M, BN, w % n_slots);
      const int ft = w / n_slots, ntok = min(BN, slot.end - slot.row0);
      const float* swp[C::kMats];
#pragma unroll
      for (int m = 0; m < C::kMats; ++m) swp[m] = p.sw[m] + ((long long)slot.e * p.Nb + ft) * p.nkb + kb0;
#pragma unroll
      for (int j = 0; j < C::kCols / 2; ++j) acc[j] = 0ull;
      // The next block's scales, tokens lane, lane + 32, ...; multiplied
      // where they are used, so that nothing waits for the loads before that.
      float sn[kLanes], wn[C::kMats];
      auto load_scales = [&](int i) {
#pragma unroll
        for (int m = 0; m < C::kMats; ++m) wn[m] = __ldg(swp[m] + i);
#pragma unroll
        for (int c = 0; c < kLanes; ++c) {
          const int t = 32 * c + lane;
          if constexpr (SRC == SRC_CODES)
            sn[c] = t < ntok ? p.sx[(long long)(kb0 + i) * p.lds + slot.row0 + t] : 0.0f;
        }
      };
      load_scales(0);
      bool ok = true;
#pragma unroll 1
      for (int i = 0; i < n_it; ++i, ++it) {
        const int b = it % C::kAcc;
        float sc[kLanes], wc[C::kMats];
#pragma unroll
        for (int c = 0; c < kLanes; ++c) sc[c] = SRC == SRC_CODES ? sn[c] : 0.0f;
#pragma unroll
        for (int m = 0; m < C::kMats; ++m) wc[m] = wn[m];
        if (i + 1 < n_it) load_scales(i + 1);
        if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[b], (it / C::kAcc) & 1, p.timeout_ns))) {
          abort_flag[0] = 1;
          ok = false;
          break;
        }
        tc::fence_after();
        // the quantizing warps wrote this block's token scales before its MMA ran
        if constexpr (SRC != SRC_CODES) sc[0] = sring[(it % C::kRing) * BN + (lane & (BN - 1))];
        // sx * sw of all tokens where every lane can read four at a time
        float* mu = mul + (it & 1) * C::kCols;
#pragma unroll
        for (int m = 0; m < C::kMats; ++m)
#pragma unroll
          for (int c = 0; c < kLanes; ++c)
            if (BN >= 32 || lane < BN) mu[m * BN + 32 * c + lane] = sc[c] * wc[m];
        __syncwarp();
        const uint32_t ta = tmem + b * C::kCols + ((uint32_t)(32 * warp) << 16);
#pragma unroll
        for (int c = 0; c < C::kCols / 16; ++c) {
          uint32_t v[16];
          tmem_ld16(ta + 16 * c, v);
          tmem_wait16(v);
          if (c == C::kCols / 16 - 1) {
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[b]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(mu + 16 * c + 4 * j);
            fma2(acc[8 * c + 2 * j], pair(v[4 * j], v[4 * j + 1]), s.x);
            fma2(acc[8 * c + 2 * j + 1], pair(v[4 * j + 2], v[4 * j + 3]), s.y);
          }
        }
      }
      if (split > 1) break;  // one item per cluster; its sums are completed below
      // The sums go to shared memory, 16 tokens at a time, and are finished
      // in loops (the epilogue's code once, not once per token: unrolled, its
      // instruction fetches took longer than the product).
      const int f0 = 128 * ft, n = f0 + feat;
      if constexpr (PAIR) {
        if (few_sync_or(!ok)) break;
      } else if (!ok) {
        break;
      }
      const float bias = (!PAIR && p.bias && n < p.N) ? __ldg(p.bias + n) : 0.0f;
#pragma unroll
      for (int c = 0; c < BN / 16; ++c) {
        if (16 * c < ntok) {
#pragma unroll
          for (int j = 0; j < 16 * C::kMats; j += 2) {
            float x, y;
            unpair(acc[(j < 16 ? 16 * c + j : BN + 16 * c + j - 16) / 2], x, y);
            red[j * 128 + feat] = x;
            red[(j + 1) * 128 + feat] = y;
          }
          const int count = min(16, ntok - 16 * c);
          if constexpr (PAIR) {
#pragma unroll 1
            for (int j = 0; j < count; ++j)
              red[j * 128 + feat] = n < p.N ? epi_act(red[j * 128 + feat], p.act) * red[(16 + j) * 128 + feat] : 0.0f;
            few_sync();
            quantize_staged(p, red, slot.row0, 16 * c, 1, count, f0, warp, lane);
            few_sync();
          } else if (n < p.N) {
#pragma unroll 1
            for (int j = 0; j < count; ++j) {
              const float a = red[j * 128 + feat] + bias;
              store1(p.Y, p.ydt, (slot.row0 + 16 * c + j) * p.ldy + n, p.act ? epi_act(a, p.act) : a);
            }
          }
        }
      }
    }
  } else if constexpr (SRC != SRC_CODES) {
    // ------------------------------------------------------------ quantize the tokens: warp q takes iterations q, q + 6, ...
    static_assert(SRC == SRC_CODES || BN == 16, "in-kernel quantization serves 16 tokens");
    // At iteration i a warp waits for the MMA of i - kStages by the parity of
    // the stage's barrier, which must not be a phase further back: the MMA of
    // i - 2 kStages has to be known complete.  The warp's last wait was for
    // the MMA of i - kQuantWarps - kStages, and a complete MMA means that all
    // those kAcc and more before it are (the sums are read in order).
    static_assert(SRC == SRC_CODES || C::kStages == kQuantWarps || C::kStages >= kQuantWarps + C::kAcc,
                  "a quantizing warp may not lap the stages");
    static_assert(C::kAcc <= C::kStages, "nor an issuing one");
    typedef typename SrcType<SRC>::T T;
    const int half = lane >> 4, l = lane & 15;
    uint32_t it = 0, mine = warp - 5 - C::kIssue;
    bool ok = true;
    for (int w = cid; w < n_items && ok; w += n_cid) {
      const Slot slot = slot_at(p.slots, p.experts, p.M, BN, w % n_slots);
      const int ntok = min(BN, slot.end - slot.row0);
      const uint32_t end = it + n_it;
      if (mine < end) {
        // lane m < 16 knows where row m is
        long long at = 0;
        if (l < ntok) {
          at = slot.row0 + l;
          if (p.order) at = p.order[at] / p.kdiv;
          at *= p.ldx;
          // The activations come into L2 ahead of the loads, which would
          // each wait behind the weights in memory otherwise.
          if (warp == 5 + C::kIssue && half == 0 && p.vec && w == cid) {
            const int n = min(p.K, kb1 * 128) - kb0 * 128;
            prefetch_l2(reinterpret_cast<const T*>(p.X) + at + kb0 * 128, (uint32_t)(n * sizeof(T)) & ~15u);
          }
        }
        for (; mine < end; mine += kQuantWarps) {
          const int s = mine % C::kStages, k0 = (kb0 + (int)(mine - it)) * 128, k = k0 + 8 * l;
          uint8_t* tile = smem + s * C::kStage + C::kMats * kATile;
          // codes of row m, whose scale this lane or another one has stored:
          // row m of the K-major SWIZZLE_128B tile, whose 16-byte chunk j sits
          // at chunk j ^ (m % 8)
          auto put = [&](int m, const float (&v)[8], float factor) {
            *reinterpret_cast<uint2*>(tile + m * 128 + (((l >> 1) ^ (m & 7)) << 4) + (l & 1) * 8) = codes8(v, factor);
          };
          float* my_scales = sring + (mine % C::kRing) * BN;
          auto stage_free = [&]() -> bool {
            return __all_sync(0xffffffffu, mine < C::kStages ||
                                               mbar_wait(&empty[s], ((mine / C::kStages) & 1) ^ 1, p.timeout_ns));
          };
          // All loads of ROUNDS row pairs in flight before the first value is
          // used; the maxima of all rows reduced together, and lane r of a
          // half warp divides for its row r alone.
          constexpr int kVec = sizeof(T) == 4 ? 2 : 1;
          auto rows = [&](auto rounds) {
            constexpr int ROUNDS = decltype(rounds)::value;
#pragma unroll 1
            for (int r0 = 0; 2 * r0 < ntok; r0 += ROUNDS) {
              uint4 raw[ROUNDS][kVec];
#pragma unroll
              for (int r = 0; r < ROUNDS; ++r) {
                const int m = 2 * (r0 + r) + half;
                const T* row = reinterpret_cast<const T*>(p.X) + __shfl_sync(0xffffffffu, at, m) + k;
#pragma unroll
                for (int q = 0; q < kVec; ++q) raw[r][q] = load16_if(reinterpret_cast<const uint4*>(row) + q, m < ntok);
              }
              uint32_t am[ROUNDS];
#pragma unroll
              for (int r = 0; r < ROUNDS; ++r) {
                float v[8];
                unpack8<T>(raw[r], v);
                am[r] = amax8(v);
              }
#pragma unroll
              for (int d = 8; d; d >>= 1)
#pragma unroll
                for (int r = 0; r < ROUNDS; ++r) am[r] = max(am[r], __shfl_xor_sync(0xffffffffu, am[r], d));
              uint32_t my_am = am[0];
#pragma unroll
              for (int r = 1; r < ROUNDS; ++r) my_am = (l & (ROUNDS - 1)) == r ? am[r] : my_am;
              const GroupScale g = group_scale(my_am);
              if (r0 == 0 && !stage_free()) ok = false;
              if (l < ROUNDS) my_scales[2 * (r0 + l) + half] = g.scale;
#pragma unroll
              for (int r = 0; r < ROUNDS; ++r) {
                const float factor = __shfl_sync(0xffffffffu, g.mul, r, 16);
                float v[8];
                unpack8<T>(raw[r], v);
                put(2 * (r0 + r) + half, v, factor);
              }
            }
          };
          if (ntok <= 0) {
            if (!stage_free()) ok = false;  // a row without an expert: nothing reads the codes
          } else if (p.vec && k0 + 128 <= p.K) {
            if (ntok <= 2) rows(std::integral_constant<int, 1>());
            else rows(std::integral_constant<int, 4 / kVec>());
          } else {
            if (!stage_free()) ok = false;
#pragma unroll 1
            for (int m = half; m < ((ntok + 1) & ~1); m += 2) {
              const long long row = __shfl_sync(0xffffffffu, at, m);
              float v[8];
              load8(reinterpret_cast<const T*>(p.X) + row + k, m < ntok ? p.K - k : 0, v);
              const GroupScale g = group_scale(half_warp_max(amax8(v)));
              put(m, v, g.mul);
              if (l == 0) my_scales[m] = g.scale;
            }
          }
          if (!ok) {
            abort_flag[0] = 1;
            break;
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[s]);
        }
      }
      it = end;
    }
  }
  __syncwarp();

  // A cluster's sums: all stages have been consumed, and their memory takes
  // the partial sums, [matrix][token][feature].
  float* part = reinterpret_cast<float*>(smem);
  const bool on = split > 1 && cid < n_items;
  const Slot slot = on ? slot_at(p.slots, p.experts, p.M, BN, cid % n_slots) : Slot{};
  const int ft = on ? cid / n_slots : 0, ntok = on ? min(BN, slot.end - slot.row0) : 0;
  const int feat = 32 * warp + lane, f0 = 128 * ft;
  if (warp < 4 && on) {
#pragma unroll
    for (int j = 0; j < C::kCols; j += 2)
      if ((j & (BN - 1)) < ntok) {
        float x, y;
        unpair(acc[j / 2], x, y);
        part[j * 128 + feat] = x;
        part[(j + 1) * 128 + feat] = y;
      }
  }
  tc::fence_before();
  __syncthreads();
  if (abort_flag[0]) {
    // A wait ran out in one of the warps (all of them see it here).  It is
    // reported, and nothing of this CTA may be in flight when it leaves:
    // neither copies into its shared memory nor MMAs that read it or write TMEM.
    if (tid == 128) {
      flag(p.status, MTC_STATUS_TIMEOUT);
      for (uint32_t j = issued > C::kStages ? issued - C::kStages : 0; j < issued; ++j)
        (void)mbar_wait(&full[j % C::kStages], (j / C::kStages) & 1, 10000000ull);
    } else if (warp >= 5 && warp < 5 + C::kIssue && lane == 0) {
      tc::commit(&drain[warp - 5]);
      (void)mbar_wait(&drain[warp - 5], 0, 100000000ull);
    }
    __syncthreads();
  }

  if (split > 1) {
    // ------------------------------------------------------------ sums over the cluster
    // Rank r completes the tokens r, r + split, ..., the partial sums added in
    // rank order; none if a rank gave up (its sums are not whole).
    tc::cluster_sync();
    // (looked at when the sums are there: in flight with them)
    const uint32_t gave_up = lane < split ? load_cluster1(abort_flag, lane) : 0u;
    if ((!PAIR || warp < 4) && on) {
      // a warp (of all, or of those that quantize) per token, 4 features per
      // lane, all ranks' loads in flight
      const int n_warps = PAIR ? 4 : (int)(blockDim.x >> 5);
      const int f4 = 4 * lane, n4 = f0 + f4;
      float bias[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) bias[q] = (!PAIR && p.bias && n4 + q < p.N) ? __ldg(p.bias + n4 + q) : 0.0f;
      const int count = rank < ntok ? (ntok - 1 - rank) / split + 1 : 0;
#pragma unroll 1
      for (int i = warp; i < count; i += n_warps) {
        const int j = rank + i * split;
        float4 x[C::kMats][kMaxCluster];
#pragma unroll
        for (int m = 0; m < C::kMats; ++m)
#pragma unroll
          for (int q = 0; q < kMaxCluster; ++q)
            if (q < split) x[m][q] = load_cluster4(part + (m * BN + j) * 128 + f4, q);
        float a[C::kMats][4];
#pragma unroll
        for (int m = 0; m < C::kMats; ++m) {
          a[m][0] = a[m][1] = a[m][2] = a[m][3] = 0.0f;
#pragma unroll
          for (int q = 0; q < kMaxCluster; ++q)
            if (q < split) {
              a[m][0] += x[m][q].x;
              a[m][1] += x[m][q].y;
              a[m][2] += x[m][q].z;
              a[m][3] += x[m][q].w;
            }
        }
        if constexpr (PAIR) {
          float h[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) h[q] = n4 + q < p.N ? epi_act(a[0][q], p.act) * a[C::kMats - 1][q] : 0.0f;
          *reinterpret_cast<float4*>(red + i * 128 + f4) = make_float4(h[0], h[1], h[2], h[3]);
        } else {
          const long long y = (slot.row0 + j) * p.ldy + n4;
          const bool bad = __any_sync(0xffffffffu, gave_up);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (n4 + q < p.N && !bad) {
              const float o = a[0][q] + bias[q];
              store1(p.Y, p.ydt, y + q, p.act ? epi_act(o, p.act) : o);
            }
        }
      }
      if constexpr (PAIR) {
        few_sync();
        if (!__any_sync(0xffffffffu, gave_up)) quantize_staged(p, red, slot.row0, rank, split, count, f0, warp, lane);
      }
    }
    tc::cluster_sync();  // no CTA leaves while another reads its partial sums
  }
  if (warp == 5) {
    tc::fence_after();
    tc::tmem_dealloc(tmem, C::kAcc * C::kCols);
  }
}

// ---------------------------------------------------------------------------
// many_kernel
// ---------------------------------------------------------------------------
constexpr int kManyStages = 4;
constexpr uint32_t kManyStage = 3 * kATile;
constexpr int kManyWarps = 8;                         // scaling warps: 2 column halves x 4 lane quadrants
constexpr int kManyThreads = 32 * (kManyWarps + 4);   // + a warpgroup: codes, 2 for MMAs, scales
// A row of each scaling thread, for values that cannot leave as vectors (the
// stride of 5 16-byte units keeps 16-byte accesses free of bank conflicts):
// 4000 x 1024 x 3001 bf16 takes 42.2 us, 95.6 with every thread storing
// its own row.
constexpr int kRowLd = 20;
constexpr uint32_t kStaging = kManyWarps * 32 * kRowLd * 4;
// Scales of an iteration: sx of 128 rows, sw of the two scale blocks of the
// features, and the tile {first row, end row, feature tile}, in a ring that
// a warp of its own fills together with a stage (4-byte asynchronous copies:
// rows start anywhere, and no copy waits for a load).  It writes iteration i after
// the MMA of i - kManyStages has completed, which was issued after the sums
// of i - kManyStages - 2 were read: more slots than kManyStages + 2 are never
// overwritten early.
constexpr int kScaleSlots = 8, kScaleLd = 132;
static_assert(kScaleSlots > kManyStages + 2, "a scale slot must outlive its reader");
constexpr uint32_t kManyScales = kManyStages * kManyStage + kStaging;
constexpr uint32_t kManyTiles = kManyScales + kScaleSlots * kScaleLd * 4;
constexpr uint32_t kManyBias = kManyTiles + kScaleSlots * 16;  // 128 values per scaling warp
constexpr uint32_t kManyBars = kManyBias + kManyWarps * 128 * 4;
constexpr size_t kManySmem = 1024 + kManyBars + 256;
static_assert(kManySmem <= 227 * 1024, "shared memory of one CTA");
// Registers: 384 threads are launched with 168 each; the scaling warps (128
// fp32 sums and the values loaded) take what the last warpgroup gives back:
// 2 x 128 x 224 + 128 x 56 <= 384 x 168.
constexpr int kScaleRegs = 224, kIssueRegs = 56;

struct ManyParams {
  int nkb, N, Nb, n_tiles;            // n_tiles: feature tiles (256 wide, or 128 of gate and up)
  const float* sw[2];
  const int32_t* slots;
  int M;
  const float* sx;
  long long lds;
  void* Y;
  int ydt, vec;                       // vec: rows of Y start on 32 bytes
  long long ldy;
  const float* bias;
  float one;                          // 1
  uint8_t* hq;                        // GATED: codes [row][ldh] and scales [n / 128][hs_ld]
  long long ldh;
  float* hs;
  long long hs_ld;
  uint32_t* status;
  unsigned long long timeout_ns;
  uint32_t withhold;                  // diagnostic: the first stage of a CTA never becomes full
};

// Barrier of the two warps that share rows (64 threads), which tells both
// whether either of them passed true.
__device__ __forceinline__ bool pair_sync_or(int id, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "bar.red.or.pred q, %1, 64, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"((uint32_t)x)
      : "memory");
  return r != 0;
}

// 32 bytes at a 32-byte aligned address (a whole sector from one thread).
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// What becomes of the sums: stored as they are, after bias and activation
// (kEpilogue + activation), or act(gate) * up, quantized (kGated + activation).
enum { kPlain = 0, kEpilogue = 4, kGated = 8 };

template <int MODE>
__global__ void __launch_bounds__(kManyThreads, 1)
    many_kernel(const __grid_constant__ CUtensorMap tw0, const __grid_constant__ CUtensorMap tw1,
                const __grid_constant__ CUtensorMap tx, const ManyParams p) {
  constexpr bool GATED = MODE >= kGated;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* staging = reinterpret_cast<float*>(smem + kManyStages * kManyStage);
  float* scales = reinterpret_cast<float*>(smem + kManyScales);  // [kScaleSlots][kScaleLd]
  int4* tiles = reinterpret_cast<int4*>(smem + kManyTiles);      // [kScaleSlots]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kManyBars);
  uint64_t* empty = full + kManyStages;
  uint64_t* acc_full = empty + kManyStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;        // [2]
  uint64_t* drain = acc_empty + 2;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(drain + 2);
  uint32_t* tmem_slot = const_cast<uint32_t*>(abort_flag) + 1;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  griddep_wait();
  griddep_launch_dependents();
  const int n_slots = slot_count(p.slots, 0, p.M, 128);
  const int n_work = n_slots * p.n_tiles;
  if ((int)blockIdx.x >= n_work) return;

  if (tid == 0) {
    for (int i = 0; i < kManyStages; ++i) {
      // the codes, the lanes' scales, the tile (and see few_kernel)
      mbar_init(&full[i], 1 + 32 + 1 + (i == 0 && p.withhold ? 1 : 0));
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kManyWarps);
      mbar_init(&drain[i], 1);
    }
    abort_flag[0] = 0;
    fence_barrier_init();
  }
  if (warp == kManyWarps + 1) tc::tmem_alloc(tmem_slot, 512);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  // All threads, once their part is over.  (In either branch: what follows it
  // would otherwise cost the scaling warps registers, and 4096 x 4096 x 14336
  // 255 us instead of 246.)
  auto finish = [&]() {
    __syncwarp();
    tc::fence_before();
    asm volatile("bar.sync 0, %0;" ::"n"(kManyThreads) : "memory");
  };

  if (warp >= kManyWarps) {
    regs_dec<kIssueRegs>();
    uint32_t issued = 0;  // the loading thread: stages it has loaded
    // Tiles in time: a dense product runs the token tiles of one feature tile
    // together (all tokens stay in L2), a grouped one the feature tiles of one
    // token tile (its expert's weights do).
    auto slot_of = [&](int t) { return p.slots ? t / p.n_tiles : t % n_slots; };
    auto feature_tile = [&](int t) { return p.slots ? t % p.n_tiles : t / n_slots; };
    // the stage of iteration `it`, once the MMA that read it before is over
    auto stage_free = [&](uint32_t it) {
      return it < kManyStages || mbar_wait(&empty[it % kManyStages], ((it / kManyStages) & 1) ^ 1, p.timeout_ns);
    };
    if (warp == kManyWarps) {
      // ------------------------------------------------------------ codes by TMA
      if (lane == 0) {
        uint32_t it = 0;
        Slot next = slot_at(p.slots, 0, p.M, 128, slot_of(blockIdx.x));  // one tile ahead
        for (int t = blockIdx.x; t < n_work && !abort_flag[0]; t += gridDim.x) {
          const Slot slot = next;
          if (t + (int)gridDim.x < n_work) next = slot_at(p.slots, 0, p.M, 128, slot_of(t + gridDim.x));
          const int f0 = slot.e * p.N + feature_tile(t) * (GATED ? 128 : 256);
          for (int kb = 0; kb < p.nkb; ++kb, ++it) {
            if (!stage_free(it)) {
              abort_flag[0] = 1;
              break;
            }
            const int s = it % kManyStages;
            uint8_t* st = smem + s * kManyStage;
            mbar_expect_tx(&full[s], kManyStage);
            tc::tma_load_2d(st, &tx, kb * 128, slot.row0, &full[s]);
            tc::tma_load_2d(st + kATile, &tw0, kb * 128, f0, &full[s]);
            tc::tma_load_2d(st + 2 * kATile, GATED ? &tw1 : &tw0, kb * 128, GATED ? f0 : f0 + 128, &full[s]);
          }
        }
        issued = it;
      }
    } else if (warp == kManyWarps + 3) {
      // ------------------------------------------------------------ scales and tiles
      uint32_t it = 0;
      Slot next = slot_at(p.slots, 0, p.M, 128, slot_of(blockIdx.x));
      for (int t = blockIdx.x; t < n_work; t += gridDim.x) {
        const Slot slot = next;
        if (t + (int)gridDim.x < n_work) next = slot_at(p.slots, 0, p.M, 128, slot_of(t + gridDim.x));
        const int nt = feature_tile(t);
        // lanes 0 and 1 fetch the features' scales, every lane those of the
        // rows lane, lane + 32, ...; a row past the end takes the last row's
        // scale (its values are never stored)
        const long long sb = (long long)slot.e * p.Nb;
        const float* sw = GATED ? p.sw[lane & 1] + (sb + nt) * p.nkb
                                : p.sw[0] + (sb + min(2 * nt + (lane & 1), p.Nb - 1)) * p.nkb;
        const float* sx[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) sx[j] = p.sx + min(slot.row0 + lane + 32 * j, slot.end - 1);
        bool ok = true;
        for (int kb = 0; kb < p.nkb; ++kb, ++it) {
          if (!__all_sync(0xffffffffu, stage_free(it))) {
            ok = false;
            break;
          }
          if (lane == 0) tiles[it % kScaleSlots] = make_int4(slot.row0, slot.end, nt, 0);
          float* sc = scales + (it % kScaleSlots) * kScaleLd;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            copy4_async(sc + lane + 32 * j, sx[j]);
            sx[j] += p.lds;
          }
          if (lane < 2) copy4_async(sc + 128 + lane, sw + kb);
          copy4_arrive(&full[it % kManyStages]);
          // (that arrival answers for the copies only: the tile, an ordinary
          // store, is published by one of its own)
          if (lane == 0) mbar_arrive(&full[it % kManyStages]);
        }
        if (!ok && lane == 0) abort_flag[0] = 1;
        if (__any_sync(0xffffffffu, !ok || abort_flag[0])) break;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp <= kManyWarps + 2 && lane == 0) {
      // ---------------------------------------------------------- MMA: one warp per accumulator
      constexpr uint32_t idesc = idesc_e4m3_f32(128, 256);
      const int b = warp - kManyWarps - 1;
      const uint32_t total = (uint32_t)((n_work - 1 - (int)blockIdx.x) / (int)gridDim.x + 1) * p.nkb;
      for (uint32_t it = b; it < total && !abort_flag[0]; it += 2) {
        const int s = it % kManyStages;
        // (the accumulator first: see few_kernel)
        if ((it >= 2 && !mbar_wait(&acc_empty[b], ((it >> 1) & 1) ^ 1, p.timeout_ns)) ||
            !mbar_wait(&full[s], (it / kManyStages) & 1, p.timeout_ns)) {
          abort_flag[0] = 1;
          break;
        }
        tc::fence_after();
        const uint32_t a0 = smem_u32(smem + s * kManyStage), b0 = a0 + kATile;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          mma_e4m3_ss(tmem + b * 256, tc::smem_desc_k_sw128(a0 + 32 * j), tc::smem_desc_k_sw128(b0 + 32 * j), idesc,
                      j > 0);
        tc::commit(&acc_full[b]);
        tc::commit(&empty[s]);
      }
    }
    finish();
    if (abort_flag[0]) {
      // a wait ran out: reported, and nothing left in flight (see few_kernel)
      if (warp == kManyWarps && lane == 0) {
        flag(p.status, MTC_STATUS_TIMEOUT);
        for (uint32_t j = issued > kManyStages ? issued - kManyStages : 0; j < issued; ++j)
          (void)mbar_wait(&full[j % kManyStages], (j / kManyStages) & 1, 10000000ull);
      } else if (warp <= kManyWarps + 2 && lane == 0) {
        tc::commit(&drain[warp - kManyWarps - 1]);
        (void)mbar_wait(&drain[warp - kManyWarps - 1], 0, 100000000ull);
      }
      asm volatile("bar.sync 5, 128;" ::: "memory");  // these four warps
    }
    if (warp == kManyWarps + 1) {
      tc::fence_after();
      tc::tmem_dealloc(tmem, 512);
    }
  } else {
    // ------------------------------------------------------------ scale and add, then store
    regs_inc<kScaleRegs>();
    const int quad = warp & 3, hf = warp >> 2;  // TMEM lanes 32 quad .., columns 128 hf ..
    float* my_row = staging + (warp * 32 + lane) * kRowLd;
    float* bias = reinterpret_cast<float*>(smem + kManyBias) + 128 * warp;
    const int my_scale = 32 * quad + lane;
    // TMEM columns of the sums 0..63 and 64..127: 128 features, or 64 of the
    // gate and the same 64 of the up matrix
    const uint32_t lanes = tmem + ((uint32_t)(32 * quad) << 16);
    const uint32_t tm_a = lanes + (GATED ? 64 : 128) * hf, tm_b = tm_a + (GATED ? 128 : 64);
    uint32_t it = 0;
    int turn = 0;
    bool stop = false;
    for (int t = blockIdx.x; t < n_work && !stop; t += gridDim.x) {
      f32x2 acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = 0ull;
      bool ok = true;
#pragma unroll 1
      for (int kb = 0; kb < p.nkb; ++kb, ++it) {
        const int b = it & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[b], (it >> 1) & 1, p.timeout_ns))) {
          abort_flag[0] = 1;
          ok = false;
          break;
        }
        tc::fence_after();
        // this block's scales were written before its MMA ran
        const float* slot = scales + (it % kScaleSlots) * kScaleLd;
        const float sa = slot[my_scale] * slot[128 + (GATED ? 0 : hf)];
        const float sb = GATED ? slot[my_scale] * slot[129] : sa;
        const f32x2 sc_a = pair(sa, sa), sc_b = pair(sb, sb);
        // (the next columns are loaded while these are added)
        uint32_t v[2][16];
        tmem_ld16(tm_a + b * 256, v[0]);
        tmem_wait16(v[0]);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (c < 7) tmem_ld16((c < 3 ? tm_a : tm_b) + b * 256 + 16 * ((c + 1) & 3), v[(c + 1) & 1]);
#pragma unroll
          for (int j = 0; j < 8; ++j) fma2(acc[8 * c + j], pair(v[c & 1][2 * j], v[c & 1][2 * j + 1]), c < 4 ? sc_a : sc_b);
          if (c < 7) tmem_wait16(v[(c + 1) & 1]);
          if (c == 6) {
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[b]);
          }
        }
      }
      const int4 tile = tiles[(it - 1) % kScaleSlots];
      const int nt = tile.z, m0 = tile.x + 32 * quad;
      const int n0 = GATED ? nt * 128 + 64 * hf : nt * 256 + 128 * hf;  // first feature of this warp
      const int left = p.N - n0;                                        // features of this warp that exist
      const bool mine = ok && m0 + lane < tile.y;                       // this thread's row exists
      if constexpr (GATED) {
        if (left < 64) {
          // the matrix ends in these columns: act(0) * 0 behind them
#pragma unroll
          for (int j = 0; j < 64; ++j) {
            float x, y;
            unpair(acc[j], x, y);
            acc[j] = pair(2 * (j & 31) < left ? x : 0.0f, 2 * (j & 31) + 1 < left ? y : 0.0f);
          }
        }
        float largest = 0.0f;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          float g[2], u[2];
          unpair(acc[j], g[0], g[1]);
          unpair(acc[32 + j], u[0], u[1]);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            g[q] = act_fast<MODE - kGated>(g[q]) * u[q];
            largest = max_abs(largest, g[q]);
          }
          acc[j] = pair(g[0], g[1]);
        }
        uint32_t am = __float_as_uint(largest);
        // The scale covers the columns of two warps.  (A slot of this
        // exchange is written again two tiles later, after a barrier that the
        // other warp reaches once it has read it.)  Both stop at the same tile.
        turn ^= 1;
        reinterpret_cast<uint32_t*>(my_row)[turn] = am;
        stop = pair_sync_or(1 + quad, !ok);
        am = max(am, reinterpret_cast<const uint32_t*>(staging + ((warp ^ 4) * 32 + lane) * kRowLd)[turn]);
        const GroupScale gs = group_scale(am);
        if (mine) {
          if (hf == 0) p.hs[(long long)nt * p.hs_ld + m0 + lane] = gs.scale;
          uint8_t* dst = p.hq + (long long)(m0 + lane) * p.ldh + n0;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float h[4];
              unpair(acc[16 * c + 2 * j], h[0], h[1]);
              unpair(acc[16 * c + 2 * j + 1], h[2], h[3]);
              w[j] = gs.mul == 0.0f ? 0u : codes2(h[0], h[1], gs.mul) | codes2(h[2], h[3], gs.mul) << 16;
            }
            // (n0 and ldh are multiples of 32; codes past N are zero)
            if (n0 + 32 * c < p.ldh) store32(dst + 32 * c, w);
          }
        }
      } else if (!ok) {
        stop = true;
      } else {
        if constexpr (MODE >= kEpilogue) {
          // the warp's 128 values of the bias, then read four at a time
          float4 f;
          f.x = p.bias && 4 * lane < left ? __ldg(p.bias + n0 + 4 * lane) : 0.0f;
          f.y = p.bias && 4 * lane + 1 < left ? __ldg(p.bias + n0 + 4 * lane + 1) : 0.0f;
          f.z = p.bias && 4 * lane + 2 < left ? __ldg(p.bias + n0 + 4 * lane + 2) : 0.0f;
          f.w = p.bias && 4 * lane + 3 < left ? __ldg(p.bias + n0 + 4 * lane + 3) : 0.0f;
          *reinterpret_cast<float4*>(bias + 4 * lane) = f;
          __syncwarp();
        }
        const long long y0 = (long long)(m0 + lane) * p.ldy + n0;
        uint8_t* y = reinterpret_cast<uint8_t*>(p.Y) + y0 * (p.ydt == MTC_F32 ? 4 : 2);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          float o[16];
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            unpair(acc[8 * c + j / 2], o[j], o[j + 1]);
            unpair(acc[8 * c + j / 2 + 1], o[j + 2], o[j + 3]);
            if constexpr (MODE >= kEpilogue) {
              const float4 f = *reinterpret_cast<const float4*>(bias + 16 * c + j);
              o[j] = act_fast<MODE - kEpilogue>(o[j] + f.x);
              o[j + 1] = act_fast<MODE - kEpilogue>(o[j + 1] + f.y);
              o[j + 2] = act_fast<MODE - kEpilogue>(o[j + 2] + f.z);
              o[j + 3] = act_fast<MODE - kEpilogue>(o[j + 3] + f.w);
            }
          }
          if (p.vec && 16 * c + 16 <= left) {
            if (p.ydt != MTC_F32) {
              uint32_t w[8];
#pragma unroll
              for (int j = 0; j < 8; ++j)
                w[j] = p.ydt == MTC_BF16 ? pack2(MTC_BF16, o[2 * j], o[2 * j + 1]) : pack2(MTC_F16, o[2 * j], o[2 * j + 1]);
              if (mine) store32(y + 32 * c, w);
            } else {
              // Sums leave through a multiplication by p.one (= 1): stored
              // directly, the compiler lays them out for the stores and moves
              // every one of them in the main loop (466 against 415 thousand
              // cycles at 4096 x 4096 x 14336).
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(o[8 * h + j] * p.one);
                if (mine) store32(y + 64 * c + 32 * h, w);
              }
            }
          } else if (16 * c < left) {
            // The last columns, or rows that do not start on 32 bytes: by way
            // of shared memory, half a warp per row, one value per lane.
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<float4*>(my_row + j) =
                  make_float4(o[j] * p.one, o[j + 1] * p.one, o[j + 2] * p.one, o[j + 3] * p.one);
            __syncwarp();
            const int col = lane & 15;
#pragma unroll
            for (int r = lane >> 4; r < 32; r += 2)
              if (m0 + r < tile.y && 16 * c + col < left)
                store1(p.Y, p.ydt, (long long)(m0 + r) * p.ldy + n0 + 16 * c + col, (my_row - lane * kRowLd)[r * kRowLd + col]);
            __syncwarp();
          }
        }
      }
    }
    finish();
  }
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
// `bound` items at most.  While they leave SMs idle their inputs are split
// over clusters of up to 8 CTAs (one SM streams at most about twice its share
// of the memory bandwidth): over as many as keep all items on the device at
// once and give every CTA at least four blocks of 128 inputs.
// 1 x 14336 x 4096, 32 items: 14.7 us split by 4, 31.3 whole; 1 x 8192 x 2048,
// 16 items: 8.2 us; split by 8, which does not fit at once, 13.6.
// 1 x 896 x 128: 4.6 us whole, 5.2 split by 2.  A split launch has one
// cluster per item.
template <int BN, int SRC, bool PAIR>
int launch_few(const CUtensorMap& tw0, const CUtensorMap& tw1, const CUtensorMap& tx, FewParams& p, long long bound,
               int sms, cudaStream_t st, const char* who) {
  static std::atomic<uint64_t> ready{0};
  static ClusterCounts clusters;
  constexpr size_t smem = FewCfg<BN, PAIR>::kSmem;
  MTC_CHECK_CUDA(allow_smem(few_kernel<BN, SRC, PAIR>, smem, ready), who);
  constexpr int threads = FewCfg<BN, PAIR>::kThreads + (SRC == SRC_CODES ? 0 : 32 * kQuantWarps);
  p.split = 1;
  for (int s = 2; s <= kMaxCluster && bound * s <= sms && p.nkb >= 4 * s; ++s)
    if (bound <= resident_clusters(few_kernel<BN, SRC, PAIR>, threads, smem, s, clusters)) p.split = s;
  const int grid = p.split > 1 ? (int)bound * p.split : (int)(bound < sms ? bound : sms);
  MTC_CHECK_CUDA(launch_chained(few_kernel<BN, SRC, PAIR>, dim3(grid), dim3(threads), smem, st, p.split, tw0, tw1, tx,
                                p),
                 who);
  return MTC_OK;
}

// Tiles that gate / up pairs come in, too: activations.
template <int BN, int SRC>
int launch_few(const CUtensorMap& tw0, const CUtensorMap& tw1, const CUtensorMap& tx, FewParams& p, long long bound,
               int sms, bool pair, cudaStream_t st, const char* who) {
  return pair ? launch_few<BN, SRC, true>(tw0, tw1, tx, p, bound, sms, st, who)
              : launch_few<BN, SRC, false>(tw0, tw1, tx, p, bound, sms, st, who);
}

template <int MODE>
int launch_many(const CUtensorMap& tw0, const CUtensorMap& tw1, const CUtensorMap& tx, const ManyParams& p, int grid,
                cudaStream_t st, const char* who) {
  static std::atomic<uint64_t> ready{0};
  MTC_CHECK_CUDA(allow_smem(many_kernel<MODE>, kManySmem, ready), who);
  MTC_CHECK_CUDA(launch_chained(many_kernel<MODE>, dim3(grid), dim3(kManyThreads), kManySmem, st, 1, tw0, tw1, tx, p),
                 who);
  return MTC_OK;
}

}  // namespace

namespace {
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
  static const EncodeTiledFn fn = []() -> EncodeTiledFn {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(p);
    return nullptr;
  }();
  return fn;
}
}  // namespace

// TMA map of rows of codes: boxes of 128 inputs x box_rows in the K-major
// 128-byte swizzle; inputs past K and rows past `rows` read as zero.
int encode_codes_map(CUtensorMap* map, const uint8_t* codes, long long ld, long long K, long long rows, int box_rows,
                     const char* who) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) {
    set_error("%s: cuTensorMapEncodeTiled unavailable from the driver", who);
    return MTC_ERR_CUDA;
  }
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r =
      enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes), dims, strides, box, estr,
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("%s: cuTensorMapEncodeTiled failed (%d)", who, (int)r);
    return MTC_ERR_CUDA;
  }
  return MTC_OK;
}

int check_matrix(const mtc_fp8_matrix* w, const char* who) {
  MTC_REQUIRE(w && w->codes && w->scales, "%s: null matrix", who);
  MTC_REQUIRE(w->K >= 1 && w->N >= 1 && w->E >= 1, "%s: bad matrix shape %d x (%d, %d)", who, w->E, w->K, w->N);
  MTC_REQUIRE(w->K <= kMaxRows && w->N <= kMaxRows, "%s: more than 2^31 inputs or outputs", who);
  MTC_REQUIRE(w->ldk >= w->K && (w->ldk & 15) == 0, "%s: row stride %lld of the codes is not a multiple of 16 >= K",
              who, (long long)w->ldk);
  MTC_REQUIRE((reinterpret_cast<uintptr_t>(w->codes) & 15) == 0, "%s: codes not 16-byte aligned", who);
  MTC_REQUIRE(aligned(w->scales), "%s: scales not aligned to their elements", who);
  MTC_REQUIRE((long long)w->E * w->N <= 0x7fffff00ll, "%s: more than 2^31 weight rows", who);
  return MTC_OK;
}

int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64 && (sms = known[dev].load(std::memory_order_relaxed)) > 0) return sms;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < 64) known[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

int launch_product(const Product& a, cudaStream_t st, const char* who) {
  const mtc_fp8_matrix* w = a.w[0];
  const int nkb = (w->K + kBlock - 1) / kBlock, Nb = (w->N + kBlock - 1) / kBlock;
  const int n_mats = a.w[1] ? 2 : 1;
  const int sms = sm_count();
  MTC_REQUIRE(sms > 0, "%s: no CUDA device", who);
  if (a.slot_bound <= 0) return MTC_OK;
  MTC_REQUIRE((long long)a.slot_bound * Nb <= kMaxRows, "%s: more than 2^31 tiles", who);
  CUtensorMap tw[2], tx;
  for (int i = 0; i < n_mats; ++i) {
    const mtc_fp8_matrix* m = a.w[i];
    if (m->map_ready) {
      memcpy(&tw[i], m->map, sizeof(CUtensorMap));
    } else {
      const int rc = encode_codes_map(&tw[i], m->codes, m->ldk, m->K, (long long)m->E * m->N, 128, who);
      if (rc != MTC_OK) return rc;
    }
  }
  if (n_mats == 1) tw[1] = tw[0];
  tx = tw[0];
  if (a.xq) {
    const int rc = encode_codes_map(&tx, a.xq, a.ldq, w->K, a.rows, a.tile, who);
    if (rc != MTC_OK) return rc;
  }
  if (a.many) {
    ManyParams p = {};
    p.nkb = nkb;
    p.N = w->N;
    p.Nb = Nb;
    p.n_tiles = n_mats == 2 ? Nb : (w->N + 255) / 256;
    p.sw[0] = w->scales;
    p.sw[1] = a.w[1] ? a.w[1]->scales : w->scales;
    p.slots = a.slots;
    p.M = a.rows;
    p.sx = a.sx;
    p.lds = a.lds;
    p.Y = a.Y;
    p.ydt = a.ydt;
    p.ldy = a.ldy;
    p.vec = (reinterpret_cast<uintptr_t>(a.Y) & 31) == 0 && (a.ldy & (a.ydt == MTC_F32 ? 7 : 15)) == 0;
    p.bias = a.bias;
    p.one = 1.0f;
    p.hq = a.hq;
    p.ldh = a.ldh;
    p.hs = a.hs;
    p.hs_ld = a.hs_ld;
    p.status = a.status;
    p.timeout_ns = wait_limit_ns();
    p.withhold = take_withheld_bytes();
    const long long work = (long long)a.slot_bound * p.n_tiles;
    const int grid = (int)(work < sms ? work : sms);
    if (n_mats == 2) {
      switch (a.gate_act) {
        case MTC_ACT_RELU: return launch_many<kGated + MTC_ACT_RELU>(tw[0], tw[1], tx, p, grid, st, who);
        case MTC_ACT_SILU: return launch_many<kGated + MTC_ACT_SILU>(tw[0], tw[1], tx, p, grid, st, who);
        case MTC_ACT_GELU_TANH: return launch_many<kGated + MTC_ACT_GELU_TANH>(tw[0], tw[1], tx, p, grid, st, who);
        default: return launch_many<kGated + MTC_ACT_NONE>(tw[0], tw[1], tx, p, grid, st, who);
      }
    }
    switch (a.act) {
      case MTC_ACT_RELU: return launch_many<kEpilogue + MTC_ACT_RELU>(tw[0], tw[1], tx, p, grid, st, who);
      case MTC_ACT_SILU: return launch_many<kEpilogue + MTC_ACT_SILU>(tw[0], tw[1], tx, p, grid, st, who);
      case MTC_ACT_GELU_TANH: return launch_many<kEpilogue + MTC_ACT_GELU_TANH>(tw[0], tw[1], tx, p, grid, st, who);
      default: break;
    }
    if (a.bias) return launch_many<kEpilogue + MTC_ACT_NONE>(tw[0], tw[1], tx, p, grid, st, who);
    return launch_many<kPlain>(tw[0], tw[1], tx, p, grid, st, who);
  }
  FewParams p = {};
  p.K = w->K;
  p.nkb = nkb;
  p.N = w->N;
  p.Nb = Nb;
  p.sw[0] = w->scales;
  p.sw[1] = a.w[1] ? a.w[1]->scales : w->scales;
  p.slots = a.slots;
  p.experts = a.experts;
  p.M = a.rows;
  p.sx = a.sx;
  p.lds = a.lds;
  p.order = a.order;
  p.kdiv = a.kdiv;
  p.Y = a.Y;
  p.ydt = a.ydt;
  p.ldy = a.ldy;
  p.bias = a.bias;
  p.act = n_mats == 2 ? a.gate_act : a.act;
  p.hq = a.hq;
  p.ldh = a.ldh;
  p.hs = a.hs;
  p.hs_ld = a.hs_ld;
  p.early = a.early;
  p.status = a.status;
  p.timeout_ns = wait_limit_ns();
  p.withhold = take_withheld_bytes();
  const long long bound = (long long)Nb * a.slot_bound;
  const bool pair = n_mats == 2;
  if (a.xq) {
    MTC_REQUIRE(!pair, "%s: codes of a gate / up pair in tiles of %d rows", who, a.tile);
    switch (a.tile) {
      case 16: return launch_few<16, SRC_CODES, false>(tw[0], tw[1], tx, p, bound, sms, st, who);
      case 32: return launch_few<32, SRC_CODES, false>(tw[0], tw[1], tx, p, bound, sms, st, who);
      case 64: return launch_few<64, SRC_CODES, false>(tw[0], tw[1], tx, p, bound, sms, st, who);
      default: return launch_few<128, SRC_CODES, false>(tw[0], tw[1], tx, p, bound, sms, st, who);
    }
  }
  p.X = a.X;
  p.ldx = a.ldx;
  p.vec = (reinterpret_cast<uintptr_t>(a.X) & 15) == 0 && a.ldx % (a.xdt == MTC_F32 ? 4 : 8) == 0;
  if (a.xdt == MTC_F32) return launch_few<16, SRC_F32>(tw[0], tw[1], tx, p, bound, sms, pair, st, who);
  if (a.xdt == MTC_BF16) return launch_few<16, SRC_BF16>(tw[0], tw[1], tx, p, bound, sms, pair, st, who);
  return launch_few<16, SRC_F16>(tw[0], tw[1], tx, p, bound, sms, pair, st, who);
}

}  // namespace fp8
}  // namespace mtc

extern "C" int mtc_fp8_matrix_init(mtc_fp8_matrix* w) {
  mtc::clear_error();
  const int rc = mtc::fp8::check_matrix(w, "mtc_fp8_matrix_init");
  if (rc != MTC_OK) return rc;
  static_assert(sizeof(CUtensorMap) == sizeof(w->map), "TMA descriptor size");
  CUtensorMap map;
  const int re = mtc::fp8::encode_codes_map(&map, w->codes, w->ldk, w->K, (long long)w->E * w->N, 128,
                                            "mtc_fp8_matrix_init");
  if (re != MTC_OK) return re;
  memcpy(w->map, &map, sizeof(map));
  w->map_ready = 1;
  return MTC_OK;
}
