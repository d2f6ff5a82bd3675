// int8 matrix product with a scale for each token and each channel, on tcgen05 (kind::i8).
//
//   out[m][n] = (sum_k xq[m][k] wq[n][k]) * xs[m] * ws[n]   (+ residual, or SwiGLU over pairs)
//
// The sums are exact int32 (k up to 2^31 / 127^2 = 133,000 values), so neither the tile shape nor
// a split of K changes a result: a row has the same bits whatever rows share its call.
//
// Layout. The weights are the M side of the tensor-core tile (128 channels = 128 TMEM lanes) and
// the tokens its N side (16 to 256 columns). So a call of few tokens pads them to 16, not 128;
// an epilogue warp holds 32 neighbouring channels of one token, whose stores are contiguous; the
// channel's scale is one register and the token's a broadcast load. Both operands arrive by TMA
// (128-byte swizzle, 128 values of K a stage; rows and values past the ends read zeros).
//
// Schedule. Warp 0 issues TMA into a ring, warp 1 issues four MMAs (K = 32 each) a stage, warps
// 2-9 drain the accumulator (two warps a TMEM lane quarter, half the tokens each; the residual's
// loads run one chunk ahead). Many tiles: a persistent grid with two accumulators, so that one
// tile's epilogue runs behind the next one's products; for a long K by pairs of CTAs, whose tensor
// cores share the tokens' rows (256 channels a tile). Few tiles (fewer than the SMs): a cluster
// of 2 to 8 CTAs splits K, each leaves its int32 partial tile in its own shared memory, and after
// one cluster barrier every CTA adds up its share of the tokens over distributed shared memory.
// No workspace, no atomics.
//
// Bound: weight bytes from DRAM up to some 100 tokens; beyond, the operands' way from L2 for single CTAs, the
// tensor cores for pairs (8192^3: 2850 TOP/s, bf16 out 3060).
#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "bulk.cuh"
#include "common.h"
#include "dev_util.cuh"
#include "ops.h"

namespace qasr {
namespace {

constexpr int kCh = 128;    // channels of a tile
constexpr int kKb = 128;    // K bytes of a stage
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kMaxCluster = 8;

template <int NT, bool PAIR = false>
struct Shape {
  static constexpr int kStage = kCh * kKb + (PAIR ? NT / 2 : NT) * kKb;
  static constexpr int kStages = PAIR ? 6 : NT >= 256 ? 4 : NT >= 128 ? 6 : NT >= 64 ? 4 : NT >= 32 ? 5 : 6;
  static constexpr int kHalf = NT / 2;                       // tokens of an epilogue warp
  static constexpr int kSmem = 1024 + kStages * kStage + kEpiWarps * kHalf * 4 + 256;
  static_assert(kStages * kStage >= NT * kCh * 4, "the partial tile reuses the ring");
};

// Instruction descriptor: int32 accumulator, signed 8-bit A and B, both K-major, M = channels, N = nt.
__device__ __forceinline__ uint32_t idesc_i8(int nt, int channels) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(nt >> 3) << 17) | ((uint32_t)(channels >> 4) << 24);
}

struct LinArgs {
  long long m;
  int n, nk, ct, tiles, split;
  int nt;  // tokens of a tile: a multiple of 16, of 32 above 64, at most the template's NT
  const float *xs, *ws;
  const void* resid;
  long long ldr, ldo;
  void* out;
  OpsErrors* err;
};

__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(1024 >> 4) << 32;  // 8-row groups 1024 bytes apart
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;            // 128-byte swizzle
  return d;
}

// The copies and products are issued by an elected lane of a warp that waits and counts together: their
// operands are uniform registers, which a branch of one lane would have to fill anew each time (8 x 12288
// x 2048 7.2 us so, 5.2 now; 64 tokens 9.1 and 7.4; 381 x 4096 x 2048 11.2 and 9.5).
// Both tiles of a stage, which are `bytes` together.
__device__ __forceinline__ void tma_pair(void* dst_w, const CUtensorMap* map_w, int ch, void* dst_x, const CUtensorMap* map_x,
                                         int m, int k, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
      " @e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%7], %8;\n"
      " @e cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%6, %2}], [%7];\n"
      " @e cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%3], [%4, {%6, %5}], [%7];\n}\n" ::"r"(
          smem_u32(dst_w)),
      "l"((uint64_t)map_w), "r"(ch), "r"(smem_u32(dst_x)), "l"((uint64_t)map_x), "r"(m), "r"(k), "r"(smem_u32(bar)),
      "r"(bytes)
      : "memory");
}

// The same for one CTA of a pair, whose shares all complete on the first CTA's barrier (`bar`, as a cluster
// address); that CTA expects the bytes of both (0: the second CTA).
__device__ __forceinline__ void tma_pair2(void* dst_w, const CUtensorMap* map_w, int ch, void* dst_x,
                                          const CUtensorMap* map_x, int m, int k, uint32_t bytes, uint64_t* own,
                                          uint32_t bar) {
  asm volatile(
      "{\n .reg .pred e, f;\n elect.sync _|e, 0xffffffff;\n setp.ne.and.u32 f, %8, 0, e;\n"
      " @f mbarrier.arrive.expect_tx.shared::cta.b64 _, [%9], %8;\n"
      " @e cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%6, %2}], [%7];\n"
      " @e cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%3], [%4, {%6, %5}], [%7];\n}\n" ::"r"(
          smem_u32(dst_w)),
      "l"((uint64_t)map_w), "r"(ch), "r"(smem_u32(dst_x)), "l"((uint64_t)map_x), "r"(m), "r"(k), "r"(bar), "r"(bytes),
      "r"(smem_u32(own))
      : "memory");
}

template <bool PAIR>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  if constexpr (PAIR)
    asm volatile(
        "{\n .reg .pred e, p;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
        " @e tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accum));
  else
    asm volatile(
      "{\n .reg .pred e, p;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum));
}

// On `bar` of this CTA, or of both CTAs of the pair.
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile(
        "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
        " @e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}\n" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    asm volatile(
      "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
      : "memory");
}

// A wait of a whole warp, as one answer.
__device__ __forceinline__ bool warp_wait(const LinArgs& a, uint64_t* bar, uint32_t parity, int code) {
  if (__all_sync(0xffffffffu, mbar_wait(bar, parity, nullptr, 0))) return true;
  if ((threadIdx.x & 31) == 0) ops_gave_up(a.err, code);
  return false;
}

#define QASR_R8(r, i) "=r"((r)[i]), "=r"((r)[i + 1]), "=r"((r)[i + 2]), "=r"((r)[i + 3]), "=r"((r)[i + 4]), \
    "=r"((r)[i + 5]), "=r"((r)[i + 6]), "=r"((r)[i + 7])
// C columns of this warp's lane quarter: lane = TMEM lane.
template <int C>
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t* r) {
  if constexpr (C == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : QASR_R8(r, 0) : "r"(addr));
  else if constexpr (C == 16)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : QASR_R8(r, 0), QASR_R8(r, 8)
        : "r"(addr));
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : QASR_R8(r, 0), QASR_R8(r, 8), QASR_R8(r, 16), QASR_R8(r, 24)
        : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;");
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ int ld_cluster(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <bool BF16>
__device__ __forceinline__ void put(void* p, long long i, float v) {
  if constexpr (BF16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
  else ((float*)p)[i] = v;
}

// Residual of tokens m0 .. m0 + C - 1 of this lane's channel, as loaded: it is converted where it
// is used, so that nothing waits for the loads before that.
template <int C, bool BF16>
__device__ __forceinline__ void load_resid(const LinArgs& a, long long m0, int ch, uint32_t* r) {
#pragma unroll
  for (int j = 0; j < C; ++j) {
    r[j] = 0u;
    if (m0 + j < a.m && ch < a.n) {
      const long long i = (m0 + j) * a.ldr + ch;
      if constexpr (BF16) r[j] = ((const uint16_t*)a.resid)[i];
      else r[j] = ((const uint32_t*)a.resid)[i];
    }
  }
}
template <bool BF16>
__device__ __forceinline__ float resid_value(uint32_t r) {
  return __uint_as_float(BF16 ? r << 16 : r);
}

// silu(g) * u by exp(-|g|), which does not overflow: far negative gates keep their small values.
// The denominator is in [1, 2], whose correctly rounded reciprocal takes no slow path (a quotient
// does for tiny exponentials); in all at most 9 * 2^-24 off.
__device__ __forceinline__ float gated(float g, float u) {
  const float t = expf(-fabsf(g));
  const float s = __fmul_rn(g >= 0.f ? 1.0f : t, __frcp_rn(__fadd_rn(1.0f, t)));
  return __fmul_rn(__fmul_rn(s, g), u);
}

// C tokens from m0 of one channel a lane: sums acc, token scales xs, residual r; all 32 lanes call it.
template <int C, int EPI, bool BF16>
__device__ __forceinline__ void finish(const LinArgs& a, const int* acc, const float* xs, const uint32_t* r,
                                       long long m0, int ch, float wsc, int lane) {
  float v[C];
#pragma unroll
  for (int j = 0; j < C; ++j) v[j] = __fmul_rn(__fmul_rn((float)acc[j], xs[j]), wsc);
  if constexpr (EPI == LINEAR_SWIGLU && C > 1) {
    // lanes 2i, 2i + 1 hold gate and up of output column (ch / 2): of two tokens the even lane
    // finishes the first and the odd lane the second
    static_assert(C % 2 == 0, "tokens in pairs");
#pragma unroll
    for (int j = 0; j < C; j += 2) {
      const float got = __shfl_xor_sync(0xffffffffu, lane & 1 ? v[j] : v[j + 1], 1);
      const float g = lane & 1 ? got : v[j], u = lane & 1 ? v[j + 1] : got;
      const long long m = m0 + j + (lane & 1);
      if (m < a.m && ch < a.n) put<BF16>(a.out, m * a.ldo + (ch >> 1), gated(g, u));
    }
  } else if constexpr (EPI == LINEAR_SWIGLU) {
    const float u = __shfl_xor_sync(0xffffffffu, v[0], 1);
    if (m0 < a.m && ch < a.n && !(lane & 1)) put<BF16>(a.out, m0 * a.ldo + (ch >> 1), gated(v[0], u));
  } else {
#pragma unroll
    for (int j = 0; j < C; ++j)
      if (m0 + j < a.m && ch < a.n)
        put<BF16>(a.out, (m0 + j) * a.ldo + ch, EPI == LINEAR_RESID ? __fadd_rn(v[j], resid_value<BF16>(r[j])) : v[j]);
  }
}

// A split tile's tokens [p0, p1) of one half: C at a time, the peers' partial sums added up.
template <int C, int EPI, bool BF16>
__device__ __forceinline__ void join(const LinArgs& a, uint32_t part, const float* xs, long long m0, int p0, int p1,
                                     int ch, float wsc, int lane) {
#pragma unroll 1
  for (int p = p0; p < p1; p += C) {
    if (m0 + p >= a.m) break;
    uint32_t r[C];
    if constexpr (EPI == LINEAR_RESID) load_resid<C, BF16>(a, m0 + p, ch, r);
    int acc[C] = {};
#pragma unroll 4
    for (int k = 0; k < a.split; ++k) {
      const uint32_t peer = map_rank(part + (uint32_t)p * (kCh * 4), k);
#pragma unroll
      for (int j = 0; j < C; ++j) acc[j] += ld_cluster(peer + j * (kCh * 4));
    }
    finish<C, EPI, BF16>(a, acc, xs + p, r, m0 + p, ch, wsc, lane);
  }
}

template <int NT, int EPI, bool BF16, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) linear_kernel(const __grid_constant__ CUtensorMap map_w,
                                                             const __grid_constant__ CUtensorMap map_x,
                                                             const LinArgs a) {
  using S = Shape<NT, PAIR>;
  constexpr int ST = S::kStages;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* xs_s = reinterpret_cast<float*>(smem + ST * S::kStage);  // [epilogue warp][kHalf]
  uint64_t* full = reinterpret_cast<uint64_t*>(xs_s + kEpiWarps * S::kHalf);
  uint64_t* empty = full + ST;
  uint64_t* acc_full = empty + ST;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int cluster = PAIR ? 2 : a.split;
  const int rank = cluster > 1 ? blockIdx.x % cluster : 0;
  const int unit0 = cluster > 1 ? blockIdx.x / cluster : blockIdx.x;
  // (a split tile's CTAs have one unit each)
  const int step = PAIR ? gridDim.x / 2 : a.split > 1 ? a.tiles : gridDim.x;
  const int k0 = PAIR ? 0 : (int)((long long)rank * a.nk / a.split);
  const int k1 = PAIR ? a.nk : (int)((long long)(rank + 1) * a.nk / a.split);
  constexpr int kTileCh = PAIR ? 2 * kCh : kCh;  // channels of a unit, this CTA's the rank-th 128

  if (tid == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], PAIR ? 2 * kEpiWarps : kEpiWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(2 * NT));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(2 * NT));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  if constexpr (PAIR) cluster_barrier();  // both CTAs' barriers are set up
  asm volatile("tcgen05.fence::after_thread_sync;");
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  pdl_launch_dependents();
  pdl_wait();

  if (warp == 0) {
    int it = 0;
    for (int u = unit0; u < a.tiles && !__any_sync(0xffffffffu, *abort_flag); u += step) {
      const int ch0 = u % a.ct * kTileCh + (PAIR ? rank * kCh : 0), m0 = u / a.ct * a.nt + (PAIR ? rank * (a.nt / 2) : 0);
      for (int kt = k0; kt < k1; ++kt, ++it) {
        const int st = it % ST;
        if (it >= ST && !warp_wait(a, &empty[st], (uint32_t)((it / ST) - 1) & 1u, 31)) {
          *abort_flag = 1;
          break;
        }
        unsigned char* sp = smem + st * S::kStage;
        if constexpr (PAIR)
          tma_pair2(sp, &map_w, ch0, sp + kCh * kKb, &map_x, m0, kt * kKb,
                    rank == 0 ? (uint32_t)(2 * kCh * kKb + a.nt * kKb) : 0u, &full[st], map_rank(smem_u32(&full[st]), 0));
        else
          tma_pair(sp, &map_w, ch0, sp + kCh * kKb, &map_x, m0, kt * kKb, kCh * kKb + a.nt * kKb, &full[st]);
      }
    }
  } else if (warp == 1) {
    const uint32_t idesc = idesc_i8(a.nt, kTileCh);
    int it = 0, lt = 0;
    // (a pair's first CTA issues for both)
    for (int u = PAIR && rank > 0 ? a.tiles : unit0; u < a.tiles && !__any_sync(0xffffffffu, *abort_flag); u += step, ++lt) {
      const int ab = lt & 1;
      if (lt >= 2 && !warp_wait(a, &acc_empty[ab], (uint32_t)((lt >> 1) - 1) & 1u, 32)) {
        *abort_flag = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;");
      const uint32_t acc = tmem + (uint32_t)(ab * NT);
      bool ok = true;
      for (int kt = k0; kt < k1; ++kt, ++it) {
        const int st = it % ST;
        if (!warp_wait(a, &full[st], (uint32_t)(it / ST) & 1u, 33)) {
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;");
        const uint32_t sw = smem_u32(smem + st * S::kStage), sx = sw + kCh * kKb;
#pragma unroll
        for (int kk = 0; kk < kKb / 32; ++kk)
          mma_i8<PAIR>(acc, sw128_desc(sw + kk * 32), sw128_desc(sx + kk * 32), idesc, (kt > k0 || kk > 0) ? 1u : 0u);
        commit<PAIR>(&empty[st]);
      }
      if (!ok) {
        *abort_flag = 1;
        break;
      }
      commit<PAIR>(&acc_full[ab]);
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;  // TMEM lane quarter and token half of this warp
    // tokens in registers at a time (16 where their residuals and the next ones' are too)
    constexpr int kMost = EPI == LINEAR_RESID || NT > 64 ? 16 : 32, C = S::kHalf < kMost ? S::kHalf : kMost;
    const int H = a.nt / 2;
    float* xs = xs_s + (warp - 2) * S::kHalf;
    int lt = 0;
    for (int u = unit0; u < a.tiles; u += step, ++lt) {
      const int ab = lt & 1;
      const int ch = u % a.ct * kTileCh + (PAIR ? rank * kCh : 0) + q * 32 + lane;
      const long long m0 = (long long)(u / a.ct) * a.nt + half * H;
      const float wsc = ch < a.n ? a.ws[ch] : 0.f;
      __syncwarp();
      for (int j = lane; j < H; j += 32) xs[j] = m0 + j < a.m ? a.xs[m0 + j] : 0.f;
      __syncwarp();
      uint32_t r[C];
      if constexpr (EPI == LINEAR_RESID)
        if (a.split == 1) load_resid<C, BF16>(a, m0, ch, r);
      if (!warp_wait(a, &acc_full[ab], (uint32_t)(lt >> 1) & 1u, 34)) {
        *abort_flag = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;");
      const uint32_t trow = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(ab * NT + half * H);
#pragma unroll 1
      for (int c = 0; c < H; c += C) {
        if (m0 + c >= a.m) break;
        int acc[C];
        tmem_ld<C>(trow + c, reinterpret_cast<uint32_t*>(acc));
        if (a.split > 1) {
          // every stage has been read by the MMAs that this accumulator waited for
          int* part = reinterpret_cast<int*>(smem);
#pragma unroll
          for (int j = 0; j < C; ++j) part[(half * H + c + j) * kCh + q * 32 + lane] = acc[j];
        } else {
          uint32_t next[C];
          if constexpr (EPI == LINEAR_RESID)
            if (c + C < H) load_resid<C, BF16>(a, m0 + c + C, ch, next);
          finish<C, EPI, BF16>(a, acc, xs + c, r, m0 + c, ch, wsc, lane);
          if constexpr (EPI == LINEAR_RESID) {
#pragma unroll
            for (int j = 0; j < C; ++j) r[j] = next[j];
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;");
      if (lane == 0) {
        if (PAIR && rank > 0) arrive_cluster(map_rank(smem_u32(&acc_empty[ab]), 0));
        else mbar_arrive(&acc_empty[ab]);
      }
    }
  }
  if (a.split > 1) {
    __syncwarp();
    cluster_barrier();  // every partial tile is in its CTA's shared memory
    if (warp >= 2) {
      const int q = warp & 3, half = (warp - 2) >> 2;
      const int ch = unit0 % a.ct * kCh + q * 32 + lane;
      const int H = a.nt / 2;
      const long long m0 = (long long)(unit0 / a.ct) * a.nt + half * H;
      const float wsc = ch < a.n ? a.ws[ch] : 0.f;
      const uint32_t part = smem_u32(smem) + (uint32_t)(half * H * kCh + q * 32 + lane) * 4u;
      const float* xs = xs_s + (warp - 2) * S::kHalf;
      const int each = H / a.split;  // tokens of a rank (H >= 8 = the largest split, and a multiple of it)
      if (each % 8 == 0)
        join<8, EPI, BF16>(a, part, xs, m0, rank * each, (rank + 1) * each, ch, wsc, lane);
      else if (each % 4 == 0)
        join<4, EPI, BF16>(a, part, xs, m0, rank * each, (rank + 1) * each, ch, wsc, lane);
      else if (each % 2 == 0)
        join<2, EPI, BF16>(a, part, xs, m0, rank * each, (rank + 1) * each, ch, wsc, lane);
      else
        join<1, EPI, BF16>(a, part, xs, m0, rank * each, (rank + 1) * each, ch, wsc, lane);
    }
    __syncwarp();
    cluster_barrier();  // no CTA leaves while a peer reads its partial
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  if constexpr (PAIR) {
    cluster_barrier();  // neither CTA leaves while the other's products read its operands or signal its barriers
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * NT));
  } else {
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * NT));
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn get_encode() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)p;
  });
  return fn;
}

bool byte_map(CUtensorMap* m, const void* base, long long rows, int cols, long long ld, int box_rows) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return false;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)kKb, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct LinCall {
  const int8_t *xq, *wq;
  long long ldx, ldw;
  int k;
  LinearEpi epi;
  bool bf16;
};

template <int NT, int EPI, bool BF16, bool PAIR>
cudaError_t launch_as(const LinArgs& a, const CUtensorMap& mw, const CUtensorMap& mx, int grid, cudaStream_t s) {
  static OncePerDevice once;
  constexpr int kSmem = Shape<NT, PAIR>::kSmem;
  const cudaError_t e = once.smem(linear_kernel<NT, EPI, BF16, PAIR>, kSmem);
  if (e != cudaSuccess) return e;
  return ops_launch(linear_kernel<NT, EPI, BF16, PAIR>, dim3(grid), dim3(kThreads), kSmem, s, PAIR ? 2 : a.split, mw, mx, a);
}

template <int NT, bool PAIR = false>
cudaError_t launch(const LinCall& c, const LinArgs& a, int grid, cudaStream_t s) {
  CUtensorMap mw, mx;
  if (!byte_map(&mw, c.wq, a.n, c.k, c.ldw, kCh) || !byte_map(&mx, c.xq, a.m, c.k, c.ldx, PAIR ? a.nt / 2 : a.nt))
    return cudaErrorInvalidValue;
  if (c.epi == LINEAR_SWIGLU)
    return c.bf16 ? launch_as<NT, LINEAR_SWIGLU, true, PAIR>(a, mw, mx, grid, s)
                  : launch_as<NT, LINEAR_SWIGLU, false, PAIR>(a, mw, mx, grid, s);
  if (c.epi == LINEAR_RESID)
    return c.bf16 ? launch_as<NT, LINEAR_RESID, true, PAIR>(a, mw, mx, grid, s)
                  : launch_as<NT, LINEAR_RESID, false, PAIR>(a, mw, mx, grid, s);
  return c.bf16 ? launch_as<NT, LINEAR_STORE, true, PAIR>(a, mw, mx, grid, s)
                : launch_as<NT, LINEAR_STORE, false, PAIR>(a, mw, mx, grid, s);
}

}  // namespace

cudaError_t linear_int8(const int8_t* xq, long long ldx, const float* xs, const int8_t* wq, long long ldw,
                        const float* ws, long long m, int n, int k, LinearEpi epi, const void* residual, long long ldr,
                        void* out, long long ldo, OpsDtype dt, OpsErrors* err, cudaStream_t s) {
  if (m <= 0 || n <= 0) return cudaSuccess;
  if (!err) return cudaErrorInvalidValue;
  LinArgs a{};
  a.err = err;
  a.m = m; a.n = n; a.xs = xs; a.ws = ws; a.resid = residual; a.ldr = ldr; a.ldo = ldo; a.out = out;
  const LinCall c{xq, wq, ldx, ldw, k, epi, dt == OPS_BF16};
  a.ct = ceil_div(n, kCh);
  a.nk = ceil_div(k, kKb);
  const int sms = ops_sm_count();
  // Tile width and K split with the least estimated time in cycles. A step of 128 bytes of K takes 2
  // for each of the 128 + nt rows it brings from L2 (64 bytes a cycle and SM; the products take 2
  // nt), a tile's epilogue about 8 nt beside the next tile's products, and a split's join 2000.
  // Measured against all widths and splits at 16 shapes, the choice is within 8 % of the best
  // (12 % at 32 x 4096 x 2048); e.g. 8191 x 2048 x 6144: 224 tokens 90 us (592 tiles, four full
  // waves), 256 or 128 tokens 94 us, 160 107 us; 381 x 2048 x 6144: 192 tokens in 4 splits 11.9 us,
  // 96 in 2 11.2 us, the worst 32 us; 8 x 2048 x 6144: 8 splits 5.2 us, 4 4.9 us, the worst 9.4 us.
  long long best = -1;
  static const int widths[] = {16, 32, 64, 96, 128, 160, 192, 224, 256};
  for (int nt : widths) {
    const long long tiles = (long long)a.ct * ((m + nt - 1) / nt);
    if (tiles > 0x7FFFFFFF / 16) continue;
    for (int split = 1; split <= kMaxCluster; split *= 2) {
      if (split > 1 && (a.nk < split * 2 || nt / 2 % split || tiles * split > 2 * sms)) break;
      const long long waves = (tiles * split + sms - 1) / sms;
      const long long loop = (long long)((a.nk + split - 1) / split) * 2 * (128 + nt);
      const long long epi = 8 * nt + (split > 1 ? 2000 : 0);
      const long long cost = waves * (loop > epi ? loop : epi) + epi;
      if (best < 0 || cost < best) {
        best = cost;
        a.nt = nt;
        a.split = split;
        a.tiles = (int)tiles;
      }
    }
  }
  if (best < 0) return cudaErrorInvalidValue;
  // A pair of CTAs (cta_group::2) works on 256 channels, each CTA with its 128 and half the tokens: it brings
  // 128 + nt / 2 rows a step, and the products of a step, 2 nt, weigh as much. For a long K and a full grid:
  // 8191 x 2048 x 6144 90 us without and 80 with pairs, 3048 x 2048 x 6144 40 and 34, 8192^3 430 and 385. At
  // K = 2048, where a tile's epilogue weighs as much as its products, the two are alike with a full grid (8191
  // x 4096: 68 and 69 us) and pairs are worse with a small one (381 x 12288: 15.6 and 18.7).
  bool pair = false;
  for (int nt = 160; nt <= 256 && a.nk >= 32 && sms > 1; nt += 32) {
    const long long tiles = (long long)ceil_div(n, 2 * kCh) * ((m + nt - 1) / nt);
    if (tiles > 0x7FFFFFFF / 16 || tiles < sms / 2) continue;
    const long long waves = (tiles + sms / 2 - 1) / (sms / 2);
    const long long step = 2 * std::max(128 + nt / 2, nt), loop = a.nk * step, epi = 8 * nt;
    const long long cost = waves * (loop > epi ? loop : epi) + epi;
    if (cost < best) {
      best = cost;
      pair = true;
      a.nt = nt;
      a.split = 1;
      a.tiles = (int)tiles;
    }
  }
  if (pair) {
    a.ct = ceil_div(n, 2 * kCh);
    return launch<256, true>(c, a, 2 * std::min(a.tiles, sms / 2), s);
  }
  const int grid = a.split > 1 ? a.tiles * a.split : (a.tiles < sms ? a.tiles : sms);
  if (a.nt <= 16) return launch<16>(c, a, grid, s);
  if (a.nt <= 32) return launch<32>(c, a, grid, s);
  if (a.nt <= 64) return launch<64>(c, a, grid, s);
  if (a.nt <= 128) return launch<128>(c, a, grid, s);
  return launch<256>(c, a, grid, s);
}

}  // namespace qasr
