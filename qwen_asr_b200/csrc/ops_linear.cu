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
// 2-5 drain the accumulator. Many tiles: a persistent grid with two accumulators, so that one
// tile's epilogue runs behind the next one's products. Few tiles (fewer than the SMs): a cluster
// of 2 to 8 CTAs splits K, each leaves its int32 partial tile in its own shared memory, and after
// one cluster barrier every CTA adds up its share of the tokens over distributed shared memory.
// No workspace, no atomics.
//
// Bound: weight bytes from DRAM up to some 100 tokens, the tensor cores beyond.
#include <cuda.h>

#include <mutex>

#include "bulk.cuh"
#include "common.h"
#include "dev_util.cuh"
#include "ops.h"

namespace qasr {
namespace {

constexpr int kCh = 128;    // channels of a tile
constexpr int kKb = 128;    // K bytes of a stage
constexpr int kEpiWarps = 4;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kMaxCluster = 8;

__device__ int g_wait_err;  // nonzero once a bounded wait gave up

template <int NT>
struct Shape {
  static constexpr int kStage = kCh * kKb + NT * kKb;
  static constexpr int kStages = NT >= 256 ? 4 : NT >= 128 ? 6 : NT >= 64 ? 4 : NT >= 32 ? 5 : 6;
  static constexpr int kSmem = 1024 + kStages * kStage + 256;
  // int32 accumulator, signed 8-bit A and B, both K-major
  static constexpr uint32_t kIdesc =
      (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(kCh >> 4) << 24);
  static_assert(kStages * kStage >= NT * kCh * 4, "the partial tile reuses the ring");
};

struct LinArgs {
  long long m;
  int n, nk, ct, tiles, split;
  int epi, bf16;
  const float *xs, *ws;
  const void* resid;
  long long ldr, ldo;
  void* out;
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

__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"((uint64_t)map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum));
}

__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ int ld_cluster(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float get(const LinArgs& a, const void* p, long long i) {
  return a.bf16 ? __bfloat162float(((const __nv_bfloat16*)p)[i]) : ((const float*)p)[i];
}
__device__ __forceinline__ void put(const LinArgs& a, long long i, float v) {
  if (a.bf16)
    ((__nv_bfloat16*)a.out)[i] = __float2bfloat16_rn(v);
  else
    ((float*)a.out)[i] = v;
}

// silu(g) * u by exp(-|g|), which does not overflow: far negative gates keep their small values.
__device__ __forceinline__ float gated(float g, float u) {
  const float t = expf(-fabsf(g));
  const float s = __fdiv_rn(g >= 0.f ? 1.0f : t, __fadd_rn(1.0f, t));
  return __fmul_rn(__fmul_rn(s, g), u);
}

// C tokens m0 .. of one channel a lane (sums acc): scales, epilogue, stores. All 32 lanes call it.
template <int C>
__device__ __forceinline__ void finish(const LinArgs& a, const int* acc, long long m0, int ch, float wsc, int lane) {
  float v[C];
#pragma unroll
  for (int j = 0; j < C; ++j)
    v[j] = __fmul_rn(__fmul_rn((float)acc[j], m0 + j < a.m ? __ldg(a.xs + m0 + j) : 0.f), wsc);
  if (a.epi == LINEAR_SWIGLU) {
    // lanes 2i, 2i + 1 hold gate and up of output column (ch / 2): of two tokens the even lane
    // finishes the first and the odd lane the second
#pragma unroll
    for (int j = 0; j < C; j += 2) {
      const float got = __shfl_xor_sync(0xffffffffu, lane & 1 ? v[j] : v[j + 1], 1);
      const float g = lane & 1 ? got : v[j], u = lane & 1 ? v[j + 1] : got;
      const long long m = m0 + j + (lane & 1);
      if (m < a.m && ch < a.n) put(a, m * a.ldo + (ch >> 1), gated(g, u));
    }
    return;
  }
  if (a.epi == LINEAR_RESID) {
    float r[C];
#pragma unroll
    for (int j = 0; j < C; ++j) r[j] = m0 + j < a.m && ch < a.n ? get(a, a.resid, (m0 + j) * a.ldr + ch) : 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] = __fadd_rn(v[j], r[j]);
  }
#pragma unroll
  for (int j = 0; j < C; ++j)
    if (m0 + j < a.m && ch < a.n) put(a, (m0 + j) * a.ldo + ch, v[j]);
}

template <int NT>
__global__ void __launch_bounds__(kThreads, 1) linear_kernel(const __grid_constant__ CUtensorMap map_w,
                                                             const __grid_constant__ CUtensorMap map_x,
                                                             const LinArgs a) {
  using S = Shape<NT>;
  constexpr int ST = S::kStages;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + ST * S::kStage);
  uint64_t* empty = full + ST;
  uint64_t* acc_full = empty + ST;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = a.split > 1 ? blockIdx.x % a.split : 0;
  const int unit0 = a.split > 1 ? blockIdx.x / a.split : blockIdx.x;
  const int step = a.split > 1 ? a.tiles : gridDim.x;  // a split tile's CTAs have one unit each
  const int k0 = (int)((long long)rank * a.nk / a.split), k1 = (int)((long long)(rank + 1) * a.nk / a.split);

  if (tid == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kEpiWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(2 * NT));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;");
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (int u = unit0; u < a.tiles && !*abort_flag; u += step) {
        const int ch0 = u % a.ct * kCh, m0 = u / a.ct * NT;
        for (int kt = k0; kt < k1; ++kt, ++it) {
          const int st = it % ST;
          if (it >= ST && !mbar_wait(&empty[st], (uint32_t)((it / ST) - 1) & 1u, &g_wait_err, 31)) {
            *abort_flag = 1;
            break;
          }
          unsigned char* sp = smem + st * S::kStage;
          mbar_expect_tx(&full[st], S::kStage);
          tma_2d(sp, &map_w, kt * kKb, ch0, &full[st]);
          tma_2d(sp + kCh * kKb, &map_x, kt * kKb, m0, &full[st]);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int it = 0, lt = 0;
      for (int u = unit0; u < a.tiles && !*abort_flag; u += step, ++lt) {
        const int ab = lt & 1;
        if (lt >= 2 && !mbar_wait(&acc_empty[ab], (uint32_t)((lt >> 1) - 1) & 1u, &g_wait_err, 32)) {
          *abort_flag = 1;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;");
        const uint32_t acc = tmem + (uint32_t)(ab * NT);
        bool ok = true;
        for (int kt = k0; kt < k1; ++kt, ++it) {
          const int st = it % ST;
          if (!mbar_wait(&full[st], (uint32_t)(it / ST) & 1u, &g_wait_err, 33)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;");
          const uint32_t sw = smem_u32(smem + st * S::kStage), sx = sw + kCh * kKb;
#pragma unroll
          for (int kk = 0; kk < kKb / 32; ++kk)
            mma_i8(acc, sw128_desc(sw + kk * 32), sw128_desc(sx + kk * 32), S::kIdesc, (kt > k0 || kk > 0) ? 1u : 0u);
          commit(&empty[st]);
        }
        if (!ok) {
          *abort_flag = 1;
          break;
        }
        commit(&acc_full[ab]);
      }
    }
  } else {
    const int q = warp & 3;  // TMEM lane quarter of this warp
    int lt = 0;
    for (int u = unit0; u < a.tiles; u += step, ++lt) {
      const int ab = lt & 1;
      const bool ok = mbar_wait(&acc_full[ab], (uint32_t)(lt >> 1) & 1u, &g_wait_err, 34);
      if (!ok) {
        *abort_flag = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;");
      const int ch = u % a.ct * kCh + q * 32 + lane;
      const long long m0 = (long long)(u / a.ct) * NT;
      const float wsc = ch < a.n ? __ldg(a.ws + ch) : 0.f;
      const uint32_t trow = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(ab * NT);
#pragma unroll 1
      for (int c = 0; c < NT; c += 16) {
        if (m0 + c >= a.m) break;
        uint32_t r[16];
        tmem_ld16(trow + c, r);
        asm volatile("tcgen05.wait::ld.sync.aligned;");
        if (a.split > 1) {
          // every stage has been read by the MMAs that this accumulator waited for
          int* part = reinterpret_cast<int*>(smem);
#pragma unroll
          for (int j = 0; j < 16; ++j) part[(c + j) * kCh + q * 32 + lane] = (int)r[j];
        } else {
          finish<16>(a, reinterpret_cast<const int*>(r), m0 + c, ch, wsc, lane);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;");
      if (lane == 0) mbar_arrive(&acc_empty[ab]);
    }
  }
  if (a.split > 1) {
    __syncwarp();
    cluster_barrier();  // every partial tile is in its CTA's shared memory
    if (warp >= 2) {
      const int q = warp & 3;
      const int ch = unit0 % a.ct * kCh + q * 32 + lane;
      const long long m0 = (long long)(unit0 / a.ct) * NT;
      const float wsc = ch < a.n ? __ldg(a.ws + ch) : 0.f;
      const uint32_t base = smem_u32(smem) + (uint32_t)(q * 32 + lane) * 4u;
      const int live = (int)min((long long)NT, a.m - m0);
      // token pairs in turn: pair p belongs to rank p % split
#pragma unroll 1
      for (int p = rank * 2; p < live; p += a.split * 2) {
        int acc[2] = {0, 0};
        for (int r = 0; r < a.split; ++r) {
          const uint32_t peer = map_rank(base + (uint32_t)p * (kCh * 4), r);
          acc[0] += ld_cluster(peer);
          acc[1] += ld_cluster(peer + kCh * 4);
        }
        finish<2>(a, acc, m0 + p, ch, wsc, lane);
      }
    }
    __syncwarp();
    cluster_barrier();  // no CTA leaves while a peer reads its partial
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * NT));
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

template <int NT>
cudaError_t launch(const int8_t* xq, long long ldx, const int8_t* wq, long long ldw, int k, LinArgs a, cudaStream_t s) {
  CUtensorMap mw, mx;
  if (!byte_map(&mw, wq, a.n, k, ldw, kCh) || !byte_map(&mx, xq, a.m, k, ldx, NT)) return cudaErrorInvalidValue;
  static OncePerDevice once;
  const cudaError_t e = once.smem(linear_kernel<NT>, Shape<NT>::kSmem);
  if (e != cudaSuccess) return e;
  a.ct = ceil_div(a.n, kCh);
  a.nk = ceil_div(k, kKb);
  const long long tiles = (long long)a.ct * ((a.m + NT - 1) / NT);
  if (tiles > 0x7FFFFFFF) return cudaErrorInvalidValue;
  a.tiles = (int)tiles;
  const int sms = ops_sm_count();
  a.split = 1;
  // few tiles: split K while the CTAs still fit one wave and each keeps two stages of K
  while (a.split < kMaxCluster && a.tiles * a.split * 2 <= sms && a.nk >= a.split * 4) a.split *= 2;
  const int grid = a.split > 1 ? a.tiles * a.split : (a.tiles < sms ? a.tiles : sms);
  return ops_launch(linear_kernel<NT>, dim3(grid), dim3(kThreads), Shape<NT>::kSmem, s, a.split, mw, mx, a);
}

}  // namespace

cudaError_t linear_int8(const int8_t* xq, long long ldx, const float* xs, const int8_t* wq, long long ldw,
                        const float* ws, long long m, int n, int k, LinearEpi epi, const void* residual, long long ldr,
                        void* out, long long ldo, OpsDtype dt, cudaStream_t s) {
  if (m <= 0 || n <= 0) return cudaSuccess;
  LinArgs a{};
  a.m = m; a.n = n; a.epi = epi; a.bf16 = dt == OPS_BF16; a.xs = xs; a.ws = ws;
  a.resid = residual; a.ldr = ldr; a.ldo = ldo; a.out = out;
  if (m <= 16) return launch<16>(xq, ldx, wq, ldw, k, a, s);
  if (m <= 32) return launch<32>(xq, ldx, wq, ldw, k, a, s);
  if (m <= 64) return launch<64>(xq, ldx, wq, ldw, k, a, s);
  const long long ct = ceil_div(n, kCh);
  if (ct * ((m + 255) / 256) < ops_sm_count()) return launch<128>(xq, ldx, wq, ldw, k, a, s);
  return launch<256>(xq, ldx, wq, ldw, k, a, s);
}

int linear_int8_error() {
  int e = 0;
  if (cudaMemcpyFromSymbol(&e, g_wait_err, sizeof(int)) != cudaSuccess) return 0;
  if (e) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_wait_err, &zero, sizeof(int));
  }
  return e;
}

}  // namespace qasr
