// Attention of many query rows over the int8 KV cache (ops_kv8.cu) on tcgen05: prompts and long chunks.
//
// One CTA owns 128 query rows of one KV head (row = query position x head of the group) and walks
// the keys they see in blocks of 64. Per block
//   S = Q K^T          M = 128, N = 64, K = head_dim                 -> TMEM columns 0 .. 63
//   p = exp2(S f - m)  f = scale * log2(e) * K scale of 16 tokens; running maximum m and sum l
//   O += P V           P = p * V scale / vref, from TMEM; N = head_dim -> TMEM columns 128 ..
// and at the end O * vref / l.
//
// Precision. int8 is exact in f16, so K and V enter the products as they are; their scales stay
// outside, in f32 (vref, a power of two above every V scale the rows see, keeps P in f16's range).
// A query row is scaled by a power of two to [1/2, 1). With PL = 2 (f32 rows) q and P are two f16
// planes, hi + lo, held to 2^-25 of the row's largest; both planes add into the same f32
// accumulator. With PL = 1 (bf16 rows) one plane: 2^-11 of a probability, an eighth of the output's
// own rounding.
// m is only raised when a score exceeds it by 2^8 (p up to 256 is as exact in f16): O is then
// rescaled in TMEM, which the first blocks of a row do and later ones hardly ever.
//
// Roles (256 threads, two CTAs an SM, so that one's softmax runs beside the other's products): warps
// 0-3 softmax, a thread a row; warps 4-6 bring K and V from global memory as int8, one block ahead in
// registers, and write them as f16 rows of a token in the 128-byte-swizzle layout, which is K-major for
// Q K^T and MN-major for P V; one thread of warp 7 issues the products, Q K^T of the next block before
// P V of this one. (Issuing takes as long as the products do, 48 cycles each at N = 64 and 64 at N = 128,
// so a softmax thread that did it kept its warp waiting: 3.1 us a block instead of 1.8.) K has two
// buffers, so that its conversion runs beside the products of the block before.
//
// Bound: f32 rows - the tensor pipe (four products of 128 x 64 x head_dim a block), bf16 rows - exp2
// and the conversions around it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bulk.cuh"
#include "dev_util.cuh"
#include "ops.h"

namespace qasr {
namespace {

constexpr int kRows = 128, kKeys = 64, kThreads = 256, kFill = 96;  // (threads that bring K and V)
constexpr float kNone = -1.0e30f;
constexpr uint32_t kColS = 0, kColP = 64, kColO = 128, kCols = 256;  // TMEM columns

__device__ int g_prompt_err;  // nonzero once a bounded wait gave up

struct PromptArgs {
  Kv8 c;
  const void* q;
  void* out;
  long long q_seq, q_row, o_seq, o_row;
  const int *starts, *counts;
  int idx_stride, rows, group;
  float scale;
  int q_vec, o_vec;  // rows start on 16-byte boundaries
};

template <int HD, int PL>
struct Smem {
  static constexpr int kPlane = kRows * HD * 2, kK = kKeys * HD * 2, kV = kK;
  // Q, two K, V, then 1024 bytes of rows' factors, V scales and barriers: two f32 CTAs fill an SM
  static constexpr int kBytes = PL * kPlane + 2 * kK + kV + 1024;
};

// 128-byte swizzle, 8-row groups 1024 bytes apart; lead: bytes from 64 columns to the next (MN-major)
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr, uint32_t lead = 16) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)(lead >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// f32 accumulator, f16 A (K-major) and B (K-major or MN-major), M = 128
__device__ __forceinline__ constexpr uint32_t idesc_f16(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accum));
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

#define R8(r, i) "=r"((r)[i]), "=r"((r)[i + 1]), "=r"((r)[i + 2]), "=r"((r)[i + 3]), "=r"((r)[i + 4]), \
    "=r"((r)[i + 5]), "=r"((r)[i + 6]), "=r"((r)[i + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : R8(r, 0), R8(r, 8), R8(r, 16), R8(r, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : R8(r, 0), R8(r, 8)
      : "r"(addr));
}
#undef R8
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two f32 in one register pair.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split(f32x2 v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return pack_f16(a - f.x, b - f.y);
}
// One tile of 16 scores: probabilities ex2(x f - m) (0 where seen says so), their sum to l, times w as f16 planes.
template <int PL, bool PARTIAL>
__device__ __forceinline__ void weigh(const float* x, float f, float m, float w, int seen, f32x2& l, uint32_t* hi,
                                      uint32_t* lo) {
  const f32x2 f2 = pair(f, f), m2 = pair(-m, -m), w2 = pair(w, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float2 t = split(fma2(pair(x[2 * i], x[2 * i + 1]), f2, m2));
    t.x = ex2(t.x);
    t.y = ex2(t.y);
    if (PARTIAL) {  // (not by the score: -inf times a zero scale is no number)
      if (2 * i >= seen) t.x = 0.f;
      if (2 * i + 1 >= seen) t.y = 0.f;
    }
    const f32x2 p = pair(t.x, t.y);
    l = add2(l, p);
    const f32x2 v = mul2(p, w2);
    const float2 u = split(v);
    hi[i] = pack_f16(u.x, u.y);
    if (PL == 2) {
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
      const float2 r = split(fma2(pair(h.x, h.y), pair(-1.f, -1.f), v));
      lo[i] = pack_f16(r.x, r.y);
    }
  }
}
// Two bytes of w (int8 + 128) as f16.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t bytes_f16(uint32_t w) {
  const uint32_t p = __byte_perm(w, 0x64646464u, SEL);  // 1024 + byte
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&p), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Bounded wait. Once one gave up nobody waits any more: the warps run through what is left of their
// loops, with the barriers between them, and leave an output that the error code disowns.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* gave_up, int code) {
  if (*gave_up) return false;
  if (mbar_wait(bar, parity, &g_prompt_err, code)) return true;
  *gave_up = 1;
  return false;
}

// N (4 or 2) neighbouring values of a query row, as loaded: converted later, so that no load waits for
// the one before.
template <bool BF16, int N>
struct LaneValues {
  uint32_t w[BF16 ? N / 2 : N];
  __device__ __forceinline__ void load(const PromptArgs& a, long long at) {
    if constexpr (BF16) {
      const uint16_t* p = (const uint16_t*)a.q + at;
      if (a.q_vec) {
        if constexpr (N == 4) {
          const uint2 v = *reinterpret_cast<const uint2*>(p);
          w[0] = v.x; w[1] = v.y;
        } else {
          w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
      } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = (uint32_t)p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
      }
    } else {
      const uint32_t* p = (const uint32_t*)a.q + at;
      if (a.q_vec) {
        if constexpr (N == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(p);
          w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(p);
          w[0] = v.x; w[1] = v.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = p[i];
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (uint32_t& x : w) x = 0u;
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (BF16) return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
    else return __uint_as_float(w[i]);
  }
};

// grid: row tiles x sequences x KV heads. PL: planes of q and P; bf16 rows have one.
template <int HD, int PL>
__global__ void __launch_bounds__(kThreads, 2) prompt_tc_kernel(const PromptArgs a) {
  using L = Smem<HD, PL>;
  constexpr bool BF16 = PL == 1;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *sq = smem, *sk = smem + PL * L::kPlane, *sv = sk + 2 * L::kK;
  float* row_fac = reinterpret_cast<float*>(sv + L::kV);  // each row's factor
  float* red = row_fac + kRows;                           // the largest V scale of each warp's tiles
  uint64_t* k_full = reinterpret_cast<uint64_t*>(red + 8);
  uint64_t *k_free = k_full + 2, *v_full = k_full + 4, *s_full = k_full + 5, *s_free = k_full + 6, *p_full = k_full + 7,
           *o_done = k_full + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(k_full + 9);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (smem_u32(smem) & 1023) {  // the swizzle's rows would not fit (never seen: no static shared memory)
    if (tid == 0) atomicExch(&g_prompt_err, 40);
    return;
  }
  if (tid == 0) {
    mbar_init(&k_full[0], kFill);
    mbar_init(&k_full[1], kFill);
    mbar_init(&k_free[0], 1);  // Q K^T of a block is done: its K may be overwritten
    mbar_init(&k_free[1], 1);
    mbar_init(v_full, kFill);
    mbar_init(s_full, 1);   // and S may be read
    mbar_init(s_free, kRows);
    mbar_init(p_full, kRows);
    mbar_init(o_done, 1);   // P V of a block is done: P and V may be overwritten, O rescaled
    *gave_up = 0;
    fence_mbar_init();
  }
  if (warp == 7) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pdl_launch_dependents();
  pdl_wait();

  // all (sequence, KV head) of a row tile in turn, and the last tiles, which see the most keys, first
  const int heads = a.c.n_kv * a.c.n_seq, row_tile = (int)(gridDim.x / heads) - 1 - (int)(blockIdx.x / heads);
  const int kvh = blockIdx.x % heads % a.c.n_kv, seq = blockIdx.x % heads / a.c.n_kv;
  const int row0 = row_tile * kRows;
  int start = a.starts[(long long)seq * a.idx_stride], count = a.rows;
  if (a.counts) count = min(max(a.counts[(long long)seq * a.idx_stride], 0), a.rows);
  if (start < 0) count = 0;
  start = min(start, a.c.capacity);
  // keys any row of the tile sees, in tiles of 16 (a scale each) and blocks of 64
  const int s_last = min(count - 1, (row0 + kRows - 1) / a.group);
  const int len = s_last >= row0 / a.group ? (int)min((long long)start + s_last + 1, (long long)a.c.capacity) : 0;
  const int tiles = (len + kKv8Block - 1) / kKv8Block, nb = (len + kKeys - 1) / kKeys;
  const long long blocks = a.c.capacity / kKv8Block;
  const float* ks = a.c.ks + seq * a.c.scale_stride + kvh * blocks;
  const float* vs = a.c.vs + seq * a.c.scale_stride + kvh * blocks;

  // ---- Q: every warp brings 16 rows, all of them in flight, a lane HD / 32 neighbouring values
  if (nb > 0) {
    constexpr int N = HD / 32;
    float top = 0.f;
    {
      const int r0 = warp * 16;
      // lane i knows where row i is (a division a row, not one for each of its values)
      const int lr = row0 + r0 + (lane & 15), ls = lr / a.group;
      const long long loff =
          ls < count ? seq * a.q_seq + (long long)ls * a.q_row + (long long)(kvh * a.group + lr - ls * a.group) * HD : -1;
      LaneValues<BF16, N> raw[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const long long off = __shfl_sync(0xffffffffu, loff, i);
        raw[i].zero();
        if (off >= 0) raw[i].load(a, off + lane * N);
      }
      // the largest V scale among the tiles (a NaN one only spoils the rows that see it)
      for (int i = tid; i < tiles; i += kThreads) top = fmaxf(top, __ldg(vs + i));
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = r0 + i;
        float f[N], mx = 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          f[e] = raw[i].get(e);
          mx = fmaxf(mx, fabsf(f[e]));
        }
        mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)));
        // 2^-e and 2^e for the exponent that puts the largest value into [1/2, 1): exact factors, two
        // of them where one would leave f32's normal range
        const int top_e = (int)(__float_as_uint(mx) >> 23);  // (0: zero or subnormal, 255: no number)
        const int e = top_e == 255 ? 0 : max(top_e, 1) - 126;
        const int e1 = e / 2, e2 = e - e1;
        // (a negative scale turns the query round, so that larger scores stay larger)
        const float d1 = copysignf(__int_as_float((127 - e1) << 23), a.scale), d2 = __int_as_float((127 - e2) << 23);
        if (lane == 0)
          row_fac[r] = fabsf(a.scale) * 1.4426950408889634f * __int_as_float((127 + e1) << 23) * __int_as_float((127 + e2) << 23);
        uint32_t hi[N / 2], lo[N / 2];
#pragma unroll
        for (int p = 0; p < N / 2; ++p) {
          const float x = f[2 * p] * d1 * d2, y = f[2 * p + 1] * d1 * d2;
          hi[p] = pack_f16(x, y);
          if (PL == 2) lo[p] = pack_rest(x, y, hi[p]);
        }
        const int col = lane * N;
        unsigned char* at = sq + (col >> 6) * (kRows * 128) + r * 128 + ((((col & 63) >> 3) ^ (r & 7)) << 4) + (col & 7) * 2;
        if constexpr (N == 4) {
          *reinterpret_cast<uint2*>(at) = make_uint2(hi[0], hi[1]);
          if (PL == 2) *reinterpret_cast<uint2*>(at + L::kPlane) = make_uint2(lo[0], lo[1]);
        } else {
          *reinterpret_cast<uint32_t*>(at) = hi[0];
          if (PL == 2) *reinterpret_cast<uint32_t*>(at + L::kPlane) = lo[0];
        }
      }
    }
    fence_async_smem();
    top = warp_max(top);
    if (lane == 0) red[warp] = top;
  }
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem = *tmem_slot;

  if (warp < 4) {
    // ---------------------------------------------------------------- softmax: thread = query row = TMEM lane
    const int rr = row0 + tid, s = rr / a.group;
    const bool live = s < count;
    const int last = live ? min(start + s, a.c.capacity - 1) : -1;
    const float fac = nb > 0 ? row_fac[tid] : 0.f;
    float top = 0.f, vref = 0.f;
    if (nb > 0)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, red[i]);
    if (top > 0.f)  // the power of two above it, 2^-100 at least
      vref = fmaxf(__uint_as_float((__float_as_uint(top) + 0x7FFFFFu) & 0xFF800000u), 7.888609e-31f);
    const float rvref = vref > 0.f ? __fdiv_rn(1.0f, vref) : 0.f;
    const uint32_t trow = tmem + ((uint32_t)(warp * 32) << 16);
    float m = kNone;
    f32x2 l = 0;  // two partial sums
    float kn[4], vn[4];  // the next block's scales
    auto scales = [&](int j) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int tl = j * 4 + b;
        kn[b] = tl < tiles ? __ldg(ks + tl) : 0.f;
        vn[b] = tl < tiles ? __ldg(vs + tl) : 0.f;
      }
    };
    scales(0);
    for (int j = 0; j < nb; ++j) {
      float f[4], w[4];
      const int pos0 = j * kKeys;
      const bool partial = __any_sync(0xffffffffu, pos0 + kKeys - 1 > last);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        f[b] = fac * kn[b];
        w[b] = vn[b] * rvref;
        // a row that sees nothing of a tile takes nothing of its scale either
        if (partial && pos0 + b * kKv8Block > last) w[b] = 0.f;
      }
      if (j + 1 < nb) scales(j + 1);
      wait(s_full, (uint32_t)j & 1u, gave_up, 43);
      __syncwarp();
      after_sync();
      float x[kKeys];
      tmem_ld32(trow + kColS, reinterpret_cast<uint32_t*>(x));
      tmem_ld32(trow + kColS + 32, reinterpret_cast<uint32_t*>(x + 32));
      tmem_ld_wait();
      before_sync();
      mbar_arrive(s_free);
      if (partial) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
          if (pos0 + i > last) x[i] = -__int_as_float(0x7F800000);
      }
      float mx = kNone;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        float t = x[16 * b];
#pragma unroll
        for (int i = 1; i < 16; ++i) t = fmaxf(t, x[16 * b + i]);
        mx = fmaxf(mx, t * f[b]);  // (a masked tile's -inf, or no number: ignored)
      }
      const bool grow = mx > m + 8.f;
      const float corr = grow ? ex2(m - mx) : 1.f;
      if (grow) m = mx;
      if (j > 0) {
        wait(o_done, (uint32_t)(j - 1) & 1u, gave_up, 44);
        __syncwarp();
        after_sync();
        if (__any_sync(0xffffffffu, grow)) {
          l = mul2(l, pair(corr, corr));
#pragma unroll 1
          for (int c = 0; c < HD; c += 16) {
            uint32_t o[16];
            tmem_ld16(trow + kColO + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
            tmem_st16(trow + kColO + c, o);
          }
          tmem_st_wait();
        }
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t hi[8], lo[8];
        if (partial)
          weigh<PL, true>(x + 16 * b, f[b], m, w[b], last + 1 - pos0 - 16 * b, l, hi, lo);
        else
          weigh<PL, false>(x + 16 * b, f[b], m, w[b], 16, l, hi, lo);
        tmem_st8(trow + kColP + 8 * b, hi);
        if (PL == 2) tmem_st8(trow + kColP + 32 + 8 * b, lo);
      }
      tmem_st_wait();
      before_sync();
      mbar_arrive(p_full);
    }
    // ---- O * vref / l
    if (nb > 0) wait(o_done, (uint32_t)(nb - 1) & 1u, gave_up, 45);
    __syncwarp();
    after_sync();
    const float2 sums = split(l);
    const float total = sums.x + sums.y;
    const float inv = total == 0.f ? 0.f : __fdiv_rn(vref, total);
    // through shared memory (operands are idle now, 32 rows a warp), so that a row's stores are contiguous
    constexpr int kPitch = HD + 4;  // floats; eight rows' 16-byte pieces hit distinct banks
    static_assert(kRows * kPitch * 4 <= PL * L::kPlane + 2 * L::kK + L::kV, "the output reuses the operands");
    float* stage = reinterpret_cast<float*>(smem);
#pragma unroll 1
    for (int c = 0; c < HD; c += 32) {
      float o[32];
      if (nb > 0) {
        tmem_ld32(trow + kColO + c, reinterpret_cast<uint32_t*>(o));
        tmem_ld_wait();
      }
#pragma unroll
      for (int i = 0; i < 32; i += 4)
        *reinterpret_cast<float4*>(stage + tid * kPitch + c + i) =
            nb > 0 ? make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncwarp();
    constexpr int kLanes = HD / 4, kPer = 32 / kLanes;  // lanes of a row, rows at a time
    // (this lane's own row: s, rr)
    const long long mine = rr < a.rows * a.group
                               ? seq * a.o_seq + (long long)s * a.o_row + (long long)(kvh * a.group + rr - s * a.group) * HD
                               : -1;
    const int col = lane % kLanes * 4;
#pragma unroll 1
    for (int i0 = 0; i0 < 32; i0 += 8 * kPer) {
      float4 o[8];  // (all read before the first store, which might alias them for all the compiler knows)
      long long off[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i0 + i * kPer + lane / kLanes;
        o[i] = *reinterpret_cast<const float4*>(stage + (warp * 32 + r) * kPitch + col);
        off[i] = __shfl_sync(0xffffffffu, mine, r);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (off[i] < 0) continue;
        const long long at = off[i] + col;
        if constexpr (BF16) {
          __nv_bfloat16* p = (__nv_bfloat16*)a.out + at;
          __nv_bfloat162 v[2] = {__floats2bfloat162_rn(o[i].x, o[i].y), __floats2bfloat162_rn(o[i].z, o[i].w)};
          if (a.o_vec) {
            *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(v);
          } else {
            p[0] = v[0].x; p[1] = v[0].y; p[2] = v[1].x; p[3] = v[1].y;
          }
        } else {
          float* p = (float*)a.out + at;
          if (a.o_vec) {
            *reinterpret_cast<float4*>(p) = o[i];
          } else {
            p[0] = o[i].x; p[1] = o[i].y; p[2] = o[i].z; p[3] = o[i].w;
          }
        }
      }
    }
  } else if (warp < 7) {
    // ---------------------------------------------------------------- K and V: int8 -> f16 operands
    const int ct = tid - 128;
    const int8_t* k = a.c.k + seq * a.c.seq_stride + (long long)kvh * a.c.capacity * HD;
    const int8_t* v = a.c.v + seq * a.c.seq_stride + (long long)kvh * a.c.capacity * HD;
    const int end = tiles * kKv8Block;  // tokens past it are zeros
    constexpr int kPieces = kKeys * HD / 16, kN = (kPieces + kFill - 1) / kFill;  // 16 bytes of K or V, a thread's
    uint4 kr[kN], vr[kN];
    auto load = [&](const int8_t* src, int j, uint4* r) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int id = ct + i * kFill, tok = j * kKeys + id / (HD / 16);
        r[i] = make_uint4(0, 0, 0, 0);
        if (id < kPieces && tok < end)
          r[i] = __ldg(reinterpret_cast<const uint4*>(src + (long long)tok * HD + id % (HD / 16) * 16));
      }
    };
    auto store = [&](unsigned char* dst, const uint4* r) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int id = ct + i * kFill, row = id / (HD / 16), c = id % (HD / 16) * 2;  // 16-byte f16 chunks c, c + 1
        if (id >= kPieces) break;
        // lanes of the second 64 columns begin with their second chunk, so that eight lanes hit distinct banks
        const bool swap = c & 8;
        const uint32_t w[4] = {(swap ? r[i].z : r[i].x) ^ 0x80808080u, (swap ? r[i].w : r[i].y) ^ 0x80808080u,
                               (swap ? r[i].x : r[i].z) ^ 0x80808080u, (swap ? r[i].y : r[i].w) ^ 0x80808080u};
        unsigned char* p = dst + (c >> 3) * (kKeys * 128) + row * 128;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<uint4*>(p + ((((c & 7) + (h ^ (int)swap)) ^ (row & 7)) << 4)) =
              make_uint4(bytes_f16<0x4140>(w[2 * h]), bytes_f16<0x4342>(w[2 * h]), bytes_f16<0x4140>(w[2 * h + 1]),
                         bytes_f16<0x4342>(w[2 * h + 1]));
      }
      fence_async_smem();
    };
    load(k, 0, kr);
    load(v, 0, vr);
    auto put_k = [&](int j) {  // into its buffer, then the next block's loads
      store(sk + (j & 1) * L::kK, kr);
      mbar_arrive(&k_full[j & 1]);
      if (j + 1 < nb) load(k, j + 1, kr);
    };
    if (nb > 0) put_k(0);
    for (int j = 0; j < nb; ++j) {
      // K of block j + 1 goes where that of j - 1 was
      if (j + 1 < nb) {
        // (a barrier of its own: that of S may be two phases on by now)
        if (j > 0 && !wait(&k_free[(j - 1) & 1], (uint32_t)((j - 1) >> 1) & 1u, gave_up, 46)) break;
        put_k(j + 1);
      }
      if (j > 0 && !wait(o_done, (uint32_t)(j - 1) & 1u, gave_up, 47)) break;
      store(sv, vr);
      mbar_arrive(v_full);
      if (j + 1 < nb) load(v, j + 1, vr);
    }
  } else if (lane == 0 && nb > 0) {
    // ---------------------------------------------------------------- products
    const uint32_t qa = smem_u32(sq), ka = smem_u32(sk), va = smem_u32(sv);
    auto qk = [&](int j) {
      if (!wait(&k_full[j & 1], (uint32_t)(j >> 1) & 1u, gave_up, 41)) return;
      after_sync();
      const uint32_t kb = ka + (uint32_t)(j & 1) * L::kK;
#pragma unroll
      for (int pl = 0; pl < PL; ++pl)
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_ss(tmem + kColS, sw128_desc(qa + pl * L::kPlane + (kk >> 2) * (kRows * 128) + (kk & 3) * 32),
                 sw128_desc(kb + (kk >> 2) * (kKeys * 128) + (kk & 3) * 32), idesc_f16(kKeys, false),
                 (pl > 0 || kk > 0) ? 1u : 0u);
      commit(s_full);
      commit(&k_free[j & 1]);
    };
    qk(0);
    for (int j = 0; j < nb && !*gave_up; ++j) {
      if (j + 1 < nb) {
        if (!wait(s_free, (uint32_t)j & 1u, gave_up, 48)) break;
        qk(j + 1);
      }
      if (!wait(v_full, (uint32_t)j & 1u, gave_up, 42) || !wait(p_full, (uint32_t)j & 1u, gave_up, 49)) break;
      after_sync();
#pragma unroll
      for (int pl = 0; pl < PL; ++pl)
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          mma_ts(tmem + kColO, tmem + kColP + pl * 32 + kk * 8, sw128_desc(va + kk * 2048, kKeys * 128),
                 idesc_f16(HD, true), (j > 0 || pl > 0 || kk > 0) ? 1u : 0u);
      commit(o_done);
    }
  }
  __syncwarp();
  before_sync();
  __syncthreads();
  if (warp == 7) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
}

template <int HD, int PL>
cudaError_t launch(const PromptArgs& a, cudaStream_t s) {
  static OncePerDevice once;
  const cudaError_t e = once.smem(prompt_tc_kernel<HD, PL>, Smem<HD, PL>::kBytes);
  if (e != cudaSuccess) return e;
  const long long ctas = ((long long)a.rows * a.group + kRows - 1) / kRows * a.c.n_kv * a.c.n_seq;
  if (ctas > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
  const dim3 g((unsigned)ctas);
  return ops_launch(prompt_tc_kernel<HD, PL>, g, dim3(kThreads), Smem<HD, PL>::kBytes, s, 1, a);
}

}  // namespace

cudaError_t kv8_prompt_attention(const Kv8& c, const void* q, long long q_seq, long long q_row, void* out,
                                 long long o_seq, long long o_row, OpsDtype dt, int rows, int heads, const int* starts,
                                 const int* counts, int idx_stride, float scale, cudaStream_t s) {
  auto vec = [&](const void* p, long long seq, long long row) {
    const int es = dt == OPS_BF16 ? 2 : 4;
    return (uintptr_t)p % 16 == 0 && seq * es % 16 == 0 && row * es % 16 == 0;
  };
  const PromptArgs a{c, q, out, q_seq, q_row, o_seq, o_row, starts, counts, idx_stride, rows, heads / c.n_kv, scale,
                     vec(q, q_seq, q_row), vec(out, o_seq, o_row)};
  if (c.head_dim == 128) return dt == OPS_BF16 ? launch<128, 1>(a, s) : launch<128, 2>(a, s);
  return dt == OPS_BF16 ? launch<64, 1>(a, s) : launch<64, 2>(a, s);
}

int kv8_prompt_error() {
  int e = 0;
  if (cudaMemcpyFromSymbol(&e, g_prompt_err, sizeof(int)) != cudaSuccess) return 0;
  if (e) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_prompt_err, &zero, sizeof(int));
  }
  return e;
}

}  // namespace qasr
