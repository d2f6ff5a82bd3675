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
// Roles (288 threads, two CTAs an SM, so that one's softmax runs beside the other's products):
// warps 0-3 softmax, a thread a row; warps 4-7 bring K and V from global memory as int8, one block
// ahead in registers, and write them as f16 rows of a token in the 128-byte-swizzle layout, which is
// K-major for Q K^T and MN-major for P V; one thread of warp 8 issues the products: Q K^T of the next block before P V of this one.
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

constexpr int kRows = 128, kKeys = 64, kThreads = 288;
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
  static constexpr int kBytes = 1024 + PL * kPlane + kK + kV + 256;
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

// Bounded wait of a whole warp, which leaves it converged (and of one mind).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, &g_prompt_err, code));
}

// 8 values of a query row.
template <bool BF16>
__device__ __forceinline__ void load8(const PromptArgs& a, long long at, float* f) {
  if constexpr (BF16) {
    const __nv_bfloat16* p = (const __nv_bfloat16*)a.q + at;
    if (a.q_vec) {
      bf16x8_to_f32(*reinterpret_cast<const uint4*>(p), f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = __bfloat162float(p[i]);
    }
  } else {
    const float* p = (const float*)a.q + at;
    if (a.q_vec) {
      const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 4);
      f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w;
      f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = p[i];
    }
  }
}

// grid (row tiles, n_kv, n_seq). PL: planes of q and P; bf16 rows have one.
template <int HD, int PL>
__global__ void __launch_bounds__(kThreads, 2) prompt_tc_kernel(const PromptArgs a) {
  using L = Smem<HD, PL>;
  constexpr bool BF16 = PL == 1;
  extern __shared__ unsigned char smem_raw[];
  __shared__ float red[4];
  unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char *sq = smem, *sk = smem + PL * L::kPlane, *sv = sk + L::kK;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sv + L::kV);
  uint64_t *k_full = q_full + 1, *v_full = q_full + 2, *s_full = q_full + 3, *s_free = q_full + 4, *p_full = q_full + 5,
           *o_done = q_full + 6;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 7);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(q_full, kRows);
    mbar_init(k_full, 128);
    mbar_init(v_full, 128);
    mbar_init(s_full, 1);   // Q K^T of a block is done: S may be read, K overwritten
    mbar_init(s_free, kRows);
    mbar_init(p_full, kRows);
    mbar_init(o_done, 1);   // P V of a block is done: P and V may be overwritten, O rescaled
    fence_mbar_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();

  const int kvh = blockIdx.y, seq = blockIdx.z;
  // the last rows see the most keys: they start first
  const int row0 = (gridDim.x - 1 - blockIdx.x) * kRows;
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

  if (warp < 4) {
    // ---------------------------------------------------------------- softmax: thread = query row = TMEM lane
    const int rr = row0 + tid, s = rr / a.group;
    const bool live = s < count;
    const int last = live ? min(start + s, a.c.capacity - 1) : -1;
    const long long qoff = seq * a.q_seq + (long long)s * a.q_row + (long long)(kvh * a.group + rr % a.group) * HD;
    float fac = 0.f, vref = 0.f;
    {
      float mx = 0.f;
      if (live)
        for (int c = 0; c < HD; c += 8) {
          float f[8];
          load8<BF16>(a, qoff + c, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(f[i]));
        }
      int e = 0;
      if (mx > 0.f && mx < __int_as_float(0x7F800000)) frexpf(mx, &e);
      fac = scalbnf(fabsf(a.scale) * 1.4426950408889634f, e);
      // (a negative scale turns the query round, so that larger scores stay larger)
      const float sign = a.scale < 0.f ? -1.f : 1.f;
      for (int c = 0; c < HD; c += 8) {
        float f[8] = {};
        if (live) load8<BF16>(a, qoff + c, f);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = scalbnf(f[2 * i], -e) * sign, y = scalbnf(f[2 * i + 1], -e) * sign;
          hi[i] = pack_f16(x, y);
          if (PL == 2) lo[i] = pack_rest(x, y, hi[i]);
        }
        const uint32_t at = (uint32_t)((c >> 6) * (kRows * 128) + tid * 128 + ((((c & 63) >> 3) ^ (tid & 7)) << 4));
        *reinterpret_cast<uint4*>(sq + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (PL == 2) *reinterpret_cast<uint4*>(sq + L::kPlane + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      fence_async_smem();
      mbar_arrive(q_full);
      // the largest V scale among the tiles (a NaN one only spoils the rows that see it)
      float top = 0.f;
      for (int i = tid; i < tiles; i += kRows) top = fmaxf(top, __ldg(vs + i));
      top = warp_max(top);
      if (lane == 0) red[warp] = top;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
      if (top > 0.f)  // the power of two above it, 2^-100 at least
        vref = fmaxf(__uint_as_float((__float_as_uint(top) + 0x7FFFFFu) & 0xFF800000u), 7.888609e-31f);
    }
    const float rvref = vref > 0.f ? __fdiv_rn(1.0f, vref) : 0.f;
    const uint32_t trow = tmem + ((uint32_t)(warp * 32) << 16);
    float m = kNone;
    f32x2 l = 0;  // two partial sums
    bool ok = true;
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
      if (!warp_wait(s_full, (uint32_t)j & 1u, 41)) {
        ok = false;
        break;
      }
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
        if (!warp_wait(o_done, (uint32_t)(j - 1) & 1u, 42)) {
          ok = false;
          break;
        }
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
    if (ok && nb > 0) ok = warp_wait(o_done, (uint32_t)(nb - 1) & 1u, 43);
    after_sync();
    const float2 sums = split(l);
    const float total = sums.x + sums.y;
    const float inv = total == 0.f ? 0.f : __fdiv_rn(vref, total);
    const long long ooff = seq * a.o_seq + (long long)s * a.o_row + (long long)(kvh * a.group + rr % a.group) * HD;
#pragma unroll 1
    for (int c = 0; c < HD; c += 16) {
      float o[16];
      if (nb > 0) {
        tmem_ld16(trow + kColO + c, reinterpret_cast<uint32_t*>(o));
        tmem_ld_wait();
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = nb > 0 ? o[i] * inv : 0.f;
      if (rr >= a.rows * a.group) {
        // a row behind the last: nothing to write
      } else if constexpr (BF16) {
        __nv_bfloat16* p = (__nv_bfloat16*)a.out + ooff + c;
        __nv_bfloat162 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
        if (a.o_vec) {
          reinterpret_cast<uint4*>(p)[0] = reinterpret_cast<uint4*>(v)[0];
          reinterpret_cast<uint4*>(p)[1] = reinterpret_cast<uint4*>(v)[1];
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = i & 1 ? v[i >> 1].y : v[i >> 1].x;
        }
      } else {
        float* p = (float*)a.out + ooff + c;
        if (a.o_vec) {
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<float4*>(p + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = o[i];
        }
      }
      __syncwarp();
    }
  } else if (warp < 8) {
    // ---------------------------------------------------------------- K and V: int8 -> f16 operands
    const int ct = tid - 128;
    const int8_t* k = a.c.k + seq * a.c.seq_stride + (long long)kvh * a.c.capacity * HD;
    const int8_t* v = a.c.v + seq * a.c.seq_stride + (long long)kvh * a.c.capacity * HD;
    const int end = tiles * kKv8Block;  // tokens past it are zeros
    constexpr int kN = kKeys * HD / 16 / 128;  // 16-byte pieces of a block's K or V a thread
    uint4 kr[kN], vr[kN];
    auto load = [&](const int8_t* src, int j, uint4* r) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int id = ct + i * 128, tok = j * kKeys + id / (HD / 16);
        r[i] = make_uint4(0, 0, 0, 0);
        if (tok < end) r[i] = __ldg(reinterpret_cast<const uint4*>(src + (long long)tok * HD + id % (HD / 16) * 16));
      }
    };
    auto store = [&](unsigned char* dst, const uint4* r) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int id = ct + i * 128, row = id / (HD / 16), c = id % (HD / 16) * 2;  // 16-byte f16 chunks c, c + 1
        const uint32_t w[4] = {r[i].x ^ 0x80808080u, r[i].y ^ 0x80808080u, r[i].z ^ 0x80808080u, r[i].w ^ 0x80808080u};
        unsigned char* p = dst + (c >> 3) * (kKeys * 128) + row * 128;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<uint4*>(p + ((((c & 7) + h) ^ (row & 7)) << 4)) =
              make_uint4(bytes_f16<0x4140>(w[2 * h]), bytes_f16<0x4342>(w[2 * h]), bytes_f16<0x4140>(w[2 * h + 1]),
                         bytes_f16<0x4342>(w[2 * h + 1]));
      }
      fence_async_smem();
    };
    load(k, 0, kr);
    load(v, 0, vr);
    for (int j = 0; j < nb; ++j) {
      if (j > 0 && !mbar_wait(s_full, (uint32_t)(j - 1) & 1u, &g_prompt_err, 44)) break;
      store(sk, kr);
      mbar_arrive(k_full);
      if (j + 1 < nb) load(k, j + 1, kr);
      if (j > 0 && !mbar_wait(o_done, (uint32_t)(j - 1) & 1u, &g_prompt_err, 45)) break;
      store(sv, vr);
      mbar_arrive(v_full);
      if (j + 1 < nb) load(v, j + 1, vr);
    }
  } else if (lane == 0 && nb > 0) {
    // ---------------------------------------------------------------- products
    const uint32_t qa = smem_u32(sq), ka = smem_u32(sk), va = smem_u32(sv);
    auto qk = [&]() {
      bool first = true;
#pragma unroll
      for (int pl = 0; pl < PL; ++pl)
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          mma_ss(tmem + kColS, sw128_desc(qa + pl * L::kPlane + (kk >> 2) * (kRows * 128) + (kk & 3) * 32),
                 sw128_desc(ka + (kk >> 2) * (kKeys * 128) + (kk & 3) * 32), idesc_f16(kKeys, false), first ? 0u : 1u);
          first = false;
        }
      commit(s_full);
    };
    bool ok = mbar_wait(q_full, 0, &g_prompt_err, 46) && mbar_wait(k_full, 0, &g_prompt_err, 47);
    if (ok) {
      after_sync();
      qk();
    }
    for (int j = 0; j < nb && ok; ++j) {
      if (j + 1 < nb) {
        ok = mbar_wait(k_full, (uint32_t)(j + 1) & 1u, &g_prompt_err, 48) &&
             mbar_wait(s_free, (uint32_t)j & 1u, &g_prompt_err, 49);
        if (!ok) break;
        after_sync();
        qk();
      }
      ok = mbar_wait(v_full, (uint32_t)j & 1u, &g_prompt_err, 50) && mbar_wait(p_full, (uint32_t)j & 1u, &g_prompt_err, 51);
      if (!ok) break;
      after_sync();
#pragma unroll
      for (int pl = 0; pl < PL; ++pl)
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          mma_ts(tmem + kColO, tmem + kColP + pl * 32 + kk * 8, sw128_desc(va + kk * 2048, kKeys * 128),
                 idesc_f16(HD, true),
                 (j > 0 || pl > 0 || kk > 0) ? 1u : 0u);
      commit(o_done);
    }
  }
  __syncwarp();
  before_sync();
  __syncthreads();
  if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
}

template <int HD, int PL>
cudaError_t launch(const PromptArgs& a, cudaStream_t s) {
  static OncePerDevice once;
  const cudaError_t e = once.smem(prompt_tc_kernel<HD, PL>, Smem<HD, PL>::kBytes);
  if (e != cudaSuccess) return e;
  const dim3 g((a.rows * a.group + kRows - 1) / kRows, a.c.n_kv, a.c.n_seq);
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
