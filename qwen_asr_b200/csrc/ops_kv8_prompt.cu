// Attention of many query rows over the int8 KV cache (ops_kv8.cu) on tcgen05: prompts and long chunks.
//
// One CTA owns 128 query rows of one KV head (row = query position x head of the group) and walks
// the keys they see in blocks of 64. Per block
//   S = Q K^T          M = 128, N = 64, K = head_dim   -> TMEM
//   p = exp2(S f - m)  f = scale * log2(e) * K scale of 16 tokens (a tile); running maximum m and sum l
//   O += P V           P = p * V scale * 2^(kTop - r), an operand in TMEM; N = head_dim
// and at the end O * 2^(r - kTop) / l.
//
// Precision. int8 is exact in f16, so K and V enter the products as they are; their scales stay
// outside, in f32. A query row is scaled by a power of two to [1/2, 1). For f32 rows q and P are two f16
// planes, hi + lo, which hold a value to 2^-22 of itself (q, or 2^-25 of the row's largest); both planes add into
// the same f32 accumulator. For bf16 rows one plane: 2^-11 of a probability, an eighth of the output's own rounding.
// f16 has no step below 2^-24, so a row's weights p * V scale are held as fractions of about the largest of them,
// 2^r, in the upper part of its range: none is off by more than 2^-30 of the row's largest so far (bf16 rows) or
// 2^-37 of the block's (f32 rows, whose blocks are added outside TMEM, each with an r of its own). Not as fractions
// of the largest V scale: a block of large values that a row gives no weight, or does not see, would cost it the
// others' bits (1e-3 of the output behind a scale 1e4 times as large); and thousands of keys that have 2^-25 of the
// weight each add up. All blocks take the same path: a score is taken relative to its tile's largest, which is exact
// for scores of any size, and a masked one is -inf (4 x 512 bf16 rows behind 1000 to 7000 112 us, f32 168; with a path
// each for whole, partly masked and large-scored blocks 125 and 178, by their length; 113 and 166 with fractions of
// the largest V scale and two paths).
// m is only raised when a score exceeds it by 2^kLag, and r of bf16 rows when a weight exceeds 2^(r + kLag): what has
// been summed is then rescaled, which the first blocks of a row do and later ones hardly ever.
//
// Two kernels. In both some warps do the softmax; others bring K and V from global memory as int8, two
// blocks ahead in registers, and write them as f16 rows of a token in the 128-byte-swizzle layout, which is
// K-major for Q K^T and MN-major for P V; the last warp issues the products, Q K^T of the next block
// before P V of this one. (One thread that did this was the longest chain of all: the operands of a product
// are uniform registers, and a branch of one lane has to fill them anew each time. A whole warp that waits
// and counts together, with an elected lane to issue, took 64 rows over 8064 f32 keys from 197 to 149 us.)
//   bf16 rows: 256 threads, a softmax thread a row; two CTAs an SM, one's softmax beside the other's
//   products. O stays in TMEM. 8 x 381 rows over up to 1403 keys, 8 KV heads of 2 x 128: 44 us; 2048 rows
//   over 8048 keys, 4 KV heads of 4 x 64: 145 us; 592 heads' rows over 8064 keys: 201 us, 773 TFLOP/s.
//   f32 rows: see below. The same shapes: 70, 214 and 310 us.
// Bound: the chain of a block's steps (scores, maximum, exp2, P V). bf16 rows: 0.9 us a block and CTA alone
// on its SM, two CTAs an SM, in which exp2 takes 0.27 us an SM and the products 0.3 to 0.35 (a quarter of the exp2 as
// polynomials on the FMA units was slower: 51 -> 55 us); f32 rows: 1.2 us, the products 0.7 of them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "bulk.cuh"
#include "dev_util.cuh"
#include "ops.h"

namespace qasr {
namespace {

constexpr int kMaxParts = 4;  // CTAs that share a row tile's keys
constexpr int kRows = 128, kKeys = 64, kThreads = 256, kFill = 96;  // (threads that bring K and V)
constexpr float kNone = -3.4028235e38f;  // running maximum before any key: the lowest number, no score is below
constexpr float kLag = 8.f;  // what a score may exceed m by, and a bf16 row's weight 2^r (log2)
constexpr int kTop1 = 7, kTop2 = 14;  // log2 of 2^r in P: 2^(kTop1 + kLag) and 2^kTop2 are in f16's range (to 65504)
constexpr float kTiny = 1.1754944e-38f;  // for a factor of 0: a masked score's -inf stays -inf
constexpr float kFaint = 80.f;  // probabilities under 2^-80 count as 2^-80 for r: P's factor stays finite
constexpr uint32_t kColS = 0, kColP = 64, kColO = 128, kCols = 256;  // TMEM columns

struct PromptArgs {
  Kv8 c;
  const void* q;
  void* out;
  long long q_seq, q_row, o_seq, o_row;
  const int *starts, *counts;
  int idx_stride, rows, group;
  float scale;
  int q_vec, o_vec;  // rows start on 16-byte boundaries
  int splits;        // CTAs of a cluster that share a row tile's keys
  OpsErrors* err;
};

template <int HD>
struct Smem {
  static constexpr int kPlane = kRows * HD * 2, kK = kKeys * HD * 2;
  // bf16 rows: Q, two K, a V; f32 rows: two planes of Q, two K, two V; then rows' factors, V scales, barriers
  static constexpr int kBytes1 = kPlane + 3 * kK + 2048;
  static constexpr int kBytes2 = 2 * kPlane + 4 * kK + 6144;
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
      "{\n .reg .pred e, p;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n .reg .pred e, p;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accum));
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
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
__device__ __forceinline__ float lg2(float x) {  // (-inf for 0 and, flushed, for what is below 2^-126)
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (NaN when a is)
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// r for weights of up to 2^e: the whole number 1/2 to 3/2 above it, within what leaves 2^r, and a V scale times
// 2^-r, in f32's range. (By 1.5 * 2^23, whose low bits are then the number.)
__device__ __forceinline__ int exponent_of(float e) {
  return __float_as_int(fminf(fmaxf(e, -100.f), 121.f) + 12582912.f) - 0x4B400000 + 1;
}
__device__ __forceinline__ float power(int r) { return __int_as_float((127 + r) << 23); }
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
// One tile of 16 scores, the largest of which is t: probabilities ex2((x - t) f + d), their sum to l, times w as f16
// planes. (Not ex2(x f - m): of large scores the rounding of m would be the largest probability's exponent.)
template <int PL>
__device__ __forceinline__ void weigh(const float* x, float t, float f, float d, float w, f32x2& l, uint32_t* hi, uint32_t* lo) {
  const f32x2 t2 = pair(-t, -t), f2 = pair(f, f), d2 = pair(d, d), w2 = pair(w, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 y = split(fma2(add2(pair(x[2 * i], x[2 * i + 1]), t2), f2, d2));
    const f32x2 p = pair(ex2(y.x), ex2(y.y));
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
// loops, with the barriers between them, and leave an output that the error code, reported at the end, disowns.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* gave_up, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  uint64_t t0 = 0;
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (i & 15) continue;  // (the timer is slow to read: never on a wait that soon ends)
    if (*gave_up) return false;
    const uint64_t now = global_timer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > 2000000000ull) {
      *gave_up = code;
      return false;
    }
  }
}

// The same for a whole warp, as one answer: what follows stays uniform to the compiler.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up, int code) {
  return __all_sync(0xffffffffu, wait(bar, parity, gave_up, code));
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

// What a CTA works on.
struct Work {
  int kvh, seq, row0, start, count, tiles, nb;  // tiles of 16 keys (a scale each), blocks of 64
  int first;                                    // the first key; scales, keys and tiles count from there
  const float *ks, *vs;
  const int8_t *k, *v;
};
// A sequence's first position (0 to the capacity) and live rows. (A skipped one's start must not be negative
// either: the order below counts from it, and would find no tile for a CTA.)
__device__ __forceinline__ void rows_of(const PromptArgs& a, int seq, int& start, int& count) {
  start = a.starts[(long long)seq * a.idx_stride];
  count = a.rows;
  if (a.counts) count = min(max(a.counts[(long long)seq * a.idx_stride], 0), a.rows);
  if (start < 0) count = 0;
  start = min(max(start, 0), a.c.capacity);
}
// All 32 lanes call it. The row tiles of up to 32 sequences are taken up by the keys they see, most first, so
// that no long one is left for the end: lane i counts those of sequence i that see at least K tiles' worth of
// keys, and a search over K finds the CTA's (8 x 381 f32 rows behind 0 to 1024 tokens 77 us with the last rows
// of all sequences as they come, 69 so; 4 x 1024 behind 6000, 0, 1000, 3000 291 and 229; where all begin alike,
// which needs no search, 37 and 39).
__device__ __forceinline__ Work work_of(const PromptArgs& a) {
  Work t;
  const int row_tiles = (int)(((long long)a.rows * a.group + kRows - 1) / kRows), id = blockIdx.x / a.splits;
  const int item = id / a.c.n_kv;
  t.kvh = id % a.c.n_kv;
  if (a.c.n_seq == 1) {
    t.seq = 0;
    t.row0 = (row_tiles - 1 - item) * kRows;
    rows_of(a, 0, t.start, t.count);
  } else {
    const int lane = threadIdx.x & 31, base = item / (32 * row_tiles) * 32, p = item % (32 * row_tiles);
    const int n = min(a.c.n_seq - base, 32), i = base + min(lane, n - 1);  // (lanes behind the last repeat it)
    int start, count;
    rows_of(a, i, start, count);
    // row tiles with live rows, and what the first sees, in rows of a tile
    int live = (int)(((long long)count * a.group + kRows - 1) / kRows);
    const int first = min(start / max(kRows / a.group, 1), 1 << 30);
    int who, tile;
    if (__all_sync(0xffffffffu, first == __shfl_sync(0xffffffffu, first, 0) && live == row_tiles)) {
      who = p % n;
      tile = row_tiles - 1 - p / n;
    } else {
      const int all = lane < n ? row_tiles : 0;
      if (lane >= n) live = 0;
      // tile x's key: first + x, or -1 - x without live rows; how many have K at least
      auto upto = [&](int K) {
        return K >= 0 ? min(max(live - max(K - first, 0), 0), live) : live + max(min(all - 1, -1 - K) - live + 1, 0);
      };
      int lo = -row_tiles, hi = __reduce_max_sync(0xffffffffu, first + live);  // more than p at lo, none at hi
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__reduce_add_sync(0xffffffffu, upto(mid)) > p) lo = mid;
        else hi = mid;
      }
      const int above = __reduce_add_sync(0xffffffffu, upto(lo + 1));
      const unsigned same = __ballot_sync(0xffffffffu, upto(lo) > upto(lo + 1));
      const bool me = (same >> lane & 1u) && __popc(same & ((1u << lane) - 1u)) == p - above;
      who = __ffs((int)__ballot_sync(0xffffffffu, me)) - 1;
      tile = lo >= 0 ? lo - __shfl_sync(0xffffffffu, first, who) : -1 - lo;
    }
    t.seq = base + who;
    t.row0 = tile * kRows;
    t.start = __shfl_sync(0xffffffffu, start, who);
    t.count = __shfl_sync(0xffffffffu, count, who);
  }
  // keys any row of the tile sees
  const int s_last = min(t.count - 1, (t.row0 + kRows - 1) / a.group);
  const int len = s_last >= t.row0 / a.group ? (int)min((long long)t.start + s_last + 1, (long long)a.c.capacity) : 0;
  // this CTA's share of their blocks
  const int all = (len + kKeys - 1) / kKeys, part = blockIdx.x % a.splits;
  const int b0 = (int)((long long)all * part / a.splits), b1 = (int)((long long)all * (part + 1) / a.splits);
  t.nb = b1 - b0;
  t.first = b0 * kKeys;
  t.tiles = (min(len, b1 * kKeys) - t.first + kKv8Block - 1) / kKv8Block;
  const long long blocks = a.c.capacity / kKv8Block;
  const long long head = ((long long)t.kvh * a.c.capacity + t.first) * a.c.head_dim;
  t.ks = a.c.ks + t.seq * a.c.scale_stride + t.kvh * blocks + t.first / kKv8Block;
  t.vs = a.c.vs + t.seq * a.c.scale_stride + t.kvh * blocks + t.first / kKv8Block;
  t.k = a.c.k + t.seq * a.c.seq_stride + head;
  t.v = a.c.v + t.seq * a.c.seq_stride + head;
  return t;
}

// Q as operand planes: each of eight warps brings 16 rows, all of them in flight, a lane HD / 32
// neighbouring values. Also the rows' factors.
template <int HD, int PL, bool BF16>
__device__ __forceinline__ void bring_q(const PromptArgs& a, const Work& t, unsigned char* sq, float* row_fac, int warp,
                                        int lane) {
  constexpr int N = HD / 32, kPlane = kRows * HD * 2;
  const int r0 = warp * 16;
  // lane i knows where row i is (a division a row, not one for each of its values)
  const int lr = t.row0 + r0 + (lane & 15), ls = lr / a.group;
  const long long loff = ls < t.count ? t.seq * a.q_seq + (long long)ls * a.q_row +
                                            (long long)(t.kvh * a.group + lr - ls * a.group) * HD
                                      : -1;
  LaneValues<BF16, N> raw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const long long off = __shfl_sync(0xffffffffu, loff, i);
    raw[i].zero();
    if (off >= 0) raw[i].load(a, off + lane * N);
  }
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
      if (PL == 2) *reinterpret_cast<uint2*>(at + kPlane) = make_uint2(lo[0], lo[1]);
    } else {
      *reinterpret_cast<uint32_t*>(at) = hi[0];
      if (PL == 2) *reinterpret_cast<uint32_t*>(at + kPlane) = lo[0];
    }
  }
  fence_async_smem();
}

// Where a query row's output starts (negative behind the last row).
__device__ __forceinline__ long long out_row(const PromptArgs& a, const Work& t, int rr, int hd) {
  if (rr >= a.rows * a.group) return -1;
  const int s = rr / a.group;
  return t.seq * a.o_seq + (long long)s * a.o_row + (long long)(t.kvh * a.group + rr - s * a.group) * hd;
}

// 16 bytes, or zeros. (Not by the read-only path, here as for the scales: what the kernel before has written must be
// seen, although this one may have started beside it.)
__device__ __forceinline__ uint4 ld_if(const int8_t* p, bool there) {
  uint4 v;
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %5, 0;\n mov.b32 %0, 0;\n mov.b32 %1, 0;\n mov.b32 %2, 0;\n mov.b32 %3, 0;\n"
      " @p ld.global.v4.b32 {%0,%1,%2,%3}, [%4];\n}\n"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"((int)there));
  return v;
}

// What one of FILL threads brings of a block of K or V: 16-byte pieces of rows (tokens) kStep apart, as int8 in
// registers, then f16 rows in shared memory. All addresses are a thread's own constants plus immediates.
template <int HD, int FILL>
struct Pieces {
  static constexpr int kRow = HD / 16, kStep = FILL / kRow, kN = (kKeys + kStep - 1) / kStep;
  static_assert(FILL % kRow == 0 && kStep % 4 == 0, "whole rows; their swizzle is one of two");
  uint4 r[kN];
  // tokens from end on are zeros
  __device__ __forceinline__ void load(const int8_t* src, int j, int end, int ct) {
    const int row = ct / kRow, left = min(end - j * kKeys, kKeys) - row;
    const int8_t* p = src + (long long)j * (kKeys * HD) + ct * 16;
#pragma unroll
    for (int i = 0; i < kN; ++i) r[i] = ld_if(p + i * (kStep * HD), i * kStep < left);
  }
  __device__ __forceinline__ void store(unsigned char* dst, int ct) const {
    const int row = ct / kRow, c = ct % kRow * 2;  // 16-byte f16 chunks c, c + 1
    // lanes of the second 64 columns begin with their second chunk, so that eight lanes hit distinct banks
    const bool swap = c & 8;
    unsigned char* p = dst + (c >> 3) * (kKeys * 128) + row * 128;
    const uint32_t at0 = (((c & 7) + (int)swap) ^ (row & 7)) << 4, at1 = at0 ^ 16;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if (kKeys % kStep && i == kN - 1 && row + i * kStep >= kKeys) break;
      const uint32_t flip = (i * kStep & 4) << 4;
      const uint32_t w[4] = {(swap ? r[i].z : r[i].x) ^ 0x80808080u, (swap ? r[i].w : r[i].y) ^ 0x80808080u,
                             (swap ? r[i].x : r[i].z) ^ 0x80808080u, (swap ? r[i].y : r[i].w) ^ 0x80808080u};
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<uint4*>(p + i * (kStep * 128) + ((h ? at1 : at0) ^ flip)) =
            make_uint4(bytes_f16<0x4140>(w[2 * h]), bytes_f16<0x4342>(w[2 * h]), bytes_f16<0x4140>(w[2 * h + 1]),
                       bytes_f16<0x4342>(w[2 * h + 1]));
    }
    fence_async_smem();
  }
};

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float peer1(uint32_t addr, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_rank(addr, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 peer4(uint32_t addr, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(map_rank(addr, rank))
               : "memory");
  return v;
}

// Four values of an output row.
template <bool BF16>
__device__ __forceinline__ void put4(const PromptArgs& a, long long at, float4 o) {
  if constexpr (BF16) {
    __nv_bfloat16* p = (__nv_bfloat16*)a.out + at;
    __nv_bfloat162 v[2] = {__floats2bfloat162_rn(o.x, o.y), __floats2bfloat162_rn(o.z, o.w)};
    if (a.o_vec) {
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(v);
    } else {
      p[0] = v[0].x; p[1] = v[0].y; p[2] = v[1].x; p[3] = v[1].y;
    }
  } else {
    float* p = (float*)a.out + at;
    if (a.o_vec) {
      *reinterpret_cast<float4*>(p) = o;
    } else {
      p[0] = o.x; p[1] = o.y; p[2] = o.z; p[3] = o.w;
    }
  }
}

// Stores 32 / PARTS rows of a warp's 32 staged rows (pitch kPitch floats), the part-th share; `mine`: the
// output offset of this lane's row, negative for none.
template <int HD>
constexpr int kPitch = HD + 4;  // floats; eight rows' 16-byte pieces hit distinct banks
template <int HD, bool BF16, int PARTS>
__device__ __forceinline__ void write_rows(const PromptArgs& a, const float* stage, long long mine, int part, int lane) {
  constexpr int kLanes = HD / 4, kPer = 32 / kLanes, kRowsEach = 32 / PARTS;  // lanes of a row, rows at a time
  const int col = lane % kLanes * 4;
#pragma unroll 1
  for (int i0 = part * kRowsEach; i0 < (part + 1) * kRowsEach; i0 += 8 * kPer) {
    float4 o[8];  // (all read before the first store, which might alias them for all the compiler knows)
    long long off[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i0 + i * kPer + lane / kLanes;
      o[i] = *reinterpret_cast<const float4*>(stage + r * kPitch<HD> + col);
      off[i] = __shfl_sync(0xffffffffu, mine, r);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (off[i] >= 0) put4<BF16>(a, off[i] + col, o[i]);
    }
  }
}

// A cluster's parts of the output rows (staged: each by itself, with its maximum and sum of p), joined by 256
// threads: a CTA finishes 128 / splits of the rows. First the weights of each row's parts, a thread each, ...
__device__ __forceinline__ void join_weights(const PromptArgs& a, uint32_t maxima, uint32_t sums, float* weights, int tid) {
  if (tid >= kRows) return;
  const int p = tid % a.splits, r = (int)(blockIdx.x % a.splits) * (kRows / a.splits) + tid / a.splits;
  const float m = peer1(maxima + r * 4, p), l = peer1(sums + r * 4, p);
  float top = m;
  for (int o = 1; o < a.splits; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float part = l * ex2(m - top);
  float total = part;
  for (int o = 1; o < a.splits; o *= 2) total += __shfl_xor_sync(0xffffffffu, total, o);
  weights[tid] = total == 0.f ? 0.f : __fdiv_rn(part, total);
}
// ... then the rows.
template <int HD, bool BF16>
__device__ __forceinline__ void join_rows(const PromptArgs& a, const Work& t, uint32_t stage, const float* weights,
                                          int warp, int lane) {
  constexpr int kLanes = HD / 4, kPer = 32 / kLanes;
  const int each = kRows / a.splits, r0 = (int)(blockIdx.x % a.splits) * each, col = lane % kLanes * 4;
  for (int i = warp * kPer + lane / kLanes; i < each; i += 8 * kPer) {
    const uint32_t at = stage + ((r0 + i) * kPitch<HD> + col) * 4;
    const long long off = out_row(a, t, t.row0 + r0 + i, HD);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4& v, float w) {
      o.x = fmaf(v.x, w, o.x); o.y = fmaf(v.y, w, o.y); o.z = fmaf(v.z, w, o.z); o.w = fmaf(v.w, w, o.w);
    };
    for (int p = 0; p < a.splits; p += 2) {
      const float4 v0 = peer4(at, p), v1 = peer4(at, p + 1);
      add(v0, weights[i * a.splits + p]);
      add(v1, weights[i * a.splits + p + 1]);
    }
    if (off >= 0) put4<BF16>(a, off + col, o);
  }
}

// ------------------------------------------------------------------ bf16 rows: one plane, two CTAs an SM
// grid: row tiles x sequences x KV heads
template <int HD>
__global__ void __launch_bounds__(kThreads, 2) prompt_bf16_kernel(const PromptArgs a) {
  using L = Smem<HD>;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *sq = smem, *sk = smem + L::kPlane, *sv = sk + 2 * L::kK;
  float* row_fac = reinterpret_cast<float*>(sv + L::kK);  // each row's factor
  float* row_sum = row_fac + kRows;                       // (a part's) each row's sum
  float* weights = row_sum + kRows;                       // the joined parts'
  uint64_t* k_full = reinterpret_cast<uint64_t*>(weights + kRows);
  uint64_t *k_free = k_full + 2, *v_full = k_full + 4, *s_full = k_full + 5, *s_free = k_full + 6, *p_full = k_full + 7,
           *o_done = k_full + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(k_full + 9);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;  // (uniform)
  if (smem_u32(smem) & 1023) {  // the swizzle's rows would not fit (never seen: no static shared memory)
    if (tid == 0) ops_gave_up(a.err, 40);
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
    pdl_launch_dependents();  // (not before: the next kernel's blocks may want TMEM too, and wait for this one's end)
  }
  pdl_wait();

  const Work t = work_of(a);
  const int row0 = t.row0, start = t.start, count = t.count, tiles = t.tiles, nb = t.nb;
  if (nb > 0) bring_q<HD, 1, true>(a, t, sq, row_fac, warp, lane);
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp < 4) {
    // ---------------------------------------------------------------- softmax: thread = query row = TMEM lane
    const int rr = row0 + tid, s = rr / a.group;
    const bool live = s < count;
    const int last = (live ? min(start + s, a.c.capacity - 1) : -1) - t.first;
    const float fac = nb > 0 ? row_fac[tid] : 0.f;
    const uint32_t trow = tmem + ((uint32_t)(warp * 32) << 16);
    // log2 of the largest weight so far, relative to m; r + kLag, and 2^(kTop1 - r)
    float m = kNone, most = -__int_as_float(0x7F800000), full = -__int_as_float(0x7F800000), up = 1.f;
    f32x2 l = 0;  // two partial sums
    float kn[4], vn[4];  // the next block's scales
    auto scales = [&](int j) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int tl = j * 4 + b;
        kn[b] = tl < tiles ? t.ks[tl] : 0.f;
        vn[b] = tl < tiles ? t.vs[tl] : 0.f;
      }
    };
    scales(0);
    for (int j = 0; j < nb; ++j) {
      float f[4], w[4];
      const int pos0 = j * kKeys;
      const bool partial = __any_sync(0xffffffffu, pos0 + kKeys - 1 > last);
      float wl[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        f[b] = fac * kn[b];
        w[b] = vn[b];
        if (f[b] == 0.f) f[b] = kTiny;
        // a row that sees nothing of a tile takes nothing of its scales either (they may be NaN)
        if (partial && pos0 + b * kKv8Block > last) f[b] = 1.f, w[b] = 0.f;
        wl[b] = lg2(w[b]);
      }
      const float faint = fmaxf(fmaxf(wl[0], wl[1]), fmaxf(wl[2], wl[3])) - kFaint;
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
      float mx = kNone, e = -__int_as_float(0x7F800000), top[4], d[4];  // a tile's largest x, and its score
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        top[b] = x[16 * b];
#pragma unroll
        for (int i = 1; i < 16; ++i) top[b] = fmaxf(top[b], x[16 * b + i]);
        top[b] = fmaxf(top[b], kNone);  // (a masked tile's -inf)
        d[b] = __fmul_rn(top[b], f[b]);
        mx = fmaxf(mx, d[b]);  // (no number: ignored)
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        d[b] -= mx;
        e = fmaxf(e, d[b] + wl[b]);  // log2 of the largest weight, for a maximum of mx
      }
      const bool grow = mx > m + kLag || fmaxf(e + (mx - m), faint) > full, rescale = __any_sync(0xffffffffu, grow);
      float corr = 1.f, corr_o = 1.f;
      if (grow) {
        const float m1 = mx > m + kLag ? mx : m;
        most = fmaxf(most + (m - m1), e + (mx - m1));
        const int r = exponent_of(fmaxf(most, faint));
        corr = ex2(m - m1);
        corr_o = ex2(m - m1 + (full - (kLag + (float)r)));
        m = m1;
        full = kLag + (float)r;
        up = power(kTop1 - r);
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) d[b] += mx - m;
#pragma unroll
      for (int b = 0; b < 4; ++b) w[b] *= up;
      if (j > 0) {
        wait(o_done, (uint32_t)(j - 1) & 1u, gave_up, 44);
        __syncwarp();
        after_sync();
        if (rescale) {
          l = mul2(l, pair(corr, corr));
#pragma unroll 1
          for (int c = 0; c < HD; c += 16) {
            uint32_t o[16];
            tmem_ld16(trow + kColO + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr_o);
            tmem_st16(trow + kColO + c, o);
          }
          tmem_st_wait();
        }
      }
      f32x2 sum = 0;  // (a block's own: one by one, small probabilities would not move a large l)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t hi[8];
        weigh<1>(x + 16 * b, top[b], f[b], d[b], w[b], sum, hi, nullptr);
        tmem_st8(trow + kColP + 8 * b, hi);
      }
      l = add2(l, sum);
      tmem_st_wait();
      before_sync();
      mbar_arrive(p_full);
    }
    // ---- O * 2^(r - kTop1) / l
    if (nb > 0) wait(o_done, (uint32_t)(nb - 1) & 1u, gave_up, 45);
    __syncwarp();
    after_sync();
    const float2 sums = split(l);
    const float total = sums.x + sums.y;
    const float inv = total == 0.f ? 0.f : __fdiv_rn(1.0f, up * total);
    if (a.splits > 1) {  // (joined below)
      row_fac[tid] = m;
      row_sum[tid] = total;
    }
    // through shared memory (operands are idle now, 32 rows a warp), so that a row's stores are contiguous
    static_assert(kRows * kPitch<HD> * 4 <= L::kPlane + 3 * L::kK, "the output reuses the operands");
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
        *reinterpret_cast<float4*>(stage + tid * kPitch<HD> + c + i) =
            nb > 0 ? make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncwarp();
    if (a.splits == 1)
      write_rows<HD, true, 1>(a, stage + warp * 32 * kPitch<HD>, out_row(a, t, rr, HD), 0, lane);
  } else if (warp < 7) {
    // ---------------------------------------------------------------- K and V: int8 -> f16 operands
    const int ct = tid - 128, end = tiles * kKv8Block;
    // two blocks ahead in registers (memory takes 1.2 us, a block 1.0 to 1.3; one ahead: 592 heads' rows over
    // 8064 tokens 240 us, two 198)
    Pieces<HD, kFill> k0, k1, v0, v1;  // of even and of odd blocks
    k0.load(t.k, 0, end, ct);
    k1.load(t.k, 1, end, ct);
    v0.load(t.v, 0, end, ct);
    v1.load(t.v, 1, end, ct);
    auto put_k = [&](int j, Pieces<HD, kFill>& k) {  // into its buffer, then the loads of the block after the next
      k.store(sk + (j & 1) * L::kK, ct);
      mbar_arrive(&k_full[j & 1]);
      k.load(t.k, j + 2, end, ct);
    };
    auto block = [&](int j, Pieces<HD, kFill>& k, Pieces<HD, kFill>& v) {
      // K of block j + 1 goes where that of j - 1 was
      if (j + 1 < nb) {
        // (a barrier of its own: that of S may be two phases on by now)
        if (j > 0 && !wait(&k_free[(j - 1) & 1], (uint32_t)((j - 1) >> 1) & 1u, gave_up, 46)) return false;
        put_k(j + 1, k);
      }
      if (j > 0 && !wait(o_done, (uint32_t)(j - 1) & 1u, gave_up, 47)) return false;
      v.store(sv, ct);
      mbar_arrive(v_full);
      v.load(t.v, j + 2, end, ct);
      return true;
    };
    if (nb > 0) put_k(0, k0);
    for (int j = 0; j < nb; j += 2)
      if (!block(j, k1, v0) || (j + 1 < nb && !block(j + 1, k0, v1))) break;
  } else if (nb > 0) {
    // ---------------------------------------------------------------- products
    const uint32_t qa = smem_u32(sq), ka = smem_u32(sk), va = smem_u32(sv);
    auto qk = [&](int j) {
      if (!warp_wait(&k_full[j & 1], (uint32_t)(j >> 1) & 1u, gave_up, 41)) return;
      after_sync();
      const uint32_t kb = ka + (uint32_t)(j & 1) * L::kK;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
        mma_ss(tmem + kColS, sw128_desc(qa + (kk >> 2) * (kRows * 128) + (kk & 3) * 32),
               sw128_desc(kb + (kk >> 2) * (kKeys * 128) + (kk & 3) * 32), idesc_f16(kKeys, false), kk > 0 ? 1u : 0u);
      commit(s_full);
      commit(&k_free[j & 1]);
    };
    qk(0);
    for (int j = 0; j < nb; ++j) {
      if (j + 1 < nb) {
        if (!warp_wait(s_free, (uint32_t)j & 1u, gave_up, 48)) break;
        qk(j + 1);
      }
      if (!warp_wait(v_full, (uint32_t)j & 1u, gave_up, 42) || !warp_wait(p_full, (uint32_t)j & 1u, gave_up, 49)) break;
      after_sync();
#pragma unroll
      for (int kk = 0; kk < kKeys / 16; ++kk)
        mma_ts(tmem + kColO, tmem + kColP + kk * 8, sw128_desc(va + kk * 2048, kKeys * 128), idesc_f16(HD, true),
               (j > 0 || kk > 0) ? 1u : 0u);
      commit(o_done);
    }
  }
  if (a.splits > 1) {
    __syncwarp();
    cluster_barrier();  // every part is staged
    join_weights(a, smem_u32(row_fac), smem_u32(row_sum), weights, tid);
    __syncthreads();
    join_rows<HD, true>(a, t, smem_u32(smem), weights, warp, lane);
    __syncwarp();
    cluster_barrier();  // no CTA leaves while a peer reads its part
  }
  __syncwarp();
  before_sync();
  __syncthreads();
  if (tid == 0 && *gave_up) ops_gave_up(a.err, *gave_up);
  if (warp == 7) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
}

// ------------------------------------------------------------------ f32 rows: two planes, one CTA an SM
constexpr int kThreads2 = 512, kFillV = 96;
// TMEM columns: S, P's planes and O of two blocks each
constexpr uint32_t kS2 = 0, kP2 = 128, kO2 = 256, kCols2 = 512;

// Warps 0-7 softmax: two threads a row, each half the block's keys and half the output's dims, whose sums
// it keeps in f32 registers: every block's product starts from zero and is added there. (Accumulated in
// TMEM over all blocks, the tensor core's rounding towards zero shrank the output by 4e-8 a product:
// 1.7e-6 at 1400 keys, and growing.) Warps 8-11 bring K and 12-14 V, two blocks ahead in registers,
// warp 15 issues the products. The softmax warps take the registers that the others leave:
// 256 x (168 + 88) = 512 x 128.
template <int HD>
__global__ void __launch_bounds__(kThreads2, 1) prompt_f32_kernel(const PromptArgs a) {
  using L = Smem<HD>;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *sq = smem, *sk = smem + 2 * L::kPlane, *sv = sk + 2 * L::kK;
  float* row_fac = reinterpret_cast<float*>(sv + 2 * L::kK);  // each row's factor
  float* row_max = row_fac + kRows;                           // [block parity][half][row] (largest score, weight)
  float* row_sum = row_max + 8 * kRows;                       // [row] the second half's sum
  uint64_t* k_full = reinterpret_cast<uint64_t*>(row_sum + kRows);
  uint64_t *k_free = k_full + 2, *v_full = k_full + 4, *v_free = k_full + 6, *s_full = k_full + 8, *s_free = k_full + 10,
           *o_full = k_full + 12, *o_free = k_full + 14, *p_full = k_full + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(k_full + 18);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;  // (uniform)
  if (smem_u32(smem) & 1023) {
    if (tid == 0) ops_gave_up(a.err, 40);
    return;
  }
  if (tid == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(&k_full[b], 128);
      mbar_init(&k_free[b], 1);
      mbar_init(&v_full[b], kFillV);
      mbar_init(&v_free[b], 1);
      mbar_init(&s_full[b], 1);
      mbar_init(&s_free[b], 256);
      mbar_init(&o_full[b], 1);  // P V of a block is done: its O may be read, P overwritten
      mbar_init(&o_free[b], 256);
      mbar_init(&p_full[b], 256);
    }
    *gave_up = 0;
    fence_mbar_init();
  }
  if (warp == 15) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kCols2));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    pdl_launch_dependents();  // (not before: the next kernel's blocks may want TMEM too, and wait for this one's end)
  }
  pdl_wait();
  const Work t = work_of(a);
  const int nb = t.nb;
  if (nb > 0 && warp < 8) bring_q<HD, 2, false>(a, t, sq, row_fac, warp, lane);
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    // ---------------------------------------------------------------- softmax: row = TMEM lane
    constexpr int kDims = HD / 2;
    const int half = warp >> 2, row = (warp & 3) * 32 + lane, rr = t.row0 + row, s = rr / a.group;
    const int last = (s < t.count ? min(t.start + s, a.c.capacity - 1) : -1) - t.first;
    const float fac = nb > 0 ? row_fac[row] : 0.f;
    const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    float m = kNone;
    f32x2 l = 0, acc[kDims / 2];
#pragma unroll
    for (f32x2& x : acc) x = 0;
    float kn[2], vn[2];  // the next block's scales, of this half's two tiles
    auto scales = [&](int j) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int tl = j * 4 + half * 2 + b;
        kn[b] = tl < t.tiles ? t.ks[tl] : 0.f;
        vn[b] = tl < t.tiles ? t.vs[tl] : 0.f;
      }
    };
    float down = 0.f;          // 2^(r - kTop2) of the last block
    auto add_o = [&](int j) {  // acc += O of block j, whose buffer is free then
      const f32x2 d2 = pair(down, down);
      const uint32_t col = trow + kO2 + (uint32_t)((j & 1) * HD + half * kDims);
#pragma unroll
      for (int c = 0; c < kDims; c += 32) {
        float o[32];
        tmem_ld32(col + c, reinterpret_cast<uint32_t*>(o));
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c / 2 + i] = fma2(pair(o[2 * i], o[2 * i + 1]), d2, acc[c / 2 + i]);
      }
      before_sync();
      mbar_arrive(&o_free[j & 1]);
    };
    scales(0);
    for (int j = 0; j < nb; ++j) {
      float f[2], w[2], wl[2];
      const int pos0 = j * kKeys + half * 32;
      const bool partial = __any_sync(0xffffffffu, pos0 + 31 > last);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        f[b] = fac * kn[b];
        w[b] = vn[b];
        if (f[b] == 0.f) f[b] = kTiny;
        // a row that sees nothing of a tile takes nothing of its scales either (they may be NaN)
        if (partial && pos0 + b * kKv8Block > last) f[b] = 1.f, w[b] = 0.f;
        wl[b] = lg2(w[b]);
      }
      if (j + 1 < nb) scales(j + 1);
      wait(&s_full[j & 1], (uint32_t)(j >> 1) & 1u, gave_up, 51);
      __syncwarp();
      after_sync();
      float x[32];
      tmem_ld32(trow + kS2 + (uint32_t)((j & 1) * kKeys + half * 32), reinterpret_cast<uint32_t*>(x));
      tmem_ld_wait();
      before_sync();
      mbar_arrive(&s_free[j & 1]);
      if (partial) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (pos0 + i > last) x[i] = -__int_as_float(0x7F800000);
      }
      float mx = kNone, top[2], d[2];  // a tile's largest x, and its score
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        top[b] = x[16 * b];
#pragma unroll
        for (int i = 1; i < 16; ++i) top[b] = fmaxf(top[b], x[16 * b + i]);
        top[b] = fmaxf(top[b], kNone);  // (a masked tile's -inf)
        d[b] = __fmul_rn(top[b], f[b]);
        mx = fmaxf(mx, d[b]);  // (no number: ignored)
      }
      d[0] -= mx;
      d[1] -= mx;
      // log2 of the largest weight, for a maximum of mx
      const float e = fmaxf(fmaxf(d[0] + wl[0], d[1] + wl[1]), fmaxf(wl[0], wl[1]) - kFaint);
      // over both halves of the row (two buffers: the next block's barrier keeps them apart)
      float2* shared_max = reinterpret_cast<float2*>(row_max) + (j & 1) * 2 * kRows;
      shared_max[half * kRows + row] = make_float2(mx, e);
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const float2 other = shared_max[(half ^ 1) * kRows + row];
      const float both = fmaxf(mx, other.x);
      const bool grow = both > m + kLag;
      const float corr = grow ? ex2(m - both) : 1.f;
      const bool rescale = __any_sync(0xffffffffu, grow);
      if (grow) m = both;
      if (rescale) l = mul2(l, pair(corr, corr));
      d[0] += mx - m;
      d[1] += mx - m;
      const int r = exponent_of(fmaxf(e + (mx - m), other.y + (other.x - m)));
#pragma unroll
      for (int b = 0; b < 2; ++b) w[b] = min_nan(w[b] * power(kTop2 - r), 1e37f);
      // (P of block j - 2 has been read: its O was added in the last round)
      const uint32_t pcol = trow + kP2 + (uint32_t)((j & 1) * 64 + half * 16);
      f32x2 sum = 0;  // (a block's own: one by one, small probabilities would not move a large l)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t hi[8], lo[8];
        weigh<2>(x + 16 * b, top[b], f[b], d[b], w[b], sum, hi, lo);
        tmem_st8(pcol + 8 * b, hi);
        tmem_st8(pcol + 32 + 8 * b, lo);
      }
      l = add2(l, sum);
      tmem_st_wait();
      before_sync();
      mbar_arrive(&p_full[j & 1]);
      if (j > 0) {  // beside this block's product
        wait(&o_full[(j - 1) & 1], (uint32_t)((j - 1) >> 1) & 1u, gave_up, 52);
        __syncwarp();
        after_sync();
        add_o(j - 1);
      }
      down = power(r - kTop2);
      if (rescale) {
#pragma unroll
        for (f32x2& y : acc) y = mul2(y, pair(corr, corr));
      }
    }
    if (nb > 0) {
      wait(&o_full[(nb - 1) & 1], (uint32_t)((nb - 1) >> 1) & 1u, gave_up, 53);
      __syncwarp();
      after_sync();
      add_o(nb - 1);
    }
    // ---- O / l, through shared memory, so that a row's stores are contiguous
    const float2 sums = split(l);
    float total = sums.x + sums.y;
    if (half == 1) row_sum[row] = total;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (half == 0) row_sum[row] += total;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    total = row_sum[row];
    const float inv = total == 0.f ? 0.f : __fdiv_rn(1.0f, total);
    if (a.splits > 1 && half == 0) row_fac[row] = m;  // (joined below)
    static_assert(kRows * kPitch<HD> * 4 <= 2 * L::kPlane + 4 * L::kK, "the output reuses the operands");
    float* stage = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int i = 0; i < kDims / 2; i += 2) {
      const float2 p = split(acc[i]), q = split(acc[i + 1]);
      *reinterpret_cast<float4*>(stage + row * kPitch<HD> + half * kDims + 2 * i) =
          make_float4(p.x * inv, p.y * inv, q.x * inv, q.y * inv);
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (a.splits == 1) {
      write_rows<HD, false, 2>(a, stage + (warp & 3) * 32 * kPitch<HD>, out_row(a, t, rr, HD), half, lane);
    } else {
      cluster_barrier();  // every part is staged
      join_weights(a, smem_u32(row_fac), smem_u32(row_sum), row_max, tid);
      asm volatile("bar.sync 1, 256;" ::: "memory");
      join_rows<HD, false>(a, t, smem_u32(smem), row_max, warp, lane);
      __syncwarp();
      cluster_barrier();  // no CTA leaves while a peer reads its part
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    const int end = t.tiles * kKv8Block;
    // one operand's blocks in turn: two in registers, each stored when its buffer is free
    auto fill = [&](auto& even, auto& odd, const int8_t* src, unsigned char* dst, uint64_t* full, uint64_t* free, int ct) {
      even.load(src, 0, end, ct);
      odd.load(src, 1, end, ct);
      for (int j = 0; j < nb; j += 2) {
        const uint32_t before = (uint32_t)((j >> 1) - 1) & 1u;  // the phase in which block j - 2 left the buffer
        if (j >= 2 && !wait(&free[0], before, gave_up, 54)) break;
        even.store(dst, ct);
        mbar_arrive(&full[0]);
        even.load(src, j + 2, end, ct);
        if (j + 1 >= nb) break;
        if (j >= 2 && !wait(&free[1], before, gave_up, 55)) break;
        odd.store(dst + L::kK, ct);
        mbar_arrive(&full[1]);
        odd.load(src, j + 3, end, ct);
      }
    };
    if (warp < 12) {
      // -------------------------------------------------------------- K: int8 -> f16 operand
      Pieces<HD, 128> even, odd;
      fill(even, odd, t.k, sk, k_full, k_free, tid - 256);
    } else if (warp < 15) {
      // -------------------------------------------------------------- V
      Pieces<HD, kFillV> even, odd;
      fill(even, odd, t.v, sv, v_full, v_free, tid - 384);
    } else if (nb > 0) {
      // ---------------------------------------------------------------- products
      const uint32_t qa = smem_u32(sq), ka = smem_u32(sk), va = smem_u32(sv);
      auto qk = [&](int j) {
        const int b = j & 1;
        if (j >= 2 && !warp_wait(&s_free[b], (uint32_t)((j - 2) >> 1) & 1u, gave_up, 56)) return;
        if (!warp_wait(&k_full[b], (uint32_t)(j >> 1) & 1u, gave_up, 57)) return;
        after_sync();
#pragma unroll
        for (int pl = 0; pl < 2; ++pl)
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            mma_ss(tmem + kS2 + (uint32_t)(b * kKeys),
                   sw128_desc(qa + pl * L::kPlane + (kk >> 2) * (kRows * 128) + (kk & 3) * 32),
                   sw128_desc(ka + b * L::kK + (kk >> 2) * (kKeys * 128) + (kk & 3) * 32), idesc_f16(kKeys, false),
                   (pl > 0 || kk > 0) ? 1u : 0u);
        commit(&s_full[b]);
        commit(&k_free[b]);
      };
      qk(0);
      for (int j = 0; j < nb; ++j) {
        const int b = j & 1;
        if (j + 1 < nb) qk(j + 1);
        if (!warp_wait(&v_full[b], (uint32_t)(j >> 1) & 1u, gave_up, 58) || !warp_wait(&p_full[b], (uint32_t)(j >> 1) & 1u, gave_up, 59)) break;
        if (j >= 2 && !warp_wait(&o_free[b], (uint32_t)((j - 2) >> 1) & 1u, gave_up, 60)) break;
        after_sync();
#pragma unroll
        for (int pl = 0; pl < 2; ++pl)
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            mma_ts(tmem + kO2 + (uint32_t)(b * HD), tmem + kP2 + (uint32_t)(b * 64) + pl * 32 + kk * 8,
                   sw128_desc(va + b * L::kK + kk * 2048, kKeys * 128), idesc_f16(HD, true), (pl > 0 || kk > 0) ? 1u : 0u);
        commit(&o_full[b]);
        commit(&v_free[b]);
      }
    }
    if (a.splits > 1) {  // (with the softmax warps)
      __syncwarp();
      cluster_barrier();
      cluster_barrier();
    }
  }
  __syncwarp();
  before_sync();
  __syncthreads();
  if (tid == 0 && *gave_up) ops_gave_up(a.err, *gave_up);
  if (warp == 15) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols2));
}

// CTAs of a row tile, 1, 2 or 4, whose parts a cluster joins through shared memory: the number with the least
// estimated time in blocks of keys, of which a CTA's prologue and output cost 8 and a joined one's 11; `room` CTAs
// run at once. (Eight wait long for a place.) 16 heads on 8 x 128, measured (us) at 1 / 2 / 4: 128 rows behind 8000
// bf16 124 / 70 / 42, f32 150 / 84 / 48, behind 100 11.5 / 12.9 / 11.1 and 13.1 / 13.7 / 12.1; 2 x 512 rows behind
// 3000 and 7000 bf16 155 / 96 / 85, f32 146 / 120 / 144; 1500 rows behind 6000 bf16 174 / 138 / 148, f32 243 / 215 /
// 247; 4 x 512 behind 1000 to 7000 bf16 169 / 113 / 139, f32 167 / 187 / 248; 8 x 381 behind 0 to 1022 bf16 45 / 65 /
// 103, f32 70 / 114 / 181.
int auto_splits(long long ctas, int room, int max_len) {
  const long long blocks = (max_len + kKeys - 1) / kKeys;
  int best = 1;
  long long least = 0;
  for (int s = 1; s <= kMaxParts; s *= 2) {
    const long long cost = std::max<long long>(room, ctas * s) * ((blocks + s - 1) / s + (s > 1 ? 11 : 8));
    if (s == 1 || cost < least) {
      best = s;
      least = cost;
    }
  }
  return best;
}

template <int HD, bool BF16>
cudaError_t launch(PromptArgs a, int max_len, cudaStream_t s) {
  const long long ctas = ((long long)a.rows * a.group + kRows - 1) / kRows * a.c.n_kv * a.c.n_seq;
  if (ctas > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
  if (a.splits < 1) a.splits = auto_splits(ctas, ops_sm_count() * (BF16 ? 2 : 1), max_len);
  const dim3 g((unsigned)ctas * a.splits);
  static OncePerDevice once;
  if constexpr (BF16) {
    const cudaError_t e = once.smem(prompt_bf16_kernel<HD>, Smem<HD>::kBytes1);
    if (e != cudaSuccess) return e;
    return ops_launch(prompt_bf16_kernel<HD>, g, dim3(kThreads), Smem<HD>::kBytes1, s, a.splits, a);
  } else {
    const cudaError_t e = once.smem(prompt_f32_kernel<HD>, Smem<HD>::kBytes2);
    if (e != cudaSuccess) return e;
    return ops_launch(prompt_f32_kernel<HD>, g, dim3(kThreads2), Smem<HD>::kBytes2, s, a.splits, a);
  }
}

}  // namespace

cudaError_t kv8_prompt_attention(const Kv8& c, const void* q, long long q_seq, long long q_row, void* out,
                                 long long o_seq, long long o_row, OpsDtype dt, int rows, int heads, const int* starts,
                                 const int* counts, int idx_stride, float scale, int max_len,
                                 int splits, OpsErrors* err, cudaStream_t s) {
  if (!err) return cudaErrorInvalidValue;
  auto vec = [&](const void* p, long long seq, long long row) {
    const int es = dt == OPS_BF16 ? 2 : 4;
    return (uintptr_t)p % 16 == 0 && seq * es % 16 == 0 && row * es % 16 == 0;
  };
  const PromptArgs a{c, q, out, q_seq, q_row, o_seq, o_row, starts, counts, idx_stride, rows, heads / c.n_kv, scale,
                     vec(q, q_seq, q_row), vec(out, o_seq, o_row), splits, err};
  if (c.head_dim == 128) return dt == OPS_BF16 ? launch<128, true>(a, max_len, s) : launch<128, false>(a, max_len, s);
  return dt == OPS_BF16 ? launch<64, true>(a, max_len, s) : launch<64, false>(a, max_len, s);
}

}  // namespace qasr
