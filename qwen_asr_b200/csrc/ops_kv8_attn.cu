// Attention over the int8 KV cache (ops_kv8.cu): o = softmax(scale q K^T) V per head, causal over
// positions 0 .. start + row, grouped query heads.
//
// Tensor-core tiles of 16 tokens, the cache's scale block, so a tile has one K and one V scale.
// int8 values are exact in f16 (the byte x + 128 under the exponent of 1024 is 1152 + x), so K
// and V enter as they are, and the scales stay in f32: the K scale multiplies the scores, the V
// scale the tile's product. A query row is first scaled by a power of two that puts its largest
// value into [1/2, 1).
//   f32 rows: q and the probabilities enter as two f16 planes, v = hi + lo, which holds them to
//     2^-22 of themselves (q: or 2^-25 of the row's largest, below f32's own rounding of it). The two planes are
//     rows r and r + 8 of the same 16-row operand: a tile holds 8 query rows and both planes cost one product.
//   bf16 rows: one plane (a bf16 value is exact in f16 down to 2^-14 of the row's largest, and
//     the probabilities' 2^-11 is an eighth of the output's own 2^-8), 16 rows a tile.
//   The probabilities of a tile are relative to the largest of the tile, 2^15 (f16 has no step below 2^-24, and
//     thousands of keys of 2^-25 each add up): what it is of the row's is in the tile's V scale.
// Scores, the running maximum and sum and the output stay in f32 registers.
//
// Fragments straight from the cache's layout: the order of the head's dimensions within the score
// product, and that of the output columns, are free as long as both operands agree. A thread takes
// 16 contiguous bytes of a token for both products; V's token pairs are interleaved in registers.
//
// Digit kernel (up to four query rows a KV head, so most single tokens): the products stay in
// integers. A query row is held as three signed 7-bit digits of q / max|q| (2^-22 of the largest),
// the weights (probability x V scale) as the four bytes of a 32-bit fraction of about the largest weight so far
// (2^-30 of it at most; not of the largest V scale, which may have no weight at all: a block 1000 times as large
// cost a row 4e-4 of its output so, and thousands of keys of 2^-25 each were lost with the three bytes of 23 bits);
// each digit is a column of its own in m16n8k32 products whose other operand is the cache's bytes:
// K as it is, V with its 4 x 4 bytes transposed in registers. Two query rows fill eight columns
// (q's fourth is not looked at), and sums are exact, so 32 tokens take 16 products
// and no conversion, against 64 and 350 conversions in f16.
// Step kernel (few query rows, more than four): the f16 tiles above.
// In both, one cluster per (KV head, row tile, sequence); its CTAs split the sequence's actual
// length, their warps take tiles in turn, each with its own ring of asynchronous copies and its own
// softmax state. States are merged in warp order, then in rank order over distributed shared
// memory: no workspace, no atomics, the same bits every time.
// More than 64 rows a KV head take the tcgen05 kernel of ops_kv8_prompt.cu.
//
// Bound: DRAM (the cache is read once per KV head and row tile) or, for short lengths, latency.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bulk.cuh"
#include "dev_util.cuh"
#include "ops.h"

namespace qasr {
namespace {

constexpr int kTok = kKv8Block;  // tokens of a tile
constexpr int kStepRows = 64;    // query rows of a KV head up to which its length is split
constexpr float kNone = -3.4028235e38f;  // running maximum before any key (finite: differences stay defined)

struct AttnArgs {
  Kv8 c;
  const void* q;
  void* out;
  long long q_seq, q_row, o_seq, o_row;
  const int *starts, *counts;
  int idx_stride, rows, heads, group, row_tiles;
  float scale;
  int vec;            // q rows start on 16-byte boundaries
  int longest_first;  // more CTAs than run at once
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_zero(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// Two bytes of w (already x + 128) as f16 values x.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t bytes_f16(uint32_t w) {
  const uint32_t p = __byte_perm(w, 0x64646464u, SEL);  // 1024 + byte
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&p), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return pack_f16(a - f.x, b - f.y);
}

// Shared-memory tile: 16 tokens of HD bytes, K then V then the two scales. 16-byte chunks are
// permuted within a row so that the fragment loads hit distinct banks.
template <int HD>
struct Tile {
  static constexpr int kChunks = HD / 16;
  static constexpr int kBytes = 2 * kTok * HD + 16;
  __device__ static uint32_t k_at(int row, int chunk) {
    return row * HD + (HD == 128 ? (chunk ^ ((row & 1) << 2)) : chunk) * 16;
  }
  __device__ static uint32_t v_at(int row, int chunk) {
    return kTok * HD + row * HD + (HD == 128 ? chunk ^ (((row >> 1) & 3) << 1) : chunk ^ ((row >> 1) & 3)) * 16;
  }
  // One tile's copies by `n` threads (n a multiple of 32, i the thread's index among them).
  __device__ static void fetch(uint32_t st, const int8_t* k, const int8_t* v, const float* ks, const float* vs,
                               int tile, int i, int n) {
    const long long off = (long long)tile * kTok * HD;
    for (int c = i; c < kTok * kChunks; c += n) {
      const int row = c / kChunks, ch = c % kChunks;
      cp16(st + k_at(row, ch), k + off + row * HD + ch * 16);
      cp16(st + v_at(row, ch), v + off + row * HD + ch * 16);
    }
    if (i == 0) cp4(st + 2 * kTok * HD, ks + tile);
    if (i == 1) cp4(st + 2 * kTok * HD + 4, vs + tile);
  }
};

// One warp's query rows and softmax state. PL planes (2: f32 accuracy, 8 rows; 1: 16 rows).
template <int HD, int PL>
struct WarpState {
  static constexpr int kRows = PL == 2 ? 8 : 16;
  static constexpr int kR = PL == 2 ? 1 : 2;    // rows a thread holds: g (and g + 8)
  static constexpr int kSteps = HD / 16;        // k steps of the score product
  static constexpr int kNt = HD / 8;            // column tiles of the output
  uint32_t q[kSteps][4];
  float fac[kR];   // scale * log2(e) * the row's power of two
  int last[kR];    // last position the row sees (-1: none)
  float m[kR], l[kR];
  float acc[kNt][2 * kR];

  // dims of k step j that thread t of a quad holds: 4 from here
  __device__ static int dim0(int t, int j) { return (j & 3) * 4 + t * 16 + (j >> 2) * 64; }
  // output dims of column tile j: column n is dim n * kNt + j
  __device__ static int out_dim(int n, int j) { return n * kNt + j; }

  __device__ void init(const AttnArgs& a, int seq, int kvh, int row0, int start, int count, bool bf16) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < kNt; ++j)
#pragma unroll
      for (int i = 0; i < 2 * kR; ++i) acc[j][i] = 0.f;
#pragma unroll
    for (int h = 0; h < kR; ++h) {
      const int rr = row0 + g + h * 8, s = rr / a.group;
      const bool live = s < count;  // rows past the operand too: count <= rows
      last[h] = live ? min(start + s, a.c.capacity - 1) : -1;
      m[h] = kNone;
      l[h] = 0.f;
      float f[kSteps][4];
      float mx = 0.f;
      const long long off =
          seq * a.q_seq + (long long)s * a.q_row + (long long)(kvh * a.group + rr % a.group) * HD;
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[j][i] = 0.f;
          if (live) {
            const long long at = off + dim0(t, j) + i;
            f[j][i] = bf16 ? __bfloat162float(((const __nv_bfloat16*)a.q)[at]) : ((const float*)a.q)[at];
          }
          mx = fmaxf(mx, fabsf(f[j][i]));
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      int e = 0;
      if (mx > 0.f && mx < __int_as_float(0x7F800000)) frexpf(mx, &e);
      // 2^-e and 2^e as two exact factors each (one alone can leave f32's normal range)
      const int e1 = e / 2, e2 = e - e1;
      const float d1 = __int_as_float((127 - e1) << 23), d2 = __int_as_float((127 - e2) << 23);
      fac[h] = a.scale * 1.4426950408889634f * __int_as_float((127 + e1) << 23) * __int_as_float((127 + e2) << 23);
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[j][i] = f[j][i] * d1 * d2;
        const uint32_t h0 = pack_f16(f[j][0], f[j][1]), h1 = pack_f16(f[j][2], f[j][3]);
        q[j][h] = h0;
        q[j][2 + h] = h1;
        if (PL == 2) {
          q[j][1] = pack_rest(f[j][0], f[j][1], h0);
          q[j][3] = pack_rest(f[j][2], f[j][3], h1);
        }
      }
    }
  }

  // One tile of 16 tokens from position pos0, staged at st.
  __device__ void tile(const unsigned char* st, int pos0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const float ks = *reinterpret_cast<const float*>(st + 2 * kTok * HD);
    const float vs = *reinterpret_cast<const float*>(st + 2 * kTok * HD + 4);
    float vr[kR];
    float s[2][4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] = 0.f;
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        const uint4 w4 = *reinterpret_cast<const uint4*>(st + Tile<HD>::k_at(nt * 8 + g, t + 4 * c));
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u = w[i] ^ 0x80808080u;
          mma16816(s[nt], q[c * 4 + i], bytes_f16<0x4140>(u), bytes_f16<0x4342>(u));
        }
      }
    }
    // scores of row g (+ 8h) at tokens nt * 8 + 2t + {0, 1}, in units of log2
    uint32_t p[4];
    bool grew = false;
    float corr[kR];
#pragma unroll
    for (int h = 0; h < kR; ++h) {
      float x[4];
      const float f = fac[h] * ks;
      float mx = kNone;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int nt = i >> 1, o = i & 1;
        const float sum = PL == 2 ? s[nt][o] + s[nt][2 + o] : s[nt][2 * h + o];
        x[i] = pos0 + nt * 8 + 2 * t + o <= last[h] ? __fmul_rn(sum, f) : -__int_as_float(0x7F800000);
        mx = fmaxf(mx, x[i]);
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[h], mx);
      corr[h] = ex2(m[h] - mn);
      grew |= mn > m[h];
      m[h] = mn;
      const float part = ex2(mx - mn);  // the tile's largest
      // a row that sees nothing of the tile takes nothing of its scale either (it may be NaN)
      vr[h] = pos0 <= last[h] ? vs * part : 0.f;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = ex2(x[i] - mx + 15.f);
        sum += x[i];
      }
      l[h] = fmaf(sum, part, l[h] * corr[h]);
      p[h] = pack_f16(x[0], x[1]);
      p[2 + h] = pack_f16(x[2], x[3]);
      if (PL == 2) {
        p[1] = pack_rest(x[0], x[1], p[0]);
        p[3] = pack_rest(x[2], x[3], p[2]);
      }
    }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int j = 0; j < kNt; ++j)
#pragma unroll
        for (int i = 0; i < 2 * kR; ++i) acc[j][i] *= corr[i >> 1];
    }
    // V: tokens 2t, 2t + 1 and 2t + 8, 2t + 9, kNt dims from g * kNt
    constexpr int W = kNt / 4;  // words a thread takes of a token
    uint32_t v[4][W];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 2 * t + (r & 1) + (r >> 1) * 8;
      if constexpr (HD == 128) {
        const uint4 w = *reinterpret_cast<const uint4*>(st + Tile<HD>::v_at(row, g));
        v[r][0] = w.x; v[r][1] = w.y; v[r][2] = w.z; v[r][3] = w.w;
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(st + Tile<HD>::v_at(row, g >> 1) + (g & 1) * 8);
        v[r][0] = w.x; v[r][1] = w.y;
      }
#pragma unroll
      for (int i = 0; i < W; ++i) v[r][i] ^= 0x80808080u;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const uint32_t a0 = __byte_perm(v[0][i], v[1][i], 0x5140), a1 = __byte_perm(v[0][i], v[1][i], 0x7362);
      const uint32_t b0 = __byte_perm(v[2][i], v[3][i], 0x5140), b1 = __byte_perm(v[2][i], v[3][i], 0x7362);
      const uint32_t lo[4] = {bytes_f16<0x4140>(a0), bytes_f16<0x4342>(a0), bytes_f16<0x4140>(a1),
                              bytes_f16<0x4342>(a1)};
      const uint32_t hi[4] = {bytes_f16<0x4140>(b0), bytes_f16<0x4342>(b0), bytes_f16<0x4140>(b1),
                              bytes_f16<0x4342>(b1)};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float o[4];
        mma16816_zero(o, p, lo[k], hi[k]);
        float* d = acc[i * 4 + k];
        if (PL == 2) {
          d[0] = fmaf(o[0] + o[2], vr[0], d[0]);
          d[1] = fmaf(o[1] + o[3], vr[0], d[1]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) d[e % (2 * kR)] = fmaf(o[e], vr[(e >> 1) % kR], d[e % (2 * kR)]);
        }
      }
    }
  }

  __device__ void finish_sum() {
#pragma unroll
    for (int h = 0; h < kR; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
  }
};

__device__ __forceinline__ void put(void* out, long long i, float v, bool bf16) {
  if (bf16)
    ((__nv_bfloat16*)out)[i] = __float2bfloat16_rn(v);
  else
    ((float*)out)[i] = v;
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_peer(uint32_t addr, int rank) {
  uint32_t r;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
  return v;
}

// A sequence's first position (at most the capacity) and live rows.
__device__ __forceinline__ void rows_of(const AttnArgs& a, int seq, int& start, int& count) {
  start = a.starts[(long long)seq * a.idx_stride];
  count = a.rows;
  if (a.counts) count = min(max(a.counts[(long long)seq * a.idx_stride], 0), a.rows);
  if (start < 0) count = 0;
  start = min(start, a.c.capacity);
}

// The CTA's sequence and its rows: a kernel's first reads. Where not all CTAs run at once, the longest of
// every 32 sequences go first, so that none of them is left for the end (32 sequences of 0 to 8191 tokens in
// ascending order: 61 us as they come, 50 so). All 32 lanes call it.
__device__ __forceinline__ int live_rows(const AttnArgs& a, int& start, int& count) {
  pdl_launch_dependents();
  pdl_wait();
  int seq = blockIdx.z;
  if (a.longest_first) {
    const int lane = threadIdx.x & 31, base = seq & ~31, i = base + lane;
    int len = -1;
    if (i < a.c.n_seq) {
      rows_of(a, i, start, count);
      len = count > 0 ? start + count : 0;
    }
    int rank = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const int other = __shfl_sync(0xffffffffu, len, j);
      rank += other > len || (other == len && j < lane);
    }
    const unsigned mine = __ballot_sync(0xffffffffu, rank == (seq & 31));  // (one lane)
    seq = base + __ffs((int)mine) - 1;
  }
  rows_of(a, seq, start, count);
  return seq;
}

// ------------------------------------------------------------------ step kernel
constexpr int kStepWarps = 4, kStepStages = 4;
template <int HD>
constexpr int step_smem() {
  return kStepWarps * kStepStages * Tile<HD>::kBytes;
}

// grid (splits, n_kv * row_tiles, n_seq), cluster (splits, 1, 1)
template <int HD, int PL>
__global__ void __launch_bounds__(kStepWarps * 32) step_kernel(const AttnArgs a) {
  using S = WarpState<HD, PL>;
  constexpr int R = S::kRows;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float wm[kStepWarps][R], wl[kStepWarps][R], cm[R], cl[R];
  __shared__ float part[R][HD];  // the CTA's merged output
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int splits = gridDim.x, rank = blockIdx.x;
  const int kvh = blockIdx.y / a.row_tiles, row0 = (blockIdx.y % a.row_tiles) * R;
  int start, count;
  const int seq = live_rows(a, start, count);
  // tokens any row of the tile sees
  const int s_last = min(count - 1, (row0 + R - 1) / a.group);
  const int len = s_last >= row0 / a.group ? (int)min((long long)start + s_last + 1, (long long)a.c.capacity) : 0;
  const int tiles = (len + kTok - 1) / kTok;
  const int t0 = (int)((long long)tiles * rank / splits), t1 = (int)((long long)tiles * (rank + 1) / splits);

  const long long blocks = a.c.capacity / kTok;
  const int8_t* k = a.c.k + seq * a.c.seq_stride + (long long)kvh * a.c.capacity * HD;
  const int8_t* v = a.c.v + seq * a.c.seq_stride + (long long)kvh * a.c.capacity * HD;
  const float* ks = a.c.ks + seq * a.c.scale_stride + kvh * blocks;
  const float* vs = a.c.vs + seq * a.c.scale_stride + kvh * blocks;
  unsigned char* ring = smem + warp * kStepStages * Tile<HD>::kBytes;
  const uint32_t ring_a = smem_u32(ring);
  const int mine = t1 - t0 > warp ? (t1 - t0 - warp + kStepWarps - 1) / kStepWarps : 0;
#pragma unroll
  for (int i = 0; i < kStepStages - 1; ++i) {
    if (i < mine) Tile<HD>::fetch(ring_a + i * Tile<HD>::kBytes, k, v, ks, vs, t0 + warp + i * kStepWarps, lane, 32);
    cp_commit();
  }
  S st;
  st.init(a, seq, kvh, row0, start, count, PL == 1);
  for (int i = 0; i < mine; ++i) {
    const int nx = i + kStepStages - 1;
    if (nx < mine)
      Tile<HD>::fetch(ring_a + nx % kStepStages * Tile<HD>::kBytes, k, v, ks, vs, t0 + warp + nx * kStepWarps, lane, 32);
    cp_commit();
    cp_wait<kStepStages - 1>();
    __syncwarp();
    st.tile(ring + i % kStepStages * Tile<HD>::kBytes, (t0 + warp + i * kStepWarps) * kTok);
    __syncwarp();
  }
  cp_wait<0>();
  st.finish_sum();
  __syncthreads();  // every ring is idle: it holds the warps' outputs now
  float* wo = reinterpret_cast<float*>(smem);  // [warp][R][HD]
  static_assert(kStepWarps * R * HD * 4 <= step_smem<HD>(), "the warps' outputs reuse the rings");
#pragma unroll
  for (int h = 0; h < S::kR; ++h) {
    const int r = g + h * 8;
    if (t == 0) {
      wm[warp][r] = st.m[h];
      wl[warp][r] = st.l[h];
    }
#pragma unroll
    for (int j = 0; j < S::kNt; ++j) {
      wo[(warp * R + r) * HD + S::out_dim(2 * t, j)] = st.acc[j][2 * h];
      wo[(warp * R + r) * HD + S::out_dim(2 * t + 1, j)] = st.acc[j][2 * h + 1];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * HD; i += kStepWarps * 32) {
    const int r = i / HD, d = i % HD;
    float mm = wm[0][r], ll = 0.f, o = 0.f;
#pragma unroll
    for (int w = 1; w < kStepWarps; ++w) mm = fmaxf(mm, wm[w][r]);
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) {
      const float f = ex2(wm[w][r] - mm);
      ll = fmaf(wl[w][r], f, ll);
      o = fmaf(wo[(w * R + r) * HD + d], f, o);
    }
    part[r][d] = o;
    if (d == 0) {
      cm[r] = mm;
      cl[r] = ll;
    }
  }
  if (splits > 1)
    cluster_barrier();
  else
    __syncthreads();
  const int n_rows = a.rows * a.group;
  for (int i = rank * kStepWarps * 32 + threadIdx.x; i < R * HD; i += splits * kStepWarps * 32) {
    const int r = i / HD, d = i % HD, rr = row0 + r;
    if (rr >= n_rows) continue;
    float ll, o;
    if (splits > 1) {
      float mm = kNone;
      for (int p = 0; p < splits; ++p) mm = fmaxf(mm, ld_peer(smem_u32(&cm[r]), p));
      ll = 0.f;
      o = 0.f;
      for (int p = 0; p < splits; ++p) {
        const float f = ex2(ld_peer(smem_u32(&cm[r]), p) - mm);
        ll = fmaf(ld_peer(smem_u32(&cl[r]), p), f, ll);
        o = fmaf(ld_peer(smem_u32(&part[r][d]), p), f, o);
      }
    } else {
      ll = cl[r];
      o = part[r][d];
    }
    const float inv = ll == 0.f ? 0.f : __fdiv_rn(1.0f, ll);
    put(a.out, seq * a.o_seq + (long long)(rr / a.group) * a.o_row + (long long)(kvh * a.group + rr % a.group) * HD + d,
        __fmul_rn(o, inv), PL == 1);
  }
  __syncwarp();
  if (splits > 1) cluster_barrier();  // no CTA leaves while a peer reads its part
}

// 16 consecutive values of a query row.
template <bool BF16>
__device__ __forceinline__ void load16(const AttnArgs& a, long long at, float* f) {
  if constexpr (BF16) {
    const __nv_bfloat16* p = (const __nv_bfloat16*)a.q + at;
    if (a.vec) {
      bf16x8_to_f32(*reinterpret_cast<const uint4*>(p), f);
      bf16x8_to_f32(*reinterpret_cast<const uint4*>(p + 8), f + 8);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = __bfloat162float(p[i]);
    }
  } else {
    const float* p = (const float*)a.q + at;
    if (a.vec) {
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(p + i);
        f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = p[i];
    }
  }
}

// ------------------------------------------------------------------ digit kernel
constexpr int kMaxSplits = 16;  // CTAs of a cluster (more than 8 need the kernel's leave)
constexpr int kDigWarps = 4, kDigStages = 3;  // 32 tokens (two tiles) a step
constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: float of a small int sum

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN when either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// D = A B + C; with C = 1.5 * 2^23 as bits at first, D is the sum as a float, exact below 2^22
// (128 dims * 127 * 128).
__device__ __forceinline__ void mma_s8(int* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8u8(int* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A unit in shared memory: two tiles' K, their V (16 tokens each, chunks permuted as in Tile), k scales, v scales.
template <int HD>
struct Unit {
  static constexpr int kTile = kTok * HD;
  static constexpr int kBytes = 4 * kTile + 16;
  static constexpr int kIter = kTile / 512;  // 16-byte copies of a lane for one tile of K or V
  // This lane's copies go to fixed places: byte lane * 16 + 512 i of a tile is row (lane * 16 + 512 i) / HD.
  static __device__ void fetch(uint32_t st, const int8_t* k, const int8_t* v, const float* ks, const float* vs,
                               int tile, int tiles, int lane) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (tile + h >= tiles) break;
      const long long off = (long long)(tile + h) * kTile + lane * 16;
#pragma unroll
      for (int i = 0; i < kIter; ++i) {
        const int row = i * (512 / HD) + lane / (HD / 16), ch = lane % (HD / 16);
        cp16(st + h * kTile + Tile<HD>::k_at(row, ch), k + off + i * 512);
        cp16(st + 2 * kTile + h * kTile + (Tile<HD>::v_at(row, ch) - kTok * HD), v + off + i * 512);
      }
      if (lane == 0) cp4(st + 4 * kTile + h * 4, ks + tile + h);
      if (lane == 1) cp4(st + 4 * kTile + 8 + h * 4, vs + tile + h);
    }
  }
};

// grid (splits, n_kv * row_tiles, n_seq), cluster (splits, 1, 1). RH: pairs of query rows. As operand
// column, lane (g, t) holds digit g % 4 of row g / 4 of a pair; as result, columns 2t and 2t + 1, so
// digits 0, 1 (t even) or 2, 3 of row t / 2, whose softmax state it keeps.
template <int HD, int RH, bool BF16>
__global__ void __launch_bounds__(kDigWarps * 32, RH == 1 ? 3 : 2) digit_kernel(const AttnArgs a) {
  constexpr int R = 2 * RH, kNt = HD / 8, kMt = HD / 16, kSteps = HD / 32, kWords = HD / 16;
  using U = Unit<HD>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float wm[kDigWarps][R], wl[kDigWarps][R], cm[R], cl[R];
  __shared__ float part[R][HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int splits = gridDim.x, rank = blockIdx.x;
  const int kvh = blockIdx.y / a.row_tiles, row0 = (blockIdx.y % a.row_tiles) * R;
  int start, count;
  const int seq = live_rows(a, start, count);
  const int s_last = min(count - 1, (row0 + R - 1) / a.group);
  const int len = s_last >= row0 / a.group ? (int)min((long long)start + s_last + 1, (long long)a.c.capacity) : 0;
  const int tiles = (len + kTok - 1) / kTok, units = (tiles + 1) / 2;
  const int u0 = (int)((long long)units * rank / splits), u1 = (int)((long long)units * (rank + 1) / splits);
  const long long blocks = a.c.capacity / kTok;
  const int8_t* k = a.c.k + seq * a.c.seq_stride + (long long)kvh * a.c.capacity * HD;
  const int8_t* v = a.c.v + seq * a.c.seq_stride + (long long)kvh * a.c.capacity * HD;
  const float* ks = a.c.ks + seq * a.c.scale_stride + kvh * blocks;
  const float* vs = a.c.vs + seq * a.c.scale_stride + kvh * blocks;
  unsigned char* ring = smem + warp * kDigStages * U::kBytes;
  const uint32_t ring_a = smem_u32(ring);
  const int mine = u1 - u0 > warp ? (u1 - u0 - warp + kDigWarps - 1) / kDigWarps : 0;
#pragma unroll
  for (int i = 0; i < kDigStages - 1; ++i) {
    if (i < mine) U::fetch(ring_a + i * U::kBytes, k, v, ks, vs, 2 * (u0 + warp + i * kDigWarps), tiles, lane);
    cp_commit();
  }

  const int plane = g & 3, hrow = t >> 1;
  uint32_t q[RH][kSteps][2];
  float fac[RH], m[RH], l[RH], top[RH], vref[RH], rv[RH];
  int last[RH];
  int all_see = 0x7FFFFFFF;  // every row of the warp sees up to here
#pragma unroll
  for (int h = 0; h < RH; ++h) {
    const int rr = row0 + 2 * h + (g >> 2), s = rr / a.group;
    const bool live = s < count;
    float f[kWords / 4][16];  // 16 dims from t * 16 (+ 64)
    float mx = 0.f;
    const long long off = seq * a.q_seq + (long long)s * a.q_row + (long long)(kvh * a.group + rr % a.group) * HD;
#pragma unroll
    for (int c = 0; c < kWords / 4; ++c) {
#pragma unroll
      for (int i = 0; i < 16; ++i) f[c][i] = 0.f;
      if (live) load16<BF16>(a, off + c * 64 + t * 16, f[c]);
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = max_nan(mx, fabsf(f[c][i]));
    }
    mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    constexpr float kTop = 127.f * 16384.f;
    const bool fine = mx > 0.f && mx < __int_as_float(0x7F800000);
    const float factor =
        mx == 0.f ? 0.f : fine ? mx * (fabsf(a.scale) * (1.4426950408889634f / kTop)) : __int_as_float(0x7FFFFFFF);
    fac[h] = __shfl_sync(0xffffffffu, factor, 16 * hrow);
    const float up = mx < 1e-30f ? 1.2676506e30f : 1.f;  // 2^100: kTop / mx stays finite
    const float inv = fine ? copysignf(__fdiv_rn(kTop, mx * up), a.scale) : 0.f;  // (the factor is positive)
    // (z + 64 + 64 * 128) >> 14, >> 7, >> 0: the lower digits with 64 added
    const int sh = plane == 0 ? 14 : plane == 1 ? 7 : 0, mask = plane == 0 ? -1 : 127, less = plane == 0 ? 0 : 64;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      uint32_t word = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int z = fine ? __float2int_rn(f[w >> 2][(w & 3) * 4 + i] * up * inv) : 0;
        const int d = (((z + 64 + 64 * 128) >> sh) & mask) - less;
        word |= ((uint32_t)d & 0xFFu) << (8 * i);
      }
      q[h][w >> 1][w & 1] = word;
    }
    const int sr = (row0 + 2 * h + hrow) / a.group;  // the row whose scores this lane gets
    last[h] = sr < count ? min(start + sr, a.c.capacity - 1) : -1;
    all_see = min(all_see, last[h]);
    m[h] = kNone;
    l[h] = top[h] = vref[h] = rv[h] = 0.f;
  }
  all_see = __reduce_min_sync(0xffffffffu, all_see);
  // weights of this lane's two result columns, for the scores and for the output
  const float wa = t & 1 ? 1.f : 16384.f, wb = t & 1 ? 0.f : 128.f, ba = -kMagic * wa, bb = -kMagic * wb;
  const float oa = t & 1 ? 0x1p-24f : 0x1p-8f, ob = t & 1 ? 0x1p-32f : 0x1p-16f;
  // the weights' bytes this lane hands out: digits 0 and 2 (t even), or 1 and 3
  const uint32_t sel = t & 1 ? 0x0062u : 0x0073u, sel2 = t & 1 ? 0x0040u : 0x0051u;
  const int from = 8 * t + 2 * (g >> 2) + (plane & 1);  // tokens 2t: lane (2t, 2 row + digit's parity)

  // The output so far is sum * vref / 2^32 + acc: integer sums for the present maximum m and the
  // power of two vref above the largest weight (about `top`), f32 for what came before they last grew. So a
  // step of 32 tokens neither converts nor rescales anything, unless its maximum or a weight is a new record.
  int sum[RH][kMt][4];
  float acc[RH][kMt][2];
#pragma unroll
  for (int h = 0; h < RH; ++h)
#pragma unroll
    for (int j = 0; j < kMt; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[h][j][i] = 0;
      acc[h][j][0] = acc[h][j][1] = 0.f;
    }
  int since = 0;  // steps since the sums were emptied (2072 of 32 * 255 * 127 fit 31 bits)

  for (int i = 0; i < mine; ++i) {
    const int nx = i + kDigStages - 1;
    if (nx < mine)
      U::fetch(ring_a + nx % kDigStages * U::kBytes, k, v, ks, vs, 2 * (u0 + warp + nx * kDigWarps), tiles, lane);
    cp_commit();
    cp_wait<kDigStages - 1>();
    __syncwarp();
    const unsigned char* st = ring + i % kDigStages * U::kBytes;
    const int pos0 = 2 * (u0 + warp + i * kDigWarps) * kTok;
    const float4 sc = *reinterpret_cast<const float4*>(st + 4 * U::kTile);  // ks, ks, vs, vs
    // ---- scores x[h][e]: token (e / 2) * 16 + (e % 2) * 8 + g
    float x[RH][4];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      uint32_t w[2][kWords];
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < kWords / 4; ++c) {
          const uint4 w4 = *reinterpret_cast<const uint4*>(st + b * U::kTile + Tile<HD>::k_at(r * 8 + g, t + 4 * c));
          w[r][4 * c] = w4.x; w[r][4 * c + 1] = w4.y; w[r][4 * c + 2] = w4.z; w[r][4 * c + 3] = w4.w;
        }
#pragma unroll
      for (int h = 0; h < RH; ++h) {
        int d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = __float_as_int(kMagic);
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
          mma_s8(d, w[0][2 * j], w[1][2 * j], w[0][2 * j + 1], w[1][2 * j + 1], q[h][j][0], q[h][j][1]);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          // (both products are exact)
          const float y = fmaf(__int_as_float(d[2 * r]), wa, ba) + fmaf(__int_as_float(d[2 * r + 1]), wb, bb);
          x[h][2 * b + r] = y + __shfl_xor_sync(0xffffffffu, y, 1);
        }
      }
    }
    // ---- softmax state
    const bool partial = pos0 + 2 * kTok - 1 > all_see;
    float v0[RH], v1[RH], mx[RH], most[RH];
    bool grew = ++since > 2048;
    // the step's largest weight, within 4 times: its largest probability times its larger V scale, unless these are
    // further apart
    const bool apart = !(fmaxf(sc.z, sc.w) <= 4.f * fminf(sc.z, sc.w));
#pragma unroll
    for (int h = 0; h < RH; ++h) {
      // a block that the row sees nothing of gives it nothing of its scales either (they may be NaN)
      const bool see0 = pos0 <= last[h], see1 = pos0 + kTok <= last[h];
      const float f0 = see0 ? fac[h] * sc.x : 0.f, f1 = see1 ? fac[h] * sc.y : 0.f;
      v0[h] = see0 ? sc.z : 0.f;
      v1[h] = see1 ? sc.w : 0.f;
      float t0 = kNone, t1 = kNone;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // (rounded before the maximum is taken off, as that was: of scores of any size its own difference is 0)
        x[h][e] = __fmul_rn(x[h][e], e < 2 ? f0 : f1);
        if (!partial || pos0 + (e >> 1) * 16 + (e & 1) * 8 + g <= last[h]) {
          if (e < 2) t0 = fmaxf(t0, x[h][e]);
          else t1 = fmaxf(t1, x[h][e]);
        }
      }
      mx[h] = fmaxf(t0, t1);
#pragma unroll
      for (int o = 4; o < 32; o *= 2) mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], o));
      const float mn = fmaxf(m[h], mx[h]);
      // (2^-80 at least, so that rv times a V scale stays finite)
      if (apart) {
#pragma unroll
        for (int o = 4; o < 32; o *= 2) {
          t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o));
          t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o));
        }
        most[h] = max_nan(ex2(fmaxf(t0 - mn, -80.f)) * v0[h], ex2(fmaxf(t1 - mn, -80.f)) * v1[h]);
      } else {
        most[h] = ex2(fmaxf(mx[h] - mn, -80.f)) * max_nan(v0[h], v1[h]);
      }
      grew |= mx[h] > m[h] || !(most[h] <= vref[h]);
    }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int h = 0; h < RH; ++h) {
        const float mn = fmaxf(m[h], mx[h]), corr = ex2(m[h] - mn);
#pragma unroll
        for (int j = 0; j < kMt; ++j)
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const float y = fmaf((float)sum[h][j][2 * o], oa, (float)sum[h][j][2 * o + 1] * ob);
            acc[h][j][o] = fmaf(y, vref[h], acc[h][j][o]) * corr;
            sum[h][j][2 * o] = sum[h][j][2 * o + 1] = 0;
          }
        l[h] *= corr;
        m[h] = mn;
        // the weights so far count less where the maximum grew; the power of two above them (2^-120 at least), or NaN
        const float w = top[h] = max_nan(top[h] * corr, most[h]);
        vref[h] = w > 0.f ? fmaxf(__uint_as_float((__float_as_uint(w) + 0x7FFFFFu) & 0xFF800000u), 0x1p-120f) : w;
        rv[h] = vref[h] > 0.f ? __fdiv_rn(1.f, vref[h]) : 0.f;
      }
      since = 0;
    }
    // ---- weights as bytes: column (row g / 4, digit g % 4) of tokens 2t, 2t + 1, 2t + 8, 2t + 9 a tile
    uint32_t pb[RH][2];
#pragma unroll
    for (int h = 0; h < RH; ++h) {
      const float r0 = v0[h] * rv[h] * 0x1p32f, r1 = v1[h] * rv[h] * 0x1p32f;
      uint32_t z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float p = ex2(x[h][e] - m[h]);
        // (not by the score: a masked one times a zero scale is no number)
        if (partial && pos0 + (e >> 1) * 16 + (e & 1) * 8 + g > last[h]) p = 0.f;
        l[h] += p;
        z[e] = __float2uint_rn(p * (e < 2 ? r0 : r1));  // (saturates: 1 becomes 1 - 2^-32)
      }
      const uint32_t first = __byte_perm(__byte_perm(z[0], z[1], sel), __byte_perm(z[2], z[3], sel), 0x5410);
      const uint32_t second = __byte_perm(__byte_perm(z[0], z[1], sel2), __byte_perm(z[2], z[3], sel2), 0x5410);
      const uint32_t a0 = __shfl_sync(0xffffffffu, first, from), a1 = __shfl_sync(0xffffffffu, first, from + 4);
      const uint32_t c0 = __shfl_sync(0xffffffffu, second, from), c1 = __shfl_sync(0xffffffffu, second, from + 4);
      const uint32_t w0 = plane >= 2 ? c0 : a0, w1 = plane >= 2 ? c1 : a1;
      pb[h][0] = __byte_perm(w0, w1, 0x5140);
      pb[h][1] = __byte_perm(w0, w1, 0x7362);
    }
    // ---- V: per tile the same tokens, kNt dims from g * kNt, four at a time
    constexpr int W = kNt / 4;
    uint32_t vb[2][W][4];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      uint32_t r[4][W];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 2 * t + (e & 1) + (e >> 1) * 8;
        const unsigned char* p = st + 2 * U::kTile + b * U::kTile - kTok * HD;
        if constexpr (HD == 128) {
          const uint4 w = *reinterpret_cast<const uint4*>(p + Tile<HD>::v_at(row, g));
          r[e][0] = w.x; r[e][1] = w.y; r[e][2] = w.z; r[e][3] = w.w;
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(p + Tile<HD>::v_at(row, g >> 1) + (g & 1) * 8);
          r[e][0] = w.x; r[e][1] = w.y;
        }
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t x0 = __byte_perm(r[0][w], r[1][w], 0x5140), x1 = __byte_perm(r[0][w], r[1][w], 0x7362);
        const uint32_t y0 = __byte_perm(r[2][w], r[3][w], 0x5140), y1 = __byte_perm(r[2][w], r[3][w], 0x7362);
        vb[b][w][0] = __byte_perm(x0, y0, 0x5410);
        vb[b][w][1] = __byte_perm(x0, y0, 0x7632);
        vb[b][w][2] = __byte_perm(x1, y1, 0x5410);
        vb[b][w][3] = __byte_perm(x1, y1, 0x7632);
      }
    }
    // rows g and g + 8 of product j: dims g * kNt + 2j and + 2j + 1
#pragma unroll
    for (int j = 0; j < kMt; ++j) {
      const int e0 = 2 * j, e1 = 2 * j + 1;
#pragma unroll
      for (int h = 0; h < RH; ++h)
        mma_s8u8(sum[h][j], vb[0][e0 >> 2][e0 & 3], vb[0][e1 >> 2][e1 & 3], vb[1][e0 >> 2][e0 & 3],
                 vb[1][e1 >> 2][e1 & 3], pb[h][0], pb[h][1]);
    }
    __syncwarp();
  }
  cp_wait<0>();

  // ---- the digits' sums joined, then the warps' states, then the cluster's
  __syncthreads();  // every ring is idle: it holds the warps' outputs now
  float* wo = reinterpret_cast<float*>(smem);  // [warp][R][HD]
  static_assert(kDigWarps * R * HD * 4 <= kDigWarps * kDigStages * U::kBytes, "the warps' outputs reuse the rings");
#pragma unroll
  for (int h = 0; h < RH; ++h) {
#pragma unroll
    for (int o = 4; o < 32; o *= 2) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
    const int r = 2 * h + hrow;
    if (g == 0 && !(t & 1)) {
      wm[warp][r] = m[h];
      wl[warp][r] = l[h];
    }
#pragma unroll
    for (int j = 0; j < kMt; ++j) {
      float y[2];
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        y[o] = fmaf((float)sum[h][j][2 * o], oa, (float)sum[h][j][2 * o + 1] * ob);
        y[o] = fmaf(y[o], vref[h], acc[h][j][o]);
        y[o] += __shfl_xor_sync(0xffffffffu, y[o], 1);
      }
      wo[(warp * R + r) * HD + g * kNt + 2 * j + (t & 1)] = t & 1 ? y[1] : y[0];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * HD; i += kDigWarps * 32) {
    const int r = i / HD, d = i % HD;
    float mm = wm[0][r], ll = 0.f, o = 0.f;
#pragma unroll
    for (int w = 1; w < kDigWarps; ++w) mm = fmaxf(mm, wm[w][r]);
#pragma unroll
    for (int w = 0; w < kDigWarps; ++w) {
      const float f = ex2(wm[w][r] - mm);
      ll = fmaf(wl[w][r], f, ll);
      o = fmaf(wo[(w * R + r) * HD + d], f, o);
    }
    part[r][d] = o;
    if (d == 0) {
      cm[r] = mm;
      cl[r] = ll;
    }
  }
  if (splits > 1)
    cluster_barrier();
  else
    __syncthreads();
  // warp r finishes query row r, this CTA a share of its dims: the peers' (max, sum) in the lanes
  const int rr = row0 + warp;
  if (warp < R && rr < a.rows * a.group) {
    const bool peer = lane < splits;
    const float pm = peer ? ld_peer(smem_u32(&cm[warp]), lane) : kNone;
    const float pl = peer ? ld_peer(smem_u32(&cl[warp]), lane) : 0.f;
    const float mm = warp_max(pm);
    float f = ex2(pm - mm);
    const float ll = warp_sum(pl * f);
    f = ll == 0.f ? 0.f : __fdiv_rn(f, ll);
    const int share = HD / splits;
    for (int d0 = 0; d0 < share; d0 += 32) {
      const int d = rank * share + d0 + lane;
      const bool in = d0 + lane < share;
      float o = 0.f;
#pragma unroll
      for (int p = 0; p < kMaxSplits; ++p) {
        if (p >= splits) break;
        const float y = in ? ld_peer(smem_u32(&part[warp][d]), p) : 0.f;
        o = fmaf(y, __shfl_sync(0xffffffffu, f, p), o);
      }
      if (in)
        put(a.out,
            seq * a.o_seq + (long long)(rr / a.group) * a.o_row + (long long)(kvh * a.group + rr % a.group) * HD + d, o,
            BF16);
    }
  }
  __syncwarp();
  if (splits > 1) cluster_barrier();  // no CTA leaves while a peer reads its part
}

// CTAs that share a sequence's length, for `ctas` CTAs unsplit: powers of two while all of them run
// at once (two an SM; one an SM for 16, which wait long for room) and each keeps 256 tokens; between one and
// two CTAs an SM two where sequences may be long, because lengths differ. 16 query heads on 8 x 128, measured
// (us) at 1 / 2 / 4 / 8 / 16 splits: 8 CTAs of 436 tokens 7.6 / 6.6 / 5.8 / 6.4 / 8.2; 8 of 8000 53 / 30 / 18 /
// 12.9 / 12.7; 16 of 0 to 8000 53 / 30 / 18 / 14 / 19; 64 of 0 to 8000 53 / 30 / 22 / 24 / 52; 256 of 0 to 8000
// 66 / 48 / 62 / 95, of 8000 93 / 90 / 101 / 131, of 1000 15 / 23 / 34 / 62; 1024 of 0 to 1000 41 / 66 / 111.
int auto_splits(long long ctas, int max_len) {
  const int sms = ops_sm_count();
  const long long room = 2LL * sms;
  int splits = 1;
  while (splits < kMaxSplits && splits * 512 <= max_len && ctas * splits * 2 <= (splits < 8 ? room : sms)) splits *= 2;
  if (splits == 1 && ctas > sms && ctas <= room && max_len >= 4096) splits = 2;
  return splits;
}

template <int HD, int RH, bool BF16>
cudaError_t launch_digit(AttnArgs a, int max_len, int splits, cudaStream_t s) {
  constexpr int kSmem = kDigWarps * kDigStages * Unit<HD>::kBytes;
  a.row_tiles = (a.rows * a.group + 2 * RH - 1) / (2 * RH);
  const long long ctas = (long long)a.c.n_kv * a.row_tiles * a.c.n_seq;
  if (splits < 1) splits = auto_splits(ctas, max_len);
  a.longest_first = a.c.n_seq > 1 && ctas * splits > 2LL * ops_sm_count();
  static OncePerDevice once;
  const cudaError_t e = once.smem(digit_kernel<HD, RH, BF16>, kSmem, true);
  if (e != cudaSuccess) return e;
  return ops_launch(digit_kernel<HD, RH, BF16>, dim3(splits, a.c.n_kv * a.row_tiles, a.c.n_seq), dim3(kDigWarps * 32),
                    kSmem, s, splits, a);
}

template <int HD, int PL>
cudaError_t launch(AttnArgs a, int max_len, int splits, cudaStream_t s) {
  constexpr int R = WarpState<HD, PL>::kRows;
  const int n_rows = a.rows * a.group;
  if (n_rows <= 2) return launch_digit<HD, 1, PL == 1>(a, max_len, splits, s);
  // (8 rows as two digit tiles: 170 us for 32 x 8191 tokens, one f16 tile 155 us)
  if (n_rows <= 4) return launch_digit<HD, 2, PL == 1>(a, max_len, splits, s);
  a.row_tiles = (n_rows + R - 1) / R;
  const long long ctas = (long long)a.c.n_kv * a.row_tiles * a.c.n_seq;
  if (splits < 1) splits = auto_splits(ctas, max_len);
  a.longest_first = a.c.n_seq > 1 && ctas * splits > 2LL * ops_sm_count();
  static OncePerDevice once;
  const cudaError_t e = once.smem(step_kernel<HD, PL>, step_smem<HD>(), true);
  if (e != cudaSuccess) return e;
  return ops_launch(step_kernel<HD, PL>, dim3(splits, a.c.n_kv * a.row_tiles, a.c.n_seq), dim3(kStepWarps * 32),
                    step_smem<HD>(), s, splits, a);
}

}  // namespace

cudaError_t kv8_attention(const Kv8& c, const void* q, long long q_seq, long long q_row, void* out, long long o_seq,
                          long long o_row, OpsDtype dt, int rows, int heads, const int* starts, const int* counts,
                          int idx_stride, float scale, int max_len, OpsErrors* err, cudaStream_t s, int splits) {
  if (rows <= 0 || c.n_seq <= 0) return cudaSuccess;
  if ((long long)rows * (heads / c.n_kv) > kStepRows)
    return kv8_prompt_attention(c, q, q_seq, q_row, out, o_seq, o_row, dt, rows, heads, starts, counts, idx_stride,
                                scale, max_len <= 0 || max_len > c.capacity ? c.capacity : max_len, splits > 0 ? 1 : 0,
                                err, s);
  AttnArgs a{c, q, out, q_seq, q_row, o_seq, o_row, starts, counts, idx_stride, rows, heads, heads / c.n_kv, 1, scale, 0, 0};
  const int es = dt == OPS_BF16 ? 2 : 4;
  a.vec = (uintptr_t)q % 16 == 0 && q_seq * es % 16 == 0 && q_row * es % 16 == 0;
  if (max_len <= 0 || max_len > c.capacity) max_len = c.capacity;
  if (c.head_dim == 128)
    return dt == OPS_BF16 ? launch<128, 1>(a, max_len, splits, s) : launch<128, 2>(a, max_len, splits, s);
  return dt == OPS_BF16 ? launch<64, 1>(a, max_len, splits, s) : launch<64, 2>(a, max_len, splits, s);
}

}  // namespace qasr
