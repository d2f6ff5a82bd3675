// The int8 KV cache as it is written and read back.
//
// Values are stored as q with x ~ q * s, one f32 scale s for each block of 16 tokens of a head.
// Appending a row to a block that already holds some makes the scale s' = max(s, max|x| / 127);
// where it grew, the held rows become rint(q s / s'). A block's first row (position % 16 == 0)
// starts from s = 0, so nothing of an earlier, longer history is left in its scale.
//
// One CTA owns one (sequence, head, block) of K or of V: it reads the new rows once, reduces
// max|x| over them, and writes the block's int8 rows and scale. No two CTAs share a scale, so
// there are no atomics, and a call's result depends on its inputs alone.
//
// Rounding. x / s in f32 is correctly rounded, and f32 holds every half up to 127.5, so the
// rounded quotient is on the right side of a half or on it; when it is on it, the sign of the
// remainder (one fma) says which side the exact quotient is on.
//
// Bound: latency for a token (one pass of 128 CTAs for 8 sequences of 8 heads), DRAM for prompts.
#include <cuda_bf16.h>

#include "bulk.cuh"
#include "dev_util.cuh"
#include "ops.h"

namespace qasr {
namespace {

struct AppendArgs {
  Kv8 c;
  const void *k, *v;
  long long k_seq, k_row, v_seq, v_row;
  const int *starts, *counts;
  int idx_stride, rows, vec;
};

__device__ __forceinline__ int quant_by(float x, float s) {
  const float v = __fdiv_rn(x, s);
  float t = rintf(v);
  if (fabsf(__fsub_rn(v, t)) == 0.5f) {
    const float rem = __fmaf_rn(-v, s, x);
    if (rem > 0.f) t = ceilf(v);
    if (rem < 0.f) t = floorf(v);
  }
  return (int)fminf(fmaxf(t, -127.f), 127.f);
}

// N consecutive values at p (N = head_dim / 8 = 8 or 16).
template <bool BF16, int N>
__device__ __forceinline__ void load_values(const void* base, long long off, bool vec, float* f) {
  if constexpr (BF16) {
    const __nv_bfloat16* p = (const __nv_bfloat16*)base + off;
    if (vec) {
#pragma unroll
      for (int i = 0; i < N; i += 8) bf16x8_to_f32(*reinterpret_cast<const uint4*>(p + i), f + i);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = __bfloat162float(p[i]);
    }
  } else {
    const float* p = (const float*)base + off;
    if (vec) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(p + i);
        f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = p[i];
    }
  }
}

template <int N>
struct alignas(N) Bytes {
  uint32_t w[N / 4];
};

// grid (blocks a sequence can touch, 2 * n_kv, n_seq), 128 threads: thread = (row of the block, eighth of the row)
template <bool BF16, int HD>
__global__ void __launch_bounds__(128) append_kernel(const AppendArgs a) {
  constexpr int N = HD / 8;
  __shared__ unsigned red[4];
  const int seq = blockIdx.z, head = blockIdx.y >> 1;
  const bool is_v = blockIdx.y & 1;
  pdl_launch_dependents();
  pdl_wait();
  const int start = a.starts[(long long)seq * a.idx_stride];
  int count = a.rows;
  if (a.counts) count = min(max(a.counts[(long long)seq * a.idx_stride], 0), a.rows);
  if (start < 0 || start >= a.c.capacity) return;
  const int end = (int)min((long long)start + count, (long long)a.c.capacity);
  const int blk = start / kKv8Block + blockIdx.x;
  const int base = blk * kKv8Block;
  if (base >= end || start >= end) return;  // (whole CTA)
  const int row = base + (threadIdx.x >> 3), part = (threadIdx.x & 7) * N;
  const bool fresh = row >= start && row < end;
  const bool held = row < start;  // only in the first block
  float* scale = (is_v ? a.c.vs : a.c.ks) + seq * a.c.scale_stride +
                 (long long)head * (a.c.capacity / kKv8Block) + blk;
  int8_t* dst = (is_v ? a.c.v : a.c.k) + seq * a.c.seq_stride +
                ((long long)head * a.c.capacity + row) * HD + part;
  float x[N];
  float mx = 0.f;
  unsigned bits = 0u;
  if (fresh) {
    const long long off = seq * (is_v ? a.v_seq : a.k_seq) + (row - start) * (is_v ? a.v_row : a.k_row) +
                          head * HD + part;
    load_values<BF16, N>(is_v ? a.v : a.k, off, a.vec, x);
#pragma unroll
    for (int i = 0; i < N; ++i) bits = max(bits, __float_as_uint(x[i]) & 0x7FFFFFFFu);  // NaN above infinity
  }
  const float s_old = start > base ? *scale : 0.f;
  Bytes<N> old{};
  if (held) old = *reinterpret_cast<const Bytes<N>*>(dst);
  bits = __reduce_max_sync(0xffffffffu, bits);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = bits;
  __syncthreads();  // also: every thread has read the old scale
  bits = max(max(red[0], red[1]), max(red[2], red[3]));
  mx = __uint_as_float(bits);
  const bool bad = bits >= 0x7F800000u || !(s_old >= 0.f && s_old < __int_as_float(0x7F800000));
  const float s = bad ? __int_as_float(0x7FFFFFFF) : fmaxf(s_old, __fdiv_rn(mx, 127.0f));
  Bytes<N> o{};
  if (fresh) {
    if (!bad && s > 0.f) {
#pragma unroll
      for (int i = 0; i < N; ++i) o.w[i >> 2] |= ((uint32_t)quant_by(x[i], s) & 0xFFu) << (8 * (i & 3));
    }
    *reinterpret_cast<Bytes<N>*>(dst) = o;
  } else if (held && !bad && s > s_old) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int q = (int)(int8_t)(old.w[i >> 2] >> (8 * (i & 3)));
      const int t = __double2int_rn((double)q * (double)s_old / (double)s);
      o.w[i >> 2] |= ((uint32_t)t & 0xFFu) << (8 * (i & 3));
    }
    *reinterpret_cast<Bytes<N>*>(dst) = o;
  }
  if (threadIdx.x == 0) *scale = s;
}

struct ReadArgs {
  Kv8 c;
  void *k, *v;
  long long k_seq, k_row, v_seq, v_row;
  const int *starts, *counts;
  int idx_stride, rows, vec;
};

// grid (row groups, K and V, n_seq): a thread writes 8 values of a row
template <bool BF16, int HD>
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs a) {
  const int seq = blockIdx.z;
  const bool is_v = blockIdx.y;
  void* out = is_v ? a.v : a.k;
  if (!out) return;
  pdl_launch_dependents();
  pdl_wait();
  const int start = a.starts[(long long)seq * a.idx_stride];
  int count = a.rows;
  if (a.counts) count = min(max(a.counts[(long long)seq * a.idx_stride], 0), a.rows);
  const int per_row = a.c.n_kv * HD / 8;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)a.rows * per_row) return;
  const int r = (int)(i / per_row), col = (int)(i % per_row) * 8, head = col / HD;
  float f[8] = {};
  const long long pos = (long long)start + r;
  if (start >= 0 && r < count && pos < a.c.capacity) {
    const int8_t* q = (is_v ? a.c.v : a.c.k) + seq * a.c.seq_stride +
                      ((long long)head * a.c.capacity + pos) * HD + col % HD;
    const float s = ((is_v ? a.c.vs : a.c.ks) + seq * a.c.scale_stride)[(long long)head * (a.c.capacity / kKv8Block) +
                                                                       pos / kKv8Block];
    const uint2 b = *reinterpret_cast<const uint2*>(q);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t w = j < 4 ? b.x : b.y;
      f[j] = __fmul_rn((float)(int8_t)(w >> (8 * (j & 3))), s);
    }
  }
  const long long off = seq * (is_v ? a.v_seq : a.k_seq) + r * (is_v ? a.v_row : a.k_row) + col;
  if constexpr (BF16) {
    __nv_bfloat16* o = (__nv_bfloat16*)out + off;
    __nv_bfloat162 p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
    if (a.vec) {
      *reinterpret_cast<uint4*>(o) = *reinterpret_cast<uint4*>(p);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = j & 1 ? p[j >> 1].y : p[j >> 1].x;
    }
  } else {
    float* o = (float*)out + off;
    if (a.vec) {
      *reinterpret_cast<float4*>(o) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(o + 4) = make_float4(f[4], f[5], f[6], f[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = f[j];
    }
  }
}

// 16-byte accesses to rows at p: aligned base and strides (a row starts every head_dim values).
bool vec_ok(const void* p, long long seq, long long row, OpsDtype dt) {
  const int es = dt == OPS_BF16 ? 2 : 4;
  return !p || ((uintptr_t)p % 16 == 0 && seq * es % 16 == 0 && row * es % 16 == 0);
}

}  // namespace

cudaError_t kv8_append(const Kv8& c, const void* k, long long k_seq, long long k_row, const void* v, long long v_seq,
                       long long v_row, OpsDtype dt, int rows, const int* starts, const int* counts, int idx_stride,
                       cudaStream_t s) {
  if (rows <= 0 || c.n_seq <= 0) return cudaSuccess;
  const bool vec = vec_ok(k, k_seq, k_row, dt) && vec_ok(v, v_seq, v_row, dt);
  AppendArgs a{c, k, v, k_seq, k_row, v_seq, v_row, starts, counts, idx_stride, rows, vec};
  const long long touch = ((long long)rows + 2 * kKv8Block - 2) / kKv8Block;
  const int blocks = (int)(touch < c.capacity / kKv8Block ? touch : c.capacity / kKv8Block);
  const dim3 g(blocks, 2 * c.n_kv, c.n_seq), t(128);
  if (c.head_dim == 128)
    return dt == OPS_BF16 ? ops_launch(append_kernel<true, 128>, g, t, 0, s, 1, a)
                          : ops_launch(append_kernel<false, 128>, g, t, 0, s, 1, a);
  return dt == OPS_BF16 ? ops_launch(append_kernel<true, 64>, g, t, 0, s, 1, a)
                        : ops_launch(append_kernel<false, 64>, g, t, 0, s, 1, a);
}

cudaError_t kv8_read(const Kv8& c, void* k_out, long long k_seq, long long k_row, void* v_out, long long v_seq,
                     long long v_row, OpsDtype dt, int rows, const int* starts, const int* counts, int idx_stride,
                     cudaStream_t s) {
  if (rows <= 0 || c.n_seq <= 0 || (!k_out && !v_out)) return cudaSuccess;
  const bool vec = vec_ok(k_out, k_seq, k_row, dt) && vec_ok(v_out, v_seq, v_row, dt);
  ReadArgs a{c, k_out, v_out, k_seq, k_row, v_seq, v_row, starts, counts, idx_stride, rows, vec};
  const long long n = (long long)rows * c.n_kv * c.head_dim / 8;
  const dim3 g((unsigned)((n + 255) / 256), 2, c.n_seq), t(256);
  if (c.head_dim == 128)
    return dt == OPS_BF16 ? ops_launch(read_kernel<true, 128>, g, t, 0, s, 1, a)
                          : ops_launch(read_kernel<false, 128>, g, t, 0, s, 1, a);
  return dt == OPS_BF16 ? ops_launch(read_kernel<true, 64>, g, t, 0, s, 1, a)
                        : ops_launch(read_kernel<false, 64>, g, t, 0, s, 1, a);
}

}  // namespace qasr
