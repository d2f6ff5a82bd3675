// RMSNorm with the residual's addition and int8 rows with a scale each.
//
//   h = x + r,  u = h * w,  top = max|u|,  q = rint(127 u / top),  scale = top / rms(h) / 127
//
// The int8 values do not depend on the norm: dividing the row by its rms changes u and top
// alike. So one pass over the row gives everything: the sum of h^2 and the maximum of |u| are
// reduced together, once, and the row, still in registers, is quantised behind that one barrier.
//
// Rounding. q is the correctly rounded quotient. In f32, v = u * (127 / top) is off by at most
// 127 * 4 * 2^-24 < 3.1e-5 (four roundings), so a v further than 3.2e-5 from a half rounds to the
// right side; the others (6e-5 of all) are rounded again from the exact products u and top, which f64 holds
// (top is the largest f32 product and its rounding error, one fma in the threads that hold it: exact down to 2^-100).
// 127 u needs up to 55 bits, so where the f64 quotient is next to a half the side comes from 254 u - (2n + 1) top,
// two products with their rounding errors (`rounded`). The sum of squares is held in 64 bits, where no
// finite row overflows it.
//
// Bound: DRAM for many rows. What it took to get near: a bf16 sum as packed adds, one fmax a
// value, rounding by the 1.5 * 2^23 trick whose low byte is the int8 value, and a warp that adds up
// the squares behind the barrier while the others quantise (they do not need the norm). 16411
// rows of 2048 bf16 values with a residual, call after call: 46 us, 5.1 TB/s; f32 68 us, 6.4 TB/s.
#include <cuda_bf16.h>

#include "bulk.cuh"
#include "dev_util.cuh"
#include "ops.h"

namespace qasr {
namespace {

template <bool BF16>
struct Elem;
template <>
struct Elem<false> {
  using T = float;
  static constexpr int kVec = 4;
  __device__ static float load(const T* p) { return *p; }
  __device__ static void store(T* p, float v) { *p = v; }
  __device__ static float round(float v) { return v; }
};
template <>
struct Elem<true> {
  using T = __nv_bfloat16;
  static constexpr int kVec = 8;
  __device__ static float load(const T* p) { return __bfloat162float(*p); }
  __device__ static void store(T* p, float v) { *p = __float2bfloat16_rn(v); }
  __device__ static float round(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }
};

struct NormArgs {
  const void *x, *r;
  void* h;
  const float* w;
  int8_t* q;
  float* scale;
  long long ldx, ldr, ldh, ldq, rows;
  int d;
  float eps;  // negative: int8 rows without a norm (w null, scale = top / 127)
};

// rint(127 u / top), correctly rounded, for exact u and top. (Of bf16 values 127 u is exact, too, and a quotient of
// such products that is not a half is 2^-42 away from one at least, so its rounding to f64 does not matter.)
template <bool BF16>
__device__ __forceinline__ int rounded(double u, double top) {
  if constexpr (BF16) return __double2int_rn(u * 127.0 / top);
  const double v = fabs(u), x = v * 127.0 / top, n = floor(x);
  double q = rint(x);
  if (fabs(x - n - 0.5) < 1e-9) {
    const double odd = 2.0 * n + 1.0, a = 254.0 * v, b = odd * top;
    // (a and b are within a few steps of each other, and all three differences exact)
    const double side = (a - b) + (fma(254.0, v, -a) - fma(odd, top, -b));
    if (side > 0.0) q = n + 1.0;
    if (side < 0.0) q = n;
    if (side == 0.0) q = 2.0 * rint(0.5 * (n + 0.5));  // the even one
  }
  return (int)copysign(q, u);
}

// Running row statistics: the sum of squares, and the largest |u|, rounded (its bits) and exact.
struct Stat {
  double ss = 0.0, exact = 0.0;
  unsigned top = 0u;
  __device__ void add(float h, float w) {
    ss = fma((double)h, (double)h, ss);
    const unsigned b = __float_as_uint(__fmul_rn(h, w)) & 0x7FFFFFFFu;
    if (b >= top) {
      exact = fmax(exact, fabs((double)h * (double)w));
      top = b;
    }
  }
  __device__ void warp() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      exact = fmax(exact, __shfl_xor_sync(0xffffffffu, exact, o));
    }
    top = __reduce_max_sync(0xffffffffu, top);
  }
  __device__ bool finite() const { return top < 0x7F800000u; }
};

template <bool BF16>
__device__ __forceinline__ int quant(float h, float w, float r127, const Stat& st) {
  const float v = __fmul_rn(__fmul_rn(h, w), r127);
  const float t = rintf(v);
  if (fabsf(fabsf(__fsub_rn(v, t)) - 0.5f) < 1e-4f) return rounded<BF16>((double)h * (double)w, st.exact);
  return (int)t;
}

__device__ __forceinline__ float scale_of(const NormArgs& a, double top, double ss) {
  const double rms = a.eps < 0.f ? 1.0 : sqrt(ss / (double)a.d + (double)a.eps);
  return (float)(top / rms / 127.0);
}

__device__ __forceinline__ void write_scale(const NormArgs& a, long long row, const Stat& st) {
  float sc = 1.0f;
  if (!st.finite())
    sc = __int_as_float(0x7FFFFFFF);
  else if (st.top)
    sc = scale_of(a, st.exact, st.ss);
  a.scale[row] = sc;
}

// Reduces the threads' statistics over the `nw` warps of a row (red: one slot a warp).
__device__ __forceinline__ void row_stat(Stat& st, Stat* red, int warp, int lane, int nw) {
  st.warp();
  if (nw == 1) return;
  if (lane == 0) red[warp] = st;
  __syncthreads();
  if (lane < nw) st = red[lane];
  else st = Stat();
  st.warp();
}

// 16 bytes of a row as loaded, and the sum of two of them rounded to the type. (Two bf16 values
// round the same from f32 as from their exact sum: where f32 cannot hold it, the smaller is below
// 2^-16 of the larger, far from a bf16 tie.)
template <bool BF16>
__device__ __forceinline__ uint4 add_packed(uint4 a, uint4 b) {
  uint32_t* x = reinterpret_cast<uint32_t*>(&a);
  const uint32_t* y = reinterpret_cast<const uint32_t*>(&b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      const __nv_bfloat162 h =
          __hadd2_rn(*reinterpret_cast<const __nv_bfloat162*>(x + i), *reinterpret_cast<const __nv_bfloat162*>(y + i));
      x[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      x[i] = __float_as_uint(__fadd_rn(__uint_as_float(x[i]), __uint_as_float(y[i])));
    }
  }
  return a;
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN when either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, in the low bits

// A thread's int8 values whose bit is set once more, from the exact products; its vectors of V are `step`
// vectors apart. (The value is read back from memory: an index into the registers would push them all to the
// stack. One row in eight has such a value: a thread that did all of its own again, one after the other, cost
// 16411 bf16 rows of 2048 68 us, finding them by a second look 47 to 51, this 44.)
template <bool BF16, int V>
__device__ __forceinline__ void fix_near(const NormArgs& a, long long row, double top64, int step, uint32_t mask) {
  using T = typename Elem<BF16>::T;
  const T* src = a.h ? (const T*)a.h + row * a.ldh : (const T*)a.x + row * a.ldx;
  int8_t* q = a.q + row * a.ldq;
  while (mask) {
    const int b = __ffs((int)mask) - 1;
    mask &= mask - 1;
    const int c = ((int)threadIdx.x + b / V * step) * V + b % V;
    if (c >= a.d) break;
    const double w = a.w ? (double)a.w[c] : 1.0;
    q[c] = (int8_t)rounded<BF16>((double)Elem<BF16>::load(src + c) * w, top64);
  }
}

// One row by W warps, its values in registers: NV vectors of V a thread. V = 1: rows of any length, stride and
// alignment (16411 x 2045 bf16 with residual 184 us by the kernel below, 87 so).
template <bool BF16, int V, int W, int NV>
__global__ void __launch_bounds__(W * 32) norm_vec_kernel(const NormArgs a) {
  using E = Elem<BF16>;
  using T = typename E::T;
  constexpr int N = W * 32;
  static_assert(NV * V <= 32, "a bit a value");
  __shared__ double parts[N];
  __shared__ unsigned tops[W];
  __shared__ unsigned low;  // ordered bits of the largest product's rounding error
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = blockIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  const T* x = (const T*)a.x + row * a.ldx;
  float h[NV][V], u[NV][V];
  uint4 raw[V > 1 ? NV : 1];
  if constexpr (V > 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (threadIdx.x + j * N) * V;
      raw[j] = make_uint4(0, 0, 0, 0);
      if (c < a.d) raw[j] = *reinterpret_cast<const uint4*>(x + c);
    }
    if (a.r) {
      const T* r = (const T*)a.r + row * a.ldr;
      uint4 add[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (threadIdx.x + j * N) * V;
        add[j] = make_uint4(0, 0, 0, 0);
        if (c < a.d) add[j] = *reinterpret_cast<const uint4*>(r + c);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) raw[j] = add_packed<BF16>(raw[j], add[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) h[j][0] = threadIdx.x + j * N < a.d ? E::load(x + threadIdx.x + j * N) : 0.f;
    if (a.r) {
      const T* r = (const T*)a.r + row * a.ldr;
      float add[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) add[j] = threadIdx.x + j * N < a.d ? E::load(r + threadIdx.x + j * N) : 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) h[j][0] = E::round(__fadd_rn(h[j][0], add[j]));
    }
  }
  float mx = 0.f;
  double ss = 0.0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (threadIdx.x + j * N) * V;
    if constexpr (V == 8) {
      bf16x8_to_f32(raw[j], h[j]);
    } else if constexpr (V == 4) {
      h[j][0] = __uint_as_float(raw[j].x);
      h[j][1] = __uint_as_float(raw[j].y);
      h[j][2] = __uint_as_float(raw[j].z);
      h[j][3] = __uint_as_float(raw[j].w);
    }
    if (V == 1) {
      u[j][0] = 0.f;
      if (c < a.d) {
        if (a.h) E::store((T*)a.h + row * a.ldh + c, h[j][0]);
        u[j][0] = __fmul_rn(h[j][0], a.w ? a.w[c] : 1.f);
      }
    } else if (c < a.d) {
#pragma unroll
      for (int i = 0; i + 3 < V; i += 4) {
        const float4 w = a.w ? *reinterpret_cast<const float4*>(a.w + c + i) : make_float4(1.f, 1.f, 1.f, 1.f);
        u[j][i] = __fmul_rn(h[j][i], w.x);
        u[j][i + 1] = __fmul_rn(h[j][i + 1], w.y);
        u[j][i + 2] = __fmul_rn(h[j][i + 2], w.z);
        u[j][i + 3] = __fmul_rn(h[j][i + 3], w.w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) u[j][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      mx = max_nan(mx, fabsf(u[j][i]));
      ss = fma((double)h[j][i], (double)h[j][i], ss);
    }
  }
  if constexpr (V > 1) {  // (behind the weights' loads, which might alias it for all the compiler knows)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (threadIdx.x + j * N) * V;
      if (a.h && c < a.d) *reinterpret_cast<uint4*>((T*)a.h + row * a.ldh + c) = raw[j];
    }
  }
  const unsigned mine = __float_as_uint(mx) & 0x7FFFFFFFu;
  const unsigned wtop = __reduce_max_sync(0xffffffffu, mine);
  parts[threadIdx.x] = ss;
  if (lane == 0) tops[warp] = wtop;
  if (threadIdx.x == 0) low = 0u;
  __syncthreads();
  unsigned top = tops[0];
#pragma unroll
  for (int i = 1; i < W; ++i) top = max(top, tops[i]);
  const bool finite = top < 0x7F800000u;
  if (mine == top && finite && top) {
    // this thread holds a largest product
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (threadIdx.x + j * N) * V;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c < a.d && (__float_as_uint(u[j][i]) & 0x7FFFFFFFu) == top) {
          const float e = a.w ? __fmaf_rn(h[j][i], a.w[c + i], -u[j][i]) : 0.f;
          atomicMax(&low, (unsigned)float_to_ordered(u[j][i] < 0.f ? -e : e) ^ 0x80000000u);
        }
    }
  }
  const float r127 = finite && top ? __fdiv_rn(127.0f, __uint_as_float(top)) : 0.f;
  uint32_t near = r127 > 3e38f ? ~0u : 0u;  // 127 / top overflowed: a row of subnormals takes the exact path
  int8_t* q = a.q + row * a.ldq;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (threadIdx.x + j * N) * V;
    uint32_t b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float v = __fmul_rn(u[j][i], r127);
      const float t = __fadd_rn(v, kRound);
      b[i] = finite ? __float_as_uint(t) : 0u;
      if (fabsf(__fsub_rn(v, __fsub_rn(t, kRound))) > 0.5f - 3.2e-5f) near |= 1u << (j * V + i);
    }
    if (c < a.d) {
      auto word = [&](int i) {
        return __byte_perm(__byte_perm(b[i], b[i + 1], 0x0040), __byte_perm(b[i + 2], b[i + 3], 0x0040), 0x5410);
      };
      if constexpr (V == 8)
        *reinterpret_cast<uint2*>(q + c) = make_uint2(word(0), word(4));
      else if constexpr (V == 4)
        *reinterpret_cast<uint32_t*>(q + c) = word(0);
      else
        q[c] = (int8_t)b[0];
    }
  }
  __syncthreads();  // `low` is complete
  const double top64 = (double)__uint_as_float(top) + (double)ordered_to_float((int)(low ^ 0x80000000u));
  if (near && finite) fix_near<BF16, V>(a, row, top64, N, near);
  if (warp == 0) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < W; ++i) sum += parts[i * 32 + lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0)
      a.scale[row] = !finite ? __int_as_float(0x7FFFFFFF)
                     : top   ? scale_of(a, top64, sum)
                             : 1.0f;
  }
}

// Any d, stride and alignment, for the longest rows: the row is staged in shared memory, one element a thread at a time.
template <bool BF16>
__global__ void __launch_bounds__(512) norm_any_kernel(const NormArgs a) {
  using E = Elem<BF16>;
  using T = typename E::T;
  extern __shared__ float hrow[];
  __shared__ Stat red[16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.ldx;
  pdl_launch_dependents();
  pdl_wait();
  const T* r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
  Stat st;
  for (int c = threadIdx.x; c < a.d; c += 512) {
    float h = E::load(x + c);
    if (r) h = E::round(__fadd_rn(h, E::load(r + c)));
    hrow[c] = h;
    if (a.h) E::store((T*)a.h + row * a.ldh + c, h);
    st.add(h, a.w ? a.w[c] : 1.0f);
  }
  row_stat(st, red, warp, lane, 16);
  const float r127 = st.finite() && st.top ? __fdiv_rn(127.0f, __uint_as_float(st.top)) : 0.f;
  const bool tiny = r127 > 3e38f;
  for (int c = threadIdx.x; c < a.d; c += 512) {
    const float h = hrow[c], w = a.w ? a.w[c] : 1.0f;
    const int v = r127 == 0.f ? 0
                  : tiny      ? rounded<BF16>((double)h * (double)w, st.exact)
                              : quant<BF16>(h, w, r127, st);
    a.q[row * a.ldq + c] = (int8_t)v;
  }
  if (threadIdx.x == 0) write_scale(a, row, st);
}

template <bool BF16>
cudaError_t launch(const NormArgs& a, bool vec, cudaStream_t s) {
  constexpr int V = Elem<BF16>::kVec;
  const int nv = vec ? a.d / V : a.d;  // vectors of a row, or single values
  const dim3 g((unsigned)a.rows);
  if (vec) {
    // two vectors a thread where rows fill the GPU anyway, one where a row's latency counts
    const bool many = a.rows >= 4 * ops_sm_count();
    if (nv <= 128) return ops_launch(norm_vec_kernel<BF16, V, 4, 1>, g, dim3(128), 0, s, 1, a);
    if (nv <= 256 && many) return ops_launch(norm_vec_kernel<BF16, V, 4, 2>, g, dim3(128), 0, s, 1, a);
    if (nv <= 256) return ops_launch(norm_vec_kernel<BF16, V, 8, 1>, g, dim3(256), 0, s, 1, a);
    if (nv <= 512) return ops_launch(norm_vec_kernel<BF16, V, 8, 2>, g, dim3(256), 0, s, 1, a);
    if (nv <= 1024) return ops_launch(norm_vec_kernel<BF16, V, 8, 4>, g, dim3(256), 0, s, 1, a);
    if (nv <= 2048) return ops_launch(norm_vec_kernel<BF16, V, 16, 4>, g, dim3(512), 0, s, 1, a);
  } else {
    if (nv <= 512) return ops_launch(norm_vec_kernel<BF16, 1, 4, 4>, g, dim3(128), 0, s, 1, a);
    if (nv <= 2048) return ops_launch(norm_vec_kernel<BF16, 1, 8, 8>, g, dim3(256), 0, s, 1, a);
    if (nv <= 8192) return ops_launch(norm_vec_kernel<BF16, 1, 16, 16>, g, dim3(512), 0, s, 1, a);
  }
  const size_t smem = (size_t)a.d * sizeof(float);
  if (smem > 40 * 1024) {
    static OncePerDevice once;
    const cudaError_t e = once.smem(norm_any_kernel<BF16>, kNormMaxD * (int)sizeof(float));
    if (e != cudaSuccess) return e;
  }
  return ops_launch(norm_any_kernel<BF16>, g, dim3(512), smem, s, 1, a);
}

}  // namespace

static cudaError_t run_rows(const NormArgs& a, OpsDtype dt, cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  const int V = dt == OPS_BF16 ? 8 : 4;
  auto ok = [&](const void* p, long long ld) { return !p || ((uintptr_t)p % 16 == 0 && ld % V == 0); };
  const bool vec = a.d % V == 0 && ok(a.x, a.ldx) && ok(a.r, a.ldr) && ok(a.h, a.ldh) && (uintptr_t)a.w % 16 == 0 &&
                   (uintptr_t)a.q % V == 0 && a.ldq % V == 0;
  return dt == OPS_BF16 ? launch<true>(a, vec, s) : launch<false>(a, vec, s);
}

cudaError_t rms_norm_int8(const void* x, long long ldx, const void* residual, long long ldr, const float* w, float eps,
                          OpsDtype dt, long long rows, int d, int8_t* q, long long ldq, float* scale, void* h,
                          long long ldh, cudaStream_t s) {
  return run_rows(NormArgs{x, residual, h, w, q, scale, ldx, ldr, ldh, ldq, rows, d, eps}, dt, s);
}

cudaError_t quant_rows_int8(const float* x, long long ldx, long long rows, int d, int8_t* q, long long ldq,
                            float* scale, cudaStream_t s) {
  return run_rows(NormArgs{x, nullptr, nullptr, nullptr, q, scale, ldx, 0, 0, ldq, rows, d, -1.0f}, OPS_F32, s);
}

}  // namespace qasr
