// RMSNorm with the residual's addition and int8 rows with a scale each.
//
//   h = x + r,  u = h * w,  top = max|u|,  q = rint(127 u / top),  scale = top / rms(h) / 127
//
// The int8 values do not depend on the norm: dividing the row by its rms changes u and top
// alike. So one pass over the row gives everything: the sum of h^2 and the maximum of |u| are
// reduced together, once, and the row, still in registers, is quantised behind that one barrier.
//
// Rounding. q is the correctly rounded quotient. In f32, v = u * (127 / top) is off by less
// than 127 * 4 * 2^-24 < 4e-5, so a v further than 1e-4 from a half rounds to the right side;
// the few others (2e-4 of all) are rounded again from the f64 product, whose factors h, w are
// exact. top is compared exactly too: the product's f32 rounding first, its error (one fma)
// between equal ones. The sum of squares is held in 64 bits, where no finite row overflows it.
//
// Bound: DRAM. A bf16 row of d values with a residual moves 7d bytes and takes ~25 operations a
// value.
#include <cuda_bf16.h>

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
  __device__ static void load_vec(const T* p, float* f) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  }
  __device__ static void store_vec(T* p, const float* f) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  }
};
template <>
struct Elem<true> {
  using T = __nv_bfloat16;
  static constexpr int kVec = 8;
  __device__ static float load(const T* p) { return __bfloat162float(*p); }
  __device__ static void store(T* p, float v) { *p = __float2bfloat16_rn(v); }
  __device__ static float round(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }
  __device__ static void load_vec(const T* p, float* f) { bf16x8_to_f32(*reinterpret_cast<const uint4*>(p), f); }
  __device__ static void store_vec(T* p, const float* f) {
    __nv_bfloat162 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(v);
  }
};

struct NormArgs {
  const void *x, *r;
  void* h;
  const float* w;
  int8_t* q;
  float* scale;
  long long ldx, ldr, ldh, ldq, rows;
  int d;
  float eps;
};

// Running row statistics: the sum of squares, and the largest |u| as (f32 rounding, error).
struct Stat {
  double ss = 0.0;
  unsigned top = 0u, low = 0u;  // bits of the rounded |u|; ordered bits of the error
  __device__ void add(float h, float w) {
    ss = fma((double)h, (double)h, ss);
    const float p = __fmul_rn(h, w);
    const unsigned b = __float_as_uint(p) & 0x7FFFFFFFu;
    if (b >= top) {
      float e = __fmaf_rn(h, w, -p);
      if (p < 0.f) e = -e;
      const unsigned o = (unsigned)float_to_ordered(e) ^ 0x80000000u;
      if (b > top || o > low) low = o;
      top = b;
    }
  }
  __device__ void warp() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const unsigned t = __reduce_max_sync(0xffffffffu, top);
    low = __reduce_max_sync(0xffffffffu, top == t ? low : 0u);
    top = t;
  }
  __device__ bool finite() const { return top < 0x7F800000u; }
  __device__ double top64() const {
    return (double)__uint_as_float(top) + (double)ordered_to_float((int)(low ^ 0x80000000u));
  }
};

__device__ __forceinline__ int quant(float h, float w, float r127, const Stat& st) {
  const float v = __fmul_rn(__fmul_rn(h, w), r127);
  const float t = rintf(v);
  if (fabsf(fabsf(__fsub_rn(v, t)) - 0.5f) < 1e-4f) return __double2int_rn((double)h * (double)w * 127.0 / st.top64());
  return (int)t;
}

__device__ __forceinline__ void write_scale(const NormArgs& a, long long row, const Stat& st) {
  float sc = 1.0f;
  if (!st.finite())
    sc = __int_as_float(0x7FFFFFFF);
  else if (st.top)
    sc = (float)(st.top64() / sqrt(st.ss / (double)a.d + (double)a.eps) / 127.0);
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

// One row by W warps, its values in registers: NV vectors a thread.
template <bool BF16, int W, int NV, int ROWS>
__global__ void __launch_bounds__(W * ROWS * 32) norm_vec_kernel(const NormArgs a) {
  using E = Elem<BF16>;
  using T = typename E::T;
  constexpr int V = E::kVec;
  __shared__ Stat red[W];
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % W;
  const long long row = (long long)blockIdx.x * ROWS + (threadIdx.x >> 5) / W;
  if (row >= a.rows) return;  // ROWS > 1 only with W == 1: no barrier below
  const T* x = (const T*)a.x + row * a.ldx;
  const T* r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
  const int t = warp * 32 + lane;
  float h[NV][V];
  bool in[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (t + j * W * 32) * V;
    in[j] = c < a.d;
    if (in[j]) E::load_vec(x + c, h[j]);
  }
  if (r) {
    float f[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (in[j]) E::load_vec(r + (t + j * W * 32) * V, f[j]);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) h[j][i] = E::round(__fadd_rn(h[j][i], f[j][i]));
  }
  Stat st;
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (in[j]) {
      const int c = (t + j * W * 32) * V;
      if (a.h) E::store_vec((T*)a.h + row * a.ldh + c, h[j]);
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 w = __ldg(reinterpret_cast<const float4*>(a.w + c + i));
        st.add(h[j][i], w.x);
        st.add(h[j][i + 1], w.y);
        st.add(h[j][i + 2], w.z);
        st.add(h[j][i + 3], w.w);
      }
    }
  row_stat(st, red, warp, lane, W);
  const float top = __uint_as_float(st.top);
  const float r127 = st.finite() && st.top ? __fdiv_rn(127.0f, top) : 0.f;
  const bool tiny = r127 > 3e38f;  // 127 / top overflowed: a row of subnormals
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (in[j]) {
      const int c = (t + j * W * 32) * V;
      uint32_t o[V / 4];
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 w = __ldg(reinterpret_cast<const float4*>(a.w + c + i));
        const float wf[4] = {w.x, w.y, w.z, w.w};
        o[i / 4] = 0u;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int v = r127 == 0.f ? 0
                        : tiny      ? __double2int_rn((double)h[j][i + k] * (double)wf[k] * 127.0 / st.top64())
                                    : quant(h[j][i + k], wf[k], r127, st);
          o[i / 4] |= ((uint32_t)v & 0xFFu) << (8 * k);
        }
      }
      int8_t* q = a.q + row * a.ldq + c;
      if constexpr (V == 8)
        *reinterpret_cast<uint2*>(q) = make_uint2(o[0], o[1]);
      else
        *reinterpret_cast<uint32_t*>(q) = o[0];
    }
  if (t == 0) write_scale(a, row, st);
}

// Any d, stride and alignment: the row is staged in shared memory, one element a thread at a time.
template <bool BF16>
__global__ void __launch_bounds__(512) norm_any_kernel(const NormArgs a) {
  using E = Elem<BF16>;
  using T = typename E::T;
  extern __shared__ float hrow[];
  __shared__ Stat red[16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.ldx;
  const T* r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
  Stat st;
  for (int c = threadIdx.x; c < a.d; c += 512) {
    float h = E::load(x + c);
    if (r) h = E::round(__fadd_rn(h, E::load(r + c)));
    hrow[c] = h;
    if (a.h) E::store((T*)a.h + row * a.ldh + c, h);
    st.add(h, a.w[c]);
  }
  row_stat(st, red, warp, lane, 16);
  const float r127 = st.finite() && st.top ? __fdiv_rn(127.0f, __uint_as_float(st.top)) : 0.f;
  const bool tiny = r127 > 3e38f;
  for (int c = threadIdx.x; c < a.d; c += 512) {
    const float h = hrow[c], w = a.w[c];
    const int v = r127 == 0.f ? 0
                  : tiny      ? __double2int_rn((double)h * (double)w * 127.0 / st.top64())
                              : quant(h, w, r127, st);
    a.q[row * a.ldq + c] = (int8_t)v;
  }
  if (threadIdx.x == 0) write_scale(a, row, st);
}

template <bool BF16>
cudaError_t launch(const NormArgs& a, bool vec, cudaStream_t s) {
  constexpr int V = Elem<BF16>::kVec;
  const int nv = a.d / V;  // vectors of a row
  const dim3 g((unsigned)a.rows);
  if (vec) {
    if (nv <= 128) return ops_launch(norm_vec_kernel<BF16, 4, 1, 1>, g, dim3(128), 0, s, 1, a);
    if (nv <= 256) return ops_launch(norm_vec_kernel<BF16, 8, 1, 1>, g, dim3(256), 0, s, 1, a);
    if (nv <= 512) return ops_launch(norm_vec_kernel<BF16, 8, 2, 1>, g, dim3(256), 0, s, 1, a);
    if (nv <= 1024) return ops_launch(norm_vec_kernel<BF16, 8, 4, 1>, g, dim3(256), 0, s, 1, a);
    if (nv <= 2048) return ops_launch(norm_vec_kernel<BF16, 16, 4, 1>, g, dim3(512), 0, s, 1, a);
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

cudaError_t rms_norm_int8(const void* x, long long ldx, const void* residual, long long ldr, const float* w, float eps,
                          OpsDtype dt, long long rows, int d, int8_t* q, long long ldq, float* scale, void* h,
                          long long ldh, cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  NormArgs a{x, residual, h, w, q, scale, ldx, ldr, ldh, ldq, rows, d, eps};
  const int V = dt == OPS_BF16 ? 8 : 4;
  auto ok = [&](const void* p, long long ld) { return !p || ((uintptr_t)p % 16 == 0 && ld % V == 0); };
  const bool vec = d % V == 0 && ok(x, ldx) && ok(residual, ldr) && ok(h, ldh) && (uintptr_t)w % 16 == 0 &&
                   (uintptr_t)q % V == 0 && ldq % V == 0;
  return dt == OPS_BF16 ? launch<true>(a, vec, s) : launch<false>(a, vec, s);
}

}  // namespace qasr
