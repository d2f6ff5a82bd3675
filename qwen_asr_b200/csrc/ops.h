// Operators of the 8-bit serving path on device pointers: RMSNorm with the residual's addition
// and int8 rows, the int8 matrix product, and the int8 KV cache (written, read back, attended).
// Every function enqueues on `s` on the current device, allocates nothing and returns the launch
// status. The argument checks are in ops_api.cpp; engine.cu calls these directly.
#pragma once
#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>

namespace qasr {

enum OpsDtype { OPS_F32 = 0, OPS_BF16 = 1 };

// Where kernels report a bounded wait that gave up: how many did, and the last one's code. Each user of the operators
// has a word of its own (an engine its buffer, the C entry points one a device) and compares the count with the one
// it saw last, so nobody takes or clears another's error.
struct OpsErrors {
  int count, code;
};
OpsErrors* ops_api_errors();                       // the C entry points' on the current device; null: not to be had
int ops_errors(const OpsErrors* word, int& seen);  // the code of errors since `seen`, 0: none, -1: unreadable
cudaError_t ops_report(OpsErrors* word, int code); // as a kernel does (for tests), and waits for it
#ifdef __CUDACC__
__device__ __forceinline__ void ops_gave_up(OpsErrors* word, int code) {
  atomicExch(&word->code, code);
  atomicAdd(&word->count, 1);
}
#endif

constexpr int kNormMaxD = 32768;  // the row is staged in shared memory as f32

// rows r < rows of x (row pitch ldx elements): h = x + residual rounded to the type (h = x
// without a residual), u = h * w, top = max |u|; q = rint(127 u / top) as if in exact
// arithmetic (where top is 2^-100 or more; below, top is taken to 2^-149), scale = top / sqrt(mean(h^2) + eps) / 127 (1 for a row of zeros). A row with a
// NaN or an infinity (or a product beyond f32) gets scale NaN and q = 0. h may be null, x or
// residual; q rows have pitch ldq bytes, of which bytes [d, ldq) are left as they were.
cudaError_t rms_norm_int8(const void* x, long long ldx, const void* residual, long long ldr, const float* w, float eps,
                          OpsDtype dt, long long rows, int d, int8_t* q, long long ldq, float* scale, void* h,
                          long long ldh, cudaStream_t s);

// int8 rows of x without a norm: q as above for u = x, scale = top / 127.
cudaError_t quant_rows_int8(const float* x, long long ldx, long long rows, int d, int8_t* q, long long ldq,
                            float* scale, cudaStream_t s);

enum LinearEpi { LINEAR_STORE = 0, LINEAR_RESID = 1, LINEAR_SWIGLU = 2 };

// out[m][n] = (sum_k xq[m][k] * wq[n][k]) * xs[m] * ws[n], exact int32 sums; LINEAR_RESID adds
// residual[m][n], LINEAR_SWIGLU writes silu(y[2j]) * y[2j + 1] (n even). xq / wq 16-byte
// aligned with row pitches that are multiples of 16 bytes. out may be residual.
cudaError_t linear_int8(const int8_t* xq, long long ldx, const float* xs, const int8_t* wq, long long ldw,
                        const float* ws, long long m, int n, int k, LinearEpi epi, const void* residual, long long ldr,
                        void* out, long long ldo, OpsDtype dt, OpsErrors* err, cudaStream_t s);

// int8 K/V of n_seq sequences: [n_seq][n_kv][capacity][head_dim] with an f32 scale for each
// block of kKv8Block tokens of a head, [n_seq][n_kv][capacity / kKv8Block].
constexpr int kKv8Block = 16;
constexpr int kKv8Splits = 4;  // the engine's decode steps: a sequence's bits do not depend on the batch
struct Kv8 {
  int8_t *k, *v;
  float *ks, *vs;
  long long seq_stride, scale_stride;  // elements between sequences
  int n_seq, n_kv, capacity, head_dim;
};

// Appends k / v rows [n_seq][rows][n_kv * head_dim] (element strides between sequences and
// rows) behind position starts[b * idx_stride] of each sequence; counts (null: rows) says how
// many of the rows a sequence has. A block's scale is max(scale so far, max|new| / 127): when
// it grows, the rows the block holds are re-coded. A block's first row starts its scale anew.
// Rows past the capacity, and sequences with a negative start, are not written.
cudaError_t kv8_append(const Kv8& c, const void* k, long long k_seq, long long k_row, const void* v, long long v_seq,
                       long long v_row, OpsDtype dt, int rows, const int* starts, const int* counts, int idx_stride,
                       cudaStream_t s);

// k_out / v_out [n_seq][rows][n_kv * head_dim] = the values of positions starts[b] + r, zeros
// from row counts[b] (null: rows) or the capacity on. Either output may be null.
cudaError_t kv8_read(const Kv8& c, void* k_out, long long k_seq, long long k_row, void* v_out, long long v_seq,
                     long long v_row, OpsDtype dt, int rows, const int* starts, const int* counts, int idx_stride,
                     cudaStream_t s);

// out[b][r] = softmax(scale * q[b][r] K^T) V per head over positions 0 .. starts[b] + r;
// q / out [n_seq][rows][heads * head_dim] (element strides). Rows from counts[b] on, and
// sequences with a negative start, get zeros. max_len: an upper bound of the positions any row
// sees (only the launch shape depends on it; <= 0: the capacity). splits: CTAs that share a
// sequence's length when there are few query rows, 1, 2, 4, 8 or 16 (0: by max_len and the sequences
// at hand; a fixed number makes a sequence's result independent of the others).
cudaError_t kv8_attention(const Kv8& c, const void* q, long long q_seq, long long q_row, void* out, long long o_seq,
                          long long o_row, OpsDtype dt, int rows, int heads, const int* starts, const int* counts,
                          int idx_stride, float scale, int max_len, OpsErrors* err, cudaStream_t s, int splits = 0);

// The same for many query rows, on tcgen05 (kv8_attention calls it for more than 64 a KV head). splits: CTAs
// that share a row tile's keys, 1, 2 or 4 (0: by max_len and the CTAs at hand).
cudaError_t kv8_prompt_attention(const Kv8& c, const void* q, long long q_seq, long long q_row, void* out,
                                 long long o_seq, long long o_row, OpsDtype dt, int rows, int heads, const int* starts,
                                 const int* counts, int idx_stride, float scale, int max_len, int splits,
                                 OpsErrors* err, cudaStream_t s);

// The current device's SM count (queried once a device).
inline int ops_sm_count() {
  static std::atomic<int> n[64];
  int dev = 0, v = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!(v = n[dev].load())) {
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) return 148;
    n[dev].store(v);
  }
  return v;
}

// Raises a kernel's dynamic shared memory limit, and allows it clusters of 16 CTAs, once a device
// (one object a kernel).
struct OncePerDevice {
  std::atomic<unsigned long long> done{0};
  template <typename K>
  cudaError_t smem(K kernel, int bytes, bool clusters16 = false) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (done.load() & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && clusters16)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) done.fetch_or(bit);
    return e;
  }
};

// Launch, optionally in clusters of `cluster` CTAs along x, with programmatic dependence on the
// stream's previous kernel: the CTAs may start while it ends, so every kernel launched here waits
// (pdl_wait) before it touches global memory, and lets its own successor start early in turn. None reads by the
// read-only path (__ldg, ld.global.nc), which is for memory that nobody writes while the kernel is there.
template <typename K, typename... A>
inline cudaError_t ops_launch(K kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t s, int cluster,
                              const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace qasr
