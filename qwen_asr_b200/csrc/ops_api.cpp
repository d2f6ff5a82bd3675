// C ABI of the 8-bit operators (include/qwen_asr_ext.h): argument checks, the caller's device,
// and the launch status as 0 / -1 with the reason in qwen_asr_last_error().
#include <cuda.h>

#include <exception>
#include <mutex>
#include <string>

#include "../../include/qwen_asr_ext.h"
#include "common.h"
#include "ops.h"

namespace {

using namespace qasr;

// Runs a call on `device` (-1: the current one) and gives the caller its CUDA context back.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (device < 0) return;
    const Driver& d = driver();
    if (!d.get || !d.set || !d.device) {
      ok_ = false;
      return;
    }
    CUdevice now = -1;
    if (d.get(&prev_) == CUDA_SUCCESS && prev_ && d.device(&now) == CUDA_SUCCESS && (int)now == device) return;
    ok_ = cudaSetDevice(device) == cudaSuccess;
    restore_ = prev_ != nullptr;
  }
  ~DeviceScope() {
    if (restore_) driver().set(prev_);
  }
  bool ok() const { return ok_; }

 private:
  struct Driver {
    CUresult (*get)(CUcontext*) = nullptr;
    CUresult (*set)(CUcontext) = nullptr;
    CUresult (*device)(CUdevice*) = nullptr;
    Driver() {
      load("cuCtxGetCurrent", (void**)&get);
      load("cuCtxSetCurrent", (void**)&set);
      load("cuCtxGetDevice", (void**)&device);
    }
    static void load(const char* name, void** fn) {
      void* p = nullptr;
      cudaDriverEntryPointQueryResult q;
      if (cudaGetDriverEntryPoint(name, &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
        *fn = p;
    }
  };
  static const Driver& driver() {  // looked up once, whichever thread comes first
    static const Driver d;
    return d;
  }
  CUcontext prev_ = nullptr;
  bool restore_ = false, ok_ = true;
};

int32_t fail(const char* op, const std::string& why) {
  set_error(std::string(op) + ": " + why);
  return -1;
}

template <typename F>
int32_t run(const char* op, int device, F&& launch) {
  try {
    DeviceScope scope(device);
    if (!scope.ok()) return fail(op, "cannot use device " + std::to_string(device));
    const cudaError_t e = launch();
    if (e == cudaSuccess) return 0;
    cudaGetLastError();  // a refused launch is reported here, not by the caller's next call
    return fail(op, std::string("launch failed: ") + cudaGetErrorString(e));
  } catch (const std::exception& ex) {
    return fail(op, ex.what());
  }
}

bool dtype_ok(int32_t t) { return t == QWEN_ASR_F32 || t == QWEN_ASR_BF16; }
bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }
size_t elem(int32_t t) { return t == QWEN_ASR_BF16 ? 2 : 4; }

// nullptr, or what is wrong with the cache.
const char* cache_fault(const QwenAsrKv8* c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return "a null cache pointer";
  if (c->n_seq < 1 || c->n_seq > 65535) return "n_seq must be 1 .. 65535";
  if (c->n_kv < 1 || c->n_kv > 4096) return "n_kv must be 1 .. 4096";
  if (c->head_dim != 64 && c->head_dim != 128) return "head_dim must be 64 or 128";
  if (c->capacity < kKv8Block || c->capacity % kKv8Block) return "capacity must be a positive multiple of 16";
  if (!aligned(c->k, 16) || !aligned(c->v, 16)) return "the int8 cache must start on 16-byte boundaries";
  if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4)) return "the scales must start on 4-byte boundaries";
  const int64_t rows = (int64_t)c->n_kv * c->capacity;
  if (c->n_seq > 1 && (c->seq_stride < rows * c->head_dim || c->seq_stride % 16))
    return "seq_stride must be a multiple of 16 and hold a sequence";
  if (c->n_seq > 1 && c->scale_stride < rows / kKv8Block) return "scale_stride must hold a sequence";
  return nullptr;
}

Kv8 cache_of(const QwenAsrKv8* c) {
  return Kv8{c->k, c->v, c->k_scale, c->v_scale, c->seq_stride, c->scale_stride, c->n_seq, c->n_kv, c->capacity,
             c->head_dim};
}

// Rows of `width` elements [n_seq][rows] at p: strides that hold a row and, when written, do not overlap.
const char* rows_fault(const QwenAsrRows* r, int n_seq, int rows, int64_t width, int32_t dtype, bool written) {
  if (!r->data) return "a null pointer";
  if (!aligned(r->data, elem(dtype))) return "a misaligned pointer";
  if (r->seq_stride < 0 || r->row_stride < 0) return "a negative stride";
  if (written) {
    if (rows > 1 && r->row_stride < width) return "overlapping output rows";
    const int64_t seq = (int64_t)(rows - 1) * r->row_stride + width;
    // sequences apart from each other: whole sequences in turn, or rows interleaved
    if (n_seq > 1 && r->seq_stride < seq &&
        !(rows > 1 && r->seq_stride >= width && r->row_stride >= (int64_t)(n_seq - 1) * r->seq_stride + width) &&
        !(rows == 1 && r->seq_stride >= width))
      return "overlapping output sequences";
  }
  return nullptr;
}

}  // namespace

extern "C" {

int32_t qwen_asr_rms_norm_int8(const void* x, int64_t ldx, const void* residual, int64_t ldr, const float* weight,
                               float eps, int32_t dtype, int64_t rows, int32_t d, int8_t* q, int64_t ldq, float* scale,
                               void* h, int64_t ldh, int32_t device, void* stream) {
  const char* op = "rms_norm_int8";
  if (!dtype_ok(dtype)) return fail(op, "dtype must be QWEN_ASR_F32 or QWEN_ASR_BF16");
  if (rows < 0 || rows > 0x7FFFFFFF) return fail(op, "rows must be 0 .. 2^31 - 1");
  if (d < 1 || d > kNormMaxD) return fail(op, "d must be 1 .. " + std::to_string(kNormMaxD));
  if (!(eps >= 0.f)) return fail(op, "eps must not be negative");
  if (rows == 0) return 0;
  if (!x || !weight || !q || !scale) return fail(op, "a null pointer");
  if (residual && !h) return fail(op, "with a residual the sum needs an output");
  if (!aligned(x, elem(dtype)) || !aligned(residual, elem(dtype)) || !aligned(h, elem(dtype)) || !aligned(weight, 4) ||
      !aligned(scale, 4))
    return fail(op, "a misaligned pointer");
  if (ldx < 0 || (residual && ldr < 0) || (rows > 1 && (ldq < d || (h && ldh < d))))
    return fail(op, "a row stride is negative or shorter than an output row");
  return run(op, device, [&] {
    return rms_norm_int8(x, ldx, residual, ldr, weight, eps, (OpsDtype)dtype, rows, d, q, ldq, scale, h, ldh,
                         (cudaStream_t)stream);
  });
}

int32_t qwen_asr_linear_int8(const int8_t* xq, int64_t ldx, const float* xs, const int8_t* wq, int64_t ldw,
                             const float* ws, int64_t m, int32_t n, int32_t k, int32_t epilogue, const void* residual,
                             int64_t ldr, void* out, int64_t ldo, int32_t dtype, int32_t device, void* stream) {
  const char* op = "linear_int8";
  if (!dtype_ok(dtype)) return fail(op, "dtype must be QWEN_ASR_F32 or QWEN_ASR_BF16");
  if (epilogue < QWEN_ASR_LINEAR_STORE || epilogue > QWEN_ASR_LINEAR_SWIGLU) return fail(op, "unknown epilogue");
  if (m < 0 || m > 0x7FFFFF00 || n < 1 || n > 0x7FFFFF00) return fail(op, "m or n is out of range");
  if (k < 1 || k > 131071) return fail(op, "k must be 1 .. 131071 (the sums are int32)");
  if (epilogue == QWEN_ASR_LINEAR_SWIGLU && n % 2) return fail(op, "SwiGLU needs an even n");
  if (m == 0) return 0;
  const int64_t width = epilogue == QWEN_ASR_LINEAR_SWIGLU ? n / 2 : n;
  if (!xq || !xs || !wq || !ws || !out) return fail(op, "a null pointer");
  if ((epilogue == QWEN_ASR_LINEAR_RESID) != (residual != nullptr))
    return fail(op, "the residual goes with the residual epilogue");
  if (!aligned(xq, 16) || !aligned(wq, 16) || ldx % 16 || ldw % 16)
    return fail(op, "int8 rows must start on 16-byte boundaries");
  if (ldx < k || ldw < k || ldo < width || (residual && ldr < width)) return fail(op, "a row stride is shorter than its row");
  if (ldx >= (1LL << 40) || ldw >= (1LL << 40)) return fail(op, "an int8 row stride of 2^40 or more");
  if (!aligned(out, elem(dtype)) || !aligned(residual, elem(dtype)) || !aligned(xs, 4) || !aligned(ws, 4))
    return fail(op, "a misaligned pointer");
  return run(op, device, [&] {
    return linear_int8(xq, ldx, xs, wq, ldw, ws, m, n, k, (LinearEpi)epilogue, residual, ldr, out, ldo,
                       (OpsDtype)dtype, ops_api_errors(), (cudaStream_t)stream);
  });
}

int32_t qwen_asr_kv8_append(const QwenAsrKv8* cache, const QwenAsrRows* k, const QwenAsrRows* v, int32_t dtype,
                            int32_t rows, const int32_t* starts, const int32_t* counts, int32_t index_stride,
                            int32_t device, void* stream) {
  const char* op = "kv8_append";
  if (const char* f = cache_fault(cache)) return fail(op, f);
  if (!dtype_ok(dtype)) return fail(op, "dtype must be QWEN_ASR_F32 or QWEN_ASR_BF16");
  if (rows < 0) return fail(op, "negative row count");
  if (rows == 0) return 0;
  if (!k || !v || !starts) return fail(op, "a null pointer");
  if (index_stride < 1) return fail(op, "index_stride must be positive");
  const int64_t width = (int64_t)cache->n_kv * cache->head_dim;
  if (const char* f = rows_fault(k, cache->n_seq, rows, width, dtype, false)) return fail(op, f);
  if (const char* f = rows_fault(v, cache->n_seq, rows, width, dtype, false)) return fail(op, f);
  return run(op, device, [&] {
    return kv8_append(cache_of(cache), k->data, k->seq_stride, k->row_stride, v->data, v->seq_stride, v->row_stride,
                      (OpsDtype)dtype, rows, starts, counts, index_stride, (cudaStream_t)stream);
  });
}

int32_t qwen_asr_kv8_read(const QwenAsrKv8* cache, const QwenAsrRows* k_out, const QwenAsrRows* v_out, int32_t dtype,
                          int32_t rows, const int32_t* starts, const int32_t* counts, int32_t index_stride,
                          int32_t device, void* stream) {
  const char* op = "kv8_read";
  if (const char* f = cache_fault(cache)) return fail(op, f);
  if (!dtype_ok(dtype)) return fail(op, "dtype must be QWEN_ASR_F32 or QWEN_ASR_BF16");
  if (rows < 0) return fail(op, "negative row count");
  if (rows == 0) return 0;
  if ((!k_out && !v_out) || !starts) return fail(op, "a null pointer");
  if (index_stride < 1) return fail(op, "index_stride must be positive");
  const int64_t width = (int64_t)cache->n_kv * cache->head_dim;
  const QwenAsrRows none{nullptr, 0, 0};
  if (k_out)
    if (const char* f = rows_fault(k_out, cache->n_seq, rows, width, dtype, true)) return fail(op, f);
  if (v_out)
    if (const char* f = rows_fault(v_out, cache->n_seq, rows, width, dtype, true)) return fail(op, f);
  const QwenAsrRows *ko = k_out ? k_out : &none, *vo = v_out ? v_out : &none;
  return run(op, device, [&] {
    return kv8_read(cache_of(cache), ko->data, ko->seq_stride, ko->row_stride, vo->data, vo->seq_stride,
                    vo->row_stride, (OpsDtype)dtype, rows, starts, counts, index_stride, (cudaStream_t)stream);
  });
}

int32_t qwen_asr_kv8_attention(const QwenAsrKv8* cache, const QwenAsrRows* q, const QwenAsrRows* out, int32_t dtype,
                               int32_t rows, int32_t heads, const int32_t* starts, const int32_t* counts,
                               int32_t index_stride, float scale, int32_t max_len, int32_t device, void* stream) {
  const char* op = "kv8_attention";
  if (const char* f = cache_fault(cache)) return fail(op, f);
  if (!dtype_ok(dtype)) return fail(op, "dtype must be QWEN_ASR_F32 or QWEN_ASR_BF16");
  if (heads < 1 || heads % cache->n_kv || heads / cache->n_kv > 256)
    return fail(op, "heads must be a multiple of n_kv, at most 256 times it");
  if (rows < 0 || rows > (1 << 22)) return fail(op, "rows must be 0 .. 2^22");
  if (rows == 0) return 0;
  if (!q || !out || !starts) return fail(op, "a null pointer");
  if (index_stride < 1) return fail(op, "index_stride must be positive");
  const int64_t width = (int64_t)heads * cache->head_dim;
  if (const char* f = rows_fault(q, cache->n_seq, rows, width, dtype, false)) return fail(op, f);
  if (const char* f = rows_fault(out, cache->n_seq, rows, width, dtype, true)) return fail(op, f);
  return run(op, device, [&] {
    return kv8_attention(cache_of(cache), q->data, q->seq_stride, q->row_stride, out->data, out->seq_stride,
                         out->row_stride, (OpsDtype)dtype, rows, heads, starts, counts, index_stride, scale, max_len,
                         ops_api_errors(), (cudaStream_t)stream);
  });
}

int32_t qwen_asr_ops_error(int32_t device) {
  const char* op = "ops_error";
  try {
    DeviceScope scope(device);
    if (!scope.ok()) return fail(op, "cannot use device " + std::to_string(device));
    // (reading the flags waits for the default stream alone)
    if (const cudaError_t s = cudaDeviceSynchronize()) {
      cudaGetLastError();
      return fail(op, std::string("cannot wait for the device: ") + cudaGetErrorString(s));
    }
    static std::mutex mutex;
    static int seen[64];  // errors of each device that an earlier call returned
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(op, "cannot use the current device");
    const std::lock_guard<std::mutex> lock(mutex);
    const int e = ops_errors(ops_api_errors(), seen[dev]);
    return e < 0 ? fail(op, "cannot read the device's error word") : e;
  } catch (const std::exception& ex) {
    return fail(op, ex.what());
  }
}

}  // extern "C"
