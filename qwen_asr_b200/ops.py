"""The 8-bit operators of the engine's int8 prefill and int8 KV cache on torch CUDA tensors.

    q, scale, h = rms_norm_int8(x, weight, eps, residual=r)     # int8 rows behind a norm
    y = linear_int8(q, scale, wq, ws)                           # int8 tensor-core product
    cache = kv8_cache(n_seq, n_kv, capacity, head_dim)
    kv8_append(cache, k, v, starts, counts)                     # quantised as it is written
    o = kv8_attention(q, cache, starts, counts)                 # attention over the int8 cache
    k, v = kv8_read(cache, starts, rows, counts)                # values read back

Calls run on the current stream of the tensors' device, enqueue and return; outputs are new
tensors. They keep no state and use no workspace, and can be captured into CUDA graphs. They
have no gradients: an input that requires one, or carries a forward-mode tangent, is refused, and
kv8_append counts as an in-place change of the cache. Arguments that do not fit raise
ValueError (TypeError for a wrong type) before anything is enqueued; a launch that CUDA refuses
raises RuntimeError. There is no CPU form.
"""
from __future__ import annotations

import math
import struct
from operator import index
from typing import NamedTuple

import torch
from torch.autograd import forward_ad as _forward_ad
from torch.autograd.graph import increment_version as _increment_version

from . import last_error, lib

try:
    from . import _ops_fast as _fast  # the same calls made in C++ (binding/ops_fast.cpp)
except ImportError:  # not built, or for another torch: every call takes the ctypes path below
    _fast = None

BLOCK = 16  # cache tokens that share a scale

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_FLOATS = (torch.float32, torch.bfloat16)
_MAX_INT32 = 2 ** 31 - 1
_F32, _INT8, _INT32 = torch.float32, torch.int8, torch.int32
_KV8 = struct.Struct("@PPPPqqiiii")  # QwenAsrKv8
_ROWS = struct.Struct("@Pqq")        # QwenAsrRows
_grad = torch.is_grad_enabled
_raw_stream = torch._C._cuda_getCurrentRawStream  # the current stream's handle, without a Stream object


class Kv8Cache(NamedTuple):
    """An int8 KV cache: k and v int8 [n_seq, n_kv, capacity, head_dim], k_scale and v_scale f32
    [n_seq, n_kv, capacity / 16], not negative. Slices along n_seq, or layers of a larger tensor, are caches too."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def kv8_cache(n_seq: int, n_kv: int, capacity: int, head_dim: int = 128, device="cuda") -> Kv8Cache:
    """A new, empty cache; capacity is rounded up to a multiple of 16."""
    capacity = -(-capacity // BLOCK) * BLOCK
    q = [torch.zeros(n_seq, n_kv, capacity, head_dim, dtype=torch.int8, device=device) for _ in range(2)]
    s = [torch.zeros(n_seq, n_kv, capacity // BLOCK, device=device) for _ in range(2)]
    return Kv8Cache(*q, *s)


def _derives(t):
    """Whether the call would have to differentiate: t requires a gradient, or has a tangent."""
    if t.requires_grad and _grad():
        return True
    return _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None


# An ordinary call is checked and made in C++, which answers None to any other: unusual strides and
# sizes, which ctypes handles here, and arguments that do not fit, which are named here.
def _tensor(t, name, dims, dtypes, device=None, shape=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, not {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device")
    if device is not None and t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, not on cuda:{device}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, not {t.dim()}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if _derives(t):
        raise ValueError(f"{name} requires a gradient or has a tangent, which the 8-bit operators do not have")
    if t.is_neg():
        raise ValueError(f"{name} is a negated view (resolve_neg() makes a tensor of it)")
    return t


def _is(t, dtype, device, shape):
    return (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == device and t.shape == shape
            and not _derives(t) and not t.is_neg())


def _pitch(t, name):
    """Row stride of a matrix whose rows are contiguous."""
    ld, one = t.stride()
    rows, width = t.shape
    if one != 1 and width > 1:
        raise ValueError(f"{name}: rows must be contiguous")
    return ld if rows > 1 else max(ld, width)


def _failed():
    """Raises what the library refused: RuntimeError where CUDA did, ValueError for the arguments."""
    why = last_error()
    raise (RuntimeError if "launch failed" in why or "cannot use device" in why else ValueError)(why)


def rms_norm_int8(x, weight, eps: float = 1e-6, residual=None):
    """(q, scale, h) of x [rows, d] (f32 or bf16): h = x + residual in x's type (x itself without a
    residual), q int8 [rows, d] and scale f32 [rows] with q * scale[:, None] the RMS-normalised
    rows times weight (f32 [d]). q's row stride is d rounded up to 16, as linear_int8 wants it."""
    if _fast is not None:
        out = _fast.rms_norm_int8(x, weight, eps, residual)
        if out is not None:
            return out
    _x = isinstance(x, torch.Tensor)
    code = _DTYPES.get(x.dtype) if _x else None
    if code is None or x.dim() != 2 or not x.is_cuda or _derives(x) or x.is_neg():
        _tensor(x, "x", 2, _FLOATS)
    dev, shape, dtype = x.get_device(), x.shape, x.dtype
    rows, d = shape
    if not _is(weight, _F32, dev, (d,)):
        _tensor(weight, "weight", 1, (_F32,), dev, (d,))
    if not 1 <= d <= 32768:
        raise ValueError("d must be 1 .. 32768")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    if d > 1 and weight.stride(0) != 1:
        weight = weight.contiguous()
    ld = -(-d // 16) * 16
    q = torch.empty((rows, ld), dtype=_INT8, device=x.device)
    scale = torch.empty(rows, dtype=_F32, device=x.device)
    if residual is None:
        h, hp, rp, ldr = x, None, None, 0
    else:
        if not _is(residual, dtype, dev, shape):
            _tensor(residual, "residual", 2, (dtype,), dev, shape)
        h = torch.empty(shape, dtype=dtype, device=x.device)
        hp, rp, ldr = h.data_ptr(), residual.data_ptr(), _pitch(residual, "residual")
    if lib().qwen_asr_rms_norm_int8(x.data_ptr(), _pitch(x, "x"), rp, ldr, weight.data_ptr(), eps, code, rows, d,
                                    q.data_ptr(), ld, scale.data_ptr(), hp, d, dev, _raw_stream(dev)):
        _failed()
    return (q if ld == d else q[:, :d]), scale, h


def linear_int8(xq, xs, wq, ws, residual=None, swiglu: bool = False, dtype=torch.float32):
    """xq int8 [m, k] with scales xs [m] times wq int8 [n, k] with scales ws [n]: [m, n] in `dtype`
    (f32 or bf16), with exact integer sums. residual [m, n] (in dtype) is added; swiglu takes the
    rows of wq as gate0, up0, gate1, ... and returns silu(gate) * up, [m, n / 2]. Rows of xq and wq
    start on 16-byte boundaries (row strides that are multiples of 16)."""
    if _fast is not None and dtype in _DTYPES:
        out = _fast.linear_int8(xq, xs, wq, ws, residual, bool(swiglu), dtype is torch.bfloat16)
        if out is not None:
            return out
    if not (isinstance(xq, torch.Tensor) and xq.dtype is _INT8 and xq.is_cuda and xq.dim() == 2 and not xq.is_neg()):
        _tensor(xq, "xq", 2, (_INT8,))
    dev, (m, k) = xq.get_device(), xq.shape
    if not (isinstance(wq, torch.Tensor) and wq.dtype is _INT8 and wq.get_device() == dev and wq.dim() == 2
            and not wq.is_neg()):
        _tensor(wq, "wq", 2, (_INT8,), dev)
    n = wq.shape[0]
    if wq.shape[1] != k:
        raise ValueError(f"xq has rows of {k} values, wq of {wq.shape[1]}")
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"dtype must be torch.float32 or torch.bfloat16, not {dtype}")
    if not (_is(xs, _F32, dev, (m,)) and _is(ws, _F32, dev, (n,))):
        _tensor(xs, "xs", 1, (_F32,), dev, (m,))
        _tensor(ws, "ws", 1, (_F32,), dev, (n,))
    if not (xs.is_contiguous() and ws.is_contiguous()):
        raise ValueError("xs and ws must be contiguous")
    if not 1 <= k <= 131071:
        raise ValueError("k must be 1 .. 131071")
    if n < 1 or (swiglu and n % 2):
        raise ValueError("n must be positive, and even for swiglu")
    epi, rp, ldr, width = 0, None, 0, n
    if swiglu:
        epi, width = 2, n // 2
    if residual is not None:
        if not _is(residual, dtype, dev, (m, n)):
            _tensor(residual, "residual", 2, (dtype,), dev, (m, n))
        if swiglu:
            raise ValueError("swiglu and residual exclude each other")
        epi, rp, ldr = 1, residual.data_ptr(), _pitch(residual, "residual")
    k16 = -(-k // 16) * 16
    ldx = _pitch(xq, "xq") if m > 1 else k16 if k == 1 or xq.stride(1) == 1 else _pitch(xq, "xq")
    ldw = _pitch(wq, "wq") if n > 1 else k16 if k == 1 or wq.stride(1) == 1 else _pitch(wq, "wq")
    xp, wp = xq.data_ptr(), wq.data_ptr()
    if (ldx | ldw | xp | wp) & 15:
        raise ValueError("rows of xq and wq must start on 16-byte boundaries")
    out = torch.empty((m, width), dtype=dtype, device=xq.device)
    if m and lib().qwen_asr_linear_int8(xp, ldx, xs.data_ptr(), wp, ldw, ws.data_ptr(), m, n, k, epi, rp, ldr,
                                        out.data_ptr(), width, code, dev, _raw_stream(dev)):
        _failed()
    return out


def _cache(cache):
    """(descriptor, device, n_seq, n_kv, head_dim) of a cache."""
    k, v, ks, vs = cache
    try:
        shape, st, ss = k.shape, k.stride(), ks.stride()
        n, h, cap, hd = shape
        dev, blocks = k.get_device(), cap // BLOCK
        if (k.dtype is _INT8 and v.dtype is _INT8 and ks.dtype is _F32 and vs.dtype is _F32 and v.shape == shape
                and v.stride() == st and st[1:] == (cap * hd, hd, 1) and ks.shape == (n, h, blocks)
                and vs.shape == ks.shape and vs.stride() == ss and ss[1:] == (blocks, 1) and (hd == 128 or hd == 64)
                and blocks > 0 and cap == blocks * BLOCK and dev >= 0 and v.get_device() == dev
                and ks.get_device() == dev and vs.get_device() == dev
                and not (_derives(ks) or _derives(vs)) and not any(t.is_neg() for t in cache)):
            return (_KV8.pack(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), st[0], ss[0], n, h, cap, hd),
                    dev, n, h, hd)
    except (AttributeError, ValueError):
        pass
    _tensor(k, "cache.k", 4, (_INT8,))
    n, h, cap, hd = k.shape
    dev = k.get_device()
    _tensor(v, "cache.v", 4, (_INT8,), dev, k.shape)
    _tensor(ks, "cache.k_scale", 3, (_F32,), dev, (n, h, cap // BLOCK))
    _tensor(vs, "cache.v_scale", 3, (_F32,), dev, (n, h, cap // BLOCK))
    if hd not in (64, 128):
        raise ValueError("head_dim must be 64 or 128")
    if cap < BLOCK or cap % BLOCK:
        raise ValueError("the capacity must be a positive multiple of 16")
    if n < 1 or h < 1:
        raise ValueError("a cache needs a sequence and a head")
    if all(t[0].is_contiguous() for t in (k, v, ks, vs)) and (
            n == 1 or (k.stride(0) == v.stride(0) and ks.stride(0) == vs.stride(0))):
        return (_KV8.pack(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), k.stride(0), ks.stride(0), n, h,
                          cap, hd), dev, n, h, hd)
    raise ValueError("each sequence of the cache must be contiguous, with the same strides for k and v")


def _indices(starts, counts, dev, n):
    """(starts, counts, address of starts, of counts or None, their stride)."""
    if not _is(starts, _INT32, dev, (n,)):
        _tensor(starts, "starts", 1, (_INT32,), dev, (n,))
    stride = starts.stride(0) if n > 1 else 1
    if stride > _MAX_INT32:
        starts, stride = starts.contiguous(), 1
    if counts is not None:
        if not _is(counts, _INT32, dev, (n,)):
            _tensor(counts, "counts", 1, (_INT32,), dev, (n,))
        if n > 1 and counts.stride(0) != stride:
            starts, counts, stride = starts.contiguous(), counts.contiguous(), 1
    if stride < 1:
        raise ValueError("starts and counts must not be expanded tensors")
    return starts, counts, starts.data_ptr(), None if counts is None else counts.data_ptr(), stride


def _rows(t, name):
    """Descriptor of rows [n_seq, rows, heads, head_dim] whose heads are contiguous."""
    seq, row, head, one = t.stride()
    if (one != 1 and t.shape[3] > 1) or (head != t.shape[3] and t.shape[2] > 1):
        raise ValueError(f"{name}: the heads of a row must be contiguous")
    return _ROWS.pack(t.data_ptr(), seq, row)


def kv8_append(cache: Kv8Cache, k, v, starts, counts=None) -> None:
    """Writes rows k and v [n_seq, rows, n_kv, head_dim] (f32 or bf16) behind position starts[b]
    (int32, on the device) of each sequence; counts[b] says how many of the rows it has (default
    all). The scale of a block of 16 tokens only grows while it fills, and what it holds is
    re-coded; rows past the capacity are dropped, and a negative start skips the sequence."""
    if _fast is not None and _fast.kv8_append(cache, k, v, starts, counts):
        return
    desc, dev, n, h, hd = _cache(cache)
    code = _DTYPES.get(k.dtype) if isinstance(k, torch.Tensor) else None
    if code is None or k.dim() != 4:
        _tensor(k, "k", 4, _FLOATS, dev)
    rows = k.shape[1]
    if rows > _MAX_INT32:
        raise ValueError("k has 2^31 rows or more")
    shape = (n, rows, h, hd)
    if not (_is(k, k.dtype, dev, shape) and _is(v, k.dtype, dev, shape)):
        _tensor(k, "k", 4, _FLOATS, dev, shape)
        _tensor(v, "v", 4, (k.dtype,), dev, shape)
    starts, counts, sp, cp, stride = _indices(starts, counts, dev, n)
    if rows and lib().qwen_asr_kv8_append(desc, _rows(k, "k"), _rows(v, "v"), code, rows, sp, cp, stride, dev,
                                          _raw_stream(dev)):
        _failed()
    if rows:
        _increment_version([t for t in cache if not t.is_inference()])


def kv8_read(cache: Kv8Cache, starts, rows: int, counts=None, dtype=torch.float32):
    """(k, v) [n_seq, rows, n_kv, head_dim]: the values of positions starts[b] + r, zeros from row
    counts[b] and from the capacity on."""
    if _fast is not None and dtype in _DTYPES:
        out = _fast.kv8_read(cache, starts, rows, counts, dtype is torch.bfloat16)
        if out is not None:
            return out
    desc, dev, n, h, hd = _cache(cache)
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"dtype must be torch.float32 or torch.bfloat16, not {dtype}")
    rows = index(rows)
    if not 0 <= rows <= _MAX_INT32:
        raise ValueError("rows must be 0 .. 2^31 - 1")
    starts, counts, sp, cp, stride = _indices(starts, counts, dev, n)
    k = torch.empty((n, rows, h, hd), dtype=dtype, device=starts.device)
    v = torch.empty_like(k)
    width = h * hd
    if rows and lib().qwen_asr_kv8_read(desc, _ROWS.pack(k.data_ptr(), rows * width, width),
                                        _ROWS.pack(v.data_ptr(), rows * width, width), code, rows, sp, cp, stride,
                                        dev, _raw_stream(dev)):
        _failed()
    return k, v


def kv8_attention(q, cache: Kv8Cache, starts, counts=None, scale: float | None = None, max_len: int = 0):
    """softmax(scale * q k^T) v of query rows q [n_seq, rows, heads, head_dim] (f32 or bf16) over
    the cache: row r of sequence b attends positions 0 .. starts[b] + r; rows from counts[b] on get
    zeros. scale defaults to 1 / sqrt(head_dim). max_len, an upper bound of starts + rows when the
    caller knows one, only shapes the launch: worth giving where the capacity is far larger (f32: 381
    rows from 0 in a cache of 2048 take 24 us without it, 16 with)."""
    if _fast is not None:
        out = _fast.kv8_attention(q, cache, starts, counts, scale, max_len)
        if out is not None:
            return out
    desc, dev, n, h, hd = _cache(cache)
    code = _DTYPES.get(q.dtype) if isinstance(q, torch.Tensor) else None
    if code is None or q.dim() != 4:
        _tensor(q, "q", 4, _FLOATS, dev)
    shape = q.shape
    rows, heads = shape[1], shape[2]
    if rows > 1 << 22:
        raise ValueError("q must have at most 2^22 rows")
    max_len = index(max_len)
    if not 0 <= max_len <= cache[0].shape[2]:
        max_len = 0  # (no bound: the capacity)
    if shape != (n, rows, heads, hd) or q.get_device() != dev or _derives(q) or q.is_neg():
        _tensor(q, "q", 4, _FLOATS, dev, (n, rows, heads, hd))
    if heads < 1 or heads % h or heads > 256 * h:
        raise ValueError(f"{heads} query heads do not fit {h} cached ones")
    starts, counts, sp, cp, stride = _indices(starts, counts, dev, n)
    scale = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    out = torch.empty(shape, dtype=q.dtype, device=q.device)
    width = heads * hd
    if rows and lib().qwen_asr_kv8_attention(desc, _rows(q, "q"), _ROWS.pack(out.data_ptr(), rows * width, width),
                                             code, rows, heads, sp, cp, stride, scale, max_len, dev,
                                             _raw_stream(dev)):
        _failed()
    return out


def check(device=None) -> None:
    """Raises RuntimeError when a bounded wait inside linear_int8 or kv8_attention gave up since the
    last check (outputs since then are not to be used), or when the device cannot be asked. Waits
    for all of the device's streams."""
    index = torch.cuda.current_device() if device is None else torch.device(device).index
    e = lib().qwen_asr_ops_error(-1 if index is None else index)
    if e < 0:
        raise RuntimeError(f"8-bit operators: {last_error()}")
    if e:
        raise RuntimeError(f"8-bit operators: a device-side wait timed out (code {e})")
