"""The 8-bit operators of the engine's int8 prefill and int8 KV cache on torch CUDA tensors.

    q, scale, h = rms_norm_int8(x, weight, eps, residual=r)     # int8 rows behind a norm
    y = linear_int8(q, scale, wq, ws)                           # int8 tensor-core product
    cache = kv8_cache(n_seq, n_kv, capacity, head_dim)
    kv8_append(cache, k, v, starts, counts)                     # quantised as it is written
    o = kv8_attention(q, cache, starts, counts)                 # attention over the int8 cache
    k, v = kv8_read(cache, starts, rows, counts)                # values read back

Calls run on the current stream of the tensors' device, enqueue and return; outputs are new
tensors. They keep no state and use no workspace, and can be captured into CUDA graphs. They
have no gradients: an input that requires one is refused. Arguments that do not fit raise
ValueError (TypeError for a wrong type) before anything is enqueued; a launch that CUDA refuses
raises RuntimeError. There is no CPU form.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple

import torch

from . import Kv8Desc, RowsDesc, last_error, lib

BLOCK = 16  # cache tokens that share a scale

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_FLOATS = (torch.float32, torch.bfloat16)


class Kv8Cache(NamedTuple):
    """An int8 KV cache: k and v int8 [n_seq, n_kv, capacity, head_dim], k_scale and v_scale f32
    [n_seq, n_kv, capacity / 16]. Slices along n_seq, or layers of a larger tensor, are caches too."""
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


def _tensor(t, name, dims, dtypes, device=None, shape=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, not {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, not {t.dim()}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which the 8-bit operators do not have")
    return t


def _rows2d(t, name):
    """Row stride of a matrix whose rows are contiguous."""
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: rows must be contiguous")
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _call(fn, *args):
    if fn(*args) != 0:
        raise RuntimeError(last_error())


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def rms_norm_int8(x, weight, eps: float = 1e-6, residual=None):
    """(q, scale, h) of x [rows, d] (f32 or bf16): h = x + residual in x's type (x itself without a
    residual), q int8 [rows, d] and scale f32 [rows] with q * scale[:, None] the RMS-normalised
    rows times weight (f32 [d]). q's row stride is d rounded up to 16, as linear_int8 wants it."""
    _tensor(x, "x", 2, _FLOATS)
    rows, d = x.shape
    _tensor(weight, "weight", 1, (torch.float32,), x.device, (d,))
    if residual is not None:
        _tensor(residual, "residual", 2, (x.dtype,), x.device, (rows, d))
    if not 1 <= d <= 32768:
        raise ValueError("d must be 1 .. 32768")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    w = weight if d == 1 or weight.stride(0) == 1 else weight.contiguous()
    ld = -(-d // 16) * 16
    q = torch.empty(rows, ld, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    h = x if residual is None else torch.empty(rows, d, dtype=x.dtype, device=x.device)
    ldx = _rows2d(x, "x")
    ldr = 0 if residual is None else _rows2d(residual, "residual")
    _call(lib().qwen_asr_rms_norm_int8, x.data_ptr(), ldx, None if residual is None else residual.data_ptr(), ldr,
          w.data_ptr(), eps, _DTYPES[x.dtype], rows, d, q.data_ptr(), ld, scale.data_ptr(),
          None if residual is None else h.data_ptr(), d, x.device.index, _stream(x.device))
    return (q if ld == d else q[:, :d]), scale, h


def linear_int8(xq, xs, wq, ws, residual=None, swiglu: bool = False, dtype=torch.float32):
    """xq int8 [m, k] with scales xs [m] times wq int8 [n, k] with scales ws [n]: [m, n] in `dtype`
    (f32 or bf16), with exact integer sums. residual [m, n] (in dtype) is added; swiglu takes the
    rows of wq as gate0, up0, gate1, ... and returns silu(gate) * up, [m, n / 2]. Rows of xq and wq
    start on 16-byte boundaries (row strides that are multiples of 16)."""
    _tensor(xq, "xq", 2, (torch.int8,))
    m, k = xq.shape
    dev = xq.device
    _tensor(wq, "wq", 2, (torch.int8,), dev)
    n = wq.shape[0]
    if wq.shape[1] != k:
        raise ValueError(f"xq has rows of {k} values, wq of {wq.shape[1]}")
    if dtype not in _DTYPES:
        raise TypeError(f"dtype must be torch.float32 or torch.bfloat16, not {dtype}")
    _tensor(xs, "xs", 1, (torch.float32,), dev, (m,))
    _tensor(ws, "ws", 1, (torch.float32,), dev, (n,))
    if not (xs.is_contiguous() and ws.is_contiguous()):
        raise ValueError("xs and ws must be contiguous")
    if residual is not None:
        _tensor(residual, "residual", 2, (dtype,), dev, (m, n))
        if swiglu:
            raise ValueError("swiglu and residual exclude each other")
    if not 1 <= k <= 131071:
        raise ValueError("k must be 1 .. 131071")
    if n < 1 or (swiglu and n % 2):
        raise ValueError("n must be positive, and even for swiglu")
    ldx, ldw = _rows2d(xq, "xq"), _rows2d(wq, "wq")
    if m == 1:
        ldx = -(-k // 16) * 16
    if n == 1:
        ldw = -(-k // 16) * 16
    if ldx % 16 or ldw % 16 or xq.data_ptr() % 16 or wq.data_ptr() % 16:
        raise ValueError("rows of xq and wq must start on 16-byte boundaries")
    width = n // 2 if swiglu else n
    out = torch.empty(m, width, dtype=dtype, device=dev)
    if m == 0:
        return out
    _call(lib().qwen_asr_linear_int8, xq.data_ptr(), ldx, xs.data_ptr(), wq.data_ptr(), ldw, ws.data_ptr(), m, n, k,
          2 if swiglu else 0 if residual is None else 1, None if residual is None else residual.data_ptr(),
          0 if residual is None else _rows2d(residual, "residual"), out.data_ptr(), width, _DTYPES[dtype], dev.index,
          _stream(dev))
    return out


def _cache(cache):
    k, v, ks, vs = cache
    _tensor(k, "cache.k", 4, (torch.int8,))
    n_seq, n_kv, cap, hd = k.shape
    dev = k.device
    _tensor(v, "cache.v", 4, (torch.int8,), dev, k.shape)
    _tensor(ks, "cache.k_scale", 3, (torch.float32,), dev, (n_seq, n_kv, cap // BLOCK))
    _tensor(vs, "cache.v_scale", 3, (torch.float32,), dev, (n_seq, n_kv, cap // BLOCK))
    if hd not in (64, 128):
        raise ValueError("head_dim must be 64 or 128")
    if cap < BLOCK or cap % BLOCK:
        raise ValueError("the capacity must be a positive multiple of 16")
    if k[0].is_contiguous() and v[0].is_contiguous() and ks[0].is_contiguous() and vs[0].is_contiguous():
        if n_seq == 1 or (k.stride(0) == v.stride(0) and ks.stride(0) == vs.stride(0)):
            return Kv8Desc(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), k.stride(0), ks.stride(0), n_seq,
                           n_kv, cap, hd), dev
    raise ValueError("each sequence of the cache must be contiguous, with the same strides for k and v")


def _index(t, name, dev, n_seq):
    _tensor(t, name, 1, (torch.int32,), dev, (n_seq,))
    if n_seq > 1 and t.stride(0) < 1:
        raise ValueError(f"{name} must not be an expanded tensor")
    return t


def _indices(starts, counts, dev, n_seq):
    """(starts, counts) with one stride for both."""
    _index(starts, "starts", dev, n_seq)
    if counts is not None:
        _index(counts, "counts", dev, n_seq)
        if n_seq > 1 and counts.stride(0) != starts.stride(0):
            starts, counts = starts.contiguous(), counts.contiguous()
    return starts, counts, (starts.stride(0) if n_seq > 1 else 1)


def _rows4d(t, name):
    if (t.shape[3] > 1 and t.stride(3) != 1) or (t.shape[2] > 1 and t.stride(2) != t.shape[3]):
        raise ValueError(f"{name}: the heads of a row must be contiguous")
    return RowsDesc(t.data_ptr(), t.stride(0), t.stride(1))


def kv8_append(cache: Kv8Cache, k, v, starts, counts=None) -> None:
    """Writes rows k and v [n_seq, rows, n_kv, head_dim] (f32 or bf16) behind position starts[b]
    (int32, on the device) of each sequence; counts[b] says how many of the rows it has (default
    all). The scale of a block of 16 tokens only grows while it fills, and what it holds is
    re-coded; rows past the capacity are dropped, and a negative start skips the sequence."""
    desc, dev = _cache(cache)
    _tensor(k, "k", 4, _FLOATS, dev)
    rows = k.shape[1]
    shape = (desc.n_seq, rows, desc.n_kv, desc.head_dim)
    _tensor(k, "k", 4, _FLOATS, dev, shape)
    _tensor(v, "v", 4, (k.dtype,), dev, shape)
    starts, counts, stride = _indices(starts, counts, dev, desc.n_seq)
    if rows == 0:
        return
    _call(lib().qwen_asr_kv8_append, C.byref(desc), C.byref(_rows4d(k, "k")), C.byref(_rows4d(v, "v")),
          _DTYPES[k.dtype], rows, starts.data_ptr(), None if counts is None else counts.data_ptr(), stride, dev.index,
          _stream(dev))


def kv8_read(cache: Kv8Cache, starts, rows: int, counts=None, dtype=torch.float32):
    """(k, v) [n_seq, rows, n_kv, head_dim]: the values of positions starts[b] + r, zeros from row
    counts[b] and from the capacity on."""
    desc, dev = _cache(cache)
    if dtype not in _DTYPES:
        raise TypeError(f"dtype must be torch.float32 or torch.bfloat16, not {dtype}")
    if rows < 0:
        raise ValueError("rows must not be negative")
    starts, counts, stride = _indices(starts, counts, dev, desc.n_seq)
    k = torch.empty(desc.n_seq, rows, desc.n_kv, desc.head_dim, dtype=dtype, device=dev)
    v = torch.empty_like(k)
    if rows:
        _call(lib().qwen_asr_kv8_read, C.byref(desc), C.byref(_rows4d(k, "k")), C.byref(_rows4d(v, "v")),
              _DTYPES[dtype], rows, starts.data_ptr(), None if counts is None else counts.data_ptr(), stride,
              dev.index, _stream(dev))
    return k, v


def kv8_attention(q, cache: Kv8Cache, starts, counts=None, scale: float | None = None, max_len: int = 0):
    """softmax(scale * q k^T) v of query rows q [n_seq, rows, heads, head_dim] (f32 or bf16) over
    the cache: row r of sequence b attends positions 0 .. starts[b] + r; rows from counts[b] on get
    zeros. scale defaults to 1 / sqrt(head_dim). max_len, an upper bound of starts + rows when the
    caller knows one, only shapes the launch."""
    desc, dev = _cache(cache)
    _tensor(q, "q", 4, _FLOATS, dev)
    rows, heads = q.shape[1], q.shape[2]
    _tensor(q, "q", 4, _FLOATS, dev, (desc.n_seq, rows, heads, desc.head_dim))
    if heads < 1 or heads % desc.n_kv or heads > 256 * desc.n_kv:
        raise ValueError(f"{heads} query heads do not fit {desc.n_kv} cached ones")
    starts, counts, stride = _indices(starts, counts, dev, desc.n_seq)
    if scale is None:
        scale = 1.0 / math.sqrt(desc.head_dim)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if rows:
        _call(lib().qwen_asr_kv8_attention, C.byref(desc), C.byref(_rows4d(q, "q")), C.byref(_rows4d(out, "out")),
              _DTYPES[q.dtype], rows, heads, starts.data_ptr(), None if counts is None else counts.data_ptr(), stride,
              scale, max_len, dev.index, _stream(dev))
    return out


def check(device=None) -> None:
    """Raises RuntimeError when a bounded wait inside linear_int8 gave up since the last check (its
    output is then not to be used). Waits for the device."""
    index = torch.cuda.current_device() if device is None else torch.device(device).index
    e = lib().qwen_asr_ops_error(-1 if index is None else index)
    if e:
        raise RuntimeError(f"linear_int8: a device-side wait timed out (code {e})")
