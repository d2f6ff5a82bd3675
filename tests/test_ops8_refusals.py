"""The 8-bit operators' C entry points refuse what they cannot run, before anything is enqueued: every
call here has one argument wrong and must return -1 with the reason (no GPU is needed for that)."""
import struct

import pytest

import qwen_asr_b200 as Q

P = 1 << 20  # an address that is never read: the call is refused first


def norm(**kw):
    a = dict(x=P, ldx=64, residual=P, ldr=64, weight=P, eps=1e-6, dtype=0, rows=4, d=64, q=P, ldq=64, scale=P, h=P,
             ldh=64, device=-1, stream=None)
    a.update(kw)
    return Q.lib().qwen_asr_rms_norm_int8(*a.values())


def linear(**kw):
    a = dict(xq=P, ldx=64, xs=P, wq=P, ldw=64, ws=P, m=4, n=8, k=64, epilogue=0, residual=None, ldr=0, out=P, ldo=8,
             dtype=0, device=-1, stream=None)
    a.update(kw)
    return Q.lib().qwen_asr_linear_int8(*a.values())


def cache(**kw):
    a = dict(k=P, v=P, k_scale=P, v_scale=P, seq_stride=2 * 32 * 128, scale_stride=4, n_seq=2, n_kv=2, capacity=32,
             head_dim=128)
    a.update(kw)
    return struct.pack("@PPPPqqiiii", *(x or 0 for x in a.values()))


def rows(data=P, seq=256, row=256):
    return struct.pack("@Pqq", data or 0, seq, row)


def append(c=None, k=None, v=None, dtype=0, n=1, starts=P, counts=None, stride=1):
    return Q.lib().qwen_asr_kv8_append(c or cache(), k or rows(), v or rows(), dtype, n, starts, counts, stride, -1, None)


def read(c=None, k=None, v=None, dtype=0, n=1, starts=P, stride=1):
    return Q.lib().qwen_asr_kv8_read(c or cache(), k, v, dtype, n, starts, None, stride, -1, None)


def attend(c=None, q=None, out=None, dtype=0, n=1, heads=4, starts=P, stride=1):
    return Q.lib().qwen_asr_kv8_attention(c or cache(), q or rows(seq=512, row=512), out or rows(seq=512, row=512),
                                          dtype, n, heads, starts, None, stride, 0.1, 0, -1, None)


CASES = [
    (lambda: norm(dtype=2), "dtype"), (lambda: norm(d=0), "d must"), (lambda: norm(d=32769), "d must"),
    (lambda: norm(rows=-1), "rows"), (lambda: norm(rows=1 << 31), "rows"), (lambda: norm(eps=-1.0), "eps"),
    (lambda: norm(eps=float("nan")), "eps"), (lambda: norm(x=None), "null"), (lambda: norm(weight=None), "null"),
    (lambda: norm(q=None), "null"), (lambda: norm(scale=None), "null"), (lambda: norm(h=None), "residual"),
    (lambda: norm(x=P + 2), "misaligned"), (lambda: norm(scale=P + 1), "misaligned"), (lambda: norm(ldq=63), "stride"),
    (lambda: norm(ldh=63), "stride"), (lambda: norm(ldx=-64), "stride"),
    (lambda: linear(dtype=-1), "dtype"), (lambda: linear(epilogue=3), "epilogue"), (lambda: linear(m=-1), "range"),
    (lambda: linear(n=0), "range"), (lambda: linear(k=0), "k must"), (lambda: linear(k=131072), "k must"),
    (lambda: linear(epilogue=2, n=7), "even"), (lambda: linear(xq=None), "null"), (lambda: linear(out=None), "null"),
    (lambda: linear(epilogue=1), "residual"), (lambda: linear(residual=P, ldr=8), "residual"),
    (lambda: linear(xq=P + 8), "16-byte"), (lambda: linear(ldw=72), "16-byte"), (lambda: linear(ldx=48), "shorter"),
    (lambda: linear(ldo=7), "shorter"), (lambda: linear(epilogue=1, residual=P, ldr=4), "shorter"),
    (lambda: linear(out=P + 2), "misaligned"), (lambda: linear(ldx=1 << 40), "2^40"),
    (lambda: append(c=cache(k=None)), "null"), (lambda: append(c=cache(n_seq=0)), "n_seq"),
    (lambda: append(c=cache(n_seq=65536)), "n_seq"), (lambda: append(c=cache(n_kv=0)), "n_kv"),
    (lambda: append(c=cache(head_dim=96)), "head_dim"), (lambda: append(c=cache(capacity=40)), "capacity"),
    (lambda: append(c=cache(capacity=0)), "capacity"), (lambda: append(c=cache(v=P + 4)), "16-byte"),
    (lambda: append(c=cache(seq_stride=2 * 32 * 128 - 16)), "seq_stride"), (lambda: append(c=cache(seq_stride=0)), "seq_stride"),
    (lambda: append(c=cache(seq_stride=2 * 32 * 128 + 8)), "seq_stride"), (lambda: append(c=cache(scale_stride=3)), "scale_stride"),
    (lambda: append(dtype=9), "dtype"), (lambda: append(n=-1), "row count"), (lambda: append(starts=None), "null"),
    (lambda: append(stride=0), "index_stride"), (lambda: append(k=rows(data=None)), "null"),
    (lambda: append(v=rows(data=P + 1)), "misaligned"), (lambda: append(k=rows(row=-1)), "negative"),
    (lambda: read(), "null"), (lambda: read(k=rows(seq=128)), "overlapping"), (lambda: read(k=rows(row=128), n=2), "overlapping"),
    (lambda: read(k=rows(seq=0)), "overlapping"), (lambda: read(v=rows(), stride=-1), "index_stride"),
    (lambda: attend(heads=3), "heads"), (lambda: attend(heads=0), "heads"), (lambda: attend(heads=1024), "heads"),
    (lambda: attend(n=-1), "rows"), (lambda: attend(n=(1 << 22) + 1), "rows"), (lambda: attend(starts=None), "null"),
    (lambda: attend(out=rows(seq=256, row=512)), "overlapping"), (lambda: attend(out=rows(seq=2048, row=256), n=2), "overlapping"),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_refused_with_the_reason(i):
    call, why = CASES[i]
    assert call() == -1
    assert why in Q.last_error(), Q.last_error()


def test_nothing_to_do_is_no_error():
    assert norm(rows=0) == 0 and linear(m=0) == 0
    assert append(n=0) == 0 and read(k=rows(), n=0) == 0 and attend(n=0) == 0


def test_tensors_off_the_gpu_are_refused():
    torch = pytest.importorskip("torch")
    from qwen_asr_b200 import ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.rms_norm_int8(torch.zeros(2, 8), torch.ones(8))
    with pytest.raises(ValueError, match="CUDA"):
        ops.linear_int8(torch.zeros(2, 16, dtype=torch.int8), torch.ones(2), torch.zeros(2, 16, dtype=torch.int8), torch.ones(2))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv8_cache(1, 1, 16, 64, device="cpu") and ops.kv8_read(
            ops.kv8_cache(1, 1, 16, 64, device="cpu"), torch.zeros(1, dtype=torch.int32), 1)


def test_library_refusals_are_value_errors():
    pytest.importorskip("torch")
    from qwen_asr_b200 import ops
    assert append(n=-1) == -1
    with pytest.raises(ValueError, match="row count"):
        ops._failed()
