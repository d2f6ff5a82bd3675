"""The 8-bit operators (qwen_asr_b200.ops) against their definitions in 64 bits: int8 rows, sums and
scales are compared exactly, results in f32 / bf16 with the rounding they are allowed (half a step
of the type, and what the formula beside each test adds up)."""
import math
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}  # largest relative error of a rounding


@pytest.fixture(params=["binding", "ctypes"])
def ops(request, monkeypatch):
    """The operators through the C++ binding, and through ctypes as where it is not built."""
    from qwen_asr_b200 import ops
    if request.param == "ctypes":
        monkeypatch.setattr(ops, "_fast", None)
    return ops


def test_binding_is_built_and_takes_ordinary_calls():
    from qwen_asr_b200 import ops
    x, w = rand(3, 64), rand(64)
    q, s, _ = ops._fast.rms_norm_int8(x, w, 1e-6, x)
    assert ops._fast.linear_int8(q, s, q, s, None, False, True).dtype == BF16
    c = ops.kv8_cache(2, 2, 32, 64)
    z = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert ops._fast.kv8_append(c, rand(2, 1, 2, 64), rand(2, 1, 2, 64), z, None) is True
    assert ops._fast.kv8_attention(rand(2, 1, 4, 64), c, z, None, None, 0).shape == (2, 1, 4, 64)
    assert len(ops._fast.kv8_read(c, z, 1, None, False)) == 2
    # and leaves the others, with their errors, to the caller
    assert ops._fast.rms_norm_int8(x.half(), w, 1e-6, None) is None
    assert ops._fast.rms_norm_int8(x.clone().requires_grad_(), w, 1e-6, None) is None
    assert ops._fast.linear_int8(q, s, q[:, :32], s, None, False, False) is None
    assert ops._fast.kv8_append(c, rand(2, 1, 2, 64), rand(2, 1, 2, 64).to(BF16), z, None) is None
    assert ops._fast.kv8_attention(rand(2, 1, 3, 64), c, z, None, None, 0) is None
    assert ops._fast.kv8_read(c, z.cpu(), 1, None, False) is None


def rand(*shape, seed=0, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + sum(shape))
    return torch.randn(*shape, generator=g, device="cuda") * std


# ------------------------------------------------------------------ RMSNorm -> int8
def norm_ref(x, w, eps, r):
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    u = h.double() * w.double()
    top = u.abs().amax(1, keepdim=True)
    some = torch.where(top > 0, top, torch.ones_like(top))
    q = torch.round(u * 127.0 / some)
    rms = torch.sqrt((h.double() ** 2).mean(1, keepdim=True) + eps)
    scale = torch.where(top > 0, top / rms / 127.0, torch.ones_like(top))
    return h, q, scale[:, 0]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (1, 64), (5, 333), (2, 1000), (1, 1024), (381, 2048), (33, 2052),
                                    (7, 4096), (300, 8192), (2, 16384), (3, 16392), (2, 32768), (4097, 256)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_rows(ops, dt, rows, d, residual):
    x, w = rand(rows, d, seed=1).to(dt), 1 + rand(d, seed=2, std=0.1)
    x[:, : max(1, d // 50)] *= 30  # strong channels, as residual streams have
    r = rand(rows, d, seed=3).to(dt) if residual else None
    q, scale, h = ops.rms_norm_int8(x, w, 1e-6, residual=r)
    rh, rq, rs = norm_ref(x, w, 1e-6, r)
    assert torch.equal(h, rh)
    assert torch.equal(q.double(), rq)
    assert q.stride(0) % 16 == 0 or rows == 1
    # scale: an f64 expression rounded once; its f64 sums differ by far less than half an f32 step
    assert ((scale.double() - rs).abs() <= rs * 2 ** -23).all()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("rows,d", [(3, 5), (9, 513), (1000, 2047), (5, 2049), (7, 8191), (3, 8193)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_rows_of_odd_lengths(ops, dt, rows, d, residual):
    """Rows without a common alignment, read value by value; also those of a wider matrix."""
    wide = rand(rows, d + 3, seed=31).to(dt)
    w = 1 + rand(d, seed=32, std=0.1)
    r = rand(rows, d, seed=33).to(dt) if residual else None
    for x in (wide[:, 1:d + 1].contiguous(), wide[:, 1:d + 1]):
        q, scale, h = ops.rms_norm_int8(x, w, 1e-6, residual=r)
        rh, rq, rs = norm_ref(x, w, 1e-6, r)
        assert torch.equal(h, rh) and torch.equal(q.double(), rq)
        assert ((scale.double() - rs).abs() <= rs * 2 ** -23).all()  # as above


def test_norm_special_rows_of_odd_length(ops):
    """As the special rows below, on the path that reads value by value, in bf16 too."""
    d = 1023
    for dt in (F32, BF16):
        x = rand(7, d, seed=34)
        x[1], x[2, 5], x[3, d - 1], x[6, 0] = 0, math.nan, math.inf, -math.inf
        x[4] *= 1e-39
        x[5] *= 1e30
        x, w = x.to(dt), torch.ones(d, device="cuda")
        q, scale, h = ops.rms_norm_int8(x, w, 1e-6)
        _, rq, rs = norm_ref(x, w, 1e-6, None)
        for i in (0, 1, 4, 5):
            assert torch.equal(q[i].double(), rq[i]), i
            # (a subnormal scale is rounded to 2^-149)
            assert abs(scale[i].double() - rs[i]) <= rs[i] * 2 ** -23 + 2.0 ** -149, i
        assert scale[1] == 1 and not q[1].any()
        for i in (2, 3, 6):
            assert torch.isnan(scale[i]) and not q[i].any()


def test_norm_exact_ties(ops):
    """Values whose quotient is exactly a half round to even, as in 64 bits."""
    x = torch.zeros(2, 256, device="cuda")
    x[0, 0], x[1, 0] = 254.0, -254.0
    x[0, 1:200] = torch.arange(1, 200, device="cuda", dtype=F32)  # u * 127 / 254 = n / 2
    x[1, 1:200] = -x[0, 1:200]
    w = torch.ones(256, device="cuda")
    q, _, _ = ops.rms_norm_int8(x, w, 0.0)
    assert torch.equal(q.double(), norm_ref(x, w, 0.0, None)[1])
    assert q[0, 1].item() == 0 and q[0, 3].item() == 2 and q[0, 5].item() == 2


@pytest.mark.parametrize("d", [333, 1024])
def test_norm_special_rows(ops, d):
    """Rows of zeros, of NaN and infinity, of subnormals and of huge values."""
    x = rand(8, d, seed=4)
    x[1] = 0
    x[2, 5] = math.nan
    x[3, d - 1] = math.inf
    x[4] *= 1e-42
    x[5] *= 1e30
    x[6, 0] = -math.inf
    w = torch.ones(d, device="cuda")
    q, scale, h = ops.rms_norm_int8(x, w, 1e-6)
    _, rq, rs = norm_ref(x, w, 1e-6, None)
    for i in (0, 1, 4, 5, 7):
        assert torch.equal(q[i].double(), rq[i]), i
        # (a subnormal scale is rounded to 2^-149)
        assert abs(scale[i].double() - rs[i]) <= rs[i] * 2 ** -23 + 2.0 ** -149, i
    assert scale[1] == 1 and not q[1].any()
    for i in (2, 3, 6):
        assert torch.isnan(scale[i]) and not q[i].any()


def test_norm_strided_and_in_place(ops):
    from qwen_asr_b200 import lib
    big = rand(20, 3, 640, seed=5)
    x, r = big[:, 1, 3:603], big[:, 2, :600]  # odd offset: the scalar path
    w = (1 + rand(1200, seed=6, std=0.1))[::2]
    q, scale, h = ops.rms_norm_int8(x, w, 1e-5, residual=r)
    rh, rq, rs = norm_ref(x, w, 1e-5, r)
    assert torch.equal(h, rh) and torch.equal(q.double(), rq)
    # the sum written over x, and q rows wider than the row keep what is behind it
    x2 = x.contiguous()
    q2 = torch.full((20, 640), 99, dtype=torch.int8, device="cuda")
    s2 = torch.empty(20, device="cuda")
    wc = w.contiguous()
    rc = r.contiguous()
    assert lib().qwen_asr_rms_norm_int8(x2.data_ptr(), 600, rc.data_ptr(), 600, wc.data_ptr(), 1e-5, 0, 20, 600,
                                        q2.data_ptr(), 640, s2.data_ptr(), x2.data_ptr(), 600, -1,
                                        torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(x2, rh) and torch.equal(q2[:, :600], q) and (q2[:, 600:] == 99).all()
    assert torch.equal(s2, scale)


# ------------------------------------------------------------------ int8 matrix product
def ints(rows, k, seed):
    """int8 values over the whole range, -128 too, with a row pitch of a multiple of 16."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    buf = torch.randint(-128, 128, (rows, -(-k // 16) * 16), generator=g, dtype=torch.int8, device="cuda")
    return buf[:, :k]


def linear_ref(xq, xs, wq, ws):
    """f32 values that the definition gives: exact sums, then two f32 products."""
    acc = (xq.double() @ wq.double().T).float()
    return (acc * xs[:, None]) * ws[None, :]


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 6, 48), (8, 12288, 2048), (16, 200, 1000), (17, 130, 129), (31, 1024, 6144),
          (33, 514, 2048), (64, 256, 16), (65, 1000, 333), (129, 128, 4096), (381, 4096, 2048), (300, 2050, 1024),
          (1000, 3000, 512), (5, 64, 131071)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_store_bits(ops, m, n, k):
    xq, wq = ints(m, k, 1), ints(n, k, 2)
    xs, ws = rand(m, seed=3).abs() * 0.01, rand(n, seed=4).abs() * 0.01
    y = ops.linear_int8(xq, xs, wq, ws)
    ref = linear_ref(xq, xs, wq, ws)
    assert torch.equal(y, ref)
    yb = ops.linear_int8(xq, xs, wq, ws, dtype=BF16)
    assert torch.equal(yb, ref.to(BF16))
    ops.check()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("m,n,k", [(1, 2, 16), (7, 130, 333), (40, 2048, 6144), (381, 2048, 1024), (700, 1026, 160)])
def test_linear_residual_and_swiglu(ops, dt, m, n, k):
    xq, wq = ints(m, k, 5), ints(n, k, 6)
    xs, ws = rand(m, seed=7).abs() * 0.01, rand(n, seed=8).abs() * (0.5 / k ** 0.5)
    ref = linear_ref(xq, xs, wq, ws)
    wide = rand(m, n + 6, seed=9).to(dt)
    r = wide[:, 3:n + 3]
    y = ops.linear_int8(xq, xs, wq, ws, residual=r, dtype=dt)
    assert torch.equal(y, (ref + r.float()).to(dt))
    s = ops.linear_int8(xq, xs, wq, ws, swiglu=True, dtype=dt)
    g, u = ref[:, 0::2].double(), ref[:, 1::2].double()
    want = g / (1 + torch.exp(-g)) * u
    # expf 2 ulp (4 * 2^-24), then a sum, a reciprocal and three products of 2^-24 each: 9 * 2^-24,
    # or 8 and the output's rounding; results under the smallest normal number may lose all bits
    tol = want.abs() * (8 * 2.0 ** -24 + HALF[dt]) + 2.0 ** -126
    assert ((s.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("m,n,k", [(2999, 1900, 4100), (20001, 130, 3970), (4100, 1794, 5000)])
def test_linear_many_rows_long_k(ops, dt, m, n, k):
    """The tiles of CTA pairs: a second CTA without channels, with two of them, odd rows and widths."""
    xq, wq = ints(m, k, 15), ints(n, k, 16)
    xs, ws = rand(m, seed=17).abs() * 0.01, rand(n, seed=18).abs() * (0.5 / k ** 0.5)
    ref = linear_ref(xq, xs, wq, ws)
    assert torch.equal(ops.linear_int8(xq, xs, wq, ws, dtype=dt), ref.to(dt))
    r = rand(m, n, seed=19).to(dt)
    assert torch.equal(ops.linear_int8(xq, xs, wq, ws, residual=r, dtype=dt), (ref + r.float()).to(dt))
    assert torch.equal(ops.linear_int8(xq[:100], xs[:100], wq, ws, dtype=dt), ref[:100].to(dt))
    s = ops.linear_int8(xq, xs, wq, ws, swiglu=True, dtype=dt)
    g, u = ref[:, 0::2].double(), ref[:, 1::2].double()
    want = g / (1 + torch.exp(-g)) * u
    # as in the test before
    tol = want.abs() * (8 * 2.0 ** -24 + HALF[dt]) + 2.0 ** -126
    assert ((s.double() - want).abs() <= tol).all()
    ops.check()


def test_linear_in_place_residual_and_rows_independent(ops):
    """out may be the residual (C call), and a row has the same bits whatever rows share its call."""
    from qwen_asr_b200 import lib
    m, n, k = 381, 2048, 2048
    xq, wq = ints(m, k, 11), ints(n, k, 12)
    xs, ws = rand(m, seed=13).abs(), rand(n, seed=14).abs()
    full = ops.linear_int8(xq, xs, wq, ws)
    for rows in (1, 5, 16, 100, 200):
        assert torch.equal(ops.linear_int8(xq[:rows], xs[:rows], wq, ws), full[:rows]), rows
    x = rand(m, n, seed=15)
    want = ops.linear_int8(xq, xs, wq, ws, residual=x)
    assert lib().qwen_asr_linear_int8(xq.data_ptr(), k, xs.data_ptr(), wq.data_ptr(), k, ws.data_ptr(), m, n, k, 1,
                                      x.data_ptr(), n, x.data_ptr(), n, 0, -1,
                                      torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(x, want)


def test_linear_largest_sums(ops):
    """The longest k with the largest products stays inside int32: 131071 * 128 * 128 = 2^31 - 2^14."""
    k = 131071
    xq = torch.full((3, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
    one = torch.ones(3, device="cuda")
    y = ops.linear_int8(xq, one, xq, one)
    assert (y == float(2 ** 31 - 2 ** 14)).all()


# ------------------------------------------------------------------ int8 KV cache
def empty_cache(n_seq, n_kv, cap, hd, fill=None):
    """Caches start as rubbish: nothing outside what was appended may matter."""
    g = torch.Generator(device="cuda")
    g.manual_seed(99)
    q = [torch.randint(-127, 128, (n_seq, n_kv, cap, hd), generator=g, dtype=torch.int8, device="cuda")
         for _ in range(2)]
    s = [torch.full((n_seq, n_kv, cap // 16), math.nan if fill is None else fill, device="cuda") for _ in range(2)]
    return q + s


def append_ref(q, s, new, starts, counts):
    """The definition, block by block, in 64 bits, on copies."""
    q, s = q.clone(), s.clone()
    cap = q.shape[2]
    for b, (st, c) in enumerate(zip(starts, counts)):
        if st < 0:
            continue
        end = min(st + min(max(c, 0), new.shape[1]), cap)
        blk = st // 16
        while blk * 16 < end:
            lo, hi = max(st, blk * 16), min(end, blk * 16 + 16)
            x = new[b, lo - st:hi - st].double().transpose(0, 1)
            was = s[b, :, blk].double() if lo > blk * 16 else torch.zeros(q.shape[1], dtype=torch.float64, device=q.device)
            now = torch.maximum(was, (x.abs().amax((1, 2)).float() / torch.full((q.shape[1],), 127.0, device=q.device)).double())
            safe = torch.where(now > 0, now, torch.ones_like(now))[:, None, None]
            if lo > blk * 16:
                held = q[b, :, blk * 16:lo].double()
                q[b, :, blk * 16:lo] = torch.round(held * was[:, None, None] / safe).to(torch.int8)
            q[b, :, lo:hi] = torch.round(x / safe).clamp(-127, 127).to(torch.int8)
            s[b, :, blk] = now.float()
            blk += 1
    return q, s


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=-7.0), torch.nan_to_num(b, nan=-7.0))


def append_and_check(ops, c, k, v, starts, counts):
    n = len(starts)
    st = torch.tensor(starts, dtype=torch.int32, device="cuda")
    ct = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    full = [k.shape[1]] * n if counts is None else counts
    want = [append_ref(c[0], c[2], k, starts, full), append_ref(c[1], c[3], v, starts, full)]
    ops.kv8_append(ops.Kv8Cache(*c), k, v, st, ct)
    for i, (q, s) in enumerate(want):
        assert torch.equal(c[i], q) and same(c[2 + i], s), ("k", "v")[i]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd,n_kv", [(128, 8), (64, 1), (128, 3)])
def test_append_token_by_token_and_prompts(ops, dt, hd, n_kv):
    n, cap = 4, 96
    c = empty_cache(n, n_kv, cap, hd)
    starts = [0, 0, 16, 0]
    append_and_check(ops, c, rand(n, 37, n_kv, hd, seed=1).to(dt), rand(n, 37, n_kv, hd, seed=2).to(dt), starts,
                     [37, 0, 20, 1])
    pos = [37, 0, 36, 1]
    for step in range(20):  # growing values: the blocks are re-coded
        k, v = rand(n, 1, n_kv, hd, seed=10 + step, std=1 + step / 4).to(dt), rand(n, 1, n_kv, hd, seed=50 + step).to(dt)
        append_and_check(ops, c, k, v, [p + step for p in pos], None)


def test_append_edges(ops):
    """Past the capacity, negative starts, negative and too large counts, an exactly filled block."""
    n, n_kv, hd, cap = 7, 2, 128, 48
    c = empty_cache(n, n_kv, cap, hd, fill=0.01)
    k, v = rand(n, 20, n_kv, hd, seed=1), rand(n, 20, n_kv, hd, seed=2)
    append_and_check(ops, c, k, v, [40, -1, 48, 47, 0, 16, 2 ** 31 - 1], [20, 20, 20, 20, 16, -3, 20])
    append_and_check(ops, c, k, v, [0, 15, 16, 31, 32, 5, -2 ** 31], [99, 1, 1, 17, 2 ** 31 - 1, 11, 1])


def test_append_special_values(ops):
    n_kv, hd = 2, 64
    c = empty_cache(1, n_kv, 64, hd)
    cache = ops.Kv8Cache(*c)
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    k = torch.zeros(1, 16, n_kv, hd, device="cuda")
    v = rand(1, 16, n_kv, hd, seed=3)
    k[0, :, 1] = 1e-44  # max / 127 rounds to zero
    ops.kv8_append(cache, k, v, z)
    assert (c[2][0, :, 0] == 0).all() and not c[0][0, :, :16].any()
    # a NaN poisons its block and head alone; a later block is fresh
    k2 = rand(1, 20, n_kv, hd, seed=4)
    k2[0, 3, 1, 7] = math.nan
    k2[0, 18, 0, 0] = math.inf
    ops.kv8_append(cache, k2, v[:, :1].expand(1, 20, n_kv, hd), z + 16)
    assert torch.isnan(c[2][0, 1, 1]) and not torch.isnan(c[2][0, 0, 1])
    assert torch.isnan(c[2][0, 0, 2]) and not torch.isnan(c[2][0, 1, 2])
    # what is appended to a poisoned block stays poisoned, and starting the block anew heals it
    ops.kv8_append(cache, rand(1, 1, n_kv, hd, seed=5), v[:, :1], z + 36)
    assert torch.isnan(c[2][0, 0, 2])
    ops.kv8_append(cache, rand(1, 1, n_kv, hd, seed=5), v[:, :1], z + 32)
    assert not torch.isnan(c[2][0, :, 2]).any()


def test_append_exact_ties(ops):
    """x / s exactly a half: s = 1 (largest value 127), values n + 1/2; and quotients that f32 rounds onto a half."""
    hd = 128
    c = empty_cache(1, 1, 32, hd)
    k = torch.zeros(1, 2, 1, hd, device="cuda")
    k[0, 0, 0, 0] = 127.0
    k[0, 0, 0, 1:101] = torch.arange(100, device="cuda") + 0.5
    s = 127.0 * (1 + 2 ** -20)
    k[0, 1, 0, 0] = s
    near = (torch.arange(100, device="cuda") + 0.5) * (1 + 2 ** -20)
    k[0, 1, 0, 1:101] = near
    k[0, 1, 0, 101:] = torch.nextafter(near[:27], torch.zeros(27, device="cuda"))
    append_and_check(ops, c, k, -k, [0], None)
    append_and_check(ops, c, k[:, 1:], -k[:, 1:], [16], None)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
def test_read_back(ops, dt, hd):
    n, n_kv, cap = 5, 3, 80
    c = empty_cache(n, n_kv, cap, hd, fill=0.0)
    c[2].copy_(rand(n, n_kv, cap // 16, seed=1).abs())
    c[3].copy_(rand(n, n_kv, cap // 16, seed=2).abs())
    starts, counts = [0, 7, 75, -1, 16], [30, 0, 30, 30, 2 ** 31 - 1]
    st, ct = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in (starts, counts))
    out = ops.kv8_read(ops.Kv8Cache(*c), st, 33, ct, dtype=dt)
    for o, q, s in ((out[0], c[0], c[2]), (out[1], c[1], c[3])):
        vals = (q.float() * s.repeat_interleave(16, 2)[..., None]).to(dt)
        want = torch.zeros(n, 33, n_kv, hd, dtype=dt, device="cuda")
        for b in range(n):
            live = min(counts[b], 33, cap - starts[b]) if starts[b] >= 0 else 0
            want[b, :live] = vals[b, :, starts[b]:starts[b] + live].transpose(0, 1)
        assert torch.equal(o, want)


# ------------------------------------------------------------------ attention over the cache
def filled_cache(ops, n, n_kv, cap, hd, lens, seed=0, kstd=1.0):
    c = empty_cache(n, n_kv, cap, hd)  # rubbish values and NaN scales behind every length
    k, v = rand(n, cap, n_kv, hd, seed=seed + 1, std=kstd), rand(n, cap, n_kv, hd, seed=seed + 2, std=0.5)
    z = torch.zeros(n, dtype=torch.int32, device="cuda")
    ops.kv8_append(ops.Kv8Cache(*c), k, v, z, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    return c


def attention_ref(q, c, starts, counts, scale, f32_planes):
    """(out, tolerance) in 64 bits. Tolerance of one output, relative to the head's largest |v|:
      the scores' error d: q is held to 2^-25 of its row's largest value in each of two planes or to 2^-22
        in digits, and the product, sum, factor and exponential of an f32 path are off by a few 2^-24 of
        sum |q k|: in all under 2^-21 * (scale * max|q| * max_t sum |k_t|), and the probabilities by that much; twice, for
        numerator and denominator;
      the probabilities: f16 planes hold them to 2^-25 of the largest, bytes of a 23-bit fraction to 2^-24,
        for each key (len * 2^-24 / l); one f16 plane (bf16 rows): 2^-11 of each;
      the sums: 2^-23 for each tile of 16 tokens (f32 accumulation, rescaling), and 2^-22 for the end."""
    k, v, ks, vs = c
    n, rows, heads, hd = q.shape
    g = heads // k.shape[1]
    out = torch.zeros_like(q, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(n):
        for r in range(min(max(counts[b], 0), rows)):
            L = min(starts[b] + r + 1, k.shape[2])
            if starts[b] < 0:
                continue
            kk = k[b, :, :L].double() * ks[b].repeat_interleave(16, 1)[:, :L, None].double()
            vv = v[b, :, :L].double() * vs[b].repeat_interleave(16, 1)[:, :L, None].double()
            kk, vv = kk.repeat_interleave(g, 0), vv.repeat_interleave(g, 0)
            qq = q[b, r].double()
            x = (kk @ qq[:, :, None])[..., 0] * scale
            p = torch.exp(x - x.amax(1, keepdim=True))
            l = p.sum(1)
            out[b, r] = (p[:, None] @ vv)[:, 0] / l[:, None]
            d = 2 * 2.0 ** -21 * scale * qq.abs().amax(1) * kk.abs().sum(2).amax(1)
            planes = L * 2.0 ** -24 / l + (0 if f32_planes else 2.0 ** -11)
            t = (d + planes + (L // 16 + 1) * 2.0 ** -23 + 2.0 ** -22) * vv.abs().amax((1, 2))
            tol[b, r] = t[:, None] + out[b, r].abs() * HALF[q.dtype]
    return out, tol


def attend_and_check(ops, q, c, starts, counts, scale=None, max_len=0):
    n = len(starts)
    st = torch.tensor(starts, dtype=torch.int32, device="cuda")
    ct = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    got = ops.kv8_attention(q, ops.Kv8Cache(*c), st, ct, scale=scale, max_len=max_len)
    want, tol = attention_ref(q, c, starts, [q.shape[1]] * n if counts is None else counts,
                              1 / math.sqrt(q.shape[3]) if scale is None else scale, q.dtype == F32)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (err / tol.clamp_min(1e-30)).max()
    return got


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,n_kv", [(16, 8), (4, 4), (6, 2), (8, 1), (16, 1), (40, 2)])
def test_attention_tokens(ops, dt, hd, heads, n_kv):
    lens = [1, 2, 16, 17, 63, 64, 65, 200, 511]
    c = filled_cache(ops, len(lens), n_kv, 512, hd, lens, seed=heads)
    q = rand(len(lens), 1, heads, hd, seed=3, std=2.0).to(dt)
    attend_and_check(ops, q, c, [L - 1 for L in lens], None)
    attend_and_check(ops, q, c, [L - 1 for L in lens], [1, 0, 1, -5, 1, 1, 9, 1, 1], scale=0.05, max_len=16)


def test_refusals_of_the_library_are_value_errors(ops):
    """Arguments that pass the first checks and fail in the library: a cache whose sequences share memory, more
    rows than a call takes."""
    c = ops.kv8_cache(1, 2, 32, 64)
    both = ops.Kv8Cache(*[t.expand(2, *t.shape[1:]) for t in c])
    z = torch.zeros(2, dtype=torch.int32, device="cuda")
    k = rand(2, 1, 2, 64)
    with pytest.raises(ValueError, match="seq_stride"):
        ops.kv8_append(both, k, k, z)
    with pytest.raises(ValueError, match="seq_stride"):
        ops.kv8_attention(k, both, z)
    with pytest.raises(ValueError, match="seq_stride"):
        ops.kv8_read(both, z, 1)
    one = ops.kv8_cache(1, 1, 16, 64)
    with pytest.raises(ValueError, match="rows"):
        ops.kv8_attention(rand(1, 1, 1, 64).to(BF16).expand(1, (1 << 22) + 1, 1, 64), one, z[:1])


@pytest.mark.parametrize("rows,heads", [(1, 16), (2, 16), (5, 32)])
def test_attention_many_sequences_of_any_order(ops, rows, heads):
    """More sequences than run at once, which are taken up by length: equal ones, empty ones, a last group of 7."""
    n, n_kv = 71, 8
    g = torch.Generator().manual_seed(rows)
    starts = torch.randint(0, 120, (n,), generator=g).tolist()
    starts[3], starts[40:44], starts[70] = -1, [77] * 4, 0
    counts = torch.randint(0, rows + 1, (n,), generator=g).tolist()
    c = filled_cache(ops, n, n_kv, 128, 64, [max(s, 0) + k for s, k in zip(starts, counts)], seed=rows)
    q = rand(n, rows, heads, 64, seed=5, std=1.5)
    live = [k if s >= 0 else 0 for s, k in zip(starts, counts)]
    want = attend_and_check(ops, q, c, [max(s, 0) for s in starts], live)
    st, ct = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (starts, counts))
    assert torch.equal(ops.kv8_attention(q, ops.Kv8Cache(*c), st, ct), want)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd,heads,n_kv,rows", [(128, 16, 8, 3), (128, 4, 2, 32), (128, 4, 2, 33), (64, 8, 2, 50),
                                                (128, 2, 2, 150), (64, 12, 4, 101)])
def test_attention_prompt_rows(ops, dt, hd, heads, n_kv, rows):
    starts, counts = [0, 5, 100, 31], [rows, rows - 2, 0, 1]
    lens = [s + c for s, c in zip(starts, counts)]
    c = filled_cache(ops, 4, n_kv, 256, hd, lens, seed=rows)
    q = rand(4, rows, heads, hd, seed=4, std=1.5).to(dt)
    got = attend_and_check(ops, q, c, starts, counts)
    assert not got[2].any() and not got[3, 1:].any()  # rows not in use are zeros


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("n,rows", [(2, 150), (33, 70), (40, 200)])
def test_attention_prompts_of_any_order(ops, dt, n, rows):
    """Row tiles of many sequences, taken up by the keys they see: any lengths, empty and equal sequences."""
    g = torch.Generator().manual_seed(n)
    starts = torch.randint(0, 300, (n,), generator=g).tolist()
    counts = torch.randint(0, rows + 1, (n,), generator=g).tolist()
    starts[0], counts[1], starts[n // 2], counts[n // 2] = 0, rows, starts[-1], counts[-1]
    c = filled_cache(ops, n, 2, 512, 64, [s + k for s, k in zip(starts, counts)], seed=n)
    q = rand(n, rows, 4, 64, seed=6, std=1.5).to(dt)
    attend_and_check(ops, q, c, starts, counts)
    c = filled_cache(ops, n, 2, 512, 64, [17 + rows] * n, seed=n)
    attend_and_check(ops, q, c, [17] * n, None)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd,heads,n_kv,rows", [(128, 2, 1, 65), (64, 8, 2, 140), (128, 6, 3, 300)])
def test_attention_few_rows_behind_many(ops, dt, hd, heads, n_kv, rows):
    """Few row tiles, whose keys several blocks share: long and short histories, parts that see nothing."""
    starts, counts = [3700, 0, 130], [rows, rows, rows // 3]
    c = filled_cache(ops, 3, n_kv, 4096, hd, [s + k for s, k in zip(starts, counts)], seed=rows)
    q = rand(3, rows, heads, hd, seed=7, std=1.5).to(dt)
    got = attend_and_check(ops, q, c, starts, counts)
    assert not got[2, rows // 3:].any()
    attend_and_check(ops, q[:1], [t[:1] for t in c], starts[:1], None)
    attend_and_check(ops, q[:1], [t[:1] for t in c], [600], None, max_len=600 + rows)
    attend_and_check(ops, q[:1], [t[:1] for t in c], starts[:1], [0])


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_ignores_what_is_masked(ops, rows):
    """NaN blocks behind a row's last position do not touch it; a NaN it does see reaches its head."""
    n_kv, hd, cap = 2, 128, 160
    c = filled_cache(ops, 1, n_kv, cap, hd, [cap], seed=8)
    q = rand(1, rows, 4, hd, seed=9)
    st = torch.tensor([30], dtype=torch.int32, device="cuda")
    want = ops.kv8_attention(q, ops.Kv8Cache(*c), st)
    first = (30 + rows - 1) // 16 + 1
    for t in c[2:]:
        t[:, :, first:] = math.nan
    assert torch.equal(ops.kv8_attention(q, ops.Kv8Cache(*c), st), want)
    if rows > 1:  # rows before the block keep their values when a block that later rows see is bad
        c[3][0, 1, first - 1] = math.nan
        got = ops.kv8_attention(q, ops.Kv8Cache(*c), st)
        seen = (first - 1) * 16 - 30
        assert torch.equal(got[:, :seen], want[:, :seen]) and torch.equal(got[:, :, :2], want[:, :, :2])
        assert torch.isnan(got[0, seen:, 2:]).all()


@pytest.mark.parametrize("dt", [F32, BF16])
def test_attention_shared_keys_with_bad_and_extreme_blocks(ops, dt):
    """Keys that several blocks share: NaN scales behind the last position, NaN in a block that only later rows
    see, one key far above all others."""
    rows, start, hd, cap = 100, 2990, 128, 4096
    c = filled_cache(ops, 1, 1, cap, hd, [cap], seed=12)
    q = rand(1, rows, 2, hd, seed=13).to(dt)
    st = torch.tensor([start], dtype=torch.int32, device="cuda")
    want = ops.kv8_attention(q, ops.Kv8Cache(*c), st)
    for t in c[2:]:
        t[:, :, (start + rows - 1) // 16 + 1:] = math.nan
    assert torch.equal(ops.kv8_attention(q, ops.Kv8Cache(*c), st), want)
    for t in c[2:]:  # K, then V
        keep = t[0, 0, (start + 50) // 16].clone()
        t[0, 0, (start + 50) // 16] = math.nan
        got = ops.kv8_attention(q, ops.Kv8Cache(*c), st)
        seen = (start + 50) // 16 * 16 - start
        assert torch.equal(got[:, :seen], want[:, :seen])
        assert torch.isnan(got[:, seen:]).all()
        t[0, 0, (start + 50) // 16] = keep
    c[2][0, 0, 70] *= 60  # (16 keys of the second part)
    attend_and_check(ops, q, c, [start], None)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("rows,cap", [(3, 64), (20, 64), (90, 128), (90, 2048)])
def test_attention_rows_without_alignment(ops, dt, rows, cap):
    """Query rows that start anywhere in a wider matrix: the bits of aligned ones."""
    heads, hd = 4, 64
    c = filled_cache(ops, 2, 2, cap, hd, [rows + 7, rows], seed=51)
    wide = rand(2, rows, heads * hd + 3, seed=52).to(dt)
    q = wide[:, :, 1:heads * hd + 1].unflatten(2, (heads, hd))
    st = torch.tensor([7, 0], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.kv8_attention(q, ops.Kv8Cache(*c), st), ops.kv8_attention(q.contiguous(), ops.Kv8Cache(*c), st))


def test_two_streams_at_once(ops):
    """Calls that fill the GPU, on two streams at the same time, give the bits of calls one after the other."""
    m, n, k = 2999, 1900, 4100
    xq, wq = ints(m, k, 41), ints(n, k, 42)
    xs, ws = rand(m, seed=43).abs() * 0.01, rand(n, seed=44).abs() * 0.01
    c = filled_cache(ops, 2, 2, 4096, 128, [4096, 4096], seed=45)
    q = rand(2, 150, 4, 128, seed=46)
    st = torch.tensor([3900, 1000], dtype=torch.int32, device="cuda")
    one = rand(2, 1, 4, 128, seed=47)
    calls = (lambda: ops.linear_int8(xq, xs, wq, ws), lambda: ops.kv8_attention(q, ops.Kv8Cache(*c), st),
             lambda: ops.kv8_attention(q.to(BF16), ops.Kv8Cache(*c), st), lambda: ops.linear_int8(xq[:9], xs[:9], wq, ws),
             lambda: ops.kv8_attention(one, ops.Kv8Cache(*c), st))
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for turn in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                order = calls if i == 0 else calls[::-1]
                got[i].append([f() for f in order])
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for a, b in zip(r if i == 0 else r[::-1], want):
                assert torch.equal(a, b)
    ops.check()


def test_attention_extreme_scores(ops):
    """One key far above the rest, queries of very different size, zero queries and zero blocks."""
    n_kv, hd, cap = 1, 128, 64
    k, v = rand(1, 64, 1, hd, seed=1), rand(1, 64, 1, hd, seed=2)
    k[0, 20] *= 40
    k[0, 32:48] = 0
    v[0, 48:] = 0
    c = empty_cache(1, n_kv, cap, hd)
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv8_append(ops.Kv8Cache(*c), k, v, z)
    q = rand(1, 1, 6, hd, seed=3)
    q[0, 0, 1] = 0
    q[0, 0, 2] *= 1e-20
    q[0, 0, 3, 5] = 3e4
    q[0, 0, 4] *= 30
    attend_and_check(ops, q, c, [63], None)


def test_attention_long_lengths_split(ops):
    """Lengths that all split sizes share out differently; the same bits on every run."""
    n, n_kv, hd, cap = 3, 2, 128, 5008
    lens = [4999, 129, 2577]
    c = filled_cache(ops, n, n_kv, cap, hd, lens, seed=5, kstd=1.5)
    q = rand(n, 1, 4, hd, seed=6, std=2.0)
    a = attend_and_check(ops, q, c, [L - 1 for L in lens], None)
    b = attend_and_check(ops, q, c, [L - 1 for L in lens], None, max_len=5000)
    assert torch.equal(a, b)
    for m in (1, 64, 200, 700, 1500):
        attend_and_check(ops, q, c, [L - 1 for L in lens], None, max_len=m)


# ------------------------------------------------------------------ strides, offsets, streams, graphs
def test_cache_slices_and_strided_rows(ops):
    """A layer of a cache of several, every second sequence, rows inside a packed q/k/v matrix and
    positions inside a table of structs."""
    n, layers, n_kv, hd, cap, rows, heads = 3, 2, 2, 128, 64, 5, 4
    big = [torch.zeros(2 * n, layers, n_kv, cap, hd, dtype=torch.int8, device="cuda") for _ in range(2)]
    sc = [torch.zeros(2 * n, layers, n_kv, cap // 16, device="cuda") for _ in range(2)]
    cache = ops.Kv8Cache(*[t[1::2, 1] for t in big + sc])
    qkv = rand(n, rows, (heads + 2 * n_kv) * hd, seed=1)
    q = qkv[..., :heads * hd].unflatten(2, (heads, hd))
    k = qkv[..., heads * hd:(heads + n_kv) * hd].unflatten(2, (n_kv, hd))
    v = qkv[..., (heads + n_kv) * hd:].unflatten(2, (n_kv, hd))
    table = torch.tensor([[0, 7, 5, 7], [16, 7, 2, 7], [20, 7, 5, 7]], dtype=torch.int32, device="cuda")
    ops.kv8_append(cache, k, v, table[:, 0], table[:, 2])
    plain = ops.Kv8Cache(*[t.contiguous() for t in (torch.zeros_like(cache.k), torch.zeros_like(cache.v),
                                                    torch.zeros_like(cache.k_scale), torch.zeros_like(cache.v_scale))])
    st, ct = table[:, 0].contiguous(), table[:, 2].contiguous()
    ops.kv8_append(plain, k.contiguous(), v.contiguous(), st, ct)
    for a, b in zip(cache, plain):
        assert torch.equal(a, b)
    for t in big + sc:
        assert not t[0::2].any() and not t[:, 0].any()
    want = ops.kv8_attention(q.contiguous(), plain, st, ct)
    assert torch.equal(ops.kv8_attention(q, cache, table[:, 0], table[:, 2]), want)
    # odd element offsets: no vector loads
    wide = torch.zeros(n, rows, heads * hd + 3, device="cuda")
    wide[..., 1:1 + heads * hd] = qkv[..., :heads * hd]
    qs = wide[..., 1:1 + heads * hd].unflatten(2, (heads, hd))
    assert torch.equal(ops.kv8_attention(qs, cache, table[:, 0], table[:, 2]), want)
    ks = torch.zeros(n, rows, n_kv * hd + 1, device="cuda")
    ks[..., 1:] = k.flatten(2)
    ops.kv8_append(cache, ks[..., 1:].unflatten(2, (n_kv, hd)), v, table[:, 0], table[:, 2])
    for a, b in zip(cache, plain):
        assert torch.equal(a, b)


def test_offsets_past_32_bits(ops):
    """The second sequence starts more than 2^31 bytes behind the first."""
    n_kv, hd, cap = 2, 128, 64
    stride = 2 ** 31 + 2 ** 20
    size = n_kv * cap * hd
    flat = [torch.zeros(stride + size, dtype=torch.int8, device="cuda") for _ in range(2)]
    q = [t.as_strided((2, n_kv, cap, hd), (stride, cap * hd, hd, 1)) for t in flat]
    s = [torch.zeros(2, n_kv, cap // 16, device="cuda") for _ in range(2)]
    cache = ops.Kv8Cache(*q, *s)
    near = ops.kv8_cache(2, n_kv, cap, hd)
    k, v = rand(2, 50, n_kv, hd, seed=1), rand(2, 50, n_kv, hd, seed=2)
    z = torch.zeros(2, dtype=torch.int32, device="cuda")
    for c in (cache, near):
        ops.kv8_append(c, k, v, z)
    assert torch.equal(cache.k, near.k) and torch.equal(cache.v, near.v)
    qr = rand(2, 50, 4, hd, seed=3)
    assert torch.equal(ops.kv8_attention(qr, cache, z), ops.kv8_attention(qr, near, z))
    assert torch.equal(ops.kv8_attention(qr[:, :1], cache, z + 49), ops.kv8_attention(qr[:, :1], near, z + 49))
    for a, b in zip(ops.kv8_read(cache, z, 50), ops.kv8_read(near, z, 50)):
        assert torch.equal(a, b)


def layer(ops, x, r, w, wq, ws, cache, starts):
    """norm -> q/k/v product -> cache -> attention -> product with residual, as a decoder layer runs them."""
    n_kv, hd = cache.k.shape[1], cache.k.shape[3]
    heads = wq.shape[0] // hd - 2 * n_kv
    q, s, h = ops.rms_norm_int8(x, w, 1e-6, residual=r)
    y = ops.linear_int8(q, s, wq, ws)[:, None].unflatten(2, (heads + 2 * n_kv, hd))
    ops.kv8_append(cache, y[:, :, heads:heads + n_kv], y[:, :, heads + n_kv:], starts)
    o = ops.kv8_attention(y[:, :, :heads], cache, starts).flatten(1)
    one = torch.ones(o.shape[1], device=o.device)
    oq, os_, _ = ops.rms_norm_int8(o, one, 1e-6)
    return ops.linear_int8(oq, os_, wq[:h.shape[1], :o.shape[1]], ws[:h.shape[1]], residual=h)


def layer_inputs(ops, n=6, d=512, n_kv=2, heads=4, hd=128, cap=64):
    x, r, w = rand(n, d, seed=1), rand(n, d, seed=2), 1 + rand(d, seed=3, std=0.1)
    wq, ws = ints((heads + 2 * n_kv) * hd, d, 4), rand((heads + 2 * n_kv) * hd, seed=5).abs() * 3e-4
    cache = ops.kv8_cache(n, n_kv, cap, hd)
    starts = torch.arange(n, dtype=torch.int32, device="cuda") * 3
    k, v = rand(n, cap, n_kv, hd, seed=6), rand(n, cap, n_kv, hd, seed=7)
    ops.kv8_append(cache, k, v, torch.zeros_like(starts))
    return x, r, w, wq, ws, cache, starts


def test_layer_of_them_all(ops):
    """A run of the operators together equals the chain of their definitions."""
    x, r, w, wq, ws, cache, starts = layer_inputs(ops)
    c = [t.clone() for t in cache]
    got = layer(ops, x, r, w, wq, ws, cache, starts)
    h, q, s = norm_ref(x, w, 1e-6, r)
    y = linear_ref(q.to(torch.int8), s.float(), wq, ws)[:, None].unflatten(2, (8, 128))
    st = starts.tolist()
    k8, ks8 = append_ref(c[0], c[2], y[:, :, 4:6], st, [1] * 6)
    v8, vs8 = append_ref(c[1], c[3], y[:, :, 6:], st, [1] * 6)
    o, tol = attention_ref(y[:, :, :4], (k8, v8, ks8, vs8), st, [1] * 6, 1 / math.sqrt(128), True)
    o, tol = o.flatten(1), tol.flatten(1)
    # through the second norm: u = o / max|o| moves by at most 2 tol / max|o|, so an int8 value by one step
    # where its quotient is within 127 * that of a half; the product by that many |w| steps
    _, oq, os_ = norm_ref(o.float(), torch.ones(512, device="cuda"), 1e-6, None)
    top = o.abs().amax(1, keepdim=True)
    shift = 127 * 2 * tol.amax(1, keepdim=True) / top + 1e-4
    frac = (o * 127 / top).abs() % 1
    flips = ((frac - 0.5).abs() < shift).double()
    wf = wq[:512, :512].double().abs() * ws[:512, None].double()
    want = linear_ref(oq.to(torch.int8), os_.float(), wq[:512, :512], ws[:512]).double() + h.double()
    slack = (flips @ wf.T) * os_[:, None] + (want - h.double()).abs() * (2 * tol.amax(1, keepdim=True) / top + 2 ** -20) + want.abs() * 2 ** -22
    assert ((got.double() - want).abs() <= slack).all()


def test_other_stream_and_graph(ops):
    """On a stream of the caller's and captured into two graphs that replay in turn: the eager bits."""
    x, r, w, wq, ws, cache, starts = layer_inputs(ops)
    keep = [t.clone() for t in cache]

    def reset():
        for t, k in zip(cache, keep):
            t.copy_(k)

    want = layer(ops, x, r, w, wq, ws, cache, starts)
    reset()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(ops, x, r, w, wq, ws, cache, starts)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    x2, starts2 = x * 0.5, starts + 1
    reset()
    want2 = layer(ops, x2, r, w, wq, ws, cache, starts2)
    graphs = []
    for xx, st in ((x, starts), (x2, starts2)):
        reset()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = layer(ops, xx, r, w, wq, ws, cache, st)
        graphs.append((g, o))
    for _ in range(2):
        for (g, o), wnt in zip(graphs, (want, want2)):
            reset()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, wnt)
    # new inputs in the captured buffers
    x.copy_(x2)
    starts.copy_(starts2)
    reset()
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want2)


def test_first_calls_inside_a_capture():
    """A process whose very first call of each operator is captured into a graph."""
    code = """
import torch
from qwen_asr_b200 import ops
x, w = torch.randn(40, 512, device='cuda'), torch.ones(512, device='cuda')
wq = torch.randint(-127, 128, (1024, 512), dtype=torch.int8, device='cuda')
ws = torch.rand(1024, device='cuda')
c = ops.kv8_cache(1, 2, 64, 128)
z = torch.zeros(1, dtype=torch.int32, device='cuda')
def run():
    q, s, h = ops.rms_norm_int8(x, w, residual=x)
    y = ops.linear_int8(q, s, wq, ws)[None].unflatten(2, (8, 128))
    ops.kv8_append(c, y[:, :, 4:6], y[:, :, 6:], z)
    return (ops.kv8_attention(y[:, :, :4], c, z), ops.kv8_attention(y[:, :1, :4], c, z + 39), *ops.kv8_read(c, z, 40))
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = run()
g.replay()
torch.cuda.synchronize()
got = [t.clone() for t in out]
for a, b in zip(got, run()):
    assert torch.equal(a, b)
print('captured')
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


# ------------------------------------------------------------------ refusals
def test_refusals(ops):
    x, w = rand(4, 64), rand(64)
    q8 = ints(4, 64, 1)
    s = torch.ones(4, device="cuda")
    c = ops.kv8_cache(2, 2, 32, 128)
    z = torch.zeros(2, dtype=torch.int32, device="cuda")
    k = rand(2, 1, 2, 128)
    bad = [
        (TypeError, lambda: ops.rms_norm_int8(x.half(), w)),
        (TypeError, lambda: ops.rms_norm_int8(x, w.to(BF16))),
        (TypeError, lambda: ops.rms_norm_int8(x, w, residual=x.to(BF16))),
        (ValueError, lambda: ops.rms_norm_int8(x, w[:63])),
        (ValueError, lambda: ops.rms_norm_int8(x.T, rand(4))),
        (ValueError, lambda: ops.rms_norm_int8(x, w, eps=-1.0)),
        (ValueError, lambda: ops.rms_norm_int8(x, w.cpu())),
        (ValueError, lambda: ops.rms_norm_int8(x.clone().requires_grad_(), w)),
        (ValueError, lambda: ops.linear_int8(q8, s, q8[:, :32], s)),
        (ValueError, lambda: ops.linear_int8(q8[:, 1:33], s, q8[:, :32], s)),
        (ValueError, lambda: ops.linear_int8(ints(4, 64, 1).flatten()[:4 * 60].view(4, 60), s, q8[:, :60], s)),
        (ValueError, lambda: ops.linear_int8(q8, s[:3], q8, s)),
        (ValueError, lambda: ops.linear_int8(q8, s, q8[:3], s[:3], swiglu=True)),
        (ValueError, lambda: ops.linear_int8(q8, s, q8, s, residual=rand(4, 4), swiglu=True)),
        (TypeError, lambda: ops.linear_int8(q8, s, q8, s, dtype=torch.float16)),
        (TypeError, lambda: ops.linear_int8(q8, s, q8, s, residual=rand(4, 4).to(BF16))),
        (ValueError, lambda: ops.kv8_append(c, k[:1], k[:1], z)),
        (ValueError, lambda: ops.kv8_append(c, k, k[..., :64], z)),
        (TypeError, lambda: ops.kv8_append(c, k, k, z.long())),
        (ValueError, lambda: ops.kv8_append(c, k, k, z[:1])),
        (ValueError, lambda: ops.kv8_append(c, k, k, z[:1].expand(2))),
        (ValueError, lambda: ops.kv8_append(ops.Kv8Cache(*[t.expand(2, *t.shape[1:]) for t in ops.kv8_cache(1, 2, 32)]), k, k, z)),
        (ValueError, lambda: ops.kv8_append(c, k.transpose(2, 3).contiguous().transpose(2, 3), k, z)),
        (ValueError, lambda: ops.kv8_attention(rand(2, 1, 3, 128), c, z)),
        (ValueError, lambda: ops.kv8_attention(rand(2, 1, 4, 64), c, z)),
        (ValueError, lambda: ops.kv8_read(c, z, -1)),
        (TypeError, lambda: ops.kv8_attention([1], c, z)),
    ]
    for i, (err, f) in enumerate(bad):
        with pytest.raises((err, RuntimeError) if err is ValueError else err):
            f()
    # sizes of zero are calls with nothing to do
    assert ops.rms_norm_int8(x[:0], w)[0].shape == (0, 64)
    assert ops.linear_int8(q8[:0], s[:0], q8, s).shape == (0, 4)
    ops.kv8_append(c, k[:, :0], k[:, :0], z)
    assert ops.kv8_attention(rand(2, 0, 4, 128), c, z).shape == (2, 0, 4, 128)
    assert ops.kv8_read(c, z, 0)[0].shape == (2, 0, 2, 128)
