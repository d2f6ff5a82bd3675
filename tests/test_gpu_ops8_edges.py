"""Calls of the 8-bit operators that their documentation allows at its edges: sequences without rows, blocks of
very different scales, tensors on other streams, errors of other users of the device."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.test_gpu_ops8 import BF16, F32, HALF, filled_cache, ops, rand  # noqa: E402,F401


def attend_into(ops, out, q, c, starts, counts):
    """kv8_attention by the C call, into `out` as it is."""
    desc, dev, _, _, hd = ops._cache(ops.Kv8Cache(*c))
    st, ct = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in (starts, counts))
    code = 0 if q.dtype == F32 else 1
    assert ops.lib().qwen_asr_kv8_attention(desc, ops._rows(q, "q"), ops._rows(out, "out"), code, q.shape[1], q.shape[2],
                                            st.data_ptr(), ct.data_ptr(), 1, 1 / math.sqrt(hd), 0, dev,
                                            torch.cuda.current_stream().cuda_stream) == 0
    return out


# ------------------------------------------------------------------ sequences without rows
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("n,live", [(1, 0), (2, 0), (32, 0), (40, 32), (64, 32), (64, 0), (33, 1)])
@pytest.mark.parametrize("group,rows", [(1, 150), (2, 150), (16, 20), (128, 3)])
def test_prompt_rows_of_skipped_sequences_are_zeros(ops, dt, n, live, group, rows):
    """Negative starts, of all sequences or of a whole group of 32 that is ordered together: rows in use have
    the bits they have beside sequences of no rows, and every other row is written with zeros."""
    hd, cap = 64, 512
    g = torch.Generator().manual_seed(n + group)
    starts = torch.randint(0, 300, (n,), generator=g).tolist()
    counts = torch.randint(1, rows + 1, (n,), generator=g).tolist()
    c = filled_cache(ops, n, 1, cap, hd, [s + k for s, k in zip(starts, counts)], seed=n)
    q = rand(n, rows, group, hd, seed=61).to(dt)
    none = [k if i < live else 0 for i, k in enumerate(counts)]
    want = attend_into(ops, torch.full_like(q, math.nan), q, c, [s if i < live else 0 for i, s in enumerate(starts)], none)
    for i, (s, k) in enumerate(zip(starts, none)):
        assert not torch.isnan(want[i]).any() and not want[i, k:].any() and (k == 0 or want[i, :k].any())
    for skip in (-1, -64, -1000, -2 ** 31):
        st = [s if i < live else skip for i, s in enumerate(starts)]
        got = attend_into(ops, torch.full_like(q, math.nan), q, c, st, counts)
        assert torch.equal(got, want), skip
    # rows of the sequences in turn: a neighbour's row is one row stride behind
    out = torch.full((rows, n, group, hd), math.nan, dtype=dt, device="cuda")
    attend_into(ops, out.transpose(0, 1), q, c, [s if i < live else -1000 for i, s in enumerate(starts)], counts)
    assert torch.equal(out.transpose(0, 1), want)
    ops.check()


# ------------------------------------------------------------------ blocks of very different V scales, long tails
def weighed_ref(q, c, starts, scale, held=29):
    """(out, tolerance) in 64 bits, the tolerance relative to what a row weighs: with weights w = p vscale of its
    keys, W the largest of them and l the sum of p,
      the scores' error d of a key, under 2^-21 scale max|q| sum|k| (q held to 2^-22 of its largest value or better,
        product, factor and exponential of an f32 path), once in the numerator and once in l;
      the weights: two f16 planes hold each to 2^-22, one to 2^-11, and none is off by more than 2^-29 of W (half of
        f16's smallest step, 2^-24, under a largest value of 2^4 and up) or half of 2^-32 of 8 W (digits), with int8
        values up to 127;
      the sums: 2^-23 for each tile of 16 tokens, and 2^-22 for the end, of sum w |v|; half a step of the output."""
    k, v, ks, vs = c
    n, rows, heads, hd = q.shape
    g = heads // k.shape[1]
    out = torch.zeros_like(q, dtype=torch.float64)
    tol = torch.zeros_like(out)
    plane = 2.0 ** -22 if q.dtype == F32 else 2.0 ** -11
    for b in range(n):
        for r in range(rows):
            L = starts[b] + r + 1
            kk = k[b, :, :L].double() * ks[b].repeat_interleave(16, 1)[:, :L, None].double()
            sv = vs[b].repeat_interleave(16, 1)[:, :L].double()
            vv = v[b, :, :L].double() * sv[:, :, None]
            kk, vv, sv = kk.repeat_interleave(g, 0), vv.repeat_interleave(g, 0), sv.repeat_interleave(g, 0)
            qq = q[b, r].double()
            x = (kk @ qq[:, :, None])[..., 0] * scale
            p = torch.exp(x - x.amax(1, keepdim=True))
            l = p.sum(1, keepdim=True)
            out[b, r] = (p[:, None] @ vv)[:, 0] / l
            d = 2.0 ** -21 * scale * qq.abs().amax(1, keepdim=True) * kk.abs().sum(2)
            size = (p[:, None] @ vv.abs())[:, 0] / l
            t = ((p * d)[:, None] @ vv.abs())[:, 0] / l + out[b, r].abs() * (p * d).sum(1, keepdim=True) / l
            t += size * (plane + (L // 16 + 1) * 2.0 ** -23 + 2.0 ** -22)
            t += L * 2.0 ** -held * 127 * (p * sv).amax(1, keepdim=True) / l
            tol[b, r] = t + out[b, r].abs() * HALF[q.dtype]
    return out, tol


def weighed_check(ops, q, c, starts, rows=None, held=29, max_len=0):
    st = torch.tensor(starts, dtype=torch.int32, device="cuda")
    got = ops.kv8_attention(q, ops.Kv8Cache(*c), st, max_len=max_len)
    rows = q.shape[1] if rows is None else rows
    want, tol = weighed_ref(q[:, :rows], c, starts, 1 / math.sqrt(q.shape[3]), held)
    err = (got[:, :rows].double() - want).abs()
    assert (err <= tol).all(), (err / tol.clamp_min(1e-300)).max()


PROMPT, STEP, DIGITS = [(70, 2), (40, 4)], [(6, 2), (1, 16), (20, 3)], [(1, 1), (1, 2), (2, 2), (1, 4)]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("times", [1e3, 1e5, 1e8, 1e30])
@pytest.mark.parametrize("hd,start,cap", [(64, 100, 256), (128, 100, 256), (128, 3000, 4096), (64, 3000, 4096)])
def test_a_large_block_that_a_row_does_not_see_leaves_it_alone(ops, dt, times, hd, start, cap):
    """Rows before the block, in the same tile as rows that see it (with and without keys shared by a cluster)."""
    rows, group = 70, 2
    c = filled_cache(ops, 1, 1, cap, hd, [start + rows], seed=71)
    q = rand(1, rows, group, hd, seed=72).to(dt)
    big = (start + 40) // 16
    c[3][0, 0, big] *= times
    weighed_check(ops, q, c, [start], big * 16 - start)
    weighed_check(ops, q, c, [start])


def weightless_cache(ops, rows, group, hd, L, cap, at, times, seed):
    """A cache of L tokens whose block `at` has V scales `times` as large, and keys with some e^-30 of the weight."""
    c = filled_cache(ops, 1, 1, cap, hd, [L], seed=seed, kstd=0.3)
    q = rand(1, rows, group, hd, seed=seed + 3, std=0.3) + 1
    k = torch.full((1, 16, 1, hd), -30 / math.sqrt(hd), device="cuda")
    end = min(16, L - at * 16)
    z = torch.full((1,), at * 16, dtype=torch.int32, device="cuda")
    v = rand(1, 16, 1, hd, seed=seed + 4, std=0.5)
    ops.kv8_append(ops.Kv8Cache(*c), k[:, :end], v[:, :end], z)
    c[3][0, 0, at] *= times
    return c, q


def weightless(ops, dt, times, rows, group, hd, long):
    L = (3000 if long else 437) + rows
    cap = 4096 if long else 512
    for i, at in enumerate((0, 1, L // 32, (L - rows) // 16 - 1)):
        c, q = weightless_cache(ops, rows, group, hd, L, cap, at, times, 80 + i)
        weighed_check(ops, q.to(dt), c, [L - rows])


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("times", [1e2, 1e3, 1e5, 1e8])
@pytest.mark.parametrize("hd,long", [(64, False), (128, False), (128, True)])
@pytest.mark.parametrize("rows,group", PROMPT)
def test_a_large_block_without_weight_prompts(ops, dt, times, hd, long, rows, group):
    weightless(ops, dt, times, rows, group, hd, long)


def tails(ops, dt, rows, group, hd, bits, held):
    """The first key holds nearly all of the weight and has no value; the others, 2^-bits each, are the output. The
    V scales are alike here, so a weight is off by no more than 2^-held of the largest. (Unsplit: a warp that does not
    meet the first key holds its weights by its own.)"""
    L, cap = 3500 + rows, 4096
    c = filled_cache(ops, 1, 1, cap, hd, [L], seed=91, kstd=0.02)
    q = rand(1, rows, group, hd, seed=92, std=0.1) + 1
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    k = torch.full((1, 1, 1, hd), bits * math.log(2) / math.sqrt(hd), device="cuda")
    ops.kv8_append(ops.Kv8Cache(*c), k, torch.zeros_like(k), z)
    c[1].abs_()  # (values of one sign, whose loss adds up)
    for first in (0.0, c[3][0, 0, 1].item()):
        c[3][0, 0, 0] = first
        weighed_check(ops, q.to(dt), c, [L - rows], held=held, max_len=16)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("bits", [20, 24, 25, 27])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,group", PROMPT)
def test_many_keys_of_little_weight_prompts(ops, dt, bits, hd, rows, group):
    tails(ops, dt, rows, group, hd, bits, 36 if dt == F32 else 30)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("times", [1e2, 1e3, 1e5, 1e8])
@pytest.mark.parametrize("hd,long", [(64, False), (128, False), (128, True)])
@pytest.mark.parametrize("rows,group", DIGITS)
def test_a_large_block_without_weight_tokens(ops, dt, times, hd, long, rows, group):
    weightless(ops, dt, times, rows, group, hd, long)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("bits", [20, 24, 25, 27])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,group", DIGITS)
def test_many_keys_of_little_weight_tokens(ops, dt, bits, hd, rows, group):
    tails(ops, dt, rows, group, hd, bits, 32)


def test_tokens_over_scales_of_every_size(ops):
    """V scales from the smallest normal numbers to the largest, in any order, alone and side by side; a NaN among
    them reaches the rows that see it."""
    hd, cap = 128, 512
    q = rand(1, 1, 2, hd, seed=95)
    for seed in range(4):
        c = filled_cache(ops, 1, 1, cap, hd, [cap], seed=96)
        g = torch.Generator().manual_seed(seed)
        c[3][0, 0] = torch.exp2(torch.randint(-120, 110, (cap // 16,), generator=g).float()).cuda()
        for L in (1, 16, 17, 300, 512):
            weighed_check(ops, q, c, [L - 1])
        c[3][0, 0, 20] = math.nan
        st = torch.tensor([500], dtype=torch.int32, device="cuda")
        assert torch.isnan(ops.kv8_attention(q, ops.Kv8Cache(*c), st)).all()
        assert not torch.isnan(ops.kv8_attention(q, ops.Kv8Cache(*c), st - 181)).any()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("times", [1e2, 1e3, 1e5, 1e8])
@pytest.mark.parametrize("hd,long", [(64, False), (128, False), (128, True)])
@pytest.mark.parametrize("rows,group", STEP)
def test_a_large_block_without_weight_steps(ops, dt, times, hd, long, rows, group):
    weightless(ops, dt, times, rows, group, hd, long)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("bits", [20, 24, 25, 27])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,group", STEP)
def test_many_keys_of_little_weight_steps(ops, dt, bits, hd, rows, group):
    tails(ops, dt, rows, group, hd, bits, 39)


# ------------------------------------------------------------------ errors of the device
def test_check_waits_for_every_stream(ops):
    """A call still running on a stream that does not wait for the default one could give up after the check."""
    ops.check()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
    assert not side.query()
    ops.check()
    assert side.query()


def test_each_user_has_its_own_errors(tiny_dir):
    """Two engines on one GPU and the operators beside them: whoever's wait gave up hears of it, once, and no other."""
    import qwen_asr_b200 as Q
    from qwen_asr_b200 import ops, synth
    x = synth.synth_audio(16000 * 3, seed=97)
    a, b = Q.Engine(tiny_dir), Q.Engine(tiny_dir)
    for e in (a, b):
        e.set_prefill_mode("int8")
        e.set_kv_mode("int8")
        e.set_force_n_tokens(4)
    want = a.transcribe_pcm(x)
    assert want is not None and b.transcribe_pcm(x) == want
    report = Q.lib().qwen_asr_debug_report_ops_error
    ops.check()
    assert report(a._h, 33) == 0
    assert b.transcribe_pcm(x) == want
    ops.check()
    assert a.transcribe_pcm(x) is None and "33" in Q.last_error()
    assert a.transcribe_pcm(x) == want
    assert report(None, 51) == 0
    assert a.transcribe_pcm(x) == want and b.transcribe_pcm(x) == want
    with pytest.raises(RuntimeError, match="51"):
        ops.check()
    ops.check()


# ------------------------------------------------------------------ calls in a row
def test_every_call_sees_what_the_one_before_wrote(ops):
    """Long runs of calls that start beside one another, each reading what its predecessor, or the one before that,
    has just written over old values: the bits of the same calls with the device waited for in between."""
    n, n_kv, hd, heads, d = 4, 2, 128, 8, 512
    wq, ws = torch.randint(-127, 128, (2, (heads + 2 * n_kv) * hd, d), dtype=torch.int8, device="cuda"), rand(2, 1536, seed=1).abs() * 3e-4
    steps = [1, 1, 40, 1, 3, 1, 1, 70, 1, 20, 1, 1] * 3

    def run(wait):
        cache = ops.kv8_cache(n, n_kv, 1024, hd)
        w, scale, pos, out = torch.ones(d, device="cuda"), ws[0].clone(), torch.zeros(n, dtype=torch.int32, device="cuda"), []
        g = torch.Generator(device="cuda")
        g.manual_seed(5)
        for i, rows in enumerate(steps):
            x = torch.randn(n * rows, d, generator=g, device="cuda") * (1 + i % 3)
            w.mul_(1.01)  # weights and their scales may have been written just before, too
            q, s, h = ops.rms_norm_int8(x, w, residual=x)
            wait()
            scale.copy_(ws[i % 2])
            y = ops.linear_int8(q, s, wq[i % 2], scale).view(n, rows, -1).unflatten(2, (heads + 2 * n_kv, hd))
            wait()
            before = ops.kv8_attention(y[:, :, :heads], cache, pos)
            wait()
            ops.kv8_append(cache, y[:, :, heads:heads + n_kv], y[:, :, heads + n_kv:], pos)
            wait()
            after = ops.kv8_attention(y[:, :, :heads], cache, pos)
            wait()
            out += [h, before, after, *ops.kv8_read(cache, pos, rows)]
            pos += rows
            wait()
        torch.cuda.synchronize()
        return out
    want = run(torch.cuda.synchronize)
    for _ in range(5):
        for a, b in zip(run(lambda: None), want):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ values next to a rounding border
# (a, b, c, d, n): 127 a b / (c d) is within half an f64 step of n + 1/2, above or below it; found by solving
# 254 a b - (2 n + 1) c d = 1, -1, 2, ... in whole numbers under 2^24
BORDER = [(9187418, 11738396, 14744709, 11124571, 83), (15514599, 11641642, 12066306, 16602699, 114),
          (9678723, 15910658, 11891262, 15738585, 104), (10220674, 12154493, 10568986, 13886037, 107),
          (15889422, 9953404, 13779419, 13948781, 104), (9270475, 8855139, 8706701, 14004943, 85),
          (12467758, 12640073, 15177441, 13808285, 95), (9870208, 14882039, 13310854, 16016901, 87),
          (13935253, 14249515, 16281284, 14543884, 106), (9350045, 8942833, 15864436, 13522678, 49),
          (13429207, 9812132, 12548494, 14735921, 90), (11504340, 8951737, 16485217, 16358231, 48)]


@pytest.mark.parametrize("d", [64, 49, 4096, 16384])
def test_norm_values_within_an_f64_step_of_a_border(ops, d):
    """int8 values as in exact arithmetic, at quotients that f64 rounds onto a half or over it."""
    x, w = torch.zeros(4 * len(BORDER), d, device="cuda"), torch.ones(d, device="cuda")
    want = []
    for i, (a, b, c, e, n) in enumerate(BORDER):
        w[2 * i], w[2 * i + 1] = b, e * 2.0 ** -20
        assert 254 * a * b != (2 * n + 1) * c * e
        q = n + 1 if 254 * a * b > (2 * n + 1) * c * e else n
        for j, (s, t) in enumerate(((1, 1), (-1, 1), (1, -1), (-1, -1))):
            x[4 * i + j, 2 * i], x[4 * i + j, 2 * i + 1] = s * a * 2.0 ** -20, t * c
            want.append((s * q, t * 127))
    q, _, _ = ops.rms_norm_int8(x, w)
    q = q.cpu()
    for r, (a, b) in enumerate(want):
        i = r // 4
        assert (q[r, 2 * i].item(), q[r, 2 * i + 1].item()) == (a, b), r


# ------------------------------------------------------------------ tensors with derivatives
def test_tangents_and_negated_views_are_refused(ops):
    """A forward-mode tangent would be dropped, a negated view read without its sign."""
    from torch.autograd import forward_ad
    x, w = rand(4, 64), rand(64)
    q8, s = torch.randint(-127, 128, (4, 64), dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda")
    c = ops.kv8_cache(2, 2, 32, 128)
    z, k = torch.zeros(2, dtype=torch.int32, device="cuda"), rand(2, 1, 2, 128)
    calls = [(lambda t: ops.rms_norm_int8(t, w), x), (lambda t: ops.rms_norm_int8(x, t), w),
             (lambda t: ops.rms_norm_int8(x, w, residual=t), x), (lambda t: ops.linear_int8(q8, t, q8, s), s),
             (lambda t: ops.linear_int8(q8, s, q8, t), s), (lambda t: ops.linear_int8(q8, s, q8, s, residual=t), rand(4, 4)),
             (lambda t: ops.kv8_append(c, t, k, z), k), (lambda t: ops.kv8_append(c, k, t, z), k),
             (lambda t: ops.kv8_attention(t, c, z), k), (lambda t: ops.kv8_attention(k, c._replace(v_scale=t), z), c.v_scale),
             (lambda t: ops.kv8_read(c._replace(k_scale=t), z, 1), c.k_scale)]
    ints = [(lambda t: ops.linear_int8(t, s, q8, s), q8), (lambda t: ops.linear_int8(q8, s, t, s), q8),
            (lambda t: ops.kv8_read(c._replace(k=t), z, 1), c.k), (lambda t: ops.kv8_append(c, k, k, t), z),
            (lambda t: ops.kv8_attention(k, c, z, t), z)]
    for i, (f, t) in enumerate(calls + ints):
        f(t)
        with pytest.raises(ValueError, match="negated"):
            f(torch._neg_view(t))
        if i < len(calls):
            with forward_ad.dual_level():
                with pytest.raises(ValueError, match="tangent"):
                    f(forward_ad.make_dual(t, torch.ones_like(t)))
                f(t)


def test_append_counts_as_a_change_of_the_cache(ops):
    """A backward pass that saved the cache's values from before must not use those after."""
    c = ops.kv8_cache(1, 1, 32, 64)
    k, z = rand(1, 3, 1, 64), torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv8_append(c, k, k, z)
    w = torch.ones(1, device="cuda", requires_grad=True)
    for t in (c.k_scale, c.v_scale):
        y = (t * w).sum()
        y.backward()
        y = (t * w).sum()
        ops.kv8_append(c, 3 * k, 3 * k, z + 3)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    versions = [t._version for t in c]
    ops.kv8_append(c, k[:, :0], k[:, :0], z)
    ops.kv8_attention(k, c, z)
    ops.kv8_read(c, z, 3)
    assert [t._version for t in c] == versions
    ops.kv8_append(c, k, k, z)
    assert all(t._version > v for t, v in zip(c, versions))
    with torch.inference_mode():
        c = ops.kv8_cache(1, 1, 32, 64)
        ops.kv8_append(c, k, k, z)
        assert c.k_scale.any()


# ------------------------------------------------------------------ arguments past 32 bits
def test_arguments_past_32_bits(ops):
    """A stride of positions, a number of rows and a length whose lower 32 bits are another number."""
    n, cap = 2, 64
    c = filled_cache(ops, n, 1, cap, 64, [cap, cap], seed=98)
    cache = ops.Kv8Cache(*c)
    q, k = rand(n, 1, 2, 64, seed=99), rand(n, 1, 1, 64, seed=100)
    near = torch.tensor([3, 40], dtype=torch.int32, device="cuda")
    table = torch.zeros(2 ** 32 + 2, dtype=torch.int32, device="cuda")
    far = table[::2 ** 32 + 1]
    far.copy_(near)
    assert far.stride(0) == 2 ** 32 + 1
    assert torch.equal(ops.kv8_attention(q, cache, far), ops.kv8_attention(q, cache, near))
    assert torch.equal(ops.kv8_attention(q, cache, near, far), ops.kv8_attention(q, cache, near, near))
    for a, b in zip(ops.kv8_read(cache, far, 5, far), ops.kv8_read(cache, near, 5, near)):
        assert torch.equal(a, b)
    before = [t.clone() for t in c]
    ops.kv8_append(cache, k, k, far)
    after = [t.clone() for t in c]
    for t, b in zip(c, before):
        t.copy_(b)
    ops.kv8_append(cache, k, k, near)
    assert all(torch.equal(a, b) for a, b in zip(c, after))
    del table, far
    many = k[:, :, :, :1].expand(n, 2 ** 32 + 1, 1, 64)
    with pytest.raises(ValueError, match="rows"):
        ops.kv8_append(cache, many, many, near)
    with pytest.raises(ValueError, match="rows"):
        ops.kv8_attention(many, cache, near)
    with pytest.raises(ValueError, match="rows"):
        ops.kv8_read(cache, near, 2 ** 31)
    want = ops.kv8_attention(q, cache, near)
    for m in (2 ** 32 + 16, 2 ** 80, -1, cap + 1):
        assert torch.equal(ops.kv8_attention(q, cache, near, max_len=m), want)
    with pytest.raises(TypeError):
        ops.kv8_attention(q, cache, near, max_len=1.5)
    assert torch.equal(ops.kv8_attention(q, cache, near, scale=torch.tensor(0.125)), want)
    assert torch.equal(ops.kv8_attention(q, cache, near, scale=0.125, max_len=torch.tensor(64)), want)


# ------------------------------------------------------------------ refusals
def test_refusals_are_of_the_documented_type(ops):
    """A wrong type is a TypeError and an argument that does not fit a ValueError, before anything is enqueued: never
    a launch that CUDA refuses, which is a RuntimeError."""
    x, w, s = rand(4, 64), rand(64), torch.ones(4, device="cuda")
    q8 = torch.ones(4, 64, dtype=torch.int8, device="cuda")
    c, z, k = ops.kv8_cache(2, 2, 32, 128), torch.zeros(2, dtype=torch.int32, device="cuda"), rand(2, 1, 2, 128)
    both = ops.Kv8Cache(*[t.expand(2, *t.shape[1:]) for t in ops.kv8_cache(1, 2, 32)])
    bad = [
        (TypeError, lambda: ops.rms_norm_int8(x.half(), w)), (TypeError, lambda: ops.rms_norm_int8(x, w.to(BF16))),
        (TypeError, lambda: ops.rms_norm_int8(x, w, residual=x.to(BF16))),
        (ValueError, lambda: ops.rms_norm_int8(x, w[:63])), (ValueError, lambda: ops.rms_norm_int8(x.T, rand(4))),
        (ValueError, lambda: ops.rms_norm_int8(x, w, eps=-1.0)), (ValueError, lambda: ops.rms_norm_int8(x, w, eps=math.nan)),
        (ValueError, lambda: ops.rms_norm_int8(x, w.cpu())), (ValueError, lambda: ops.rms_norm_int8(x.cpu(), w)),
        (ValueError, lambda: ops.rms_norm_int8(x.clone().requires_grad_(), w)), (ValueError, lambda: ops.rms_norm_int8(x[0], w)),
        (ValueError, lambda: ops.rms_norm_int8(rand(1, 40000), rand(40000))), (ValueError, lambda: ops.rms_norm_int8(x[:, :0], w[:0])),
        (ValueError, lambda: ops.linear_int8(q8, s, q8[:, :32], s)), (ValueError, lambda: ops.linear_int8(q8[:, 1:33], s, q8[:, :32], s)),
        (ValueError, lambda: ops.linear_int8(q8[:, :60].contiguous(), s, q8[:, :60], s)),
        (ValueError, lambda: ops.linear_int8(q8, s[:3], q8, s)), (ValueError, lambda: ops.linear_int8(q8, s, q8[:3], s[:3], swiglu=True)),
        (ValueError, lambda: ops.linear_int8(q8, s, q8, s, residual=rand(4, 4), swiglu=True)),
        (ValueError, lambda: ops.linear_int8(q8, s, q8, s, residual=rand(4, 5))), (ValueError, lambda: ops.linear_int8(q8, s, q8[:0], s[:0])),
        (ValueError, lambda: ops.linear_int8(q8[:1].expand(4, 64), s, q8, s)),
        (TypeError, lambda: ops.linear_int8(q8, s, q8, s, dtype=torch.float16)), (TypeError, lambda: ops.linear_int8(x, s, q8, s)),
        (TypeError, lambda: ops.linear_int8(q8, s, q8, s, residual=rand(4, 4).to(BF16))),
        (ValueError, lambda: ops.kv8_append(c, k[:1], k[:1], z)), (ValueError, lambda: ops.kv8_append(c, k, k[..., :64], z)),
        (TypeError, lambda: ops.kv8_append(c, k, k, z.long())), (TypeError, lambda: ops.kv8_append(c, k, k.to(BF16), z)),
        (ValueError, lambda: ops.kv8_append(c, k, k, z[:1])), (ValueError, lambda: ops.kv8_append(c, k, k, z[:1].expand(2))),
        (ValueError, lambda: ops.kv8_append(both, k, k, z)), (ValueError, lambda: ops.kv8_read(both, z, 1)),
        (ValueError, lambda: ops.kv8_append(c, k.transpose(2, 3).contiguous().transpose(2, 3), k, z)),
        (ValueError, lambda: ops.kv8_append(c._replace(v=c.v.transpose(1, 2)), k, k, z)),
        (ValueError, lambda: ops.kv8_append(c, k, k, z, z.cpu())), (ValueError, lambda: ops.kv8_attention(k, both, z)),
        (ValueError, lambda: ops.kv8_attention(rand(2, 1, 3, 128), c, z)), (ValueError, lambda: ops.kv8_attention(rand(2, 1, 4, 64), c, z)),
        (ValueError, lambda: ops.kv8_attention(rand(2, 1, 1024, 128), c, z)), (ValueError, lambda: ops.kv8_read(c, z, -1)),
        (ValueError, lambda: ops.kv8_read(ops.kv8_cache(1, 1, 16, 96), z[:1], 1)), (TypeError, lambda: ops.kv8_read(c, z, 1, dtype=torch.float16)),
        (TypeError, lambda: ops.kv8_attention([1], c, z)), (TypeError, lambda: ops.kv8_read(c, z, 1.5)),
    ]
    for i, (err, f) in enumerate(bad):
        with pytest.raises(Exception) as e:
            f()
        assert type(e.value) is err, (i, e.value)
    assert not c.k.any() and not c.k_scale.any()


def test_a_mode_that_does_not_fit_leaves_the_engine_as_it_was(tiny_dir):
    """set_kv_mode without memory for the other cache: -1, and what follows runs as before."""
    import qwen_asr_b200 as Q
    from qwen_asr_b200 import synth
    x = synth.synth_audio(16000 * 3, seed=101)
    eng = Q.Engine(tiny_dir)
    eng.set_force_n_tokens(4)
    eng.grow_kv(1 << 18)  # (caches that do not fit into what the fill below leaves)
    want, ids = eng.transcribe_pcm(x), eng.last_tokens()
    torch.cuda.empty_cache()
    for mode in (1, 0):
        held = []
        for size in (8 << 30, 1 << 30, 128 << 20, 16 << 20, 2 << 20):
            try:
                while True:
                    held.append(torch.empty(size, dtype=torch.uint8, device="cuda"))
            except torch.OutOfMemoryError:
                pass
        failed = Q.lib().qwen_asr_set_kv_mode(eng._h, mode)
        del held
        torch.cuda.empty_cache()
        assert failed == -1
        assert eng.transcribe_pcm(x) == want, Q.last_error()
        if mode == 1:
            assert eng.last_tokens() == ids
            eng.set_kv_mode("int8")
            want, ids = eng.transcribe_pcm(x), eng.last_tokens()
        else:
            assert eng.last_tokens() == ids


# ------------------------------------------------------------------ scores of any size
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("size", [1e3, 1e5, 1e7, 1e9, 1e15, 1e25, 1e33])
@pytest.mark.parametrize("near,far", [(1.0, -0.5), (-0.25, -1.0), (1.0, 0.5)])
@pytest.mark.parametrize("rows,group", [(1, 2), (1, 4), (3, 5), (70, 2)])
def test_one_key_far_above_the_others(ops, dt, size, near, far, rows, group):
    """Scores of about near * size, of one key, and far * size, of all others, as far as f32 goes: the output is the
    one key's value (the weights of the others are 0 in f32), whatever the rounding of such scores."""
    hd, cap = 64, 512
    L = 300 + rows
    for at in (0, 5, 299):
        c = filled_cache(ops, 1, 1, cap, hd, [L], seed=102)
        k = far * (1 + 0.1 * rand(1, L, 1, hd, seed=103).clamp(-2, 2))
        k[0, at] = near
        z = torch.zeros(1, dtype=torch.int32, device="cuda")
        ops.kv8_append(ops.Kv8Cache(*c), k, rand(1, L, 1, hd, seed=104), z)
        # (one sign and no cancellation: a score is off by 2^-6 of itself at most, int8 keys and rounding together)
        q = (size / math.sqrt(hd) * (1 + 0.1 * rand(1, rows, group, hd, seed=105).clamp(-2, 2))).to(dt)
        got = ops.kv8_attention(q, ops.Kv8Cache(*c), z + 300)
        want = (c[1][0, 0, at].double() * c[3][0, 0, at // 16].double()).expand_as(got)
        assert ((got.double() - want).abs() <= want.abs() * (2.0 ** -20 + HALF[dt])).all(), at


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("rows,group", [(1, 2), (1, 4), (3, 5), (70, 2)])
def test_equal_scores_of_any_size(ops, dt, rows, group):
    """Equal keys far below zero: the mean of the values."""
    hd, cap, L = 64, 512, 300 + rows
    v = rand(1, L, 1, hd, seed=106)
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    for size in (1.0, 1e6, 1e12, 1e31, 1e36):
        c = filled_cache(ops, 1, 1, cap, hd, [L], seed=107)
        ops.kv8_append(ops.Kv8Cache(*c), torch.full_like(v, -math.sqrt(size)), v, z)
        q = torch.full((1, rows, group, hd), math.sqrt(size) / math.sqrt(hd), device="cuda", dtype=dt)
        got = ops.kv8_attention(q, ops.Kv8Cache(*c), z + 300)
        vv = c[1][0, 0, :L].double() * c[3][0, 0].repeat_interleave(16)[:L, None].double()
        for r in range(rows):
            want = vv[:301 + r].mean(0)
            # weights alike: 2^-11 of each in one f16 plane, 2^-22 in two and the f32 sums
            slack = vv[:301 + r].abs().mean(0) * (2.0 ** -19 if dt == F32 else 2.0 ** -11)
            assert ((got[0, r].double() - want).abs() <= slack + want.abs() * HALF[dt]).all(), (size, r)


# ------------------------------------------------------------------ the largest shapes
def test_heads_past_2_gib_in_a_sequence_of_a_million_tokens():
    """Positions near the end of a cache whose last heads start more than 2^31 bytes behind the first."""
    from qwen_asr_b200 import ops
    n_kv, hd, cap, new = 18, 128, (1 << 20) + 16, 100
    c = ops.kv8_cache(1, n_kv, cap, hd)
    assert (n_kv - 1) * cap * hd > 2 ** 31
    start = (1 << 20) - 37
    z = torch.full((1,), start, dtype=torch.int32, device="cuda")
    k, v = rand(1, new, n_kv, hd, seed=110), rand(1, new, n_kv, hd, seed=111)
    k *= 6  # (some of the new keys outweigh the million zeros)
    ops.kv8_append(c, k, v, z)
    kr, vr = ops.kv8_read(c, z, new)
    assert not kr[0, cap - start:].any() and not vr[0, cap - start:].any()
    for rows, heads, dt in ((1, 18, F32), (1, 36, BF16), (3, 36, F32), (6, 54, BF16), (60, 36, F32), (40, 54, BF16)):
        q = rand(1, rows, heads, hd, seed=112).to(dt) * 2
        got = ops.kv8_attention(q, c, z)
        for h in (0, heads - 1):
            kk, vv = kr[0, :, h * n_kv // heads].double(), vr[0, :, h * n_kv // heads].double()
            x = q[0, :, h].double() @ kk.T / math.sqrt(hd)                      # the zeros before have a score of 0
            x = x.masked_fill(torch.arange(new, device="cuda") > torch.arange(rows, device="cuda")[:, None], -math.inf)
            top = x.amax(1, keepdim=True).clamp_min(0)
            p = torch.exp(x - top)
            l = p.sum(1, keepdim=True) + start * torch.exp(-top)
            # scores off by d, weights held to 2^-22 or 2^-11 and by 2^-29 of the largest (the zeros have no value); l
            # by at most 4096 sums in f32 one after the other (a million keys in blocks of 64, four parts): 2^-12
            d = 2 * 2.0 ** -21 / math.sqrt(hd) * (q[0, :, h].double().abs().amax(1) * kk.abs().sum(1).amax())[:, None]
            held = 2.0 ** -22 if dt == F32 else 2.0 ** -11
            size = p @ vv.abs() / l
            tol = size * (d + held + 2.0 ** -12 + 2.0 ** -22) + (p @ vv / l).abs() * HALF[dt]
            tol += new * 2.0 ** -29 * vv.abs().max() / l
            assert ((got[0, :, h].double() - p @ vv / l).abs() <= tol).all(), (rows, heads, dt, h)


def test_many_sequences_and_many_heads():
    """65535 sequences, and 4096 KV heads: the last ones as the first."""
    from qwen_asr_b200 import ops
    for n, n_kv, rows, group in ((65535, 1, 1, 1), (65535, 1, 7, 2), (65535, 1, 70, 1), (2, 4096, 1, 1), (2, 4096, 5, 2), (2, 4096, 40, 2)):
        cap = 96
        c = ops.kv8_cache(n, n_kv, cap, 64)
        st = torch.randint(0, 20, (n,), generator=torch.Generator().manual_seed(n), dtype=torch.int32).cuda()
        k = rand(n, rows + 20, n_kv, 64, seed=113)
        ops.kv8_append(c, k, k, torch.zeros_like(st))
        q = rand(n, rows, n_kv * group, 64, seed=114)
        got = ops.kv8_attention(q, c, st)
        for i in sorted({0, 1, n // 2, n - 1}):
            for h in sorted({0, n_kv - 1}):
                few = [t[i:i + 1, h:h + 1].contiguous() for t in c]
                want, tol = weighed_ref(q[i:i + 1, :, h * group:(h + 1) * group], few, [st[i].item()], 1 / 8)
                assert ((got[i:i + 1, :, h * group:(h + 1) * group].double() - want).abs() <= tol).all(), (n, rows, i, h)
        back = ops.kv8_read(c, st, 2)[0]
        assert torch.equal(back[-1, :, -1], few[0][0, 0, st[-1]:st[-1] + 2].float() * few[2][0, 0].repeat_interleave(16)[st[-1]:st[-1] + 2, None])


def test_first_calls_of_many_threads_at_once():
    """Threads whose first calls come together, through the interface that does not hold the interpreter's lock."""
    import os
    import subprocess
    import sys
    code = """
import threading
import torch
from qwen_asr_b200 import ops
ops._fast = None
x, w = torch.randn(40, 512, device='cuda'), torch.ones(512, device='cuda')
wq = torch.randint(-127, 128, (1024, 512), dtype=torch.int8, device='cuda')
ws = torch.rand(1024, device='cuda')
z = torch.zeros(1, dtype=torch.int32, device='cuda')
start, out = threading.Barrier(16), [None] * 16
torch.cuda.synchronize()
def run(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        c = ops.kv8_cache(1, 2, 64, 128)
        start.wait()
        q, s, h = ops.rms_norm_int8(x, w, residual=x)
        y = ops.linear_int8(q, s, wq, ws)[None].unflatten(2, (8, 128))
        ops.kv8_append(c, y[:, :, 4:6], y[:, :, 6:], z)
        out[i] = (ops.kv8_attention(y[:, :, :4], c, z), ops.kv8_attention(y[:, :1, :4], c, z + 39))
        torch.cuda.current_stream().synchronize()
threads = [threading.Thread(target=run, args=(i,)) for i in range(16)]
[t.start() for t in threads]
[t.join() for t in threads]
ops.check()
assert all(o is not None and all(torch.equal(a, b) for a, b in zip(o, out[0])) for o in out)
print('alike')
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "alike" in r.stdout, r.stderr[-2000:]
