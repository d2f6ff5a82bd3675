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
