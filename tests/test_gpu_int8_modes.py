"""The engine's int8 prefill (set_prefill_mode) and int8 KV cache (set_kv_mode).

Their definition is the oracle's decoder with the same quantisation steps written in; a step may
fall on the other side of a rounding border (f32 against numpy's order of sums), so results are
compared by distance: what separates the engine from its definition must be under a quarter of
what the mode itself changes against the engine without it. Layer 0's cache, whose inputs both
modes compute alike, is compared exactly, and so is everything that the engine promises bit for
bit: batched against single sequences, streams together against streams alone, a grown cache."""
import numpy as np
import pytest

from qwen_asr_b200 import synth

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.fixture(scope="module")
def Q():
    import qwen_asr_b200 as Q
    return Q


def int8_rows(u):
    u = u.astype(np.float64)
    top = np.abs(u).max(axis=1, keepdims=True)
    top[top == 0] = 1
    return np.rint(u * 127.0 / top), top[:, 0]


def int8_linear(q, s, L, key):
    return ((q @ L[key + "_i8"].astype(np.float64).T).astype(F32) * s[:, None]).astype(F32) * L[key + "_s"]


def make_decoder(O, int8_prefill, int8_kv):
    class Dec(O.Decoder):
        def __init__(self, model):
            super().__init__(model)
            c = model.cfg
            self.codes = np.zeros((2, c.dec_layers, c.dec_kv_heads, self.kv.max_seq, 128))
            self.scales = np.zeros((2, c.dec_layers, c.dec_kv_heads, self.kv.max_seq // 16), dtype=F32)

        def write(self, i, li, start, rows):  # rows [n, heads, 128] behind `start`
            cache = (self.kv.k, self.kv.v)[i]
            if not int8_kv:
                cache[li, :, start:start + len(rows)] = rows.transpose(1, 0, 2)
                return
            q, s = self.codes[i, li], self.scales[i, li]
            end = start + len(rows)
            for b in range(start // 16, -(-end // 16)):
                lo, hi = max(start, b * 16), min(end, b * 16 + 16)
                x = rows[lo - start:hi - start].transpose(1, 0, 2).astype(np.float64)
                was = s[:, b].astype(np.float64) if lo > b * 16 else np.zeros(len(s))
                now = np.maximum(was, (np.abs(x).max(axis=(1, 2)).astype(F32) / F32(127)).astype(np.float64))
                safe = np.where(now > 0, now, 1)[:, None, None]
                q[:, b * 16:lo] = np.rint(q[:, b * 16:lo] * was[:, None, None] / safe)
                q[:, lo:hi] = np.clip(np.rint(x / safe), -127, 127)
                s[:, b] = now
                cache[li, :, b * 16:hi] = q[:, b * 16:hi].astype(F32) * s[:, b, None, None]

        def prefill(self, embeds):
            m, c = self.m, self.m.cfg
            seq = embeds.shape[0]
            x = embeds.astype(F32).copy()
            cos, sin = self._rope(0, seq)
            for li, L in enumerate(m.dec_layers):
                if int8_prefill:
                    def norm(w):
                        q, top = int8_rows(x.astype(np.float64) * w)
                        rms = np.sqrt((x.astype(np.float64) ** 2).mean(axis=1) + float(c.eps))
                        return q, (top / rms / 127).astype(F32)

                    def rows(v):
                        q, top = int8_rows(v)
                        return q, (top / 127).astype(F32)
                    a = norm(L["n1"])
                    q, k, v = (int8_linear(*a, L, key) for key in ("wq", "wk", "wv"))
                else:
                    xn = O.rms_norm(x, L["n1"], c.eps)
                    q, k, v = (O._mm(xn, L[key]) for key in ("wq", "wk", "wv"))
                q = self._apply_rope(O.rms_norm(q.reshape(seq, -1, 128), L["qn"], c.eps), cos, sin)
                k = self._apply_rope(O.rms_norm(k.reshape(seq, -1, 128), L["kn"], c.eps), cos, sin)
                self.write(0, li, 0, k)
                self.write(1, li, 0, v.reshape(seq, -1, 128))
                att = self._attend(q, li, 0, seq).reshape(seq, -1)
                if int8_prefill:
                    x = (x + int8_linear(*rows(att), L, "wo")).astype(F32)
                    gu = int8_linear(*norm(L["n2"]), L, "gu")
                    x = (x + int8_linear(*rows(O.silu_mul(gu[:, 0::2], gu[:, 1::2])), L, "down")).astype(F32)
                else:
                    x = (x + O._mm(att, L["wo"])).astype(F32)
                    gu = O._mm(O.rms_norm(x, L["n2"], c.eps), L["gu"])
                    x = (x + O._mm(O.silu_mul(gu[:, 0::2], gu[:, 1::2]), L["down"])).astype(F32)
            self.kv.len = seq
            return x

        def step(self, embed):  # decoder_forward with bf16 weights
            m, c = self.m, self.m.cfg
            pos = self.kv.len
            x = embed.astype(F32).copy()
            cos, sin = self._rope(pos, 1)
            for li, L in enumerate(m.dec_layers):
                xn = O.rms_norm(x, L["n1"], c.eps)
                q, k, v = (((L[key] @ xn).astype(F32)).reshape(1, -1, 128) for key in ("wq", "wk", "wv"))
                q = self._apply_rope(O.rms_norm(q, L["qn"], c.eps), cos, sin)
                k = self._apply_rope(O.rms_norm(k, L["kn"], c.eps), cos, sin)
                self.write(0, li, pos, k)
                self.write(1, li, pos, v)
                x = ((L["wo"] @ self._attend(q, li, pos, 1).reshape(-1)).astype(F32) + x).astype(F32)
                gu = (L["gu"] @ O.rms_norm(x, L["n2"], c.eps)).astype(F32)
                x = ((L["down"] @ O.silu_mul(gu[0::2], gu[1::2])).astype(F32) + x).astype(F32)
            self.kv.len = pos + 1
            return (O.bf16_to_f32(m.lm_bits) @ O.rms_norm(x, m.norm, c.eps)).astype(F32)
    return Dec


def prompt(O, d, seconds, seed):
    model = O.Model(d, decode_mode="int8")
    c = O.Ctx.__new__(O.Ctx)
    c.model, c.tok, c.prompt, c.force_language = model, None, None, None
    return model, O.prompt_rows(c, model.encode(O.mel_spectrogram(synth.synth_audio(int(16000 * seconds), seed=seed))))


def dist(a, b):
    return float(np.linalg.norm(a.astype(np.float64) - b) / np.linalg.norm(b.astype(np.float64)))


@pytest.mark.parametrize("prefill,kv", [("int8", "f32"), ("bf16", "int8"), ("int8", "int8")])
def test_modes_match_their_definition(Q, tiny_dir, prefill, kv):
    from oracle import qwen_oracle as O
    model, rows = prompt(O, tiny_dir, 5.0, 81)
    n, steps = rows.shape[0], 20
    forced = np.random.default_rng(81).integers(0, 151643, steps).astype(np.int32)

    def engine(prefill, kv):
        eng = Q.Engine(tiny_dir)
        eng.set_decode_mode("bf16")
        eng.set_prefill_mode(prefill)
        eng.set_kv_mode(kv)
        _, lg, hid = eng.debug_decode(rows, steps, forced=forced, want_logits=True, want_hidden=True)
        return eng, lg, hid[:n - 1]

    eng, lg, hid = engine(prefill, kv)
    _, lg0, hid0 = engine("bf16", "f32")
    dec = make_decoder(O, prefill == "int8", kv == "int8")(model)
    ref = dec.prefill(rows[:-1])
    want, x = [], rows[-1]
    for i in range(steps):
        want.append(dec.step(x))
        x = model.embed(int(forced[i]))
    want = np.stack(want)
    assert dist(hid, ref) < dist(hid, hid0) / 4, (dist(hid, ref), dist(hid, hid0))
    assert dist(lg, want) < dist(lg, lg0) / 4, (dist(lg, want), dist(lg, lg0))
    # the modes cost what int8 costs: well under the 10 % at which the tokens' order would suffer
    assert dist(hid, hid0) < 0.1 and dist(lg, lg0) < 0.1


def test_kv8_first_layer_is_the_quantised_f32_cache(Q, tiny_dir):
    """Layer 0's keys and values are computed alike in both modes: its int8 cache holds exactly what
    quantising the f32 cache gives, prompt rows and decoded tokens."""
    from oracle import qwen_oracle as O
    model, rows = prompt(O, tiny_dir, 4.0, 82)
    steps = 37
    forced = np.random.default_rng(82).integers(0, 151643, steps).astype(np.int32)
    kept = {}
    for kv in ("f32", "int8"):
        eng = Q.Engine(tiny_dir)
        eng.set_decode_mode("bf16")
        eng.set_kv_mode(kv)
        eng.debug_decode(rows, steps, forced=forced, want_logits=True)
        kept[kv] = eng.debug_kv(0, rows.shape[0] - 1 + steps)
    dec = make_decoder(O, False, True)(model)
    n = rows.shape[0] - 1
    for i in range(2):
        full = kept["f32"][i].transpose(1, 0, 2)
        dec.write(i, 0, 0, full[:n])
        for p in range(n, n + steps):
            dec.write(i, 0, p, full[p:p + 1])
        want = (dec.kv.k, dec.kv.v)[i][0, :, :n + steps]
        assert np.array_equal(kept["int8"][i], want)


def test_kv8_batched_equals_single(Q, tiny_dir, m06_dir):
    """Segments decoded together give the final-step logits of one at a time bit for bit."""
    for d in (tiny_dir, m06_dir):
        for mode in ("int8", "bf16"):
            x = synth.synth_audio(16000 * 80, seed=83)
            kept = []
            for batch in (1, 0):
                eng = Q.Engine(d)
                eng.set_decode_mode(mode)
                eng.set_prefill_mode("int8")
                eng.set_kv_mode("int8")
                eng.set_language("English")
                eng.set_segment_sec(26.0)
                eng.set_force_n_tokens(12)
                used = eng.set_decode_batch(batch)
                eng.set_record_logits(True)
                eng.transcribe_pcm(x)
                kept.append((eng.recorded_logits(), used))
            (a, _), (b, ub) = kept
            assert ub >= 2 and a.size > 0 and a.shape == b.shape
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32)), (d, mode)


def test_kv8_streams_together_equal_streams_alone(Q, tiny_dir):
    n_streams, n_chunks, chunk = 3, 4, 32000
    audio = [synth.synth_audio(chunk * n_chunks, seed=320 + i) for i in range(n_streams)]

    def make():
        eng = Q.Engine(tiny_dir)
        eng.set_kv_mode("int8")
        eng.set_prefill_mode("int8")
        eng.set_language("English")
        eng.set_record_logits(True)
        return eng

    a, b = make(), make()
    many, singles = ([Q.Stream() for _ in range(n_streams)] for _ in range(2))
    for c in range(n_chunks):
        part = [x[c * chunk:(c + 1) * chunk] for x in audio]
        fin = c == n_chunks - 1
        assert Q.stream_push_many(a, many, part, finalize=fin) == [s.push(b, p, finalize=fin) for s, p in zip(singles, part)]
    assert a.last_tokens() == b.last_tokens()
    la, lb = a.recorded_logits(), b.recorded_logits()
    assert la.size > 0 and np.array_equal(la.view(np.uint32), lb.view(np.uint32))


def test_kv8_graph_and_plain_steps_and_grow(Q, tiny_dir):
    """Graph replays and plain launches give the same tokens; a grown cache keeps every value, and
    steps after the grow give the same logits."""
    from oracle import qwen_oracle as O
    x = synth.synth_audio(16000 * 6, seed=84)
    ids = []
    for graph in (True, False):
        eng = Q.Engine(tiny_dir)
        eng.set_kv_mode("int8")
        eng.set_use_graph(graph)
        eng.set_force_n_tokens(40)
        eng.transcribe_pcm(x)
        ids.append(eng.last_tokens())
    assert ids[0] == ids[1] and len(ids[0][0]) == 40
    model, rows = prompt(O, tiny_dir, 2.0, 85)
    eng = Q.Engine(tiny_dir)
    eng.set_kv_mode("int8")
    forced = np.random.default_rng(85).integers(0, 151643, 10).astype(np.int32)
    _, lg0, _ = eng.debug_decode(rows, 10, forced=forced, want_logits=True)
    P = rows.shape[0] - 1 + 10
    before = [eng.debug_kv(layer, P) for layer in range(model.cfg.dec_layers)]
    cap = eng.kv_capacity()
    assert eng.grow_kv(cap + 1) == 2 * cap
    for layer, (k, v) in enumerate(before):
        k2, v2 = eng.debug_kv(layer, P)
        assert np.array_equal(k, k2) and np.array_equal(v, v2)
    _, lg1, _ = eng.debug_decode(rows, 10, forced=forced, want_logits=True)
    assert np.array_equal(lg0.view(np.uint32), lg1.view(np.uint32))


def test_mode_switches_leave_the_other_path_as_it_was(Q, tiny_dir):
    """After int8 modes were on and off again, the default path gives its own logits bit for bit; a
    stream whose cache was emptied by a switch goes on from its prompt; bad modes are refused."""
    from oracle import qwen_oracle as O
    _, rows = prompt(O, tiny_dir, 3.0, 86)
    forced = np.random.default_rng(86).integers(0, 151643, 8).astype(np.int32)
    eng = Q.Engine(tiny_dir)
    _, lg0, _ = eng.debug_decode(rows, 8, forced=forced, want_logits=True)
    eng.set_kv_mode("int8")
    eng.set_prefill_mode("int8")
    _, lg1, _ = eng.debug_decode(rows, 8, forced=forced, want_logits=True)
    eng.set_kv_mode("f32")
    eng.set_prefill_mode("bf16")
    _, lg2, _ = eng.debug_decode(rows, 8, forced=forced, want_logits=True)
    assert np.array_equal(lg0.view(np.uint32), lg2.view(np.uint32)) and not np.array_equal(lg0, lg1)
    assert Q.lib().qwen_asr_set_kv_mode(eng._h, 2) == -1 and Q.lib().qwen_asr_set_prefill_mode(eng._h, -1) == -1
    x = synth.synth_audio(16000 * 8, seed=87)

    def push(switch):
        e = Q.Engine(tiny_dir)
        e.set_decode_mode("bf16")
        e.set_language("English")
        s = Q.Stream()
        for i in range(4):
            if switch and i == 2:
                e.set_kv_mode("int8")
                e.set_kv_mode("f32")
            s.push(e, x[i * 32000:(i + 1) * 32000], finalize=i == 3)
        return s.result()
    assert push(True) == push(False)


def test_kv8_forced_align(Q):
    """The aligner's whole-prompt prefill runs in both modes, with the words in order."""
    from tests.conftest import model_dir
    eng = Q.Engine(model_dir("tiny-aligner", 0))
    eng.set_kv_mode("int8")
    eng.set_prefill_mode("int8")
    out = eng.forced_align(synth.synth_audio(16000 * 4, seed=88), "one two three four", "English")
    assert [w["text"] for w in out] == ["one", "two", "three", "four"]
    starts = [w["start_ms"] for w in out]
    assert starts == sorted(starts)
