"""mc_sm100_logits_process bit for bit against the fp32 restatement of its stated order (and within rounding of 64 bits),
mc_sm100_token_history exactly, and a step that uses both with the linears and the sampler around them."""
import numpy as np
import pytest

import oracle_np as onp

SENTINEL = 0x1234


# ---- CPU -------------------------------------------------------------------------------------------------------------
def test_restatement_known_answers():
    l = onp.f32_to_bf16(np.float32([2.0, -2.0, 1.0, 4.0, -1.0]))
    counts, seen = np.int32([0, 3, 0, 2, 0]), np.array([True, True, False, True, False])
    out = onp.bf16_to_f32(onp.logits_process_f32(l, (2.0, 0.5, 0.25), counts, seen, np.array([1, 1, 1, 1, 0], bool), [2, 3, 2], [1.0, 8.0, 0.5]))
    assert out.tolist() == [1.0, -4.0 - 1.5 - 0.25, 2.5, 2.0 - 1.0 - 0.25 + 8.0, -np.inf]
    assert onp.pack_bits(np.arange(40)[None] % 2 == 1).tolist() == [[0xAAAAAAAA, 0xAA]]
    counts, seen = np.full((2, 4), 9, np.int32), np.ones((2, 4), bool)
    onp.token_history(counts, seen, [(1, [0, 2, 2, -1, 2, 7], 2)], True)
    assert counts.tolist() == [[9] * 4, [0, 0, 2, 0]] and seen[1].tolist() == [True, False, True, False]


FIELDS = ("struct_size", "table_vocab", "n_slots", "n_masks", "n_bias", "reserved", "d_counts", "d_seen", "d_mask", "d_bias_token", "d_bias_value", "d_status")


def _tables(pkg, **kw):
    return pkg.LOGITS_TABLES.pack(*[{"struct_size": 72, "table_vocab": 100, **kw}.get(f, 0) for f in FIELDS])


def test_logits_refusals(pkg):
    def call(logits=16, out=16, rows=1, vocab=100, rs=100, os=100, cfg=16, base=0, t=None):
        with pytest.raises(pkg.McError) as e:
            pkg.logits_process(logits, out, rows, vocab, rs, os, cfg, t if t is not None else _tables(pkg), index_base=base, stream=16)
        assert e.value.status == pkg.MC_E_INVALID_ARGUMENT
        return e.value.message
    for kw in (dict(logits=None), dict(out=None), dict(cfg=None), dict(rows=0), dict(rows=65536), dict(vocab=0), dict(rs=99), dict(out=32, os=99),
               dict(rs=100, os=101), dict(base=-1)):
        assert "invalid args" in call(**kw), kw
    for t in (dict(struct_size=8), dict(reserved=1), dict(table_vocab=99), dict(n_slots=1), dict(n_slots=1, d_counts=16), dict(n_masks=1),
              dict(n_bias=3, d_bias_token=16)):
        assert "invalid tables" in call(t=_tables(pkg, **t)), t
    assert "invalid tables" in call(base=1)                        # columns beyond the tables' vocabulary
    assert "invalid args" in call(logits=17) and "invalid args" in call(out=17)
    lib, good = pkg.lib(), [48, 1, 8, 8, 8, 0, 16, 16, 16]
    assert lib.mc_sm100_logits_process(pkg.LOGITS_CALL.pack(*good), None, None, 0) == pkg.MC_E_INVALID_ARGUMENT
    assert lib.mc_sm100_logits_process(None, _tables(pkg), None, 0) == pkg.MC_E_INVALID_ARGUMENT
    good[0] = 40
    assert lib.mc_sm100_logits_process(pkg.LOGITS_CALL.pack(*good), _tables(pkg), None, 0) == pkg.MC_E_INVALID_ARGUMENT
    assert "struct_size=40" in pkg.last_error()


def test_tables_take_what_every_tensor_holds(pkg):
    """The binding counts rows that all tensors of a table have; a table that misses one is refused."""
    import torch
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)   # noqa: E731
    f = pkg.LOGITS_TABLES.unpack(pkg.logits_tables(100, counts=i32(300), seen=i32(8), masks=i32(12), bias_token=i32(5), bias_value=torch.zeros(3)))
    assert f[:6] == (72, 100, 2, 3, 3, 0)
    for kw in (dict(counts=i32(300)), dict(seen=i32(8)), dict(bias_token=i32(5)), dict(bias_value=torch.zeros(3))):
        with pytest.raises(pkg.McError) as e:
            pkg.logits_process(16, 16, 1, 100, 100, 100, 16, pkg.logits_tables(100, **kw), stream=16)
        assert e.value.status == pkg.MC_E_INVALID_ARGUMENT and "invalid tables" in e.value.message


def test_misaligned_tables_are_refused(pkg):
    for i in range(6, 12):
        t = [72, 100, 1, 1, 1, 0, 16, 16, 16, 16, 16, 16]
        t[i] = 18
        with pytest.raises(pkg.McError) as e:
            pkg.logits_process(16, 16, 1, 100, 100, 100, 16, pkg.LOGITS_TABLES.pack(*t), stream=16)
        assert e.value.status == pkg.MC_E_INVALID_ARGUMENT and "invalid tables" in e.value.message
    ok = dict(counts=16, seen=16, tokens=16, offsets=16, prompt_len=16, slots=16, status=16)
    for bad in [{k: 18} for k in ok] + [dict(n_tokens=2 ** 31)]:
        kw = dict(ok, n_seqs=1, table_vocab=100, n_slots=1, n_tokens=4, stream=16)
        kw.update(bad)
        with pytest.raises(pkg.McError) as e:
            pkg.token_history(**kw)
        assert e.value.status == pkg.MC_E_INVALID_ARGUMENT and "invalid args" in e.value.message


def test_history_refusals(pkg):
    base = dict(counts=16, seen=16, tokens=16, n_seqs=2, table_vocab=10, n_tokens=2, n_slots=2)
    for kw in (dict(counts=None), dict(seen=None), dict(tokens=None), dict(n_seqs=0), dict(table_vocab=0), dict(n_tokens=1), dict(n_slots=0),
               dict(n_slots=1), dict(table_vocab=1 << 31), dict(n_slots=1 << 31)):
        with pytest.raises(pkg.McError) as e:
            pkg.token_history(**{**base, **kw}, stream=16)
        assert e.value.status == pkg.MC_E_INVALID_ARGUMENT and "invalid args" in e.value.message, kw
    for head in ((76, 2, 10, 2, 2, 0), (80, 2, 10, 2, 2, 2)):
        assert pkg.lib().mc_sm100_token_history(pkg.HISTORY_CALL.pack(*head, 16, 16, 16, 0, 0, 0, 0), None, 0) == pkg.MC_E_INVALID_ARGUMENT
        assert "invalid call struct" in pkg.last_error()
    assert pkg.lib().mc_sm100_token_history(None, None, 0) == pkg.MC_E_INVALID_ARGUMENT


def test_tensors_of_other_widths_are_refused(pkg):
    """Truth values for bits, 64-bit tokens or offsets, fp32 logits: refused by the binding before the call (nothing is launched: the
    tensors are the host's)."""
    import torch
    t = lambda dtype, *s: torch.zeros(s, dtype=dtype)  # noqa: E731
    i32, i64, bf, f32, f64, yes = torch.int32, torch.int64, torch.bfloat16, torch.float32, torch.float64, torch.bool
    for bad in (dict(counts=t(i64, 2, 100)), dict(counts=t(torch.int16, 2, 100)), dict(seen=t(yes, 2, 100)), dict(seen=t(i64, 2, 4)), dict(masks=t(yes, 2, 100)),
                dict(bias_token=t(i64, 3)), dict(bias_value=t(bf, 3)), dict(bias_value=t(f64, 3))):
        kw = {**dict(counts=t(i32, 2, 100), seen=t(i32, 2, 4), masks=t(i32, 2, 4), bias_token=t(i32, 3), bias_value=t(f32, 3)), **bad}
        with pytest.raises(pkg.McError) as e:
            pkg.logits_tables(100, **kw)
        assert e.value.status == pkg.MC_E_INVALID_ARGUMENT and "logits_tables: " in e.value.message, list(bad)
    for bad in (dict(logits=t(f32, 1, 100)), dict(out=t(f32, 1, 100)), dict(cfg=t(i64, 1, 8)), dict(cfg=t(bf, 1, 8))):
        kw = {**dict(logits=t(bf, 1, 100), out=t(bf, 1, 100), cfg=t(i32, 1, 8)), **bad}
        with pytest.raises(pkg.McError) as e:
            pkg.logits_process(**kw, n_rows=1, vocab=100, row_stride=100, out_stride=100, tables=_tables(pkg), stream=16)
        assert e.value.status == pkg.MC_E_INVALID_ARGUMENT and "logits_process: " in e.value.message, list(bad)
    for bad in [{k: t(i64, 8)} for k in ("counts", "seen", "tokens", "offsets", "prompt_len", "slots")] + [dict(seen=t(yes, 8)), dict(tokens=t(torch.int16, 8))]:
        kw = {**{k: t(i32, 8) for k in ("counts", "seen", "tokens", "offsets", "prompt_len", "slots")}, **bad}
        with pytest.raises(pkg.McError) as e:
            pkg.token_history(**kw, n_seqs=1, table_vocab=4, n_slots=1, n_tokens=4, stream=16)
        assert e.value.status == pkg.MC_E_INVALID_ARGUMENT and "token_history: " in e.value.message, list(bad)


# ---- GPU: logits -----------------------------------------------------------------------------------------------------
def _config(rows):
    a = np.zeros((len(rows), 8), np.uint32)
    for i, (rep, freq, pres, slot, mask, begin, count) in enumerate(rows):
        a[i, :3] = np.float32([rep, freq, pres]).view(np.uint32)
        a[i, 3:7] = np.array([slot, mask, begin, count], np.int64).astype(np.uint32)
    return a


class Case:
    """Rows with every rule in turn: none, penalties, mask, biases, all; tables with more rows than are used."""

    def __init__(self, rows, vocab, seed, table_vocab=None, nb=20):
        g = np.random.default_rng(seed)
        self.rows, self.vocab, self.tv = rows, vocab, table_vocab or vocab
        self.logits = onp.f32_to_bf16((g.standard_normal((rows, vocab)) * 3).astype(np.float32))
        slots = rows + 2
        self.counts = g.integers(0, 4, (slots, self.tv)).astype(np.int32) * (g.random((slots, self.tv)) < 0.3)
        self.counts = self.counts.astype(np.int32)
        self.seen = (self.counts > 0) | (g.random((slots, self.tv)) < 0.1)
        self.mask = g.random((rows + 1, self.tv)) < np.linspace(0.0, 1.0, rows + 1)[:, None]      # row 0 leaves nothing
        self.bt, self.bv, cfg = [], [], []
        for r in range(rows):
            k = r % 5
            n = nb if k in (3, 4) else 0
            tok = g.integers(-2, self.tv + 2, n)
            if n > 3:
                tok[n // 2] = tok[0]                                    # the same token twice
                tok[n - 1] = tok[0]
            cfg.append((1.0 + 0.5 * g.random() if k in (1, 4) else 1.0, g.random() if k in (1, 4) else 0.0, g.random() if k in (1, 4) else 0.0,
                        int(g.integers(0, slots)) if k in (1, 4) else -1, int(g.integers(0, rows + 1)) if k in (2, 4) else -1, len(self.bt), n))
            self.bt += tok.tolist()
            self.bv += (g.standard_normal(n) * 5).astype(np.float32).tolist()
        self.cfg = cfg

    def want(self, base=0, columns=None, logits=None):
        out = []
        lg = self.logits if logits is None else logits
        for r, (rep, freq, pres, slot, mask, begin, count) in enumerate(self.cfg):
            hist = 0 <= slot < len(self.counts)
            cols = slice(base, base + (columns or self.vocab))
            out.append(onp.logits_process_f32(lg[r][cols] if columns else lg[r], (rep, freq, pres), self.counts[slot] if hist else None,
                                              self.seen[slot] if hist else None, self.mask[mask] if 0 <= mask < len(self.mask) else None,
                                              self.bt[begin:begin + count], self.bv[begin:begin + count], base))
        return np.stack(out)

    def run(self, pkg, in_place=False, in_pad=0, out_pad=0, base=0, columns=None, in_off=0, out_off=0, status=None, logits=None, pdl=False):
        import gpu_util as g
        import torch
        n = columns or self.vocab
        lg = (self.logits if logits is None else logits)[:, base:base + n]
        buf = torch.full((in_off + self.rows * (n + in_pad),), SENTINEL, dtype=torch.int16, device="cuda")
        buf[in_off:].view(self.rows, n + in_pad)[:, :n] = g.dev(lg)
        before = buf.clone()
        if in_place:
            out, out_pad, out_off = buf, in_pad, in_off
        else:
            out = torch.full((out_off + self.rows * (n + out_pad),), SENTINEL, dtype=torch.int16, device="cuda")
        bt, bv = np.int32(self.bt or [0]), np.float32(self.bv or [0])
        keep = [g.dev(self.counts), g.dev(onp.pack_bits(self.seen)), g.dev(onp.pack_bits(self.mask)), g.dev(bt), g.dev(bv), g.dev(_config(self.cfg))]
        t = pkg.logits_tables(self.tv, counts=keep[0], seen=keep[1], masks=keep[2], bias_token=keep[3], bias_value=keep[4], status=status)
        pkg.logits_process(buf[in_off:], out[out_off:], self.rows, n, n + in_pad, n + out_pad, keep[5], t, index_base=base, pdl=pdl)
        g.sync()
        got = g.host_u16(out)
        assert np.all(got[:out_off] == SENTINEL)
        got = got[out_off:].reshape(self.rows, n + out_pad)
        assert np.all(got[:, n:] == SENTINEL), "columns between the rows were written"
        if not in_place:
            assert torch.equal(before, buf), "the logits were written"
        return got[:, :n]


def _same(got, want):
    f, h = onp.bf16_to_f32(got), onp.bf16_to_f32(want)
    bad = ~((got == want) | (np.isnan(f) & np.isnan(h)))
    assert not bad.any(), [(tuple(i), float(f[tuple(i)]), float(h[tuple(i)])) for i in np.argwhere(bad)[:4]]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 32, 33, 255, 1000, 2048, 4099, 20000, 122753])
@pytest.mark.parametrize("rows", [1, 5, 12])
def test_logits_all_rules(pkg, rows, vocab):
    c = Case(rows, vocab, rows * 1000 + vocab)
    _same(c.run(pkg), c.want())
    _same(c.run(pkg, in_place=True), c.want())
    _same(c.run(pkg, in_pad=3, out_pad=6), c.want())
    _same(c.run(pkg, pdl=True), c.want())


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [(0, 0), (1, 1), (3, 5), (0, 7), (8, 4)])
def test_logits_alignment(pkg, offsets):
    for vocab in (8, 9, 515, 4097):
        c = Case(5, vocab, vocab)
        _same(c.run(pkg, in_off=offsets[0], out_off=offsets[1]), c.want())
        _same(c.run(pkg, in_off=offsets[0], out_off=offsets[1], in_pad=1, out_pad=2), c.want())
        _same(c.run(pkg, in_off=offsets[0], in_place=True), c.want())


@pytest.mark.gpu
def test_logits_within_rounding_of_64_bits(pkg):
    """Up to five fp32 operations on values below 64, then one rounding: 6 * 2^-24 * 64 + 2^-8 |l|."""
    c = Case(10, 5000, 4)
    got = onp.bf16_to_f32(c.run(pkg)).astype(np.float64)
    for r, (rep, freq, pres, slot, mask, begin, count) in enumerate(c.cfg):
        l = onp.bf16_to_f32(c.logits[r]).astype(np.float64)
        if slot >= 0:
            rep, freq, pres = (float(np.float32(v)) for v in (rep, freq, pres))
            l = np.where(c.seen[slot], np.where(l > 0, l / rep, l * rep), l) - freq * c.counts[slot] - pres * (c.counts[slot] > 0)
        for t, v in zip(c.bt[begin:begin + count], c.bv[begin:begin + count]):
            if 0 <= t < 5000:
                l[t] += v
        if mask >= 0:
            l[~c.mask[mask]] = -np.inf
        fin = np.isfinite(l)
        assert np.array_equal(fin, np.isfinite(got[r]))
        assert np.all(np.abs(got[r][fin] - l[fin]) <= 6 * 2.0 ** -24 * 64 + 2.0 ** -8 * np.abs(l[fin]))


@pytest.mark.gpu
def test_logits_values_at_the_edge(pkg):
    """Infinities, NaN, the type's lowest and highest values, zeros of both signs under every rule; biases of -infinity."""
    c = Case(5, 700, 9)
    special = np.uint16([0x7F80, 0xFF80, 0x7FC0, 0xFF7F, 0x7F7F, 0x0000, 0x8000, 0x0001, 0x8001])
    c.logits[:] = special[np.arange(700) % len(special)]
    c.bv[::3] = [float("-inf")] * len(c.bv[::3])
    _same(c.run(pkg), c.want())
    _same(c.run(pkg, in_place=True), c.want())


@pytest.mark.gpu
def test_logits_long_bias_lists(pkg):
    """Lists longer than a block, of one token only, and over every token."""
    g = np.random.default_rng(3)
    for vocab, tokens in ((300, [7] * 900), (5000, list(range(5000)) + list(range(0, 5000, 3))), (5000, g.integers(0, 40, 3000).tolist())):
        c = Case(1, vocab, 5)
        c.bt, c.bv = tokens, (g.standard_normal(len(tokens)) * 2).astype(np.float32).tolist()
        c.cfg = [(1.3, 0.2, 0.1, 0, -1, 0, len(tokens))]
        _same(c.run(pkg), c.want())
        _same(c.run(pkg, in_place=True), c.want())


@pytest.mark.gpu
def test_logits_vocab_shards(pkg):
    """Each shard against its columns of the whole; the tables are the whole vocabulary's."""
    c = Case(6, 3001, 21)
    whole = c.run(pkg)
    for base, columns in ((0, 1000), (1000, 1001), (2001, 1000)):
        _same(c.run(pkg, base=base, columns=columns), whole[:, base:base + columns])
        _same(c.run(pkg, base=base, columns=columns), c.want(base, columns))


@pytest.mark.gpu
def test_logits_rows_outside_the_tables_are_reported(pkg):
    import torch
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    c = Case(4, 500, 2)
    c.cfg = [(1.5, 0, 0, 2, -1, 0, 0)] * 4
    _same(c.run(pkg, status=status), c.want())
    assert status.item() == 0
    for bad in ((1.5, 0, 0, len(c.counts), -1, 0, 0), (1.5, 0, 0, 1, len(c.mask), 0, 0), (1.0, 0, 0, -1, -1, 0, len(c.bt) + 2),
                (1.0, 0, 0, -1, -1, 0xFFFFFFFF, 0xFFFFFFFF)):
        c.cfg[2] = bad
        status.zero_()
        if not c.bt:
            c.bt, c.bv = [0], [0.0]
        _same(c.run(pkg, status=status), c.want())
        assert status.item() == 1, bad
        _same(c.run(pkg), c.want())                                # without a status word


@pytest.mark.gpu
def test_a_row_without_tokens_still_gives_the_samplers_one(pkg):
    import gpu_util as g
    import torch
    c = Case(3, 600, 8)
    c.cfg = [(1, 0, 0, -1, 0, 0, 0)] * 3                           # mask row 0 allows nothing
    got = c.run(pkg)
    assert np.all(got == 0xFF80)
    d, out = g.dev(got), torch.full((3,), -7, dtype=torch.int32, device="cuda")
    stage = torch.zeros(pkg.argmax_stage_bytes(3), dtype=torch.uint8, device="cuda")
    pkg.launch_argmax_bf16(d, 3, 600, 600, 0, stage, out)
    assert all(0 <= v < 600 or v == 2 ** 31 - 1 for v in out.tolist())


# ---- GPU: history ----------------------------------------------------------------------------------------------------
def _history(pkg, slots, vocab, seqs, rebuild, seed=0, null=(), status=None):
    import gpu_util as g
    import torch
    r = np.random.default_rng(seed)
    counts, seen = r.integers(0, 5, (slots, vocab)).astype(np.int32), r.random((slots, vocab)) < 0.4
    words = (vocab + 31) // 32
    dc, ds = g.dev(counts), g.dev(onp.pack_bits(seen))
    flat = np.int32([t for s in seqs for t in s[1]])
    off = np.cumsum([0] + [len(s[1]) for s in seqs]).astype(np.uint32)
    dev = {"offsets": g.dev(off), "prompt_len": g.dev(np.uint32([s[2] for s in seqs])), "slots": g.dev(np.int32([s[0] for s in seqs]))}
    for k in null:
        dev[k] = None
    pkg.token_history(dc, ds, g.dev(flat), len(seqs), vocab, **dev, n_tokens=flat.size, rebuild=rebuild, status=status)
    g.sync()
    good = [s for s in seqs if 0 <= s[0] < slots]
    onp.token_history(counts, seen, good, rebuild)
    assert np.array_equal(dc.cpu().numpy(), counts)
    got = ds.cpu().numpy().view(np.uint32).reshape(slots, words)
    want = onp.pack_bits(seen)
    assert np.array_equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("rebuild", [False, True])
@pytest.mark.parametrize("vocab", [1, 31, 33, 1000, 50000, 122753])
def test_history(pkg, vocab, rebuild):
    r = np.random.default_rng(vocab)
    tok = lambda n: (r.random(n) ** 3 * vocab).astype(np.int64).tolist()  # noqa: E731
    _history(pkg, 3, vocab, [(1, tok(700), 300)], rebuild)
    _history(pkg, 6, vocab, [(5, tok(1), 0), (0, [], 0), (2, tok(3000), 3000), (3, tok(257), 9999), (1, tok(64) + [-1, vocab, vocab + 5, -2 ** 31], 1)], rebuild)
    _history(pkg, 4, vocab, [(2, tok(500), 10), (0, tok(5), 0), (2, tok(400), 0), (2, [], 0), (0, tok(90), 90)], rebuild)   # a slot named three times
    _history(pkg, 2, vocab, [(1, [0] * 5000, 4), (0, [vocab - 1] * 33, 0)], rebuild)                                       # one token only


@pytest.mark.gpu
def test_history_without_the_optional_arrays(pkg):
    for rebuild in (False, True):
        _history(pkg, 5, 300, [(i, [t], 0) for i, t in enumerate((4, -1, 299, 300))], rebuild, null=("offsets", "prompt_len", "slots"))
        _history(pkg, 5, 300, [(i, [t], 0) for i, t in ((4, 7), (0, 7), (2, 9))], rebuild, null=("offsets", "prompt_len"))
        _history(pkg, 5, 300, [(i, [t], 1) for i, t in ((4, 7), (0, 7), (4, 9))], rebuild, null=("offsets",))
        _history(pkg, 5, 300, [(0, [1, 2, 1], 0), (1, [], 0), (2, [5] * 70, 0)], rebuild, null=("slots", "prompt_len"))


@pytest.mark.gpu
def test_history_reports_what_it_passes_over(pkg):
    import gpu_util as g
    import torch
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for rebuild in (False, True):
        _history(pkg, 3, 200, [(1, [5, 6], 0), (2, [7], 0)], rebuild, status=status)
        assert status.item() == 0
        for bad in (-1, 3, 2 ** 31 - 1):
            _history(pkg, 3, 200, [(1, [5, 6], 0), (bad, [7, 8], 0), (2, [7], 0)], rebuild, status=status)
            assert status.item() == 1
            status.zero_()
        # offsets that leave the tokens, or run backwards: the sequence is passed over, its slot stays as it was
        for off in ([0, 2, 9], [0, 2, 1]):
            counts, seen = torch.full((2, 40), 3, dtype=torch.int32, device="cuda"), torch.zeros((2, 2), dtype=torch.int32, device="cuda")
            pkg.token_history(counts, seen, g.dev(np.int32([1, 1, 2])), 2, 40, offsets=g.dev(np.uint32(off)), rebuild=rebuild, status=status)
            assert status.item() == 1 and bool((counts[1] == 3).all()) and int(counts[0, 1]) == (2 if rebuild else 5)
            status.zero_()


@pytest.mark.gpu
def test_tables_beyond_32_bits(pkg):
    """Counts of slots whose entries lie beyond 2^32: rebuilt, added to, and read by the penalties."""
    import gpu_util as g
    import torch
    vocab, slots = 122753, 35100
    assert (slots - 1) * vocab > 2 ** 32
    words = (vocab + 31) // 32
    counts, seen = torch.zeros(slots * vocab, dtype=torch.int32, device="cuda"), torch.zeros(slots * words, dtype=torch.int32, device="cuda")
    d_slots = g.dev(np.int32([slots - 1, 2]))
    tok = np.int32([5, 7, 7, vocab - 1, 0, 0])
    pkg.token_history(counts, seen, g.dev(tok), 2, vocab, offsets=g.dev(np.uint32([0, 4, 6])), prompt_len=g.dev(np.uint32([1, 1])), slots=d_slots, rebuild=True)
    pkg.token_history(counts, seen, g.dev(np.int32([9, 9])), 2, vocab, slots=d_slots)
    last, third = counts[-vocab:].cpu().numpy(), counts[2 * vocab:3 * vocab].cpu().numpy()
    assert last.nonzero()[0].tolist() == [7, 9, vocab - 1] and last[[7, 9, vocab - 1]].tolist() == [2, 1, 1]
    assert third.nonzero()[0].tolist() == [0, 9] and int(torch.count_nonzero(counts)) == 5
    known = np.unpackbits(seen[-words:].cpu().numpy().view(np.uint8), bitorder="little")[:vocab].astype(bool)
    assert known.nonzero()[0].tolist() == [5, 7, 9, vocab - 1]
    logits = onp.f32_to_bf16(np.random.default_rng(1).standard_normal((1, vocab)).astype(np.float32) * 3)
    out = g.empty_u16(1, vocab)
    pkg.logits_process(g.dev(logits), out, 1, vocab, vocab, vocab, g.dev(_config([(1.5, 0.5, 0.25, slots - 1, -1, 0, 0)])), pkg.logits_tables(vocab, counts=counts, seen=seen))
    _same(g.host_u16(out), onp.logits_process_f32(logits[0], (1.5, 0.5, 0.25), last, known, None, [], [])[None])


# ---- GPU: together ---------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_prompt_then_steps_eager_and_replayed(pkg):
    """Prompt chunk through gated MLP, residual and lm_head, then sampled steps whose history feeds the next step's
    penalties: every stage against its restatement, and a captured step replayed against the eager ones."""
    import gpu_util as g
    import torch
    H, I, V, P, B = 256, 320, 1003, 37, 4
    f = onp.bf16_to_f32
    w1, w2, w3 = onp.seeded_bf16(1, (2 * I, H), 0.05), onp.seeded_bf16(2, (H, I), 0.05), onp.seeded_bf16(3, (V, H), 0.1)
    bias, x = onp.seeded_bf16(4, (V,), 0.3), onp.seeded_bf16(5, (P, H), 1.0)
    dx, h, logits = g.dev(x), g.empty_u16(P, I), g.empty_u16(B, V)
    y = g.empty_u16(P, H)
    d1, d2, d3, db = g.dev(w1), g.dev(w2), g.dev(w3), g.dev(bias)
    pkg.launch_linear_epilogue(d1, None, dx, h, P, 2 * I, H, activation="silu", gated=True)
    pkg.launch_linear_epilogue(d2, None, h, y, P, H, I, residual=dx)
    pkg.launch_linear_epilogue(d3, None, y[P - B:], logits, B, V, H, bias=db)
    g.sync()
    for got, args in ((h, (f(w1), f(x), None, None, None, "silu", True)), (y, (f(w2), f(g.host_u16(h)), None, None, f(x))),
                      (logits, (f(w3), f(g.host_u16(y))[P - B:], None, f(bias)))):
        want, bound = onp.linear_epilogue_f64(*args)
        assert np.all(np.abs(f(g.host_u16(got)).reshape(want.shape) - want) <= bound)
    prompt = [np.random.default_rng(r).integers(0, V, 11 * r).tolist() for r in range(B)]
    slots = [2, 0, 3, 1]
    mask = np.random.default_rng(9).random((1, V)) < 0.2
    cfg = g.dev(_config([(1.3, 0.4, 0.6, slots[r], 0 if r == 1 else -1, 3 * r, 3) for r in range(B)]))
    bt, bv = [5, 7, 5] * B, [2.0, float("-inf"), 1.0] * B
    d_mask, d_bt, d_bv = g.dev(onp.pack_bits(mask)), g.dev(np.int32(bt)), g.dev(np.float32(bv))
    scfg = np.zeros((B, 6), np.uint32)
    scfg[:, 0], scfg[:, 1], scfg[:, 2], scfg[:, 3] = np.float32(0.9).view(np.uint32), np.float32(0.95).view(np.uint32), 50, np.float32(1).view(np.uint32)
    d_scfg, d_slots = g.dev(scfg), g.dev(np.int32(slots))

    def session():
        s = {"counts": torch.full((B, V), 99, dtype=torch.int32, device="cuda"), "seen": torch.full((B, (V + 31) // 32), -1, dtype=torch.int32, device="cuda"),
             "edited": g.empty_u16(B, V), "token": torch.zeros(B, dtype=torch.int32, device="cuda"),
             "rng": g.dev(np.array([onp.splitmix64(70 + r) for r in range(B)], np.uint64).view(np.int64))}
        off = np.cumsum([0] + [len(p) for p in prompt]).astype(np.uint32)
        s["keep"] = [g.dev(np.int32(sum(prompt, []))), g.dev(off), g.dev(np.uint32([len(p) for p in prompt]))]
        pkg.token_history(s["counts"], s["seen"], s["keep"][0], B, V, offsets=s["keep"][1], prompt_len=s["keep"][2], slots=d_slots, rebuild=True)
        s["tables"] = pkg.logits_tables(V, counts=s["counts"], seen=s["seen"], masks=d_mask, bias_token=d_bt, bias_value=d_bv)
        return s

    def step(s):
        pkg.logits_process(logits, s["edited"], B, V, V, V, cfg, s["tables"], pdl=True)
        pkg.sample_topk_topp(s["edited"], B, V, V, d_scfg, s["rng"], s["token"], pdl=True)
        pkg.token_history(s["counts"], s["seen"], s["token"], B, V, slots=d_slots, pdl=True)

    s = session()
    counts, seen = np.zeros((B, V), np.int32), np.zeros((B, V), bool)
    onp.token_history(counts, seen, [(slots[r], prompt[r], len(prompt[r])) for r in range(B)], True)
    raw, drawn = g.host_u16(logits), []
    for _ in range(8):
        step(s)
        g.sync()
        want = np.stack([onp.logits_process_f32(raw[r], (1.3, 0.4, 0.6), counts[slots[r]], seen[slots[r]], mask[0] if r == 1 else None,
                                                bt[3 * r:3 * r + 3], bv[3 * r:3 * r + 3]) for r in range(B)])
        _same(g.host_u16(s["edited"]), want)
        tok = s["token"].tolist()
        assert mask[0, tok[1]] and 7 not in tok
        onp.token_history(counts, seen, [(slots[r], [tok[r]], 0) for r in range(B)], False)
        assert np.array_equal(s["counts"].cpu().numpy(), counts)
        drawn.append(tok)
    again = session()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(again)
    again2 = []
    for _ in range(8):
        graph.replay()
        torch.cuda.synchronize()
        again2.append(again["token"].tolist())
    assert again2 == drawn
    assert torch.equal(again["counts"], s["counts"]) and torch.equal(again["seen"], s["seen"])


def _many_slots(pkg, slots, vocab, seed):
    """As many sequences as slots, in turned order, a few tokens each: every entry of the rebuilt tables."""
    import gpu_util as g
    import torch
    r = np.random.default_rng(seed)
    tokens = r.integers(0, vocab, (slots, 50)).astype(np.int32)
    tokens[:, 0], tokens[:, 1], tokens[:, 2] = 0, vocab - 1, -1
    counts = torch.full((slots, vocab), 9, dtype=torch.int32, device="cuda")
    seen = torch.full((slots, (vocab + 31) // 32), -1, dtype=torch.int32, device="cuda")
    order = r.permutation(slots).astype(np.int32)
    pkg.token_history(counts, seen, g.dev(tokens.reshape(-1)), slots, vocab, offsets=g.dev(np.arange(slots + 1, dtype=np.uint32) * 50),
                      prompt_len=g.dev(np.full(slots, 20, np.uint32)), slots=g.dev(order), rebuild=True)
    g.sync()
    want, known = np.zeros((slots, vocab), np.int32), np.zeros((slots, vocab), bool)
    onp.token_history(want, known, [(int(order[i]), tokens[i].tolist(), 20) for i in range(slots)], True)
    assert np.array_equal(counts.cpu().numpy(), want)
    assert np.array_equal(seen.cpu().numpy().view(np.uint32), onp.pack_bits(known))


# A CTA of the rebuild takes ceil(vocab / floor(4 * 148 / slots)) tokens, a multiple of 32 between 2048 and 13664: sizes in front of, inside
# and behind the spans (11904 .. 11936) whose counters and bits pass 48 KB only together with the kernel's static shared memory.
@pytest.mark.gpu
@pytest.mark.parametrize("slots,vocab", [(64, 106800), (64, 107000), (64, 107136), (64, 107200), (52, 130800), (33, 202048), (64, 122753), (64, 20000), (148, 54657), (300, 30001)])
def test_history_of_many_slots(pkg, slots, vocab):
    _many_slots(pkg, slots, vocab, slots + vocab)


@pytest.mark.gpu
def test_history_of_many_slots_is_a_process_s_first_call():
    """No earlier call has raised the kernel's shared memory."""
    import subprocess
    import sys
    code = ("import sys; sys.path[:0] = %r\nimport importlib, test_logits_rules as t\n"
            "t._many_slots(importlib.import_module('minicpm5-5080fast_b200'), 64, 107000, 1)") % [p for p in sys.path if p]
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr[-2000:]
