"""The operators behind a step's answer, as they are timed: linears with a fused epilogue, the edit of the logits, and
the token history that the edit reads.

Three kinds of case.  "linear": y = act(x W^T scale + bias) + residual, bf16 or e4m3 weights, optionally gated over
interleaved (gate, up) rows.  "logits": repetition / frequency / presence penalties, sparse biases and grammar masks on
bf16 logits.  "history": the token counts and seen bits of a batch's slots, rebuilt from token lists.
"""
import importlib
import math

import torch

own = False

HIDDEN, QKV, GATE_UP, INTER, VOCAB = 2304, 3456, 11520, 5760, 122753   # the decode stack's configuration


def _pkg():
    return importlib.import_module("minicpm5-5080fast_b200")


# ---- cases ----------------------------------------------------------------------------------------------------------
def _linear(name, m, n, k, weights="bf16", bias=False, residual=False, act="none", gated=False, x_pad=0):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "weights": weights, "bias": bias, "residual": residual,
            "act": act, "gated": gated, "x_pad": x_pad}


def _logits(name, rows, vocab, past=0, bias=0, allowed=1.0, penalties=True, in_place=False):
    return {"name": name, "op": "logits", "rows": rows, "vocab": vocab, "past": past, "bias": bias, "allowed": allowed,
            "penalties": penalties, "in_place": in_place}


def _history(name, seqs, longest, vocab):
    return {"name": name, "op": "history", "seqs": seqs, "longest": longest, "vocab": vocab}


def listed():
    return [
        # one token of one session: down projection added to the residual stream
        _linear("down_m1_bf16", 1, HIDDEN, INTER, residual=True),
        # one token, e4m3 weights: gate and up with the SwiGLU behind them
        _linear("gate_up_m1_e4m3", 1, GATE_UP, HIDDEN, weights="e4m3", act="silu", gated=True),
        # a decode batch: fused qkv with a bias
        _linear("qkv_m16_bf16", 16, QKV, HIDDEN, bias=True),
        # the last positions of a batch of prompts through the lm_head; the vocabulary is odd, so rows of y are unaligned
        _linear("lm_head_m33_bf16", 33, VOCAB, HIDDEN, bias=True),
        # a short prompt: the output projection reads a column block of the wider qkv result
        _linear("o_m301_bf16", 301, HIDDEN, HIDDEN, bias=True, residual=True, x_pad=QKV - HIDDEN),
        # a long prompt chunk, e4m3 weights: down projection added to the residual stream
        _linear("down_m2048_e4m3", 2048, HIDDEN, INTER, weights="e4m3", residual=True),
        # the largest: a long prompt chunk through gate and up
        _linear("gate_up_m4096_bf16", 4096, GATE_UP, HIDDEN, act="silu", gated=True),
        # one session that writes under a grammar: few tokens allowed, a repetition penalty over a short history
        _logits("logits_1_row", 1, VOCAB, past=500, allowed=0.01),
        # grammar masks alone, applied in place
        _logits("logits_8_rows_mask_in_place", 8, VOCAB, allowed=0.3, penalties=False, in_place=True),
        # a full batch with every rule on
        _logits("logits_64_rows", 64, VOCAB, past=4000, bias=300, allowed=0.9),
        # a session comes back: its history is laid out again
        _history("history_1", 1, 1200, VOCAB),
        # a full batch comes back after a pause
        _history("history_64", 64, 8192, VOCAB),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "logits", "logits", "history"])
    if op == "linear":
        weights = rng.choice(["bf16", "e4m3"])
        step = 8 if weights == "bf16" else 16
        while True:
            m = _log_int(rng, 1, 8192)
            k = _log_int(rng, 256, 8192) // step * step
            n = _log_int(rng, 64, 24000)
            if 2 * 10 ** 5 <= m * n * k <= 4096 * GATE_UP * HIDDEN:
                break
        gated = rng.random() < 0.3
        return {"op": "linear", "m": m, "n": n // 2 * 2 if gated else n, "k": k, "weights": weights, "bias": rng.random() < 0.5,
                "residual": rng.random() < 0.5, "act": rng.choice(["silu", "gelu", "gelu_tanh", "relu"] + ([] if gated else ["none"] * 4)),
                "gated": gated, "x_pad": rng.choice([0, 0, 0, 64, 1152])}
    vocab = _log_int(rng, 1000, 160000)
    if op == "logits":
        in_place = rng.random() < 0.2
        return {"op": "logits", "rows": _log_int(rng, 1, 64), "vocab": vocab, "past": 0 if in_place else rng.choice([0, _log_int(rng, 1, 8192)]),
                "bias": 0 if in_place else rng.choice([0, _log_int(rng, 1, 400)]), "allowed": rng.choice([0.999, 0.5, 0.02] + ([] if in_place else [1.0])),
                "penalties": not in_place, "in_place": in_place}
    return {"op": "history", "seqs": _log_int(rng, 1, 64), "longest": _log_int(rng, 1, 8192), "vocab": vocab}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _tokens(shape, vocab, g):
    """Token ids as text has them: few ids make up most of it."""
    return (torch.rand(shape, generator=g, device="cuda") ** 3 * vocab).to(torch.int32).clamp_(max=vocab - 1)


def _pack_bits(flags):
    """[rows, vocab] truth values as 32-bit words, token t in bit t % 32 of word t // 32."""
    rows, vocab = flags.shape
    words = (vocab + 31) // 32
    padded = torch.zeros((rows, words * 32), dtype=torch.int64, device=flags.device)
    padded[:, :vocab] = flags
    value = (padded.view(rows, words, 32) << torch.arange(32, device=flags.device)).sum(2)
    return (value - ((value >> 31) << 32)).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    state = dict(case)
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        n_out = n // 2 if case["gated"] else n
        w = (randn(n, k) * 0.02).to(torch.bfloat16)
        state["w"], state["scale"] = w, None
        if case["weights"] == "e4m3":
            amax = w.float().abs().amax(1)
            state["scale"] = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
            state["w"] = (w.float() / state["scale"][:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        state["x"] = randn(m, k + case["x_pad"]).to(torch.bfloat16)       # the operator reads its first k columns
        state["bias_v"] = (randn(n) * 0.5).to(torch.bfloat16) if case["bias"] else None
        state["res"] = randn(m, n_out).to(torch.bfloat16) if case["residual"] else None
        state["y"] = torch.empty((m, n_out), dtype=torch.bfloat16, device="cuda")
    elif case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        state["logits"] = (randn(rows, vocab) * 2.5).to(torch.bfloat16)
        state["out"] = state["logits"] if case["in_place"] else torch.empty_like(state["logits"])
        slots = torch.randperm(rows, generator=g, device="cuda")
        counts = torch.zeros((rows, vocab), dtype=torch.int32, device="cuda")
        seen = torch.zeros((rows, vocab), dtype=torch.bool, device="cuda")
        if case["past"]:
            past = _tokens((rows, case["past"]), vocab, g).long()
            said = past[:, case["past"] // 2:]                            # the first half is the prompt
            seen.scatter_(1, past, True)
            counts.scatter_add_(1, said, torch.ones_like(said, dtype=torch.int32))
        state["counts"], state["seen"] = counts, _pack_bits(seen)
        masked = case["allowed"] < 1.0
        state["masks"] = _pack_bits(torch.rand(rows, vocab, generator=g, device="cuda") < case["allowed"]) if masked else None
        nb = case["bias"]
        state["bias_token"] = _tokens((rows * nb,), vocab, g) if nb else None
        state["bias_value"] = randn(rows * nb) * 4.0 if nb else None
        cfg = torch.zeros((rows, 8), dtype=torch.float32, device="cuda")
        if case["penalties"]:
            cfg[:, 0] = 1.0 + 0.4 * torch.rand(rows, generator=g, device="cuda")
            cfg[:, 1:3] = torch.rand(rows, 2, generator=g, device="cuda")
        else:
            cfg[:, 0] = 1.0
        cfg = cfg.view(torch.int32)
        cfg[:, 3] = slots.int() if case["past"] else -1
        cfg[:, 4] = torch.randperm(rows, generator=g, device="cuda").int() if masked else -1
        cfg[:, 5] = torch.arange(rows, device="cuda", dtype=torch.int32) * nb
        cfg[:, 6] = nb
        state["cfg"] = cfg
    else:
        seqs, vocab = case["seqs"], case["vocab"]
        lens = torch.randint(case["longest"] // 2, case["longest"] + 1, (seqs,), generator=g, device="cuda")
        state["offsets"] = torch.cat([torch.zeros_like(lens[:1]), lens.cumsum(0)]).int()
        state["n_tokens"] = int(state["offsets"][-1])
        state["tokens"] = _tokens((max(1, state["n_tokens"]),), vocab, g)
        state["prompt_len"] = (lens * 3 // 4).int()
        state["slots"] = torch.randperm(seqs, generator=g, device="cuda").int()
        state["counts"] = torch.full((seqs, vocab), 7, dtype=torch.int32, device="cuda")     # what the last sessions left
        state["seen"] = torch.full((seqs, (vocab + 31) // 32), -1, dtype=torch.int32, device="cuda")
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------
def _act(v, kind):
    if kind == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if kind == "gelu":
        return v * 0.5 * (1.0 + torch.erf(v * (1.0 / math.sqrt(2.0))))
    if kind == "gelu_tanh":
        return v * 0.5 * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if kind == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _bits(words, vocab):
    """[rows, vocab] truth values out of 32-bit words."""
    t = torch.arange(vocab, device=words.device)
    return (words[:, t // 32] >> (t % 32).int()) & 1 != 0


def _linear_plain(s):
    w = s["w"].float() if s["scale"] is None else s["w"].view(torch.float8_e4m3fn).float() * s["scale"][:, None]
    v = s["x"][:, :s["k"]].float() @ w.T
    if s["bias_v"] is not None:
        v = v + s["bias_v"].float()
    v = _act(v[:, 0::2], s["act"]) * v[:, 1::2] if s["gated"] else _act(v, s["act"])
    if s["res"] is not None:
        v = v + s["res"].float()
    return v.to(torch.bfloat16)


def _logits_plain(s):
    cfg, vocab = s["cfg"], s["vocab"]
    v = s["logits"].float()
    if s["past"]:
        slot = cfg[:, 3].long()
        rep, freq, pres = (cfg[:, i:i + 1].view(torch.float32) for i in range(3))
        c = s["counts"][slot].float()
        v = torch.where(_bits(s["seen"][slot], vocab), torch.where(v > 0, v / rep, v * rep), v)
        v = v - freq * c - pres * (c > 0)
    if s["bias_token"] is not None:
        j = torch.arange(s["bias_token"].numel(), device=v.device)
        row = (cfg[:, 5].long()[None, :] <= j[:, None]).sum(1) - 1
        v = v + torch.zeros_like(v).index_put_((row, s["bias_token"].long()), s["bias_value"], accumulate=True)
    if s["masks"] is not None:
        v = torch.where(_bits(s["masks"][cfg[:, 4].long()], vocab), v, torch.full_like(v, -math.inf))
    return v.to(torch.bfloat16)


def _history_plain(s):
    vocab, n = s["vocab"], s["n_tokens"]
    t = s["tokens"][:n].long()
    j = torch.arange(n, device=t.device)
    seq = torch.searchsorted(s["offsets"][1:].contiguous(), j.int(), right=True)
    slot = s["slots"].long()[seq]
    said = (j - s["offsets"].long()[seq] >= s["prompt_len"].long()[seq]).int()
    counts = torch.zeros_like(s["counts"]).index_put_((slot, t), said, accumulate=True)
    seen = torch.zeros(counts.shape, dtype=torch.bool, device=t.device).index_put_((slot, t), torch.ones_like(t, dtype=torch.bool))
    return counts, _pack_bits(seen)


def run(state):
    s = state
    if s["op"] == "linear":
        if not own:
            return _linear_plain(s)
        _pkg().launch_linear_epilogue(s["w"], s["scale"], s["x"], s["y"], s["m"], s["n"], s["k"], bias=s["bias_v"], residual=s["res"],
                                      activation=s["act"], gated=s["gated"], x_stride=s["k"] + s["x_pad"])
        return s["y"]
    if s["op"] == "logits":
        if not own:
            out = _logits_plain(s)
            return s["logits"].copy_(out) if s["in_place"] else out
        pkg = _pkg()
        tables = pkg.logits_tables(s["vocab"], counts=s["counts"], seen=s["seen"], masks=s["masks"], bias_token=s["bias_token"],
                                   bias_value=s["bias_value"])
        pkg.logits_process(s["logits"], s["out"], s["rows"], s["vocab"], s["vocab"], s["vocab"], s["cfg"], tables)
        return s["out"]
    if not own:
        return _history_plain(s)
    _pkg().token_history(s["counts"], s["seen"], s["tokens"], s["seqs"], s["vocab"], offsets=s["offsets"], prompt_len=s["prompt_len"],
                         slots=s["slots"], n_tokens=s["n_tokens"], rebuild=True)
    return s["counts"], s["seen"]


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        n_out = n // 2 if case["gated"] else n
        w = n * k * 2 if case["weights"] == "bf16" else n * k + 4 * n
        return {"bytes": w + 2 * m * k + 2 * m * n_out * (2 if case["residual"] else 1) + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    vocab = case["vocab"]
    if case["op"] == "logits":
        known = vocab * (1.0 - math.exp(-case["past"] / vocab)) if case["past"] else 0
        masked = case["allowed"] < 1.0
        row = 8 * case["bias"] + (vocab // 8 if case["past"] else 0) + int(4 * known) + (vocab // 8 if masked else 0) + 32
        row += int(2 * vocab * (1.0 - case["allowed"])) if case["in_place"] else 4 * vocab
        return {"bytes": case["rows"] * row, "flops": case["rows"] * vocab}
    tokens = case["seqs"] * case["longest"] * 3 // 4
    return {"bytes": 4 * tokens + case["seqs"] * (4 * vocab + vocab // 8 + 12), "flops": tokens}


# ---- 64 bits --------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        w = s["w"].double() if s["scale"] is None else s["w"].view(torch.float8_e4m3fn).double() * s["scale"].double()[:, None]
        z = torch.einsum("mk,nk->mn", s["x"][:, :case["k"]].double(), w)
        if s["bias_v"] is not None:
            z += s["bias_v"].double()
        a, other = (z[:, ::2], z[:, 1::2]) if case["gated"] else (z, 1.0)
        if case["act"] == "relu":
            a = a.clamp(min=0)
        elif case["act"] == "gelu":
            a = 0.5 * a * torch.erfc(-a / math.sqrt(2.0))
        elif case["act"] == "gelu_tanh":
            a = a * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (a + 0.044715 * a ** 3))
        elif case["act"] == "silu":
            a = a * torch.sigmoid(a)
        y = a * other
        return y if s["res"] is None else y + s["res"].double()
    vocab = case["vocab"]
    shifts = torch.arange(32, device="cuda", dtype=torch.int32)

    def unpack(words):
        return ((words[:, :, None] >> shifts) & 1).flatten(1)[:, :vocab].bool()

    if case["op"] == "logits":
        l, cfg = s["logits"].double(), s["cfg"]
        for r in range(case["rows"]):
            rep, freq, pres = cfg[r, :3].view(torch.float32).double()
            if case["past"]:
                h = int(cfg[r, 3])
                known, c = unpack(s["seen"][h:h + 1])[0], s["counts"][h].double()
                l[r] = torch.where(known & (l[r] > 0), l[r] / rep, torch.where(known, l[r] * rep, l[r])) - freq * c - pres * (c > 0)
            if case["bias"]:
                part = slice(int(cfg[r, 5]), int(cfg[r, 5]) + case["bias"])
                l[r].index_add_(0, s["bias_token"][part].long(), s["bias_value"][part].double())
            if s["masks"] is not None:
                k = int(cfg[r, 4])
                l[r][~unpack(s["masks"][k:k + 1])[0]] = -math.inf
        return l
    counts, seen = torch.zeros_like(s["counts"]), torch.zeros((case["seqs"], vocab), dtype=torch.bool, device="cuda")
    for i in range(case["seqs"]):
        a, b, p, h = int(s["offsets"][i]), int(s["offsets"][i + 1]), int(s["prompt_len"][i]), int(s["slots"][i])
        counts[h] = torch.bincount(s["tokens"][a + p:b], minlength=vocab).int()
        seen[h, s["tokens"][a:b].unique().long()] = True
    return counts, _pack_bits(seen)
