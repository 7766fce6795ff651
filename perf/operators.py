"""The timed operators between a model's logits and the choice of its next token.

A user who generates DNA over a tokenizer's vocabulary penalises what a row has seen, adds a bias and lets only those
tokens follow that an automaton over bases allows; a user who trains through that distribution needs its gradient.  Five
operators: ``process_logits``, its backward pass, ``TokenHistory`` (which tokens a row has seen, how often it generated
each), ``Grammar.allowed`` (the mask of an automaton's states) and ``Grammar.step`` (states after a token, and their
masks).  Where ``own`` is false ``run`` computes them from elementary torch operations.

Vocabularies are those of the tokenizers here: 10 ids (single bases), 512 (bytes), 4,106 (6-mers), 4,096 and 32,000
(BPE; tokens of 1 to 14 random bases).  The first five ids are specials, id 3 ends a sequence.
"""
import math

import numpy as np
import torch

own = False

LETTERS = np.frombuffer(b"ACGTN", dtype=np.uint8)      # classes 0..4 of the automata; every other byte counts as N
END = 3
DEAD, FINISHED = -1, -2
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


def _logits(name, rows, width, dtype, out="", penalties="row", seen=0.05, bias="shared", keep=0.9, last=False):
    """seen: share of the vocabulary in a row's history; penalties: "row" (a tensor with one value a row), "all" (one
    number) or "repetition" (only that one); keep: share of the tokens the mask allows, 0 for no mask; last: the logits are
    the last position of a [rows, 2, width] tensor."""
    return {"name": name, "op": "logits", "rows": rows, "width": width, "dtype": dtype, "out": out or dtype, "penalties": penalties,
            "seen": seen, "bias": bias, "keep": keep, "last": last}


def _grad(name, rows, width, dtype, bias="shared", seen=0.05, keep=0.9):
    c = _logits(name, rows, width, dtype, seen=seen, bias=bias, keep=keep)
    return {**c, "op": "grad"}


def _history(name, vocab, width, rows, layout, lo, hi, ids, generated):
    """rows of lo..hi tokens (log-uniform); layout: "right" or "left" (padded to hi) or "ragged"; ids: bits of an id."""
    return {"name": name, "op": "history", "vocab": vocab, "width": width, "rows": rows, "layout": layout, "lo": lo, "hi": hi,
            "ids": ids, "generated": generated}


def _mask(name, vocab, width, rows, automaton, size):
    """automaton: "avoid" (size motifs of 4 to 8 bases may not occur) or "pattern" (size positions, each with the bases
    it may hold)."""
    return {"name": name, "op": "mask", "vocab": vocab, "width": width, "rows": rows, "automaton": automaton, "size": size}


def _step(name, vocab, width, rows, dtype, automaton, size, lo, hi):
    """The step after a prompt of lo..hi tokens and a first generated token."""
    return {"name": name, "op": "step", "vocab": vocab, "width": width, "rows": rows, "dtype": dtype, "automaton": automaton,
            "size": size, "lo": lo, "hi": hi, "ids": 64}


def listed():
    return [
        # interactive generation with a byte-level model: one row, where latency is all
        _logits("logits_one_row", 1, 512, "float32", penalties="all", seen=0.02, keep=0.02),
        # a serving batch over 6-mers (rows whose length is no multiple of 16 bytes), every request with its own penalties
        _logits("logits_serving", 64, 4106, "bfloat16", seen=0.2),
        # a large sampling batch over BPE tokens, repetition penalty only, straight from the last position of a prefill
        _logits("logits_repetition", 333, 32000, "float16", penalties="repetition", bias="none", keep=0, last=True),
        # rollouts: thousands of samples a step, masked by a pattern, results in 32 bits for the sampler
        _logits("logits_rollouts", 2048, 32000, "bfloat16", out="float32", keep=0.25),
        # fine-tuning through the constrained distribution, a small batch in 32 bits, a learned bias
        _grad("grad_small", 32, 4096, "float32", seen=0.3),
        # the same with thousands of positions and a large vocabulary
        _grad("grad_large", 4096, 32000, "bfloat16"),
        # prompts of a serving batch: 6-mer windows of different lengths, padded, only what was seen
        _history("history_windows", "kmer", 4106, 256, "left", 100, 1000, 64, False),
        # chromosome windows a byte-level model has generated so far: few rows of a million ids, ten of them in use
        _history("history_chromosome", "byte", 512, 8, "right", 524288, 1048576, 32, True),
        # a packed batch of generated reads, flat ids and offsets, BPE
        _history("history_reads", "bpe", 32000, 1000, "ragged", 25, 1700, 64, True),
        # restriction sites that may not occur, 6-mer tokens, a serving batch
        _mask("mask_sites_kmer", "kmer", 4106, 64, "avoid", 40),
        # a designed element with degenerate positions, BPE tokens, a large sampling batch, rows at every position
        _mask("mask_pattern_bpe", "bpe", 32000, 1024, "pattern", 2000),
        # everything a generation loop does between two forward passes, the first time after a prompt
        _step("step_serving", "bpe", 32000, 48, "bfloat16", "avoid", 60, 20, 700),
    ]


def draw(rng):
    """One more case of these ranges: sizes spread over their logarithm, odd ones among them."""
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    def vocabulary():
        kind = rng.choice(["char", "byte", "kmer", "bpe", "bpe"])
        return kind, {"char": 10, "byte": 512, "kmer": 10 + 4 ** rng.randint(1, 6), "bpe": log(100, 32000)}[kind]

    op = rng.choice(["logits", "logits", "grad", "history", "mask", "step"])
    if op in ("logits", "grad"):
        width = rng.choice([10, 512, 4106, log(5, 32000), log(5, 32000)])
        most = 60_000_000 if op == "logits" else 130_000_000
        rows = log(1, max(2, min(4096, most // width)))
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        seen, keep = rng.choice([0.01, 0.1, 0.6]), rng.choice([0, 0.03, 0.5, 0.97])
        bias = rng.choice(["shared", "row"])
        if op == "grad":
            return _grad("", rows, width, dtype, bias=bias, seen=seen, keep=keep)
        return _logits("", rows, width, dtype, out=rng.choice(["", "float32"]), penalties=rng.choice(["row", "all", "repetition"]), seen=seen,
                       bias=rng.choice([bias, "none"]), keep=keep, last=rng.random() < 0.4)
    kind, width = vocabulary()
    if op == "history":
        hi = log(12, 1048576)
        rows = log(1, max(2, min(1024, 8_000_000 // hi, 30_000_000 // width)))
        # what was seen alone says little where a row has seen all there is
        return _history("", kind, width, rows, rng.choice(["right", "left", "ragged"]), max(1, hi // log(1, 60)), hi, rng.choice([32, 64]),
                        width < 4 * hi or rng.random() < 0.5)
    automaton = rng.choice(["avoid", "pattern"])
    size = log(1, 100) if automaton == "avoid" else log(5, 4000)
    if op == "mask":
        return _mask("", kind, width, log(max(1, 2000 // width), min(1024, 32_000_000 // width)), automaton, size)
    return _step("", kind, width, log(1, 48), rng.choice(["float32", "bfloat16", "float16"]), automaton, size, 1, log(2, 700))


# --------------------------------------------------------------------------- inputs

def _generator(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 16 + salt)
    return g


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _pack(ok):
    """Truth values [rows, width] -> words: bit v % 32 of word v // 32."""
    rows, width = ok.shape
    words = -(-width // 32)
    full = torch.zeros((rows, words * 32), dtype=torch.int64, device=ok.device)
    full[:, :width] = ok
    shift = torch.arange(32, device=ok.device)
    return (full.view(rows, words, 32) << shift).sum(-1).to(torch.int32)


def _unpack(words, width):
    v = torch.arange(width, device=words.device)
    return ((words[:, v >> 5] >> (v & 31).to(torch.int32)) & 1).bool()


def _tokens(kind, width, rng):
    """(classes [width, longest] with 5 past a token's end, lengths [width], flat bytes, offsets)."""
    if kind == "byte":
        flat = np.arange(256, dtype=np.uint8)
        lengths = np.zeros(width, dtype=np.int64)
        lengths[:256] = 1
    else:
        lengths = np.zeros(width, dtype=np.int64)
        if kind == "char":
            lengths[5:10] = 1
            codes = np.arange(5)
        elif kind == "kmer":
            k = round(math.log(width - 10, 4))
            lengths[5:10], lengths[10:] = 1, k
            grid = (np.arange(4 ** k)[:, None] >> (2 * np.arange(k - 1, -1, -1))) & 3
            codes = np.concatenate([np.arange(5), grid.reshape(-1)])
        else:
            lengths[5:9] = 1
            lengths[9:] = 2 + rng.binomial(12, 0.38, width - 9)
            codes = np.concatenate([np.arange(4), rng.integers(0, 4, int(lengths[9:].sum()))])
        flat = LETTERS[codes]
    offsets = np.zeros(width + 1, dtype=np.int64)
    np.cumsum(lengths, out=offsets[1:])
    table = _byte_classes()
    longest = int(lengths.max())
    at = np.minimum(offsets[:-1, None] + np.arange(longest), flat.size - 1)
    classes = np.where(np.arange(longest) < lengths[:, None], table[flat[at]], 5)
    return classes, lengths, flat, offsets


def _byte_classes():
    table = np.full(256, 4, dtype=np.uint8)
    table[LETTERS] = np.arange(5)
    return table


def _automaton(kind, size, rng):
    """(next state [states, 5], -1 for none; accepting [states])."""
    if kind == "pattern":
        nxt = np.full((size + 1, 5), -1, dtype=np.int32)
        most = rng.choice([1, 2, 4], size, p=[0.6, 0.2, 0.2])
        order = np.argsort(rng.random((size, 4)), axis=1)
        for j in range(4):
            rows = np.flatnonzero(most > j)
            nxt[rows, order[rows, j]] = rows + 1
        nxt[size, :4] = size                                       # anything may follow the element
        accepting = np.arange(size + 1) == size
        return nxt, accepting
    to, fail, bad = [[-1] * 4], [0], [False]                       # motifs: trie, then the links of the longest suffixes
    for _ in range(size):
        s, n = 0, int(rng.integers(4, 9))
        for c in rng.integers(0, 4, n).tolist():
            if to[s][c] < 0:
                to[s][c] = len(to)
                to.append([-1] * 4)
                fail.append(0)
                bad.append(False)
            s = to[s][c]
        bad[s] = True
    queue = []
    for c in range(4):
        if to[0][c] < 0:
            to[0][c] = 0
        else:
            queue.append(to[0][c])
    for s in queue:
        bad[s] = bad[s] or bad[fail[s]]
        for c in range(4):
            t = to[s][c]
            if t < 0:
                to[s][c] = to[fail[s]][c]
            else:
                fail[t] = to[fail[s]][c]
                queue.append(t)
    nxt = np.array(to, dtype=np.int32)
    nxt[np.array(bad)[nxt]] = -1
    nxt = np.concatenate([nxt, np.zeros((len(to), 1), dtype=np.int32)], axis=1)     # an N starts again
    return nxt, np.ones(len(to), dtype=bool)


def _grammar_state(case, seed):
    rng = np.random.default_rng([seed, 7])
    classes, lengths, flat, offsets = _tokens(case["vocab"], case["width"], rng)
    nxt, accepting = _automaton(case["automaton"], case["size"], rng)
    states = rng.integers(0, len(nxt), case["rows"])
    odd = rng.random(case["rows"])
    states = np.where(odd < 0.03, DEAD, np.where(odd < 0.06, FINISHED, states)).astype(np.int32)
    n = len(nxt)                                                   # rows n: dead; column 5: past a token's end
    full = np.full((n + 1, 6), n, dtype=np.int64)
    full[:n, :5] = np.where(nxt < 0, n, nxt)
    full[:n, 5] = np.arange(n)
    s = {"next": torch.from_numpy(full).cuda(), "classes": torch.from_numpy(classes).long().cuda(),
         "has": torch.from_numpy(lengths > 0).cuda(), "accepting": torch.from_numpy(np.append(accepting, False)).cuda(),
         "states": torch.from_numpy(states).cuda(), "host": (nxt, accepting, flat, offsets)}
    if own:
        from dnatok_b200 import Automaton, Grammar
        s["grammar"] = Grammar(Automaton(nxt, accepting, byte_class=_byte_classes()), (flat, offsets), end_id=END, width=case["width"])
    return s


def _ids(case, seed, g, count):
    width = case["width"]
    if case["vocab"] == "byte":
        letters = torch.tensor(list(b"ACGTacgtN"), device="cuda")
        at = (_rand(g, count) * 8.02).long()
        return letters[at]
    u = _rand(g, count).double()
    low = min(5, width - 1)
    if case["vocab"] == "bpe":
        u = u ** 3                                                 # few tokens make up most of a text
    return low + (u * (width - low)).long()


def _rows_state(case, seed):
    rng = np.random.default_rng([seed, 9])
    rows, lo, hi = case["rows"], case["lo"], case["hi"]
    lengths = np.exp(rng.uniform(math.log(lo), math.log(hi + 0.99), rows)).astype(np.int64).clip(lo, hi)
    g = _generator(seed, 2)
    kind = torch.int64 if case["ids"] == 64 else torch.int32
    layout = case.get("layout", "right")
    if layout == "ragged":
        offsets = np.zeros(rows + 1, dtype=np.int64)
        np.cumsum(lengths, out=offsets[1:])
        return {"ids": _ids(case, seed, g, int(offsets[-1])).to(kind), "offsets": torch.from_numpy(offsets).cuda()}
    ids = _ids(case, seed, g, rows * hi).view(rows, hi)
    n = torch.from_numpy(lengths).to(torch.int32).cuda()
    at = torch.arange(hi, device="cuda")
    inside = at >= hi - n[:, None] if layout == "left" else at < n[:, None]
    return {"ids": torch.where(inside, ids, 0).to(kind), "lengths": n}


def _logits_state(case, seed):
    g = _generator(seed, 3)
    rows, width, dtype = case["rows"], case["width"], TYPES[case["dtype"]]
    x = torch.randn((rows, 2 if case.get("last") else 1, width), generator=g, device="cuda").mul_(4).to(dtype)
    s = {"logits": x[:, -1]}
    per_row = case.get("penalties", "row") == "row"
    s["repetition"] = 1 + _rand(g, rows) / 2 if per_row else 1.25
    s["frequency"] = _rand(g, rows) if per_row else 0.5
    s["presence"] = _rand(g, rows) if per_row else 0.25
    if case.get("penalties") == "repetition":
        s["frequency"] = s["presence"] = 0.0
    return s


def prepare(case, seed):
    op, rows, width = case["op"], case["rows"], case["width"]
    if op == "history":
        return {"case": case, **_rows_state(case, seed)}
    if op == "mask":
        return {"case": case, **_grammar_state(case, seed)}
    if op == "step":
        s = {"case": case, **_grammar_state(case, seed), **_rows_state(case, seed), **_logits_state(case, seed)}
        # the token a sampler took: one that the mask before it allowed, where it allowed any
        ok = _plain_allowed(s, s["states"])
        s["tokens"] = (ok * (1 + _rand(_generator(seed, 5), rows, width))).argmax(1)
        return s
    s = {"case": case, **_logits_state(case, seed)}
    g = _generator(seed, 4)
    seen = _rand(g, rows, width) < case["seen"]
    s["seen"] = _pack(seen)
    # half of what a row has seen it generated itself, mostly once or twice
    s["counts"] = torch.where(seen & (_rand(g, rows, width) < 0.5), (1 - 2 * torch.log(1 - _rand(g, rows, width))).to(torch.int32), 0).to(torch.int32)
    if case["bias"] != "none":
        s["bias"] = torch.randn((width,) if case["bias"] == "shared" else (rows, width), generator=g, device="cuda")
    if case["keep"]:
        s["allowed"] = _pack(_rand(g, rows, width) < case["keep"])
    if op == "grad":
        s["logits"].requires_grad_()
        s["bias"].requires_grad_()
        s["gradient"] = torch.randn((rows, width), generator=g, device="cuda").to(TYPES[case["dtype"]])
    if own:
        from dnatok_b200 import TokenHistory
        s["history"] = TokenHistory(rows, width)
        s["history"].seen.copy_(s["seen"])
        s["history"].counts.copy_(s["counts"])
    return s


# --------------------------------------------------------------------------- the framework's calls

def _run_own(s):
    case = s["case"]
    from dnatok_b200 import TokenHistory, process_logits
    if case["op"] == "history":
        h = TokenHistory(case["rows"], case["width"], counts=case["generated"])
        h.add(s["ids"], s.get("lengths"), offsets=s.get("offsets"), pad_left=case["layout"] == "left", generated=case["generated"])
        return {"seen": h.seen, "counts": h.counts} if case["generated"] else {"seen": h.seen}
    if case["op"] == "mask":
        return {"allowed": s["grammar"].allowed(s["states"])}
    kw = {"repetition": s["repetition"], "frequency": s["frequency"], "presence": s["presence"]}
    if case["op"] == "step":
        h = TokenHistory(case["rows"], case["width"])
        h.add(s["ids"], s["lengths"])
        h.append(s["tokens"])
        states, allowed = s["grammar"].step(s["states"], s["tokens"])
        y = process_logits(s["logits"], history=h, allowed=allowed, **kw)
        return {"logits": y, "states": states, "allowed": allowed, "seen": h.seen, "counts": h.counts}
    y = process_logits(s["logits"], history=s["history"], bias=s.get("bias"), allowed=s.get("allowed"), out_dtype=TYPES[case["out"]], **kw)
    if case["op"] == "logits":
        return {"logits": y}
    dx, db = torch.autograd.grad(y, (s["logits"], s["bias"]), s["gradient"])
    return {"logits": y, "dlogits": dx, "dbias": db}


# --------------------------------------------------------------------------- the plain forms

def _column(v):
    return v[:, None] if isinstance(v, torch.Tensor) else v


def _plain_logits(x, seen, counts, s, bias, ok):
    x = x.float()
    r = _column(s["repetition"])
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    if s["case"].get("penalties") != "repetition":
        x = torch.where(counts > 0, x - _column(s["frequency"]) * counts - _column(s["presence"]), x)
    if bias is not None:
        x = x + bias
    return x if ok is None else torch.where(ok, x, -math.inf)


def _plain_gradients(s, seen, ok):
    g, x, r = s["gradient"].float(), s["logits"].detach().float(), _column(s["repetition"])
    if ok is not None:
        g = torch.where(ok, g, 0.0)
    dx = torch.where(seen, torch.where(x > 0, g / r, g * r), g)
    return dx.to(s["logits"].dtype), g.sum(0) if s["case"]["bias"] == "shared" else g


def _plain_counts(s, rows, width):
    ids = s["ids"]
    if "offsets" in s:
        at = torch.arange(ids.shape[0], device=ids.device)
        key = (torch.searchsorted(s["offsets"], at, right=True) - 1) * width + ids
    else:
        at = torch.arange(ids.shape[1], device=ids.device)
        n = s["lengths"][:, None]
        inside = at >= ids.shape[1] - n if s["case"].get("layout") == "left" else at < n
        key = (torch.arange(rows, device=ids.device)[:, None] * width + ids)[inside]
    return torch.zeros(rows * width, dtype=torch.int32, device=ids.device).scatter_add_(0, key, torch.ones_like(key, dtype=torch.int32)).view(rows, width)


def _plain_allowed(s, states):
    nxt, dead = s["next"], s["next"].shape[0] - 1
    first = torch.where(states >= 0, states, dead).long()
    at = first[:, None].expand(-1, s["classes"].shape[0])
    for j in range(s["classes"].shape[1]):                         # a token's bases one after the other
        at = nxt[at, s["classes"][:, j]]
    ok = (at != dead) & s["has"]
    ok[:, END] = s["accepting"][first] | (states == FINISHED)
    return ok


def _plain_advance(s, states, tokens):
    nxt, dead = s["next"], s["next"].shape[0] - 1
    first = torch.where(states >= 0, states, dead).long()
    at = first
    for j in range(s["classes"].shape[1]):
        at = nxt[at, s["classes"][tokens, j]]
    at = torch.where(s["has"][tokens] & (at != dead), at, DEAD)
    ends = s["accepting"][first] | (states == FINISHED)
    return torch.where(tokens == END, torch.where(ends, FINISHED, DEAD), at).to(torch.int32)


def _run_plain(s):
    case = s["case"]
    rows, width = case["rows"], case["width"]
    if case["op"] == "history":
        counts = _plain_counts(s, rows, width)
        seen = _pack(counts > 0)
        return {"seen": seen, "counts": counts} if case["generated"] else {"seen": seen}
    if case["op"] == "mask":
        return {"allowed": _pack(_plain_allowed(s, s["states"]))}
    if case["op"] == "step":
        counts = torch.zeros((rows, width), dtype=torch.int32, device="cuda")
        counts.scatter_add_(1, s["tokens"][:, None], torch.ones((rows, 1), dtype=torch.int32, device="cuda"))
        seen = (_plain_counts(s, rows, width) > 0) | (counts > 0)
        states = _plain_advance(s, s["states"], s["tokens"])
        ok = _plain_allowed(s, states)
        y = _plain_logits(s["logits"], seen, counts, s, None, ok).to(s["logits"].dtype)
        return {"logits": y, "states": states, "allowed": _pack(ok), "seen": _pack(seen), "counts": counts}
    seen = _unpack(s["seen"], width)
    ok = _unpack(s["allowed"], width) if "allowed" in s else None
    bias = s["bias"].detach() if "bias" in s else None
    y = _plain_logits(s["logits"].detach(), seen, s["counts"], s, bias, ok).to(TYPES[case["out"]])
    if case["op"] == "logits":
        return {"logits": y}
    dx, db = _plain_gradients(s, seen, ok)
    return {"logits": y, "dlogits": dx, "dbias": db}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------- floors and 64 bits

def work(case):
    rows, width = case["rows"], case["width"]
    cells, words = rows * width, rows * (-(-width // 32)) * 4
    if case["op"] == "history":
        mean = (case["hi"] - case["lo"]) / math.log(case["hi"] / case["lo"]) if case["hi"] > case["lo"] else case["hi"]
        ids = rows * mean
        return {"bytes": ids * case["ids"] // 8 + words + (4 * cells if case["generated"] else 0), "flops": 0}
    if case["op"] == "mask":
        # the tokens' bases and the automaton once, a word of mask for 32 tokens
        bases = {"char": 5, "byte": 256, "kmer": 6 * width}.get(case["vocab"], 6.5 * width)
        states = case["size"] + 1 if case["automaton"] == "pattern" else 4.5 * case["size"]
        return {"bytes": words + bases + 10 * states + 4 * rows, "flops": 0}
    if case["op"] == "step":
        prompt = rows * 8 * (case["hi"] - case["lo"]) / math.log(max(case["hi"] / case["lo"], 1.01))
        return {"bytes": 2 * cells * SIZE[case["dtype"]] + 2 * words + 4 * cells + prompt + 20 * rows, "flops": 0}
    es, counted = SIZE[case["dtype"]], case["penalties"] != "repetition"
    keep = case["keep"] or 1                                       # a masked logit need not be read
    b = words * (1 + bool(case["keep"])) + cells * (keep * es + SIZE[case["out"]] + (4 * case["seen"] * keep if counted else 0))
    b += {"none": 0, "shared": 4 * width, "row": 4 * cells * keep}[case["bias"]]
    flops = cells * keep * (1 + 4 * case["seen"])
    if case["op"] == "grad":
        # the gradient at the allowed places, the signs of what was seen, both results
        b += cells * (keep * es + keep * case["seen"] * es + es) + words * 2 + (4 * width if case["bias"] == "shared" else 4 * cells)
        flops *= 2
    return {"bytes": b, "flops": flops}


def _bits(words, width):
    return np.unpackbits(words.cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :width].astype(bool)


def _exact_logits(x, seen, counts, r, f, p, bias, ok, counted):
    """float64 on the GPU: a factor and an offset for every place, then one product and one sum."""
    x = x.detach().to(torch.float64)
    wide = lambda v: v.to(torch.float64).reshape(-1, 1) if isinstance(v, torch.Tensor) else torch.tensor(v, dtype=torch.float64, device="cuda")  # noqa: E731
    r, f, p = wide(r), wide(f), wide(p)
    # (a product with a rounded 1 / r in 64 bits is good to 2^-52)
    y = x * (1 + seen.to(torch.float64) * (torch.where(x > 0, 1 / r, r) - 1))
    if counted:
        y -= counts * f + counts.clamp(max=1) * p
    if bias is not None:
        y += bias.detach()
    if ok is not None:
        y.masked_fill_(~ok, -math.inf)
    return y


def exact(case, seed):
    if case["op"] in ("history", "mask"):
        return None                                                # whole numbers only
    s = prepare(case, seed)
    rows, width = case["rows"], case["width"]
    counted = case.get("penalties") != "repetition"
    if case["op"] == "step":
        ids, n, tokens = s["ids"].cpu().numpy(), s["lengths"].cpu().numpy(), s["tokens"].cpu().numpy()
        seen = np.zeros((rows, width), dtype=bool)
        for i in range(rows):
            seen[i, ids[i, :n[i]]] = True
        counts = np.zeros((rows, width), dtype=np.int64)
        counts[np.arange(rows), tokens] = 1
        seen |= counts > 0
        nxt, accepting, flat, offsets = s["host"]
        table = _byte_classes()
        ok = np.zeros((rows, width), dtype=bool)
        for i, state in enumerate(s["states"].cpu().numpy().tolist()):
            token = int(tokens[i])
            ended = state == FINISHED or (state >= 0 and bool(accepting[state]))
            if token == END:
                state = FINISHED if ended else DEAD
            elif state >= 0 and offsets[token] < offsets[token + 1]:
                for c in flat[offsets[token]:offsets[token + 1]].tolist():
                    state = int(nxt[state, table[c]]) if state >= 0 else DEAD
            else:
                state = DEAD
            if state >= 0:
                at = np.full(width, state)
                left = offsets[1:] - offsets[:-1]
                for j in range(int(left.max())):
                    go = (left > j) & (at >= 0)
                    at[go] = nxt[at[go], table[flat[offsets[:-1][go] + j]]]
                ok[i] = (at >= 0) & (left > 0)
            ok[i, END] = state == FINISHED or (state >= 0 and bool(accepting[state]))
        seen, counts, ok = (torch.from_numpy(a).cuda() for a in (seen, counts, ok))
        y = _exact_logits(s["logits"], seen, counts, s["repetition"], s["frequency"], s["presence"], None, ok, True)
        return {"logits": y, "states": None, "allowed": None, "seen": None, "counts": None}
    seen = torch.from_numpy(_bits(s["seen"], width)).cuda()
    ok = torch.from_numpy(_bits(s["allowed"], width)).cuda() if "allowed" in s else None
    y = _exact_logits(s["logits"], seen, s["counts"], s["repetition"], s["frequency"], s["presence"], s.get("bias"), ok, counted)
    if case["op"] == "logits":
        return {"logits": y}
    g = s["gradient"].to(torch.float64)
    if ok is not None:
        g.masked_fill_(~ok, 0.0)
    r = s["repetition"].to(torch.float64).reshape(-1, 1).expand(rows, width)
    x = s["logits"].detach()
    up, down = seen & (x > 0), seen & ~(x > 0)
    db = g.sum(0) if case["bias"] == "shared" else g.clone()
    g[up] /= r[up]
    g[down] *= r[down]
    return {"logits": y, "dlogits": g, "dbias": db}
