"""The operators as a generation loop uses them together: encode, history, grammar, logits, the next token."""
import re

import numpy as np
import pytest

import generate_reference as R
import helpers as H

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from dnatok_b200 import Automaton, B200Tokenizer, process_logits  # noqa: E402
from dnatok_b200.tables import token_bytes  # noqa: E402


@pytest.mark.parametrize("name,side", [("char", "right"), ("kmer6", "left"), ("bpe4096", "right"), ("byte", "left"), ("bpe32000", "right")])
def test_generated_rows_obey_the_grammar_and_the_penalties(name, side):
    tok = B200Tokenizer(H.spec(name))
    tok.padding_side = side
    text = token_bytes(tok.spec)
    width, n, steps = tok.vocab_size + 6, 5, 12                    # the model pads its vocabulary
    rng = np.random.default_rng(4)
    prompts = ["".join(rng.choice(list("ACGT"), k)) for k in (40, 1, 333, 18, 90)]
    d_bytes, d_off, offsets = tok.to_device(prompts)
    enc = tok.encode_device(d_bytes, d_off, host_offsets=offsets, padding="longest")
    motifs = ["GAATTC", "TTT", "CCWGG"]
    automaton = Automaton.avoiding(motifs)
    grammar = tok.grammar(automaton, width=width)
    history = tok.token_history(n, width=width)
    history.add(enc["input_ids"], enc["lengths"], pad_left=side == "left")
    ids, mask = enc["input_ids"].cpu().numpy(), enc["attention_mask"].cpu().numpy()
    seen, counts = R.history(n, width, [r[m == 1] for r, m in zip(ids, mask)], False)
    states = grammar.start(n)
    allowed = grammar.allowed(states)
    host_states = states.cpu().numpy()
    rows = [b""] * n
    g = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(steps):
        model = torch.randn((n, 3, width), generator=g, device="cuda").mul_(3).bfloat16()
        y = process_logits(model[:, -1], history=history, repetition=1.5, frequency=0.25, presence=0.5, allowed=allowed)
        ok = R.allowed(automaton, text, grammar.end_id, host_states, width)
        want, bound = R.logits(R.host(model[:, -1]), seen, counts, 1.5, 0.25, 0.5, None, ok)
        R.close(y, want, bound, torch.bfloat16)
        tokens = y.float().argmax(-1)
        history.append(tokens)
        states, allowed = grammar.step(states, tokens)
        chosen = tokens.cpu().numpy()
        s, c = R.history(n, width, [[v] for v in chosen], True)
        seen, counts = seen | s, counts + c
        host_states = R.advance(automaton, text, grammar.end_id, host_states, chosen, width)
        assert np.array_equal(states.cpu().numpy(), host_states) and (host_states != -1).all()
        rows = [r + text[v] for r, v in zip(rows, chosen)]
    assert np.array_equal(R.unpack(history.seen.cpu().numpy(), width), seen) and np.array_equal(history.counts.cpu().numpy(), counts)
    for r, s in zip(rows, host_states):
        assert not re.search(b"GAATTC|TTT|CC[AT]GG", r.upper()), r
        assert s == -2 or automaton.walk(r) == s


def test_a_pattern_is_completed():
    """Rows that follow a pattern until only the end token is left."""
    tok = B200Tokenizer(H.spec("bpe4096"))
    text = token_bytes(tok.spec)
    grammar = tok.grammar(Automaton.from_pattern("ATG(NNN){3,6}(TAA|TAG|TGA)"))
    states = grammar.start(64)
    allowed = grammar.allowed(states)
    rows = [b""] * 64
    g = torch.Generator(device="cuda").manual_seed(2)
    for _ in range(40):
        y = process_logits(torch.randn((64, tok.vocab_size), generator=g, device="cuda"), allowed=allowed)
        tokens = y.argmax(-1)
        states, allowed = grammar.step(states, tokens)
        rows = [r + text[v] for r, v in zip(rows, tokens.tolist())]
        if (states == -2).all():
            break
    assert (states == -2).all()
    for r in rows:
        assert re.fullmatch(b"ATG([ACGT]{3}){3,6}(TAA|TAG|TGA)", r), r


def test_the_loop_as_one_captured_graph():
    tok = B200Tokenizer(H.spec("kmer6"))
    n, width = 6, tok.vocab_size
    grammar = tok.grammar(Automaton.avoiding(["GAATTC"]))

    def begin():
        states = grammar.start(n)
        return tok.token_history(n), states, grammar.allowed(states), torch.empty(n, dtype=torch.int32, device="cuda")

    def step(model, history, states, allowed, new):
        y = process_logits(model, history=history, repetition=1.3, frequency=0.5, allowed=allowed)
        tokens = y.argmax(-1)
        history.append(tokens)
        grammar.step(states, tokens, out=new, out_allowed=allowed)
        states.copy_(new)
        return tokens
    g = torch.Generator(device="cuda").manual_seed(3)
    inputs = [torch.randn((n, width), generator=g, device="cuda") for _ in range(6)]
    eager = begin()
    want = [step(x, *eager).clone() for x in inputs]
    again = begin()
    model = inputs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens = step(model, *again)
    got = []
    for x in inputs:
        model.copy_(x)
        graph.replay()
        got.append(tokens.clone())
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    assert torch.equal(eager[0].seen, again[0].seen) and torch.equal(eager[0].counts, again[0].counts) and torch.equal(eager[1], again[1])
