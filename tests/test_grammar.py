"""Grammar masks and states against a walk along every token's bytes (whole numbers: exact)."""
import numpy as np
import pytest

import generate_reference as R
import helpers as H

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from dnatok_b200 import Automaton, Grammar  # noqa: E402
from dnatok_b200.tables import token_bytes  # noqa: E402


def random_automaton(rng, states, classes, dead=0.3):
    nxt = rng.integers(0, states, (states, classes))
    nxt[rng.random((states, classes)) < dead] = -1
    return Automaton(nxt, rng.random(states) < 0.5, byte_class=rng.integers(0, classes, 256))


def random_tokens(rng, n, longest, alphabet=b"ACGTN"):
    letters = np.frombuffer(alphabet, dtype=np.uint8)
    return [b"" if rng.random() < 0.05 else letters[rng.integers(0, len(letters), int(rng.integers(1, longest + 1)))].tobytes() for _ in range(n)]


def some_states(rng, automaton, n):
    s = rng.integers(0, automaton.n_states, n)
    odd = rng.random(n)
    s = np.where(odd < 0.1, -1, np.where(odd < 0.2, -2, s))
    if n > 6:
        s[:4] = [automaton.n_states, 2 ** 31 - 1, -3, -2 ** 31]         # no states
    return s.astype(np.int32)


def check(automaton, tokens, end_id, states, chosen=None, width=None):
    g = Grammar(automaton, tokens, end_id=end_id, width=width)
    ds = torch.from_numpy(states).cuda()
    mask = g.allowed(ds)
    assert np.array_equal(mask.cpu().numpy(), R.pack(R.allowed(automaton, tokens, end_id, states, width)))
    if chosen is not None:
        for dtype in (torch.int32, torch.int64):
            dc = torch.from_numpy(chosen).to(dtype).cuda()
            want = R.advance(automaton, tokens, end_id, states, chosen, width)
            new = g.advance(ds, dc)
            assert np.array_equal(new.cpu().numpy(), want)
            new, mask = g.step(ds, dc)
            assert np.array_equal(new.cpu().numpy(), want)
            assert np.array_equal(mask.cpu().numpy(), R.pack(R.allowed(automaton, tokens, end_id, want, width)))
        assert np.array_equal(ds.cpu().numpy(), states)
        moved = ds.clone()
        assert g.advance(moved, dc, out=moved) is moved and np.array_equal(moved.cpu().numpy(), want)
    g.close()


@pytest.mark.parametrize("states,classes,longest", [(1, 1, 3), (2, 5, 1), (9, 5, 14), (40, 5, 15), (40, 6, 16), (300, 16, 17), (300, 17, 20), (1000, 256, 9),
                                                    (70, 4, 100), (9000, 5, 14), (5000, 9, 8), (40000, 5, 14)])
@pytest.mark.parametrize("width", [1, 31, 32, 33, 300, 1030])
def test_random_automata(states, classes, longest, width):
    rng = np.random.default_rng([states, classes, longest, width])
    automaton = random_automaton(rng, states, classes, dead=0.02 if longest > 6 else 0.3)
    tokens = random_tokens(rng, width, longest, bytes(range(256)) if classes > 16 else b"ACGTN")
    for n in (1, 23):
        chosen = rng.integers(-2, width + 2, n)
        if n > 5:
            chosen[:2] = [2 ** 31 - 1, -2 ** 31]
        check(automaton, tokens, None if width < 5 else 3, some_states(rng, automaton, n), chosen)
    check(automaton, tokens, 0, some_states(rng, automaton, 5), width=width + 45)


@pytest.mark.parametrize("n", [1, 2, 7, 64, 65, 700])
def test_every_number_of_rows(n):
    rng = np.random.default_rng(n)
    automaton = Automaton.avoiding(["GAATTC", "GANTC", "AAAAAA"])
    tokens = [None] * 5 + [b"A", b"C", b"G", b"T", b"N"] + random_tokens(rng, 500, 14, b"ACGT")
    tokens = [t or b"" for t in tokens]
    check(automaton, tokens, 3, some_states(rng, automaton, n), rng.integers(0, len(tokens), n))


@pytest.mark.parametrize("name", H.TOKENIZERS)
def test_the_tokenizers_vocabularies(name):
    from dnatok_b200 import B200Tokenizer
    tok = B200Tokenizer(H.spec(name))
    text = token_bytes(tok.spec)
    rng = np.random.default_rng(3)
    for automaton in (Automaton.avoiding(["GAATTC", "CCWGG"], reverse_complement=True), Automaton.from_pattern("ATG(NNN){0,40}TAA(R|Y){0,3}")):
        g = tok.grammar(automaton)
        states = some_states(rng, automaton, 12)
        end = tok.sep_token_id
        assert g.end_id == end and g.width == tok.vocab_size
        mask = g.allowed(torch.from_numpy(states).cuda())
        assert np.array_equal(mask.cpu().numpy(), R.pack(R.allowed(automaton, text, end, states)))
    # a width beyond the vocabulary: the further columns are never allowed
    g = tok.grammar(automaton, width=tok.vocab_size + 70)
    mask = R.unpack(g.allowed(torch.from_numpy(states).cuda()).cpu().numpy(), tok.vocab_size + 70)
    assert not mask[:, tok.vocab_size:].any()
    assert np.array_equal(mask[:, :tok.vocab_size], R.allowed(automaton, text, end, states))
    with pytest.raises(ValueError):
        tok.grammar(automaton, width=tok.vocab_size - 1)


@pytest.mark.parametrize("n", [1, 60, 300, 700])
@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("vocabulary", ["kmer", "words"])
def test_vocabularies_and_batches(vocabulary, large, n):
    """Every way of dividing a call: a row over several blocks or one, small and large tables, tokens whose ids follow one
    another in the order of their text (at any place of a word) and others."""
    import itertools
    rng = np.random.default_rng([n, large])
    tokens = [b""] * 7 + [bytes(t) for t in itertools.product(b"ACGT", repeat=6)] if vocabulary == "kmer" else random_tokens(rng, 9000, 12, b"ACGT")
    if large:
        nxt = np.full((3001, 5), -1)
        for c in range(4):
            keep = rng.random(3000) < 0.6
            nxt[:3000][keep, c] = np.arange(1, 3001)[keep]
        nxt[3000, :4] = 3000                                       # after the pattern, anything
        automaton = Automaton(nxt, np.arange(3001) == 3000)
    else:
        automaton = Automaton.avoiding(["GAATTC", "TTT", "CCWGG", "ACGT"])
    states = some_states(rng, automaton, n)
    states[-1] = automaton.n_states - 1
    check(automaton, tokens, 3, states, rng.integers(0, len(tokens), n))


def test_a_grammar_is_closed_while_a_graph_is_captured():
    a = Automaton.avoiding(["ACG"])
    tokens = [b"A", b"AC", b"ACG", b"T"]
    keep, gone = Grammar(a, tokens), Grammar(a, tokens)
    states = torch.zeros(3, dtype=torch.int32, device="cuda")
    want = keep.allowed(states)
    gone.allowed(states)
    torch.cuda.synchronize()
    graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(want)
    with torch.cuda.graph(graph):
        keep.allowed(states, out=out)
        gone.close()
    graph.replay()
    assert torch.equal(out, want)
    fresh = Grammar(a, tokens)
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        keep.allowed(states, out=out)
        with pytest.raises(RuntimeError, match="outside of stream capture"):
            fresh.allowed(states, out=out)
    out.zero_()
    other.replay()
    assert torch.equal(out, want)


def test_long_tokens_and_a_long_pattern():
    """Tokens of hundreds of bases among short ones; a pattern of thousands of positions."""
    rng = np.random.default_rng(6)
    bases = np.frombuffer(b"ACGT", dtype=np.uint8)[rng.integers(0, 4, 12000)].tobytes()
    nxt = np.full((12001, 5), -1)
    nxt[np.arange(12000), [b"ACGT".index(c) for c in bases]] = np.arange(1, 12001)
    automaton = Automaton(nxt, np.arange(12001) == 12000)
    starts = rng.integers(0, 11000, 40)
    tokens = random_tokens(rng, 200, 3, b"ACGT")
    for k, s in enumerate(starts.tolist()):
        tokens[k * 5] = bases[s:s + [1, 14, 15, 16, 30, 255, 256, 700][k % 8]]
    check(automaton, tokens, 7, np.concatenate([starts, [0, 12000, -2, -1]]).astype(np.int32), np.concatenate([np.arange(40) * 5, [7, 7, 7, 7]]))


def test_finished_and_dead_rows():
    a = Automaton.from_pattern("AC")
    g = Grammar(a, [b"", b"A", b"C", b"AC", b"ACA"], end_id=0)
    states = g.start(1)
    assert states.tolist() == [a.start]
    states, allowed = g.step(states, torch.tensor([3], device="cuda"))
    assert a.accepting[states.item()] and allowed.tolist() == [[1]]        # only the end may follow
    done, allowed = g.step(states, torch.tensor([0], device="cuda"))
    assert done.tolist() == [-2] and allowed.tolist() == [[1]]
    assert g.advance(done, torch.tensor([0], device="cuda")).tolist() == [-2]
    assert g.advance(done, torch.tensor([-1], device="cuda")).tolist() == [-2]
    dead, allowed = g.step(done, torch.tensor([1], device="cuda"))
    assert dead.tolist() == [-1] and allowed.tolist() == [[0]]
    assert g.advance(dead, torch.tensor([0], device="cuda")).tolist() == [-1]
    assert g.advance(g.start(1), torch.tensor([0], device="cuda")).tolist() == [-1]    # the end where the row may not end
    none = Grammar(a, [b"", b"A"])
    assert none.allowed(torch.tensor([-2, 2, -1], dtype=torch.int32, device="cuda")).tolist() == [[0]] * 3


def test_streams_graphs_and_outputs():
    rng = np.random.default_rng(8)
    automaton = Automaton.avoiding(["ACG", "TTT"])
    tokens = random_tokens(rng, 400, 9, b"ACGT")
    g = Grammar(automaton, tokens, end_id=3)
    graph = torch.cuda.CUDAGraph()
    states = torch.zeros(9, dtype=torch.int32, device="cuda")
    chosen = torch.full((9,), -1, dtype=torch.int64, device="cuda")
    new, mask = torch.empty_like(states), torch.empty((9, 13), dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = g.allowed(states)
    torch.cuda.current_stream().wait_stream(side)
    s = np.zeros(9, np.int32)
    assert np.array_equal(first.cpu().numpy(), R.pack(R.allowed(automaton, tokens, 3, s)))
    with torch.cuda.graph(graph):
        assert g.step(states, chosen, out=new, out_allowed=mask)[1] is mask
        states.copy_(new)
    other = Grammar(automaton, tokens)
    for _ in range(5):
        c = rng.integers(0, 400, 9)
        chosen.copy_(torch.from_numpy(c))
        graph.replay()
        s = R.advance(automaton, tokens, 3, s, c)
        assert np.array_equal(states.cpu().numpy(), s)
        assert np.array_equal(mask.cpu().numpy(), R.pack(R.allowed(automaton, tokens, 3, s)))
    out = torch.empty((9, 13), dtype=torch.int32, device="cuda")
    assert g.allowed(states, out=out) is out and torch.equal(out, mask)
    other.close()


def test_refusals():
    g = Grammar(Automaton.from_pattern("A*"), [b"A"] * 40)
    s, t = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (s.long(), s.cpu(), s[:, None], torch.zeros(6, dtype=torch.int32, device="cuda")[::2], 3):
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            g.allowed(bad)
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            g.advance(bad, t)
    for bad in (t[:2], t.short(), t.cpu(), t[:, None], 3):
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            g.step(s, bad)
    m = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    for bad in (m[:2], m.long(), m[:, :1], m.cpu(), m.t()):
        with pytest.raises((ValueError, RuntimeError)):
            g.allowed(s, out=bad)
    with pytest.raises((ValueError, RuntimeError)):
        g.step(s, t, out=s)
    for bad in (s[:2], s.long(), s.cpu()):
        with pytest.raises((ValueError, RuntimeError)):
            g.advance(s, t, out=bad)
    assert g.allowed(s[:0]).shape == (0, 2)
    assert g.step(s[:0], t[:0])[1].shape == (0, 2)
