"""Outputs of a grammar's calls that overlap what they read: refused (no GPU; the checks of the C ABI)."""

import numpy as np
import pytest

from dnatok_b200 import Automaton, Grammar, _cabi

from test_logits_overlap import no_gpu, refused  # noqa: F401

AT = 1 << 20


@pytest.fixture(scope="module")
def grammar():
    g = Grammar(Automaton.avoiding(["ACG"]), [b"A", b"C"] * 20)
    yield g
    g.close()


def step(g, states=AT, tokens=2 * AT, bits=32, n=10, out=3 * AT, allowed=4 * AT):
    return refused(_cabi.lib().dnatok_grammar_step(g.ptr, states, tokens, bits, n, out, allowed, None))


def test_states_and_masks_over_what_is_read(no_gpu, grammar):  # noqa: F811
    assert not step(grammar)
    # every block of a row reads its state and its token, while the first writes the new state
    for bits in (32, 64):
        for d in (-36, -4, 0, 4, 10 * bits // 8 - 4):
            assert step(grammar, tokens=AT, bits=bits, states=2 * AT, out=AT + d) == (d + 40 > 0)
        assert not step(grammar, tokens=AT, bits=bits, states=2 * AT, out=AT - 40) and not step(grammar, tokens=AT, bits=bits, states=2 * AT, out=AT + 10 * bits // 8)
    for d in (-36, 4, 36):
        assert step(grammar, out=AT + d)
    assert not step(grammar, out=AT - 40) and not step(grammar, out=AT + 40)
    for name, size in (("states", 40), ("tokens", 40), ("out", 40)):
        for d in (-76, -4, 0, 4, size - 4):
            assert step(grammar, **{name: 8 * AT}, allowed=8 * AT + d)
        assert not step(grammar, **{name: 8 * AT}, allowed=8 * AT - 80) and not step(grammar, **{name: 8 * AT}, allowed=8 * AT + size)
    call = _cabi.lib().dnatok_grammar_allowed
    for d, want in ((-80, False), (-76, True), (0, True), (36, True), (40, False)):
        assert refused(call(grammar.ptr, AT, 10, AT + d, None)) == want


def test_states_alone(no_gpu, grammar):  # noqa: F811
    """Without a mask a thread takes a row: the new states may be the old ones or, as wide, the tokens; shifted ones may not."""
    for name in ("states", "tokens"):
        assert not step(grammar, **{name: AT, "out": AT, "allowed": None, "states" if name == "tokens" else "tokens": 2 * AT})
        for d in (-36, -4, 4, 36):
            assert step(grammar, **{name: AT, "out": AT + d, "allowed": None, "states" if name == "tokens" else "tokens": 2 * AT})
    for d in (-36, 0, 4, 76):
        assert step(grammar, tokens=8 * AT, bits=64, out=8 * AT + d, allowed=None)
    assert not step(grammar, tokens=8 * AT, bits=64, out=8 * AT + 80, allowed=None)


@pytest.mark.gpu
def test_views_of_one_array():
    import torch
    g = Grammar(Automaton.avoiding(["ACG"]), [b"A", b"C", b"G", b"AC"] * 10)
    buffer = torch.zeros(61, dtype=torch.int32, device="cuda")
    states, tokens = buffer[:20], buffer[20:40]
    tokens.copy_(torch.arange(20))
    want, mask = g.step(states, tokens)
    for bad in (tokens, buffer[19:39], buffer[1:21], buffer[39:59]):
        with pytest.raises(RuntimeError, match="overlap"):
            g.step(states, tokens, out=bad)
    for bad in (buffer[19:39], buffer[1:21], buffer[39:59]):
        with pytest.raises(RuntimeError, match="overlap"):
            g.advance(states, tokens, out=bad)
    for bad in (buffer[:40].view(20, 2), buffer[21:].view(20, 2)):
        with pytest.raises(RuntimeError, match="overlap"):
            g.allowed(states, out=bad) if bad.data_ptr() == states.data_ptr() else g.step(states, tokens, out_allowed=bad)
    assert not states.any() and np.array_equal(tokens.cpu().numpy(), np.arange(20))
    new, m = g.step(states, tokens, out=buffer[40:60])
    assert torch.equal(new, want) and torch.equal(m, mask)
    assert torch.equal(g.advance(states, tokens, out=states), want)
