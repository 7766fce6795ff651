"""Tables that callers give: whole numbers that would not fit are refused instead of wrapped (no GPU)."""
import numpy as np
import pytest

from dnatok_b200 import Automaton, Grammar

NEXT = np.array([[0, 1, -1, 0, 0], [1, -1, 0, 1, 1]])


def test_tables_keep_their_values():
    for dtype in (np.int8, np.int16, np.int32, np.int64, np.float32, np.float64, object):
        a = Automaton(NEXT.astype(dtype), np.array([0, 1]).astype(dtype))
        assert a.next_state.dtype == np.int32 and np.array_equal(a.next_state, NEXT) and a.accepting.tolist() == [0, 1]
    assert np.array_equal(Automaton(NEXT.tolist(), [True, False]).next_state, NEXT)
    # accepting is a truth value
    for yes in (1, 2, 256, -1, 2 ** 40, 0.5):
        assert Automaton(NEXT, np.array([0, yes])).accepting.tolist() == [0, 1]


@pytest.mark.parametrize("wrong", [2 ** 32, 2 ** 32 + 1, -2 ** 32, 2 ** 31, 0.5, np.nan, np.inf])
def test_next_states_that_are_none(wrong):
    bad = NEXT.astype(np.float64 if isinstance(wrong, float) else np.int64)
    bad[0, 0] = wrong
    with pytest.raises(ValueError, match="next_state"):
        Automaton(bad, [1, 1])


@pytest.mark.parametrize("wrong", [256, 257, -256, -1, 0.5])
def test_classes_that_are_none(wrong):
    bad = np.zeros(256, dtype=np.float64 if isinstance(wrong, float) else np.int64)
    bad[65] = wrong
    with pytest.raises(ValueError, match="byte_class"):
        Automaton(NEXT, [1, 1], byte_class=bad)


def test_token_bytes_that_are_none():
    a = Automaton(NEXT, [1, 1])
    for flat, offsets, what in [(np.array([65, 256 + 65]), [0, 1, 2], "bytes"), (np.array([65, -1]), [0, 1, 2], "bytes"), (np.array([65, 66.5]), [0, 1, 2], "bytes"),
                                (np.array([65, 66], np.uint8), [0, 1.5, 2], "offsets")]:
        with pytest.raises(ValueError, match=what):
            Grammar(a, (flat, np.array(offsets)))
    for flat in (np.array([65, 66]), np.array([65, 66], np.int8), np.array([65.0, 66.0])):
        Grammar(a, (flat, np.array([0, 1, 2], np.int32))).close()


def test_ids_in_place_of_bytes():
    """A number is no text: bytes(5) would be five zeros."""
    a = Automaton(NEXT, [1, 1])
    for tokens in ([b"A", 5], [0, 1, 2], [np.int64(3)], [True]):
        with pytest.raises(TypeError, match="token"):
            Grammar(a, tokens)
    g = Grammar(a, [b"A", bytearray(b"CG"), None, b"", memoryview(b"T"), [65, 67]])
    assert g.width == 6
    g.close()
