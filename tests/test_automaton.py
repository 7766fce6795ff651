"""Automata over bases against Python's own regular expressions, and the bytes of every token (no GPU)."""
import itertools
import random
import re

import numpy as np
import pytest

from dnatok_b200 import Automaton
from dnatok_b200.automaton import IUPAC
from dnatok_b200.tables import Specials, TokenizerSpec, token_bytes

import helpers as H

PATTERNS = ["ACGT", "ATG(NNN)*T(RA|AG)", "A*", "(AC|GT)+N?", "[RY]{2,4}C", "N{3}", "N{2,}T", "((A|C)*G)?", "A|", "", "(A*)*C",
            "S{0}W{1,2}.", "B(D|H)V{0,2}"]


def as_python(pattern):
    out = ""
    inside = False
    for i, c in enumerate(pattern):
        if c in "[]":
            inside = c == "["
            out += c
        elif c == ".":
            out += "[ACGT]"
        elif c in IUPAC:
            out += IUPAC[c] if inside else "[%s]" % IUPAC[c]
        else:
            out += c
    return re.compile("(?:%s)" % out)


@pytest.mark.parametrize("pattern", PATTERNS)
def test_patterns_accept_what_regular_expressions_match(pattern):
    a, rx = Automaton.from_pattern(pattern), as_python(pattern)
    texts = ["".join(t) for n in range(6) for t in itertools.product("ACGT", repeat=n)]
    rng = random.Random(1)
    texts += ["".join(rng.choice("ACGT") for _ in range(rng.randint(6, 15))) for _ in range(500)] + ["ATG" + "ACG" * 3 + "TAA", "AN", "N"]
    for t in texts:
        want = rx.fullmatch(t) is not None
        assert a.accepts(t) == want, t
        assert a.accepts(t.lower()) == want
    # a live state can be completed: the text so far is the beginning of a match
    for s in range(a.n_states):
        if (a.next_state == s).any():
            todo, got = [s], {s}
            while todo:
                for t in a.next_state[todo.pop()]:
                    if t >= 0 and int(t) not in got:
                        got.add(int(t))
                        todo.append(int(t))
            assert any(a.accepting[t] for t in got)


def test_case_matters_where_asked():
    assert not Automaton.from_pattern("ACG", lowercase=False).accepts("acg")
    assert Automaton.avoiding("ACG", lowercase=False).accepts("acgacg")


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("motifs", [["GAATTC"], ["A"], ["GANTC", "TTAA", "CCWGG"], ["AAAA", "CAAAAC", "AC"], ["NN"]])
def test_avoided_motifs_never_occur(motifs, both):
    a = Automaton.avoiding(motifs, reverse_complement=both)
    turn = str.maketrans("ACGTURYSWKMBDHVN", "TGCAAYRSWMKVHDBN")
    every = motifs + ([m.translate(turn)[::-1] for m in motifs] if both else [])
    bad = re.compile("|".join("".join("[%s]" % IUPAC[c] for c in m) for m in every))
    rng = random.Random(2)
    texts = ["".join(t) for n in range(7) for t in itertools.product("ACGT", repeat=n)]
    texts += ["".join(rng.choice("ACGTACGTN") for _ in range(30)) for _ in range(500)]
    for t in texts:
        assert a.accepts(t) == (bad.search(t) is None), t


def test_both_of_two():
    orf, free = Automaton.from_pattern("ATG(NNN)*TAA"), Automaton.avoiding(["GAATTC", "CCC"])
    both = orf & free
    rng = random.Random(3)
    for _ in range(3000):
        t = "ATG" + "".join(rng.choice("ACGT") for _ in range(rng.randint(0, 12))) + rng.choice(["TAA", "TAG", ""])
        assert both.accepts(t) == (orf.accepts(t) and free.accepts(t))
    odd = Automaton(np.array([[0, 1], [-1, 1]]), [1, 1], byte_class=np.arange(256) % 2, start=0)
    two = odd & orf
    for t in ("ATGTAA", "ATG", "A"):
        assert two.accepts(t) == (odd.accepts(t) and orf.accepts(t))


def test_refusals():
    for bad in ("AX", "(A", "A)", "[A", "[]", "A{2", "A{,2}", "A{3,2}", "*A", "A{x}", "A B"):
        with pytest.raises(ValueError):
            Automaton.from_pattern(bad)
    for bad in ([""], ["AXC"], ["A*"]):
        with pytest.raises(ValueError):
            Automaton.avoiding(bad)
    for args, kw in [((np.zeros((2,), int), [1, 1]), {}), ((np.zeros((2, 5), int), [1]), {}), ((np.full((2, 5), 2), [1, 1]), {}),
                     ((np.full((2, 5), -2), [1, 1]), {}), ((np.zeros((2, 4), int), [1, 1]), {}), ((np.zeros((2, 5), int), [1, 1]), {"start": 2})]:
        with pytest.raises(ValueError):
            Automaton(*args, **kw)


@pytest.mark.parametrize("name", H.TOKENIZERS)
def test_token_bytes_are_the_vocabulary(name):
    s = H.spec(name)
    text = token_bytes(s)
    words = {i: w for w, i in s.vocab.items()}
    special = {s.specials.pad_id, s.specials.unk_id, s.specials.cls_id, s.specials.sep_id}
    assert len(text) == s.vocab_size
    for i, t in enumerate(text):
        if i in special or not t:
            assert not t
        else:
            assert t.decode("latin-1") == words[i]
    assert sum(map(bool, text)) >= {"char": 5, "kmer6": 4101, "bpe4096": 4091, "byte": 100, "bpe32000": 31995}[name]


def test_token_bytes_of_shared_and_late_ids():
    lut = np.full(256, 1, np.int32)
    for i, c in enumerate("ACGT"):
        lut[ord(c)] = lut[ord(c.lower())] = 4 + i
    start = lut.copy()
    start[ord("A")] = 9
    text = token_bytes(TokenizerSpec("char", Specials(0, 1, 2, 3), 10, lut, start_lut256=start))
    assert text == [b"", b"", b"", b"", b"A", b"C", b"G", b"T", b"", b"A"]
    # merges whose operands are created by a later rank
    text = token_bytes(TokenizerSpec("bpe", Specials(0, 1, 2, 3), 12, lut, merge_a=np.array([9, 4]), merge_b=np.array([6, 5]), merge_out=np.array([10, 9])))
    assert text[9] == b"AC" and text[10] == b"ACG" and text[11] == b""
    table = np.full(25, -1, np.int32)
    for i, w in enumerate(itertools.product("ACGTN", repeat=2)):
        table[i] = 1 if "N" in w else 10 + i
    text = token_bytes(TokenizerSpec("kmer", Specials(0, 1), 40, lut, k=2, kmer_table5=table))
    assert text[10] == b"AA" and text[10 + 5 * 3 + 3] == b"TT" and text[1] == b""
