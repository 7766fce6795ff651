"""Which text the ids of less usual tokenizers stand for in a grammar."""
import numpy as np
import pytest

from dnatok_b200 import Automaton
from dnatok_b200.tables import bpe_spec_from_json, following_bytes, spec_from_tokenizer, token_bytes


class Letters:
    """One id per character, an optional other one at the start of a text, pad and unknown ids only where given."""

    def __init__(self, words, other, first=None, pad=None, unk=None, sep=None):
        self.words, self.other, self.first, self.sep = words, other, first or {}, sep
        self.pad_token_id, self.unk_token_id, self.vocab_size = pad, unk, 1 + max(list(words.values()) + list(self.first.values()) + [other])

    def get_vocab(self):
        return {**{("^" + w): i for w, i in self.first.items()}, **self.words}

    def __call__(self, texts, add_special_tokens=False, **kw):
        rows = [[self.words.get(c.upper(), self.other) for c in t] for t in ([texts] if isinstance(texts, str) else texts)]
        for r, t in zip(rows, texts):
            if t and t[0].upper() in self.first:
                r[0] = self.first[t[0].upper()]
            if add_special_tokens and self.sep is not None:
                r.append(self.sep)
        return {"input_ids": rows}


BASES = {"A": 0, "C": 1, "G": 2, "T": 3, "N": 4}


def test_without_pad_and_unknown_ids_every_id_has_its_text():
    """Where a tokenizer names neither, 0 takes their place in the tables; it may be a base all the same."""
    s = spec_from_tokenizer(Letters(BASES, 4))
    assert (s.specials.pad_id, s.specials.unk_id) == (0, 0)
    assert token_bytes(s)[:4] == [b"A", b"C", b"G", b"T"] and len(token_bytes(s)[4]) == 1
    # one that names them has none there
    assert token_bytes(spec_from_tokenizer(Letters(BASES, 4, pad=0)))[:4] == [b"", b"C", b"G", b"T"]
    assert token_bytes(spec_from_tokenizer(Letters(BASES, 4, unk=0)))[:4] == [b"", b"C", b"G", b"T"]
    assert token_bytes(spec_from_tokenizer(Letters(BASES, 4, pad=4, unk=4))) == [b"A", b"C", b"G", b"T", b""]


@pytest.mark.parametrize("pad", [None, 0, 9])
def test_merges_without_a_pad_id(pad):
    vocab = {"A": 0, "C": 1, "G": 2, "T": 3, "[UNK]": 4, "AC": 5, "ACG": 6}
    cfg = {"model": {"type": "BPE", "vocab": vocab, "merges": [["A", "C"], ["AC", "G"]], "unk_token": "[UNK]"}}
    text = token_bytes(bpe_spec_from_json(cfg, pad_id=pad))
    assert text[1:5] == [b"C", b"G", b"T", b""]
    assert (text[0], text[5], text[6]) == ((b"", b"", b"") if pad == 0 else (b"A", b"AC", b"ACG"))


FIRST = {"A": 10, "C": 11, "G": 12, "T": 13}


def split_tokenizer():
    """Ids 10 .. 13 at the start of a text, 5 .. 8 behind it, N (9) at both; 3 ends a row."""
    return Letters({"A": 5, "C": 6, "G": 7, "T": 8, "N": 9}, 9, first=FIRST, pad=0, unk=1, sep=3)


def test_ids_of_the_start_and_of_what_follows():
    s = spec_from_tokenizer(split_tokenizer())
    assert s.start_lut256 is not None and s.specials.sep_id == 3
    both = token_bytes(s)
    assert [both[i] for i in (5, 6, 7, 8, 10, 11, 12, 13)] == [b"A", b"C", b"G", b"T"] * 2
    follow, first = following_bytes(s), following_bytes(s, first=True)
    assert len(follow) == len(first) == len(both)
    for i in range(len(both)):
        assert follow[i] == (b"" if i in FIRST.values() else both[i]) and first[i] == (b"" if i in (5, 6, 7, 8) else both[i])
    plain = spec_from_tokenizer(Letters(BASES, 4))
    assert following_bytes(plain) == following_bytes(plain, first=True) == token_bytes(plain)


@pytest.mark.gpu
def test_rows_never_start_again():
    """A grammar's masks hold the ids that follow, those of a row's first token where asked for; states are the same."""
    import torch
    from dnatok_b200 import B200Tokenizer, process_logits
    tok = B200Tokenizer(spec_from_tokenizer(split_tokenizer()))
    automaton = Automaton.avoiding(["AA"])
    first, follow = tok.grammar(automaton, first=True), tok.grammar(automaton)
    bits = lambda words: {v for v in range(tok.vocab_size) if words.view(-1)[v // 32].item() >> (v % 32) & 1}  # noqa: E731
    states = first.start(1)
    assert bits(first.allowed(states)) == {3, 9, 10, 11, 12, 13} and bits(follow.allowed(states)) == {3, 5, 6, 7, 8, 9}
    states, allowed = follow.step(first.advance(states, torch.tensor([10], device="cuda")), torch.tensor([-1], device="cuda"))
    assert bits(allowed) == {3, 6, 7, 8, 9}                        # no A behind the A, and no start again
    n, g = 32, torch.Generator(device="cuda").manual_seed(1)
    states, rows = first.start(n), []
    allowed = first.allowed(states)
    for k in range(20):
        tokens = process_logits(torch.randn((n, tok.vocab_size), generator=g, device="cuda"), allowed=allowed).argmax(-1)
        rows.append(tokens.cpu().numpy())
        states = (first if k == 0 else follow).advance(states, tokens)
        allowed = follow.allowed(states)
    assert (states != -1).all()
    text = token_bytes(tok.spec)
    for r in np.stack(rows, 1):
        r = r[:list(r).index(3)] if 3 in r else r
        word = b"".join(text[v] for v in r).decode()
        assert "AA" not in word and r.tolist() == (split_tokenizer()([word])["input_ids"][0] if word else [])
