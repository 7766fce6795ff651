"""Which text the ids of less usual tokenizers stand for in a grammar."""
import numpy as np
import pytest

from dnatok_b200 import Automaton
from dnatok_b200.tables import bpe_spec_from_json, spec_from_tokenizer, token_bytes


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
