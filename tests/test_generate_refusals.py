"""What the operators around logits refuse, without a GPU: the Python checks and the C ABI's own."""
import ctypes

import numpy as np
import pytest
import torch

from dnatok_b200 import Automaton, Grammar, TokenHistory, _cabi, process_logits, process_logits_backward

INVALID = -1


def logits_struct(**kw):
    a = _cabi.Logits(logits=4096, dtype=0, n_rows=2, width=40, stride=40, repetition=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change", [dict(logits=None), dict(dtype=3), dict(dtype=-1), dict(n_rows=-1), dict(width=0), dict(width=1 << 31),
                                    dict(stride=-1), dict(logits=4098), dict(counts=4096, history_rows=2), dict(seen=4096, history_rows=3),
                                    dict(seen=4096, history_rows=2, rows=4096, rows_bits=16), dict(seen=4096, history_rows=-1, rows=4096, rows_bits=32),
                                    dict(seen=4096, history_rows=9, rows=4100, rows_bits=64), dict(bias=4096, bias_stride=39),
                                    dict(allowed=4096, allowed_stride=1), dict(allowed=4097), dict(repetition=0.0), dict(repetition=-1.0),
                                    dict(repetition=float("nan")), dict(d_presence=4097)])
def test_c_abi_refuses_bad_logits(change):
    L = _cabi.lib()
    a = logits_struct(**change)
    assert L.dnatok_process_logits(ctypes.byref(a), 8192, 0, 40, None) == INVALID
    assert L.dnatok_last_error()
    assert L.dnatok_process_logits_backward(ctypes.byref(a), 8192, 0, 40, 12288, 40, None, None, 0, None) == INVALID


def test_c_abi_refuses_bad_outputs():
    L = _cabi.lib()
    a = logits_struct()
    for out, dtype, stride in [(None, 0, 40), (8192, 1, 40), (8192, 2, 40), (8194, 0, 40), (8192, 0, 39), (4096, 0, 41)]:
        assert L.dnatok_process_logits(ctypes.byref(a), out, dtype, stride, None) == INVALID
    half = logits_struct(dtype=2)
    assert L.dnatok_process_logits(ctypes.byref(half), 4096, 0, 40, None) == INVALID         # in place as another type
    for args in [(None, 0, 40, 12288, 40, None), (8192, 1, 40, 12288, 40, None), (8192, 0, -1, 12288, 40, None), (8192, 0, 40, 12288, 39, None),
                 (8193, 0, 40, 12288, 40, None), (8192, 0, 40, 12288, 40, 6), (8192, 0, 41, 8192, 40, None), (8192, 0, 40, 4096, 40, None)]:
        assert L.dnatok_process_logits_backward(ctypes.byref(a), *args, None, 0, None) == INVALID
    assert L.dnatok_process_logits(None, 8192, 0, 40, None) == INVALID


def test_c_abi_refuses_a_bad_history():
    L = _cabi.lib()
    good = dict(seen=4096, history_rows=2, width=40, ids=8192, id_bits=64, n_rows=2, columns=5, id_stride=5)
    for change in [dict(width=0), dict(width=1 << 31), dict(n_rows=-1), dict(history_rows=-1), dict(id_bits=16), dict(history_rows=3), dict(columns=-1),
                   dict(id_stride=-1), dict(seen=None), dict(ids=None), dict(ids=8196), dict(seen=4098), dict(offsets=4096, lengths=4096, total=9),
                   dict(offsets=4096, total=-1), dict(rows=4096, rows_bits=8), dict(rows=4098, rows_bits=32), dict(offsets=4100, total=9),
                   dict(lengths=4098), dict(counts=4098)]:
        h = _cabi.History(**{**good, **change})
        assert L.dnatok_history_add(ctypes.byref(h), 1, None) == INVALID, change
    assert L.dnatok_history_add(None, 1, None) == INVALID
    for nothing in [dict(columns=0), dict(n_rows=0, history_rows=0), dict(offsets=4096, total=0)]:
        h = _cabi.History(**{**good, **nothing})
        assert L.dnatok_history_add(ctypes.byref(h), 1, None) == 0


def create(next=((0, 1), (1, -1)), accepting=(1, 0), byte_class=None, text=b"AC", offsets=(0, 1, 2), width=None, end_id=-1, n_classes=None):
    L = _cabi.lib()
    nxt = np.array(next, dtype=np.int32)
    acc = np.array(accepting, dtype=np.uint8)
    bc = np.zeros(256, np.uint8) if byte_class is None else byte_class
    off = np.array(offsets, dtype=np.int64)
    flat = np.frombuffer(text, dtype=np.uint8)
    h = ctypes.c_void_p()
    rc = L.dnatok_create_grammar(_cabi.np_ptr(nxt), nxt.shape[0], nxt.shape[1] if n_classes is None else n_classes, _cabi.np_ptr(acc), _cabi.np_ptr(bc),
                                 _cabi.np_ptr(flat) if flat.size else None, _cabi.np_ptr(off), len(off) - 1 if width is None else width, end_id, ctypes.byref(h))
    return rc, h


def test_c_abi_refuses_bad_grammars():
    L = _cabi.lib()
    rc, h = create()
    assert rc == 0
    assert L.dnatok_grammar_allowed(h, None, 3, 4096, None) == INVALID
    assert L.dnatok_grammar_allowed(h, 4096, -1, 4096, None) == INVALID
    assert L.dnatok_grammar_allowed(h, 4096, 3, None, None) == INVALID
    assert L.dnatok_grammar_allowed(h, 4098, 3, 4096, None) == INVALID
    assert L.dnatok_grammar_allowed(None, 4096, 3, 4096, None) == INVALID
    assert L.dnatok_grammar_allowed(h, None, 0, None, None) == 0
    assert L.dnatok_grammar_step(h, 4096, 8192, 16, 3, 12288, None, None) == INVALID
    assert L.dnatok_grammar_step(h, 4096, None, 32, 3, 12288, None, None) == INVALID
    assert L.dnatok_grammar_step(h, 4096, 8192, 32, 3, None, None, None) == INVALID
    assert L.dnatok_grammar_step(h, 4096, 8196, 64, 3, 12288, None, None) == INVALID
    assert L.dnatok_grammar_step(h, 4096, 8192, 32, 3, 4096, 16384, None) == INVALID      # in place with a mask
    assert L.dnatok_grammar_step(h, None, None, 32, 0, None, None, None) == 0
    L.dnatok_destroy_grammar(h)
    L.dnatok_destroy_grammar(None)
    for kw in [dict(next=((0, 2), (0, 0))), dict(next=((0, -2), (0, 0))), dict(byte_class=np.full(256, 2, np.uint8)), dict(offsets=(1, 1, 2)),
               dict(offsets=(0, 2, 1)), dict(end_id=2), dict(end_id=-2), dict(width=0), dict(n_classes=0), dict(n_classes=257), dict(text=b"")]:
        assert create(**kw)[0] == INVALID, kw


def test_python_refuses_what_is_not_on_a_gpu():
    x = torch.zeros(2, 40)
    with pytest.raises(RuntimeError, match="no CPU path"):
        process_logits(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        process_logits_backward(x, x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        TokenHistory(2, 40, device="cpu")
    with pytest.raises(ValueError):
        TokenHistory(-1, 40)
    with pytest.raises(ValueError):
        TokenHistory(1, 0)
    a = Automaton.from_pattern("ACGT")
    g = Grammar(a, [None, b"A", b"CG", b""], end_id=3, width=9)
    assert g.width == 9
    with pytest.raises(RuntimeError, match="no CPU path"):
        g.allowed(torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        g.step(torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int64))
    for kw in [dict(end_id=4), dict(end_id=-1), dict(width=3)]:
        with pytest.raises(ValueError):
            Grammar(a, [None, b"A", b"CG", b""], **kw)
    with pytest.raises(ValueError):
        Grammar(a, (np.zeros(3, np.uint8), np.array([0, 2])))
    g.close()
    g.close()
