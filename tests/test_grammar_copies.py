"""Copies of a grammar share its tables, which are freed once (no GPU)."""
import copy
import ctypes

from dnatok_b200 import Automaton, Grammar, _cabi

from generate_host import library  # noqa: F401


def test_copies_are_the_grammar_itself(library):  # noqa: F811
    g = Grammar(Automaton.avoiding(["ACG"]), [b"A", b"C"])
    g.ptr = ctypes.c_void_p(4096)
    for other in (copy.copy(g), copy.deepcopy(g), copy.deepcopy({"of a model": [g]})["of a model"][0]):
        assert other is g
    del other
    library.calls.clear()
    g.close()
    g.close()
    assert [c[0] for c in library.calls] == ["dnatok_destroy_grammar"] and _cabi.lib() is library
    del g
    assert len(library.calls) == 1
