"""A grammar's first use on a device, which uploads its tables, beside a capture that it is no part of."""
import threading

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from dnatok_b200 import Automaton, Grammar  # noqa: E402


@pytest.mark.parametrize("where", ["stream", "thread"])
def test_first_use_while_another_stream_is_captured(where):
    a = Automaton.avoiding(["ACG"])
    tokens = [b"A", b"AC", b"ACG", b"T"]
    keep, fresh = Grammar(a, tokens), Grammar(a, tokens)
    states = torch.zeros(3, dtype=torch.int32, device="cuda")
    want = keep.allowed(states)
    out, mask, side = torch.zeros_like(want), torch.zeros_like(want), torch.cuda.Stream()
    torch.cuda.synchronize()
    failed = []

    def use():
        try:
            with torch.cuda.stream(side):
                fresh.allowed(states, out=mask)
        except Exception as e:
            failed.append(e)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep.allowed(states, out=out)
        if where == "stream":
            use()
        else:
            other = threading.Thread(target=use)
            other.start()
            other.join()
        keep.advance(states, torch.full((3,), -1, device="cuda"), out=states)
    assert not failed, failed
    side.synchronize()
    assert torch.equal(mask, want) and not out.any()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and not states.any()
