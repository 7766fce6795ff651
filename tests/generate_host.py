"""The host path of the operators around logits without a GPU: CPU tensors in place of device ones, a library that takes calls down."""
import pytest
import torch

from dnatok_b200 import TokenHistory, _cabi, generate


class Library:
    """Every C entry point returns ``rc`` and is taken down in ``calls`` with its arguments."""

    def __init__(self):
        self.calls, self.rc = [], 0

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name,) + args)
            return self.rc
        return entry


@pytest.fixture
def library(monkeypatch):
    made = Library()
    monkeypatch.setattr(_cabi, "lib", lambda: made)
    monkeypatch.setattr(generate, "_device_of", lambda t, what: t.get_device())
    monkeypatch.setattr(generate, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(generate, "_current_device", lambda: -1)                # the device of a CPU tensor
    return made


def history(rows, width):
    h = TokenHistory.__new__(TokenHistory)
    h.n_rows, h.width = rows, width
    h.seen = torch.zeros((rows, (width + 31) // 32), dtype=torch.int32)
    h.counts = torch.zeros((rows, width), dtype=torch.int32)
    return h
