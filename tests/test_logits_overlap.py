"""Outputs that overlap what the same call reads: refused, since other threads still read what one has written (no GPU; the
checks of the C ABI)."""
import ctypes

import numpy as np
import pytest

from dnatok_b200 import _cabi

INVALID, BASE = -1, 1 << 20


def cells(base, n, stride, row, size):
    """The bytes of n rows, each of them as a range."""
    return [(base + i * stride * size, base + (i * stride + row) * size) for i in range(n)]


def overlap(a, b):
    return any(x < v and u < y for x, y in a for u, v in b)


@pytest.fixture
def no_gpu():
    """These calls may come as far as a launch, which must not happen with addresses that are none."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("addresses that are none, where there is a GPU")


def refused(rc):
    """Whether the arguments were; without a GPU the others fail at their launch."""
    text = _cabi.lib().dnatok_last_error() or b""
    assert rc != 0
    assert (rc == INVALID) == (b"overlap" in text), text
    return rc == INVALID


def forward(out=BASE, out_dtype=0, out_stride=40, **kw):
    a = _cabi.Logits(logits=16 * BASE, dtype=0, n_rows=3, width=40, stride=40, repetition=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return refused(_cabi.lib().dnatok_process_logits(ctypes.byref(a), out, out_dtype, out_stride, None))


def test_rows_of_an_output_between_those_of_the_logits(no_gpu):
    """Against every byte of every row."""
    rng = np.random.default_rng(1)
    got = {True: 0, False: 0}
    for _ in range(3000):
        size, out_size = (2, 2) if rng.random() < 0.4 else (2, 4) if rng.random() < 0.5 else (4, 4)
        width, n = int(rng.integers(1, 9)), int(rng.integers(1, 6))
        stride, out_stride = int(rng.integers(0, 30)), int(rng.integers(width, 30))
        if rng.random() < 0.5:
            stride = out_stride * out_size // size
        at = BASE + int(rng.integers(-40, 41)) * out_size
        same = at == BASE and size == out_size and (stride == out_stride or n == 1)
        if at == BASE and not same:
            continue                                               # (refused for another reason)
        want = not same and overlap(cells(at, n, out_stride, width, out_size), cells(BASE, n, stride, width, size))
        kind = {(2, 2): (2, 2), (2, 4): (2, 0), (4, 4): (0, 0)}[size, out_size]
        assert forward(at, kind[1], out_stride, logits=BASE, dtype=kind[0], n_rows=n, width=width, stride=stride) == want
        got[want] += 1
    assert min(got.values()) > 500


@pytest.mark.parametrize("name,kw,first,last", [
    ("bias", dict(bias_stride=0), 0, 159), ("bias", dict(bias_stride=40), 0, 479), ("bias", dict(bias_stride=44), 0, 511),
    ("allowed", dict(allowed_stride=0), 0, 7), ("allowed", dict(allowed_stride=2), 0, 23),
    ("seen", dict(history_rows=3), 0, 23), ("seen", dict(history_rows=9, rows=64 * BASE, rows_bits=64), 0, 71),
    ("counts", dict(history_rows=3, seen=64 * BASE), 0, 479), ("rows", dict(history_rows=9, seen=64 * BASE, rows_bits=64), 0, 23),
    ("rows", dict(history_rows=9, seen=64 * BASE, rows_bits=32), 0, 11), ("d_repetition", {}, 0, 11), ("d_frequency", {}, 0, 11), ("d_presence", {}, 0, 11)])
def test_an_output_over_another_argument(no_gpu, name, kw, first, last):
    """The output's 480 bytes begin, end or lie inside of the argument's."""
    at = 8 * BASE
    for out, want in [(at, True), (at - 476, True), (at + (last & ~3), True), (at - 480, False), (at + (last + 8 & ~7), False)]:
        assert forward(out, **{name: at}, **kw) == want, out - at


def test_rows_that_are_not_used_may_be_written_over(no_gpu):
    """History rows are named only where there is a history."""
    assert not forward(8 * BASE, rows=8 * BASE, rows_bits=32)
    assert not forward(8 * BASE, logits=8 * BASE)


@pytest.mark.gpu
def test_views_of_one_array():
    """Outputs beside the logits are written, outputs over a part of them or of another argument refused."""
    import torch
    from dnatok_b200 import TokenHistory, process_logits
    n, width = 70, 500
    big = torch.randn(n, 3 * width, device="cuda")
    x = big[:, :width]
    h = TokenHistory(n, width)
    h.append(torch.randint(0, width, (n,), device="cuda"))
    kw = dict(history=h, repetition=1.5, frequency=torch.full((n,), 0.5, device="cuda"), bias=torch.randn(n, width, device="cuda"))
    want = process_logits(x, **kw)
    before = x.clone()
    for out in (big[:, width:2 * width], big[:, 2 * width:]):
        assert torch.equal(process_logits(x, out=out, **kw), want) and torch.equal(x, before)
    for out in (big[:, 1:width + 1], big[:, width - 1:2 * width - 1]):
        with pytest.raises(RuntimeError, match="overlap"):
            process_logits(x, out=out, **kw)
    rows = torch.randn(2 * n, width, device="cuda")
    assert torch.equal(process_logits(rows[::2], out=rows[1::2]), rows[::2])
    with pytest.raises(RuntimeError, match="overlap"):
        process_logits(rows[:n], out=rows[1:n + 1])
    with pytest.raises(RuntimeError, match="in place"):            # (the same address, another stride)
        process_logits(rows[::2], out=rows[:n])
    with pytest.raises(RuntimeError, match="output and bias overlap"):
        process_logits(x, out=kw["bias"], **kw)
    with pytest.raises(RuntimeError, match="counts overlap"):
        process_logits(x, out=h.counts.view(torch.float32), **kw)
    assert torch.equal(x, before) and torch.equal(process_logits(x, **kw), want)
    assert torch.equal(process_logits(x, out=x, **kw), want)


def backward(grad=2 * BASE, grad_stride=40, dlogits=4 * BASE, dlogits_stride=40, dbias=6 * BASE, scratch=None, scratch_bytes=0, **kw):
    a = _cabi.Logits(logits=16 * BASE, dtype=0, n_rows=3, width=40, stride=40, seen=32 * BASE, history_rows=3, allowed=48 * BASE, allowed_stride=2, repetition=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return refused(_cabi.lib().dnatok_process_logits_backward(ctypes.byref(a), grad, 0, grad_stride, dlogits, dlogits_stride, dbias, scratch, scratch_bytes, None))


def test_gradients_over_what_the_call_reads(no_gpu):
    at = 8 * BASE
    assert not backward()
    assert not backward(grad=at, dlogits=at)                       # in place
    assert not backward(grad=at, dlogits=at + 160, grad_stride=80, dlogits_stride=80)
    assert backward(grad=at, dlogits=at + 156, grad_stride=80, dlogits_stride=80)
    for move in (-476, -4, 4, 476):
        assert backward(grad=at, dlogits=at + move)
        assert backward(logits=at, dlogits=at + move)
        assert backward(grad=at, dlogits=at + move, seen=None)
        assert not backward(logits=at, dlogits=at + move, seen=None)           # these are not read then
        assert not backward(logits=at, dbias=at, dlogits=None)
        assert backward(dbias=at, dlogits=at + move, bias_stride=40)
    for out in ("dlogits", "dbias"):
        for name, kw, bytes_ in [("allowed", {}, 24), ("seen", {}, 24), ("rows", dict(rows_bits=64, history_rows=3), 24), ("d_repetition", {}, 12)]:
            for here, want in [(at, True), (at + bytes_ - 4, True), (at + bytes_, False)]:
                assert backward(**{name: at, out: here}, **kw) == want
        for name in ("bias", "counts", "d_frequency", "d_presence"):           # not read
            assert not backward(**{name: at, out: at}, bias_stride=0)
    assert backward(grad=at, dbias=at) and backward(grad=at, dbias=at + 476) and not backward(grad=at, dbias=at + 480)
    assert backward(logits=at, dbias=at + 476) and backward(dlogits=at, dbias=at + 476) and not backward(dlogits=at, dbias=at + 480)


def test_scratch_over_what_the_call_reads_or_writes(no_gpu):
    n, width, at = 1000, 40, 8 * BASE
    need = _cabi.lib().dnatok_logits_scratch_bytes(n, width)
    assert need > 1024
    good = dict(n_rows=n, history_rows=n, scratch=at, scratch_bytes=need + 10 ** 6)
    assert not backward(**good)
    for name, bytes_ in [("grad", n * 160), ("dlogits", n * 160), ("dbias", 160), ("logits", n * 160), ("allowed", n * 8), ("seen", n * 8), ("d_repetition", n * 4)]:
        end = at + (need + 7 & ~7)
        for here, want in [(at, True), (at + need - 4 & ~3, True), (end, False), (at - bytes_ + 4, True), (at - bytes_, False)]:
            assert backward(**{**good, name: here}) == want, (name, here - at)
