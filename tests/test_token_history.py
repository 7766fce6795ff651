"""Which tokens rows have seen and how often they generated each, against plain counting (whole numbers: exact)."""
import numpy as np
import pytest

import generate_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from dnatok_b200 import TokenHistory  # noqa: E402


def check(h, seen, counts):
    assert np.array_equal(R.unpack(h.seen.cpu().numpy(), h.width), seen)
    if h.width % 32:
        assert (h.seen[:, -1].cpu().numpy().view(np.uint32) >> (h.width % 32) == 0).all()
    if h.counts is not None:
        assert np.array_equal(h.counts.cpu().numpy(), counts)


def batch(rng, lengths, width, layout, dtype, hot=False, columns=None, wild=False):
    lengths = np.asarray(lengths)
    low, high = (-3, width + 3) if wild else (0, min(width, 6) if hot else width)
    rows = [rng.integers(low, high, n) for n in lengths]
    if layout == "ragged":
        flat = np.concatenate(rows + [np.zeros(0, np.int64)])
        offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
        return rows, (torch.from_numpy(flat).to(dtype).cuda(),), dict(offsets=torch.from_numpy(offsets).cuda())
    T = max([int(lengths.max()) if len(lengths) else 0, columns or 0])
    ids = rng.integers(0, width, (len(lengths), T))                # what stands in the padding must not be entered
    for i, r in enumerate(rows):
        if len(r):
            ids[i, T - len(r) if layout == "left" else 0:][:len(r)] = r
    return rows, (torch.from_numpy(ids).to(dtype).cuda(), torch.from_numpy(lengths.astype(np.int32)).cuda()), dict(pad_left=layout == "left")


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("layout", ["right", "left", "ragged"])
@pytest.mark.parametrize("width", [1, 10, 31, 32, 33, 512, 4106, 32000, 70001])
def test_rows_are_entered(width, layout, dtype):
    rng = np.random.default_rng([width, len(layout)])
    for lengths, hot in [([5], False), ([0, 1, 2, 33, 0, 700], False), ([0, 0], False), (rng.integers(0, 90, 301), True), ([20001, 3, 9000], True),
                         ([1] * 1000, False)]:
        rows, args, kw = batch(rng, lengths, width, layout, dtype, hot)
        for generated in (True, False):
            h = TokenHistory(len(rows), width, counts=generated)
            h.add(*args, generated=generated, **kw)
            check(h, *R.history(len(rows), width, rows, generated))
        h = TokenHistory(len(rows), width)                          # counts are kept, but nothing was generated
        h.add(*args, **kw)
        check(h, R.history(len(rows), width, rows, True)[0], np.zeros((len(rows), width), dtype=np.int64))


def test_prompt_then_tokens():
    rng = np.random.default_rng(1)
    n, width = 37, 600
    rows, args, kw = batch(rng, rng.integers(0, 50, n), width, "left", torch.int64)
    h = TokenHistory(n, width)
    h.add(*args, **kw)
    seen, counts = R.history(n, width, rows, False)
    for k in range(20):
        tokens = rng.integers(-2, width + 2, n) if k % 3 == 0 else rng.integers(0, 7, n)
        h.append(torch.from_numpy(tokens).to(torch.int32 if k % 2 else torch.int64).cuda())
        s, c = R.history(n, width, [[t] for t in tokens], True)
        seen, counts = seen | s, counts + c
    check(h, seen, counts)
    more, args, kw = batch(rng, rng.integers(0, 50, n), width, "ragged", torch.int32)
    h.add(*args, generated=True, **kw)                              # on top of what is there
    s, c = R.history(n, width, more, True)
    check(h, seen | s, counts + c)
    h.clear()
    check(h, seen & False, counts * 0)


@pytest.mark.parametrize("layout", ["right", "ragged"])
def test_ids_outside_the_vocabulary_and_rows_outside_the_history(layout):
    rng = np.random.default_rng(2)
    for width, lengths in [(40, [30, 30, 9, 30, 0, 30]), (300, [5000, 10, 4000, 3, 0, 6000])]:
        rows, args, kw = batch(rng, lengths, width, layout, torch.int64, wild=True)
        for bits in (torch.int32, torch.int64):
            target = np.array([2, 2, 0, -1, 1, 4])                  # two rows share one history row
            h = TokenHistory(4, width)
            h.add(*args, rows=torch.from_numpy(target).to(bits).cuda(), generated=True, **kw)
            check(h, *R.history(4, width, rows, True, target))
            h.append(torch.tensor([1, 1, 2, 3, 4, 5], device="cuda"), rows=torch.from_numpy(target).to(bits).cuda())
            s, c = R.history(4, width, [list(r) + [t] for r, t in zip(rows, [1, 1, 2, 3, 4, 5])], True, target)
            check(h, s, c)
    h = TokenHistory(3, 10)
    h.append(torch.tensor([2 ** 40 + 1, -2 ** 40, 2 ** 32], device="cuda"))
    h.append(torch.tensor([1, 1, 1], device="cuda"), rows=torch.tensor([2 ** 32, -2 ** 32, 2 ** 40], device="cuda"))
    assert not h.seen.any() and not h.counts.any()


def test_offsets_and_lengths_out_of_order_read_nothing_outside():
    """Rows whose offsets decrease are empty and offsets past the ids end there; lengths are cut to 0 .. T."""
    ids = torch.arange(10, device="cuda")
    h = TokenHistory(4, 16)
    h.add(ids, offsets=torch.tensor([-5, 3, 2, 12, 8], device="cuda"), generated=True)
    check(h, *R.history(4, 16, [[0, 1, 2], [], list(range(2, 10)), []], True))
    for left in (False, True):
        h = TokenHistory(3, 16)
        h.add(ids[:9].view(3, 3), torch.tensor([-1, 2, 7], dtype=torch.int32, device="cuda"), pad_left=left, generated=True)
        check(h, *R.history(3, 16, [[], [4, 5] if left else [3, 4], [6, 7, 8]], True))


@pytest.mark.parametrize("width", [5, 512, 4106, 32000])
def test_few_long_rows(width):
    rng = np.random.default_rng(width)
    lengths = [300001, 0, 131072, 77777]
    for layout in ("left", "ragged"):
        rows, args, kw = batch(rng, lengths, width, layout, torch.int32, hot=True)
        h = TokenHistory(4, width)
        h.add(*args, generated=True, **kw)
        seen, counts = np.zeros((4, width), dtype=bool), np.zeros((4, width), dtype=np.int64)
        for i, r in enumerate(rows):
            counts[i] = np.bincount(r, minlength=width)
        check(h, counts > 0, counts)
        h = TokenHistory(4, width, counts=False)
        h.add(*args, **kw)
        check(h, counts > 0, None)


def test_views_of_ids():
    """Rows further apart than they are long, ids that begin at any place, one row that several rows read."""
    rng = np.random.default_rng(4)
    for dtype in (torch.int32, torch.int64):
        big = torch.from_numpy(rng.integers(0, 50, (6, 4100))).to(dtype).cuda()
        for a, b in [(0, 7), (1, 4099), (3, 4), (5, 2050)]:
            view = big[:, a:b]
            h = TokenHistory(6, 50)
            h.add(view, generated=True)
            check(h, *R.history(6, 50, view.cpu().numpy(), True))
        h = TokenHistory(6, 50)
        h.add(big[:1].expand(6, 4100), generated=True)
        check(h, *R.history(6, 50, big[:1].expand(6, 4100).cpu().numpy(), True))
        h = TokenHistory(6, 50)
        h.add(big[:, :0])
        assert not h.seen.any()
    h = TokenHistory(0, 50)
    h.add(big[:0])
    h.append(torch.zeros(0, dtype=torch.int64, device="cuda"))


def test_streams_and_graphs():
    rng = np.random.default_rng(5)
    rows, args, kw = batch(rng, rng.integers(0, 400, 20), 300, "right", torch.int64)
    h = TokenHistory(20, 300)
    tokens = torch.zeros(20, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h.add(*args, generated=True, **kw)
    torch.cuda.current_stream().wait_stream(side)
    check(h, *R.history(20, 300, rows, True))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h.append(tokens)
    seen, counts = R.history(20, 300, rows, True)
    check(h, seen, counts)
    for k in range(3):
        tokens.fill_(k)
        graph.replay()
        seen[:, k] = True
        counts[:, k] += 1
    check(h, seen, counts)


def test_refusals():
    h = TokenHistory(3, 20)
    ids = torch.zeros(3, 4, dtype=torch.int64, device="cuda")
    n = torch.zeros(3, dtype=torch.int32, device="cuda")
    flat, offsets = ids.view(-1), torch.zeros(4, dtype=torch.int64, device="cuda")
    for args, kw in [((ids.cpu(),), {}), ((ids.short(),), {}), ((ids.float(),), {}), ((flat,), {}), ((ids[:2],), {}), ((ids.t(),), {}), ((ids[:, ::2],), {}),
                     ((ids, n.long()), {}), ((ids, n[:2]), {}), ((ids, n.cpu()), {}), ((flat, n), dict(offsets=offsets)), ((flat,), dict(offsets=offsets.int())),
                     ((flat,), dict(offsets=offsets, pad_left=True)), ((flat,), dict(offsets=offsets[:0])), ((flat,), dict(offsets=offsets[:3])),
                     ((ids,), dict(offsets=offsets)), ((flat[::2],), dict(offsets=offsets)), ((ids,), dict(rows=n[:2])), ((ids,), dict(rows=n.short())), ((None,), {})]:
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            h.add(*args, **kw)
    for t in (flat[:2], ids, flat[:3].short(), flat[:3].cpu(), flat[::4], 5):
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            h.append(t)
    h.counts = h.counts[:, :10]
    with pytest.raises(ValueError):
        h.append(flat[:3])
