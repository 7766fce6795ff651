"""Penalties, bias and mask on logits, and their gradient, against 64 bits."""
import math

import numpy as np
import pytest

import generate_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from dnatok_b200 import TokenHistory, process_logits, process_logits_backward  # noqa: E402

WIDTHS = [1, 2, 5, 10, 31, 32, 33, 63, 257, 512, 1000, 2049, 4106]


def make(n, width, dtype, seed=0, shift=0, pad=0, history_rows=None):
    """Random arguments; ``shift``: columns in front of the view, ``pad``: behind it."""
    rng = np.random.default_rng([seed, n, width])
    hr = n if history_rows is None else history_rows
    big = torch.from_numpy(rng.normal(0, 4, (n, shift + width + pad)).astype(np.float32)).cuda().to(dtype)
    seen = rng.random((hr, width)) < 0.4
    counts = np.where(seen & (rng.random((hr, width)) < 0.6), rng.integers(1, 9, (hr, width)), 0)
    h = TokenHistory(hr, width)
    h.seen.copy_(torch.from_numpy(R.pack(seen)))
    h.counts.copy_(torch.from_numpy(counts))
    return dict(x=big[:, shift:shift + width], h=h, seen=seen, counts=counts, ok=rng.random((n, width)) < 0.7,
                r=rng.uniform(0.7, 1.6, n).astype(np.float32), f=rng.uniform(-0.5, 1, n).astype(np.float32), p=rng.uniform(-0.5, 1, n).astype(np.float32),
                bias=rng.normal(0, 2, (n, width)).astype(np.float32), grad=rng.normal(0, 1, (n, width)).astype(np.float32))


def words(ok):
    return torch.from_numpy(R.pack(ok)).cuda()


def cuda(a):
    return torch.from_numpy(a).cuda()


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_everything_together(width, dtype):
    for n, shift, pad, out_dtype in [(1, 0, 0, None), (3, 0, 0, torch.float32), (7, 1, 2, None), (5, 3, 0, torch.float32), (2, 0, 1, None)]:
        d = make(n, width, dtype, shift=shift, pad=pad)
        y = process_logits(d["x"], history=d["h"], repetition=cuda(d["r"]), frequency=cuda(d["f"]), presence=cuda(d["p"]),
                           bias=cuda(d["bias"]), allowed=words(d["ok"]), out_dtype=out_dtype)
        want, bound = R.logits(R.host(d["x"]), d["seen"], d["counts"], d["r"], d["f"], d["p"], d["bias"], d["ok"])
        assert y.dtype == (out_dtype or dtype) and y.is_contiguous()
        R.close(y, want, bound, y.dtype)


@pytest.mark.parametrize("width", [10, 33, 4106, 32000])
@pytest.mark.parametrize("which", ["nothing", "repetition", "frequency", "presence", "bias", "shared_bias", "mask", "shared_mask", "numbers"])
def test_each_alone(which, width):
    n, dtype = 6, torch.bfloat16
    d = make(n, width, dtype, seed=1)
    kw, ref = {}, {}
    if which == "repetition":
        kw, ref = dict(history=d["h"], repetition=cuda(d["r"])), dict(seen=d["seen"], r=d["r"])
    elif which in ("frequency", "presence"):
        kw, ref = {"history": d["h"], which: 0.75}, {"seen": d["seen"], "counts": d["counts"], which[0]: 0.75}
    elif which == "numbers":
        kw = dict(history=d["h"], repetition=1.3, frequency=0.5, presence=-0.25)
        ref = dict(seen=d["seen"], counts=d["counts"], r=np.float32(1.3), f=0.5, p=-0.25)
    elif which == "bias":
        kw, ref = dict(bias=cuda(d["bias"])), dict(bias=d["bias"])
    elif which == "shared_bias":
        kw, ref = dict(bias=cuda(d["bias"][0])), dict(bias=d["bias"][:1])
    elif which == "mask":
        kw, ref = dict(allowed=words(d["ok"])), dict(ok=d["ok"])
    elif which == "shared_mask":
        kw, ref = dict(allowed=words(d["ok"][:1])[0]), dict(ok=np.broadcast_to(d["ok"][:1], (n, width)))
    y = process_logits(d["x"], **kw)
    want, bound = R.logits(R.host(d["x"]), **ref)
    R.close(y, want, bound, dtype)
    # without a penalty a history changes nothing, and one without counts does for the repetition penalty
    if which == "nothing":
        assert torch.equal(process_logits(d["x"], history=d["h"]), y) and torch.equal(y, d["x"])
    if which == "repetition":
        h = TokenHistory(n, width, counts=False)
        h.seen.copy_(d["h"].seen)
        assert torch.equal(process_logits(d["x"], history=h, repetition=cuda(d["r"])), y)


@pytest.mark.parametrize("dtype", R.TYPES)
def test_masked_logits_have_no_influence(dtype):
    n, width = 5, 1000
    d = make(n, width, dtype, seed=2)
    x, ok = d["x"].clone(), d["ok"].copy()
    ok[0] = False                                                 # a row without an allowed token
    ok[1] = True
    ok[2] = False
    ok[2, 999] = True
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).max, torch.finfo(dtype).min], dtype=dtype, device="cuda")
    hidden = cuda(~ok)
    x[hidden] = bad[torch.arange(int(hidden.sum()), device="cuda") % 5]
    kw = dict(history=d["h"], repetition=cuda(d["r"]), frequency=0.5, presence=0.5, bias=cuda(d["bias"]), allowed=words(ok))
    y = process_logits(x, **kw)
    assert torch.equal(y, process_logits(d["x"], **kw))
    assert torch.isinf(y[0]).all() and (y[0] < 0).all() and torch.isfinite(y[2]).sum() == 1
    g = d["grad"].copy()
    g[~ok] = np.nan
    dx, db = process_logits_backward(cuda(g).to(dtype), x, **kw)
    assert (dx[hidden] == 0).all() and (db[hidden] == 0).all() and torch.isfinite(dx).all()


@pytest.mark.parametrize("dtype", R.TYPES)
def test_values_that_are_not_finite(dtype):
    """NaN and infinities that are allowed follow the formula; biases of -inf and of the lowest value mask too."""
    top = float(torch.finfo(dtype).max)
    x = torch.tensor([[math.nan, math.inf, -math.inf, top, -top, 0.0, -0.0, 1.0, -1.0, 2.0]], dtype=dtype, device="cuda")
    seen = np.ones((1, 10), dtype=bool)
    counts = np.array([[0, 1, 1, 0, 0, 3, 0, 2 ** 31 - 1, 1, 0]])
    h = TokenHistory(1, 10)
    h.seen.copy_(cuda(R.pack(seen)))
    h.counts.copy_(cuda(counts))
    for bias in (0.0, -math.inf, float(np.finfo(np.float32).min)):
        b = np.full((1, 10), bias, dtype=np.float32)
        y = process_logits(x, history=h, repetition=1.5, frequency=0.5, presence=0.25, bias=cuda(b))
        want, bound = R.logits(R.host(x), seen, counts, 1.5, 0.5, 0.25, b)
        with np.errstate(all="ignore"):
            want = np.where(np.abs(want) > top * 1.01, np.sign(want) * np.inf, want)
        bound = np.where(np.isfinite(want), bound, 0.0)
        R.close(y, want, bound, dtype)
    assert torch.signbit(process_logits(x)[0, 6]) and not torch.signbit(process_logits(x)[0, 5])


def test_history_rows():
    """Rows name their history row: shared, in another order, and outside the history (no history)."""
    n, width = 7, 700
    for bits in (torch.int32, torch.int64):
        d = make(n, width, torch.float32, seed=3, history_rows=4)
        target = np.array([3, 3, 0, -1, 4, 2, 2 ** 31 - 1])
        inside = (target >= 0) & (target < 4)
        at = np.where(inside, target, 0)
        seen, counts = d["seen"][at] & inside[:, None], d["counts"][at] * inside[:, None]
        rows = torch.from_numpy(target).to(bits).cuda()
        kw = dict(history=d["h"], rows=rows, repetition=cuda(d["r"]), frequency=cuda(d["f"]), presence=cuda(d["p"]))
        want, bound = R.logits(R.host(d["x"]), seen, counts, d["r"], d["f"], d["p"])
        R.close(process_logits(d["x"], **kw), want, bound, torch.float32)
        dx, _ = process_logits_backward(cuda(d["grad"]), d["x"], **kw)
        want, _ = R.gradients(R.host(d["x"]), d["grad"], seen, d["r"])
        R.close(dx, want, np.abs(want) * 2 * R.U32, torch.float32)
    with torch.no_grad():
        far = torch.tensor([2 ** 40 + 1] * n, device="cuda")
        assert torch.equal(process_logits(d["x"], history=d["h"], rows=far, repetition=2.0), d["x"])


def test_views_outputs_and_in_place():
    n, width = 9, 333
    d = make(n, width, torch.bfloat16, seed=4)
    kw = dict(history=d["h"], repetition=1.4, presence=0.5, allowed=words(d["ok"]))
    y = process_logits(d["x"], **kw)
    # the last position of a prefill, and rows that repeat (an expanded view)
    three = torch.randn(n, 5, width, device="cuda").to(torch.bfloat16)
    three[:, -1] = d["x"]
    assert torch.equal(process_logits(three[:, -1], **kw), y)
    one = d["x"][:1].expand(n, width)
    assert torch.equal(process_logits(one, **kw), process_logits(one.contiguous(), **kw))
    # into a wider array, whose other columns stay
    wide = torch.full((n, width + 7), 5.0, dtype=torch.bfloat16, device="cuda")
    assert process_logits(d["x"], out=wide[:, 3:3 + width], **kw).data_ptr() == wide[:, 3:].data_ptr()
    assert torch.equal(wide[:, 3:3 + width], y) and (wide[:, :3] == 5).all() and (wide[:, 3 + width:] == 5).all()
    wide32 = torch.full((n, width + 7), 5.0, device="cuda")
    process_logits(d["x"], out=wide32[:, 1:1 + width], **kw)
    assert torch.equal(wide32[:, 1:1 + width].bfloat16(), y) and (wide32[:, 0] == 5).all() and (wide32[:, 1 + width:] == 5).all()
    x = d["x"].clone()
    assert process_logits(x, out=x, **kw) is x and torch.equal(x, y)
    empty = TokenHistory(0, width)
    assert process_logits(d["x"][:0], history=empty, repetition=2.0).shape == (0, width)
    assert d["x"].isfinite().all()


def test_words_behind_the_last_token_are_not_looked_at():
    d = make(3, 40, torch.float32, seed=5)
    ok = words(d["ok"])
    kw = dict(history=d["h"], repetition=1.5)
    y = process_logits(d["x"], allowed=ok, **kw)
    ok[:, 1] |= ~0xff
    d["h"].seen[:, 1] |= ~0xff
    assert torch.equal(process_logits(d["x"], allowed=ok, **kw), y)


# Calls beyond what a thread a logit serves: tiles of one and of two parts, vectors of 16 bits, halves beside 32 bits, columns
# apart; tiles and pieces that end anywhere; more rows than a grid has blocks for.
LARGE = [(40, 8192, 0, 0), (40, 8192, 1, 7), (40, 8192, 8, 8), (400, 4096, 0, 0), (400, 4100, 0, 0), (700, 1001, 0, 0), (90, 4106, 0, 0),
         (61000, 5, 0, 0), (3, 120007, 0, 0), (500, 616, 0, 0), (12, 32000, 0, 4), (530001, 1, 0, 0)]


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("n,width,shift,pad", LARGE)
def test_large_calls(n, width, shift, pad, dtype):
    d = make(n, width, dtype, seed=13, shift=shift, pad=pad, history_rows=n if n < 1000 else 50)
    seen, counts, rows = d["seen"], d["counts"], None
    if n >= 1000:
        target = np.random.default_rng(1).integers(-5, 55, n)
        inside = (target >= 0) & (target < 50)
        at = np.where(inside, target, 0)
        seen, counts = seen[at] & inside[:, None], counts[at] * inside[:, None]
        rows = torch.from_numpy(target).cuda()
    x = R.host(d["x"])
    pen = dict(history=d["h"], rows=rows, repetition=cuda(d["r"]), frequency=cuda(d["f"]), presence=cuda(d["p"]))
    ref = dict(seen=seen, counts=counts, r=d["r"], f=d["f"], p=d["p"])
    for out_dtype in {dtype, torch.float32}:
        for kw, more in [(dict(bias=cuda(d["bias"]), allowed=words(d["ok"]), **pen), dict(bias=d["bias"], ok=d["ok"], **ref)),
                         (dict(bias=cuda(d["bias"][0]), allowed=words(d["ok"][:1])), dict(bias=d["bias"][:1], ok=np.broadcast_to(d["ok"][:1], (n, width)))),
                         (pen, ref)]:
            want, bound = R.logits(x, **more)
            y = process_logits(d["x"], out_dtype=out_dtype, **kw)
            R.close(y, want, bound, out_dtype)
            if out_dtype == dtype:
                z = d["x"].clone() if shift == 0 else d["x"]
                assert torch.equal(process_logits(z, out=z, **kw), y)
                if z is d["x"]:
                    d["x"].copy_(torch.from_numpy(x).to(dtype))
    g = cuda(d["grad"]).to(dtype)
    for bias in (cuda(d["bias"]), cuda(d["bias"][0]), None):
        dx, db = process_logits_backward(g, d["x"], bias=bias, allowed=words(d["ok"]), **pen)
        want, each = R.gradients(x, R.host(g), seen, d["r"], d["ok"])
        R.close(dx, want, np.abs(want) * 2 * R.U32, dtype)
        if bias is None:
            assert db is None
        elif bias.dim() == 2:
            R.close(db, each, 0.0, torch.float32)
        else:
            R.close(db, each.sum(0), 1.01 * n * R.U32 * np.abs(each).sum(0), torch.float32)
    dx, _ = process_logits_backward(g, d["x"])                     # nothing but the identity
    assert torch.equal(dx, g)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("n,width,shift,pad", LARGE)
def test_large_calls_with_the_repetition_penalty_alone(n, width, shift, pad, dtype):
    """No counts are needed: another kernel than with them.  A hundredth of the logits are no ordinary numbers."""
    d = make(n, width, dtype, seed=29, shift=shift, pad=pad, history_rows=n if n < 1000 else 50)
    rng = np.random.default_rng(31)
    odd = torch.from_numpy(rng.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0]), (n, width)))
    d["x"].copy_(torch.where(torch.from_numpy(rng.random((n, width)) < 0.01).cuda(), odd.to(dtype).cuda(), d["x"]))
    target = rng.integers(-5, 55, n) if n >= 1000 else rng.permutation(n)
    inside = (target >= 0) & (target < len(d["seen"]))
    seen, rows = d["seen"][np.where(inside, target, 0)] & inside[:, None], torch.from_numpy(target).cuda()
    x = R.host(d["x"])
    pen, ref = dict(history=d["h"], rows=rows, repetition=cuda(d["r"])), dict(seen=seen, r=d["r"])
    for out_dtype in {dtype, torch.float32}:
        for kw, more in [(pen, ref),
                         (dict(allowed=words(d["ok"]), **pen), dict(ok=d["ok"], **ref)),
                         (dict(bias=cuda(d["bias"]), allowed=words(d["ok"][:1])[0], **pen), dict(bias=d["bias"], ok=np.broadcast_to(d["ok"][:1], (n, width)), **ref)),
                         (dict(bias=cuda(d["bias"][0]), **pen), dict(bias=d["bias"][:1], **ref))]:
            want, bound = R.logits(x, **more)
            y = process_logits(d["x"], out_dtype=out_dtype, **kw)
            R.close(y, want, bound, out_dtype)
            if kw is pen:
                zeros = want == 0
                assert (np.signbit(R.host(y))[zeros] == np.signbit(want)[zeros]).all()
            if out_dtype == dtype and shift == 0:
                z = d["x"].clone()
                process_logits(z, out=z, **kw)
                R.close(z, R.host(y), 0.0, dtype)


def test_offsets_beyond_32_bits():
    """70,001 x 32,000 logits and a history as large: the last rows as in a call of their own."""
    n, width, last = 70001, 32000, 3
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty((n, width), dtype=torch.bfloat16, device="cuda").normal_(0, 3, generator=g)
    h = TokenHistory(n, width)
    h.append(torch.randint(0, width, (n,), generator=g, device="cuda"))
    h.append(torch.randint(0, width, (n,), generator=g, device="cuda"))
    small = TokenHistory(last, width)
    small.seen.copy_(h.seen[-last:])
    small.counts.copy_(h.counts[-last:])
    assert small.counts.sum() == 2 * last and h.counts[0].sum() == 2
    bias = torch.randn(width, generator=g, device="cuda")
    ok = torch.randint(-2 ** 31, 2 ** 31, (n, width // 32), generator=g, device="cuda").int()
    kw = dict(repetition=1.5, frequency=0.25, presence=0.5, bias=bias)
    y = process_logits(x, history=h, allowed=ok, **kw)
    assert torch.equal(y[-last:], process_logits(x[-last:], history=small, allowed=ok[-last:], **kw))
    dx, db = process_logits_backward(y.nan_to_num_(0, 0, 0), x, history=h, allowed=ok, **kw)
    want, _ = process_logits_backward(y[-last:], x[-last:], history=small, allowed=ok[-last:], **kw)
    assert torch.equal(dx[-last:], want) and torch.isfinite(db).all()


@pytest.mark.parametrize("width", [512, 4106, 32000])
def test_rows_that_have_seen_everything(width):
    n = 3 * 10 ** 5 // width + 30
    d = make(n, width, torch.bfloat16, seed=14)
    d["h"].seen.fill_(-1)
    d["h"].counts.fill_(7)
    full = np.ones((n, width), dtype=bool)
    kw = dict(history=d["h"], repetition=cuda(d["r"]), frequency=cuda(d["f"]), presence=0.125)
    want, bound = R.logits(R.host(d["x"]), full, full * 7, d["r"], d["f"], 0.125)
    R.close(process_logits(d["x"], **kw), want, bound, torch.bfloat16)
    g = cuda(d["grad"]).to(torch.bfloat16)
    want, _ = R.gradients(R.host(d["x"]), R.host(g), full, d["r"])
    R.close(process_logits_backward(g, d["x"], **kw)[0], want, np.abs(want) * 2 * R.U32, torch.bfloat16)


# --------------------------------------------------------------------------- gradients

@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("n,width", [(1, 1), (1, 512), (3, 33), (64, 10), (17, 1000), (130, 257), (300, 4106), (5, 4096), (2, 32000)])
def test_gradients_against_the_formula(n, width, dtype):
    for shared in (True, False):
        for out_dtype in {dtype, torch.float32}:
            d = make(n, width, dtype, seed=6, shift=0 if shared else 1, pad=0 if shared else 2)
            x = d["x"].detach().requires_grad_()
            b = cuda(d["bias"][0] if shared else d["bias"]).requires_grad_()
            kw = dict(history=d["h"], repetition=cuda(d["r"]), frequency=0.5, presence=cuda(d["p"]), allowed=words(d["ok"]))
            y = process_logits(x, bias=b, out_dtype=out_dtype, **kw)
            g = cuda(d["grad"]).to(out_dtype)
            dx, db = torch.autograd.grad(y, (x, b), g)
            assert dx.dtype == dtype and db.dtype == torch.float32 and db.shape == b.shape
            want, rows = R.gradients(R.host(x), R.host(g), d["seen"], d["r"], d["ok"])
            R.close(dx, want, np.abs(want) * 2 * R.U32, dtype)
            if shared:                      # n - 1 additions of what is at most the sum of the sizes
                R.close(db, rows.sum(0), 1.01 * n * R.U32 * np.abs(rows).sum(0), torch.float32)
            else:
                R.close(db, rows, 0.0, torch.float32)
            ex, eb = process_logits_backward(g, x.detach(), bias=b.detach(), **kw)
            assert torch.equal(ex, dx) and torch.equal(eb, db)
            again = torch.autograd.grad(process_logits(x, bias=b, out_dtype=out_dtype, **kw), (x, b), g)
            assert torch.equal(again[0], dx) and torch.equal(again[1], db)


def test_gradients_against_differences():
    """y is linear in each logit on either side of 0 and in the bias: with a step that does not cross 0, differences are
    exact but for two roundings of y, here of sums below 64 in size."""
    n, width, step = 4, 200, 0.25
    d = make(n, width, torch.float32, seed=7)
    x = torch.where(d["x"] >= 0, d["x"] + 0.5, d["x"] - 0.5).detach().requires_grad_()
    b = cuda(d["bias"][0]).requires_grad_()
    kw = dict(history=d["h"], repetition=cuda(d["r"]), frequency=cuda(d["f"]), presence=cuda(d["p"]), allowed=words(d["ok"]))
    g = cuda(d["grad"])
    dx, db = torch.autograd.grad(process_logits(x, bias=b, **kw), (x, b), g)

    def value(x, b):
        y = process_logits(x.detach(), bias=b.detach(), **kw).double()
        return torch.where(torch.isinf(y), 0.0, y * g.double())
    err = 8 * 64 * R.U32 / (2 * step) * float(g.abs().max())
    slope = (value(x + step, b) - value(x - step, b)) / (2 * step)
    assert (slope - dx.double()).abs().max() <= err
    slope = ((value(x, b + step) - value(x, b - step)) / (2 * step)).sum(0)
    assert (slope - db.double()).abs().max() <= n * err


def test_gradient_layouts():
    """Gradients as autograd hands them over: expanded, transposed, of only one input, of a shared mask or bias of one row."""
    n, width = 6, 200
    d = make(n, width, torch.bfloat16, seed=8)
    ok = words(d["ok"][:1])
    x = d["x"].detach().requires_grad_()
    y = process_logits(x, history=d["h"], repetition=1.5, allowed=ok, out_dtype=torch.float32)
    torch.where(torch.isinf(y), 0.0, y).sum().backward()
    want, _ = R.gradients(R.host(x), np.ones((n, width)), d["seen"], 1.5, np.broadcast_to(d["ok"][:1], (n, width)))
    R.close(x.grad, want, np.abs(want) * 2 * R.U32, torch.bfloat16)
    y = process_logits(x, history=d["h"], repetition=1.5)
    g = torch.randn(width, n, device="cuda").to(torch.bfloat16).t()
    dx, = torch.autograd.grad(y, x, g)
    assert torch.equal(dx, process_logits_backward(g.contiguous(), x.detach(), history=d["h"], repetition=1.5)[0])
    b = cuda(d["bias"][:1]).requires_grad_()
    y = process_logits(x.detach(), bias=b, allowed=ok)
    db, = torch.autograd.grad(y, b, torch.ones_like(y))
    assert db.shape == (1, width) and torch.equal(db[0], torch.where(cuda(d["ok"][0]), float(n), 0.0))
    empty = torch.empty(0, width, device="cuda", requires_grad=True)
    db, = torch.autograd.grad(process_logits(empty, bias=b), b, torch.empty(0, width, device="cuda"))
    assert (db == 0).all()
    with pytest.raises(RuntimeError):                              # no gradient of the gradient
        dx, = torch.autograd.grad(process_logits(x, history=d["h"], repetition=1.5), x, g, create_graph=True)
        dx.sum().backward()


def test_a_history_that_went_on_has_no_gradient():
    d = make(3, 50, torch.float32, seed=9)
    x = d["x"].detach().requires_grad_()
    y = process_logits(x, history=d["h"], repetition=1.5)
    d["h"].append(torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_through_checkpoint_and_saved_elsewhere():
    from torch.utils.checkpoint import checkpoint
    d = make(4, 100, torch.float32, seed=10, shift=1, pad=3)
    kw = dict(history=d["h"], repetition=cuda(d["r"]), allowed=words(d["ok"]), bias=cuda(d["bias"]))
    x = d["x"].detach().requires_grad_()
    g = cuda(d["grad"])
    want, = torch.autograd.grad(process_logits(x, **kw), x, g)
    got, = torch.autograd.grad(checkpoint(lambda t: process_logits(t, **kw), x, use_reentrant=False), x, g)
    assert torch.equal(got, want)
    with torch.autograd.graph.save_on_cpu():
        y = process_logits(x, **kw)
    got, = torch.autograd.grad(y, x, g)
    assert torch.equal(got, want)


# --------------------------------------------------------------------------- streams, graphs, refusals

def test_another_stream_and_a_captured_graph():
    n, width = 8, 4106
    d = make(n, width, torch.bfloat16, seed=11)
    kw = dict(history=d["h"], repetition=cuda(d["r"]), frequency=0.5, bias=cuda(d["bias"][0]), allowed=words(d["ok"]))
    x, g = d["x"].clone(), cuda(d["grad"]).to(torch.bfloat16)
    want, grads = process_logits(x, **kw), process_logits_backward(g, x, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = process_logits(x, **kw)
    side.synchronize()
    assert torch.equal(got, want)
    live = x.clone().requires_grad_()
    alive = process_logits(live, **kw)                             # an eager graph over the same leaf
    out = torch.empty_like(x)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        process_logits(x, out=out, **kw)
        static = process_logits_backward(g, live.detach(), **kw)
    with torch.cuda.graph(other):
        static2 = process_logits_backward(g, live.detach(), **kw)
    for k in range(2):
        out.zero_()
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for s in (static, static2):
            assert torch.equal(s[0], grads[0]) and torch.equal(s[1], grads[1])
    x.mul_(0.5)
    graph.replay()
    assert torch.equal(out, process_logits(x, **kw))
    assert alive.requires_grad


def test_forward_and_gradient_in_one_captured_graph():
    n, width = 20, 1000
    d = make(n, width, torch.float32, seed=15)
    kw = dict(history=d["h"], repetition=cuda(d["r"]), frequency=0.5, presence=0.5, allowed=words(d["ok"]))
    x, b, g = d["x"].clone().requires_grad_(), cuda(d["bias"][0]).requires_grad_(), cuda(d["grad"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = process_logits(x, bias=b, **kw)
        dx, db = torch.autograd.grad(y, (x, b), g)
    for k in range(2):
        with torch.no_grad():
            x.add_(k)
        dx.zero_()
        graph.replay()
        want, each = R.gradients(R.host(x), d["grad"], d["seen"], d["r"], d["ok"])
        R.close(dx, want, np.abs(want) * 2 * R.U32, torch.float32)
        R.close(db, each.sum(0), 1.01 * n * R.U32 * np.abs(each).sum(0), torch.float32)


def test_refusals():
    d = make(3, 64, torch.float32, seed=12)
    x, h = d["x"], d["h"]
    ok = words(d["ok"])
    other = TokenHistory(3, 63)
    plain = TokenHistory(3, 64, counts=False)
    for kw in [dict(repetition=1.5), dict(frequency=0.5), dict(rows=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(history=other, repetition=1.5),
               dict(history=TokenHistory(4, 64), repetition=1.5), dict(history=plain, frequency=0.5), dict(history=h, repetition=0.0),
               dict(history=h, repetition=math.inf), dict(history=h, presence=math.nan), dict(history=h, frequency=1e300), dict(history=h, repetition=1e-60), dict(history=h, repetition=torch.ones(2, device="cuda")),
               dict(history=h, repetition=torch.ones(3, device="cuda", dtype=torch.float64)), dict(history=h, repetition=torch.ones(3)),
               dict(history=h, repetition=torch.ones(3, device="cuda", requires_grad=True)), dict(history=h, repetition=torch.ones(6, device="cuda")[::2]),
               dict(history=h, rows=torch.zeros(2, dtype=torch.int32, device="cuda"), repetition=1.5),
               dict(history=h, rows=torch.zeros(3, dtype=torch.int16, device="cuda"), repetition=1.5),
               dict(bias=torch.zeros(63, device="cuda")), dict(bias=torch.zeros(64, device="cuda", dtype=torch.bfloat16)), dict(bias=torch.zeros(64)),
               dict(bias=torch.zeros(2, 64, device="cuda")), dict(bias=torch.zeros(128, device="cuda")[::2]), dict(bias=torch.zeros(1, 64, device="cuda").expand(3, 64)),
               dict(allowed=ok[:, :1]), dict(allowed=ok.long()), dict(allowed=ok.cpu()), dict(allowed=ok[:2]), dict(allowed=d["ok"]),
               dict(out=torch.empty(3, 64, device="cuda", dtype=torch.float16)), dict(out=torch.empty(3, 63, device="cuda")), dict(out=torch.empty(3, 64)),
               dict(out=torch.empty(64, device="cuda").expand(3, 64)), dict(out_dtype=torch.float16),
               dict(out=torch.empty(3, 64, device="cuda"), out_dtype=torch.bfloat16)]:
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            process_logits(x, **kw)
    for bad in (x[0], x.double(), x.long(), x[:, ::2], x.t(), torch.empty(3, 0, device="cuda")):
        with pytest.raises((ValueError, RuntimeError)):
            process_logits(bad)
    with pytest.raises(ValueError):
        process_logits(x.clone().requires_grad_(), out=torch.empty_like(x))
    with torch.no_grad():
        process_logits(x.clone().requires_grad_(), out=torch.empty_like(x))
    for g in (x[:2], x.half(), x[:, :63]):
        with pytest.raises(ValueError):
            process_logits_backward(g, x)
    h.seen = h.seen[:, :1]
    with pytest.raises(ValueError):
        process_logits(x, history=h, repetition=1.5)
