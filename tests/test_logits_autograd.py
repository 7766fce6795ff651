"""What autograd and tracing may make of the operators around logits (refused where they would be wrong without a word)."""
import pytest

torch = pytest.importorskip("torch")

from dnatok_b200 import Automaton, Grammar, TokenHistory, process_logits, process_logits_backward  # noqa: E402

from generate_host import history, library  # noqa: E402,F401


@pytest.mark.parametrize("name", ["repetition", "frequency", "presence"])
@pytest.mark.parametrize("leaf", ["logits", "bias", "neither"])
def test_a_penalty_that_needs_a_gradient_is_refused(library, name, leaf):  # noqa: F811
    x, b = torch.randn(3, 40, requires_grad=leaf == "logits"), torch.randn(40, requires_grad=leaf == "bias")
    h, v = history(3, 40), torch.ones(3, requires_grad=True)
    with pytest.raises(ValueError, match="%s has no gradient" % name):
        process_logits(x, history=h, bias=b, **{name: v})
    assert not library.calls
    with torch.no_grad():
        process_logits(x, history=h, bias=b, **{name: v})
    process_logits(x, history=h, bias=b, **{name: v.detach()})
    assert [c[0] for c in library.calls] == ["dnatok_process_logits"] * 2


@pytest.mark.parametrize("leaf", [True, False])
def test_an_output_that_is_part_of_a_graph_is_refused(library, leaf):  # noqa: F811
    """Its new values would not be those that its graph differentiates."""
    x, w = torch.randn(3, 40), torch.randn(3, 40, requires_grad=True)
    out = w if leaf else w * 2
    with pytest.raises(ValueError, match="out= has no gradient"):
        process_logits(x, out=out)
    assert not library.calls and (leaf or out.grad_fn is not None)
    with torch.no_grad():
        assert process_logits(x, out=out) is out


@pytest.mark.parametrize("name", ["logits", "bias", "repetition", "frequency", "presence"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(library, name, grad):  # noqa: F811
    from torch.autograd import forward_ad
    args = {"logits": torch.randn(3, 40, requires_grad=grad), "bias": torch.randn(40), "repetition": torch.ones(3), "frequency": torch.ones(3),
            "presence": torch.ones(3)}
    h = history(3, 40)
    with forward_ad.dual_level():
        dual = dict(args)
        dual[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(RuntimeError, match="%s has a tangent" % name):
            process_logits(history=h, **dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="%s has a tangent" % name):
            process_logits(history=h, **dual)
        with pytest.raises(RuntimeError, match="%s has a tangent" % name):
            process_logits_backward(torch.ones(3, 40), history=h, **dual)
        assert not library.calls
        process_logits(history=h, **args)                          # no tangent anywhere: nothing is lost
        with pytest.raises(RuntimeError, match="grad has a tangent"):
            process_logits_backward(forward_ad.make_dual(torch.ones(3, 40), torch.ones(3, 40)), args["logits"])
        with torch.no_grad(), pytest.raises(RuntimeError, match="out has a tangent"):
            process_logits(args["logits"], out=forward_ad.make_dual(torch.ones(3, 40), torch.ones(3, 40)))
    assert [c[0] for c in library.calls] == ["dnatok_process_logits"]


CALLS = {"process_logits": lambda x, h, g: process_logits(x, history=h, repetition=1.5),
         "process_logits_backward": lambda x, h, g: process_logits_backward(x, x, history=h, repetition=1.5)[0],
         "add": lambda x, h, g: (h.add(x.long()), x)[1],
         "append": lambda x, h, g: (h.append(x[:, 0].long()), x)[1],
         "allowed": lambda x, h, g: g.allowed(x[:, 0].int()),
         "advance": lambda x, h, g: g.advance(x[:, 0].int(), x[:, 1].long()),
         "step": lambda x, h, g: g.step(x[:, 0].int(), x[:, 1].long())[1]}


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("call", CALLS)
def test_traces_are_refused(library, call):  # noqa: F811
    """They would hold the allocation of the output and nothing that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    h, g = history(3, 40), Grammar(Automaton.avoiding(["ACG"]), [b"A", b"C"] * 20)
    library.calls.clear()
    x = torch.zeros(3, 40)
    for trace in (lambda f: torch.jit.trace(f, x, check_trace=False), lambda f: make_fx(f)(x), lambda f: make_fx(f, pre_dispatch=True)(x)):
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            trace(lambda z: CALLS[call](z, h, g))
        assert not library.calls
    CALLS[call](x, h, g)                                           # and nothing is left of it
    assert len(library.calls) == 1


def test_a_bias_may_change_before_the_backward_pass(library):  # noqa: F811
    """Its gradient does not depend on its values: an optimiser may step in between."""
    for shape in ((40,), (1, 40), (3, 40)):
        x, b = torch.randn(3, 40, requires_grad=True), torch.randn(shape, requires_grad=True)
        y = process_logits(x, bias=b)
        with torch.no_grad():
            b.add_(1)
        dx, db = torch.autograd.grad(y, (x, b), torch.ones(3, 40))
        assert db.shape == b.shape and db.dtype == torch.float32 and db.is_contiguous()


def test_without_a_repetition_penalty_nothing_but_the_mask_is_kept(library):  # noqa: F811
    """Frequency, presence and bias have derivatives that depend on no logit and no history: both may change."""
    for kw in (dict(frequency=0.5), dict(presence=torch.ones(3), repetition=1.0), {}):
        w, b = torch.randn(3, 40, requires_grad=True), torch.randn(40, requires_grad=True)
        x, h, ok, rows = w * 2, history(3, 40), torch.zeros((3, 2), dtype=torch.int32), torch.arange(3)
        y = process_logits(x, history=h, rows=rows, bias=b, allowed=ok, **kw)
        h.append(torch.zeros(3, dtype=torch.int64))
        rows.zero_()
        with torch.no_grad():
            x.mul_(2)
        library.calls.clear()
        dw, db = torch.autograd.grad(y, (w, b), torch.ones(3, 40))
        a = library.calls[-1][1]
        assert library.calls[-1][0] == "dnatok_process_logits_backward"
        assert (a.n_rows, a.width, a.dtype, a.seen, a.rows, a.allowed) == (3, 40, 0, None, None, ok.data_ptr()) and a.logits
        assert dw.shape == (3, 40) and db.shape == (40,)
        y = process_logits(x, history=h, allowed=ok, **kw)
        ok.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


@pytest.mark.parametrize("change", ["logits", "seen", "rows", "repetition"])
def test_what_the_repetition_penalty_depends_on_stays(library, change):  # noqa: F811
    w, h, rows, r = torch.randn(3, 40, requires_grad=True), history(3, 40), torch.arange(3), torch.ones(3)
    x = w * 2
    y = process_logits(x, history=h, rows=rows, repetition=r)
    with torch.no_grad():
        {"logits": x, "seen": h.seen, "rows": rows, "repetition": r}[change].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_bias_alone_keeps_no_logits(library):  # noqa: F811
    x, h, r = torch.randn(3, 40), history(3, 40), torch.ones(3)
    b = torch.randn(40, requires_grad=True)
    y = process_logits(x, history=h, repetition=r, bias=b)
    x.zero_()
    r.zero_()
    h.append(torch.zeros(3, dtype=torch.int64))
    db, = torch.autograd.grad(y, b, torch.ones(3, 40))
    assert db.shape == (40,) and library.calls[-1][1].seen is None


def wrapper(t):
    """A tensor that stands for others and has no memory of its own, as torch's distributed ones."""
    class Wrapper(torch.Tensor):
        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise AssertionError("no operation of it is expected: %s" % func)
    return torch.Tensor._make_wrapper_subclass(Wrapper, t.shape, strides=t.stride(), dtype=t.dtype, device=t.device)


@pytest.mark.parametrize("name", ["logits", "bias", "allowed", "repetition", "frequency", "presence", "rows", "out", "seen", "counts"])
def test_tensors_without_memory_are_refused(library, name):  # noqa: F811
    """An address of 0 means an argument that is not there."""
    h = history(3, 40)
    args = dict(logits=torch.randn(3, 40), bias=torch.randn(40), allowed=torch.zeros((3, 2), dtype=torch.int32), repetition=torch.ones(3), frequency=torch.ones(3),
                presence=torch.ones(3), rows=torch.zeros(3, dtype=torch.int64), out=torch.empty(3, 40))
    process_logits(history=h, **args)
    library.calls.clear()
    if name in args:
        args[name] = wrapper(args[name])
    else:
        setattr(h, name, wrapper(getattr(h, name)))
    with pytest.raises(ValueError, match="%s has no memory" % name):
        process_logits(history=h, **args)
    assert not library.calls


def test_histories_and_grammars_refuse_tensors_without_memory(library):  # noqa: F811
    h, g = history(3, 40), Grammar(Automaton.avoiding(["ACG"]), [b"A", b"C"] * 20)
    library.calls.clear()
    ids, n, t = torch.zeros((3, 5), dtype=torch.int64), torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int64)
    offsets = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: h.add(wrapper(ids)), lambda: h.add(ids, wrapper(n)), lambda: h.add(t, offsets=wrapper(offsets)), lambda: h.append(wrapper(t)),
                 lambda: h.append(t, rows=wrapper(t)), lambda: g.allowed(wrapper(n)), lambda: g.allowed(n, out=wrapper(torch.zeros((3, 2), dtype=torch.int32))),
                 lambda: g.advance(n, wrapper(t)), lambda: g.advance(n, t, out=wrapper(n)), lambda: g.step(n, t, out_allowed=wrapper(torch.zeros((3, 2), dtype=torch.int32))),
                 lambda: process_logits_backward(wrapper(torch.zeros(3, 40)), torch.zeros(3, 40))):
        with pytest.raises(ValueError, match="has no memory"):
            call()
    assert not library.calls
    empty = torch.zeros((0, 40))
    process_logits(empty, bias=torch.zeros((0, 40)), allowed=torch.zeros((0, 2), dtype=torch.int32))


def test_counts_and_seen_change_by_themselves(library):  # noqa: F811
    """The backward pass reads what was seen: counts that are cleared in between do not matter to it, marks do."""
    seen, counts = TokenHistory._cleared(3, 40, torch.device("cpu"))
    assert seen.shape == (3, 2) and counts.shape == (3, 40) and seen.is_contiguous() and counts.is_contiguous()
    assert seen.dtype == counts.dtype == torch.int32 and not seen.any() and not counts.any()
    assert counts.untyped_storage().data_ptr() == seen.untyped_storage().data_ptr() and counts.data_ptr() - seen.data_ptr() == 32
    h = history(3, 40)
    for write, refused in ((lambda: h.counts.zero_(), False), (lambda: h.seen.zero_(), True)):
        h.seen, h.counts = TokenHistory._cleared(3, 40, torch.device("cpu"))
        x = torch.randn(3, 40, requires_grad=True)
        y = process_logits(x, history=h, repetition=1.5, frequency=0.5)
        write()
        if refused:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.sum().backward()
        else:
            y.sum().backward()
            assert x.grad.shape == x.shape
    with torch.inference_mode():
        seen, counts = TokenHistory._cleared(0, 40, torch.device("cpu"))
    assert seen.shape == (0, 2) and counts.shape == (0, 40)


@pytest.mark.gpu
def test_counts_may_be_cleared_before_the_backward_pass():
    x, g = torch.randn(5, 700, device="cuda", requires_grad=True), torch.randn(5, 700, device="cuda")
    h = TokenHistory(5, 700)
    h.add(torch.randint(0, 700, (5, 300), device="cuda"), generated=True)
    want, = torch.autograd.grad(process_logits(x, history=h, repetition=1.5, frequency=0.5), x, g)
    y = process_logits(x, history=h, repetition=1.5, frequency=0.5)
    h.counts.zero_()
    assert torch.equal(torch.autograd.grad(y, x, g)[0], want) and not torch.equal(want, g)
