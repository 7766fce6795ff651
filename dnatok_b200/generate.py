"""Between a model's logits and the choice of its next token.

``process_logits`` applies penalties for repeated tokens, a bias and a mask to logits over a tokenizer's vocabulary in one
pass, and has a gradient; ``TokenHistory`` keeps which tokens a row has seen and how often it generated each;
``Grammar`` gives the mask of an automaton over bases (``Automaton``) for the tokens of a vocabulary, and a row's state
after its chosen token.  A generation loop:

    history = tok.token_history(batch)              # tok: a B200Tokenizer
    grammar = tok.grammar(Automaton.avoiding(["GAATTC"]))
    history.add(enc["input_ids"], enc["lengths"])
    states = grammar.start(batch)
    allowed = grammar.allowed(states)
    for _ in range(steps):
        logits = process_logits(model(...)[:, -1], history=history, repetition=1.2, allowed=allowed)
        tokens = choose(logits)
        history.append(tokens)
        states, allowed = grammar.step(states, tokens)

Everything numeric happens in ``libdnatok_b200.so``; work is enqueued on the current stream of the tensors' device and
nothing waits for it, but for a ``Grammar``'s first use on a device, which allocates and uploads its tables.
(``torch.jit.trace`` and ``make_fx`` cannot record that work: the calls refuse to be traced.)
Sets of tokens are int32 words: bit ``v % 32`` of word ``v // 32`` stands for token ``v``.

The calls can be captured into a CUDA graph (use a ``Grammar`` on the device once before, and keep it as long as the graph).
To capture a gradient while an eager graph over the same leaf tensors is alive, call ``process_logits_backward``, which needs
no autograd graph: autograd's own accumulation into a leaf waits on the stream of the older graph, which a capture does not
allow.
"""
from __future__ import annotations

import ctypes
import sys
from typing import Optional, Sequence, Tuple, Union

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _cabi
from .automaton import Automaton, whole_numbers

DEAD, FINISHED = _cabi.STATE_DEAD, _cabi.STATE_FINISHED
_TYPES = {torch.float32: _cabi.F32, torch.float16: _cabi.F16, torch.bfloat16: _cabi.BF16}
_BITS = {torch.int32: 32, torch.int64: 64}

Number = Union[float, int, torch.Tensor]
_LEAST, _MOST = 2.0 ** -126, 2.0 ** 126              # a repetition penalty whose reciprocal is a normal number too


# The current device, and the current stream of a device, as numbers (the public calls look whether CUDA is up, which it is where
# there are tensors, and build a Stream object on the way: 0.3 and 2 us instead of 0.1).
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _words(width: int) -> int:
    return (width + 31) // 32


def _device_of(t, what: str) -> int:
    """The number of a tensor's GPU."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor" % what)
    d = t.get_device()
    if d < 0:
        raise RuntimeError("%s must be a CUDA tensor; there is no CPU path" % what)
    return d


def _on(t, what: str, dev: int) -> None:
    d = _device_of(t, what)
    if d != dev:
        raise ValueError("%s is on cuda:%d, the call on cuda:%d" % (what, d, dev))


def _nowhere(t: torch.Tensor, what: str) -> int:
    """For ``t.data_ptr() or _nowhere(t, what)``: 0 means an argument that is not there, so only a tensor without elements may
    have that address."""
    if t.numel():
        raise ValueError("%s has no memory of its own (a distributed, fake or otherwise wrapped tensor)" % what)
    return 0


# make_fx records under a mode for functions; where there is none it need not be asked for (0.05 us instead of 1).
_modes = getattr(torch._C, "_len_torch_function_stack", None) or (lambda: 1)
_tracing = getattr(torch._C, "_is_tracing", None) or torch.jit.is_tracing


def _traced() -> bool:
    """Whether ``make_fx`` is recording the operations of this thread."""
    proxies = sys.modules.get("torch.fx.experimental.proxy_tensor")
    return proxies is not None and proxies.get_proxy_mode() is not None


def _call(fn, dev: int, *args) -> None:
    """A C entry point with the device current and its current stream as the last argument."""
    if _tracing() or (_modes() and _traced()):
        # (the trace would hold the output's allocation and nothing that fills it)
        raise RuntimeError("kernels of this library cannot be recorded by torch.jit.trace or make_fx")
    if _current_device() == dev:
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        _cabi.check(rc)


def _no_tangents(**named) -> None:
    """Forward mode would read a result without a tangent as one that does not change."""
    for name, t in named.items():
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("%s has a tangent; there is no forward-mode derivative" % name)


def _no_gradient(name: str, v) -> None:
    if getattr(v, "requires_grad", False):
        raise ValueError("%s has no gradient; detach it or call under torch.no_grad()" % name)


def _written(t: torch.Tensor) -> None:
    """A kernel has written into ``t``: a graph that saved it before must not use it."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _tokens(t, what: str, n: int, dev: int) -> int:
    """[n] whole numbers, int32 or int64, contiguous: their bits."""
    _on(t, what, dev)
    bits = _BITS.get(t.dtype)
    if bits is None or t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        raise ValueError("%s must be a contiguous int32 or int64 tensor [%d]" % (what, n))
    return bits


# --------------------------------------------------------------------------- history

class TokenHistory:
    """What each of ``n_rows`` rows has seen: ``seen`` int32 [n_rows, words] (a bit per token) and, unless ``counts`` is
    false, ``counts`` int32 [n_rows, width] (how often the row generated each token).  Both are ordinary tensors; rows may
    be copied, reordered or cleared with torch's own operations."""

    def __init__(self, n_rows: int, width: int, *, device=None, counts: bool = True):
        n_rows, width = int(n_rows), int(width)
        if n_rows < 0 or width < 1:
            raise ValueError("a history has 0 or more rows and 1 or more tokens")
        device = torch.device("cuda" if device is None else device if not isinstance(device, int) else "cuda:%d" % device)
        if device.type != "cuda":
            raise RuntimeError("a history is kept in CUDA tensors; there is no CPU path")
        self.n_rows, self.width = n_rows, width
        self.counts: Optional[torch.Tensor] = None
        if counts:
            self.seen, self.counts = self._cleared(n_rows, width, device)
        else:
            self.seen = torch.zeros((n_rows, _words(width)), dtype=torch.int32, device=device)

    @staticmethod
    def _cleared(n_rows: int, width: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
        """(seen, counts) in one array, cleared at once: the words, then the counts."""
        words = _words(width)
        split = (n_rows * words + 3) // 4 * 4
        both = torch.zeros(split + n_rows * width, dtype=torch.int32, device=device)
        # (.data: views of one array would share its version, and a write to the counts would count as one to the words)
        return both.as_strided((n_rows, words), (words, 1)), both.as_strided((n_rows, width), (width, 1), split).data

    @property
    def device(self) -> torch.device:
        return self.seen.device

    def clear(self) -> None:
        self.seen.zero_()
        if self.counts is not None:
            self.counts.zero_()

    def _check(self) -> int:
        """The number of its GPU."""
        seen, counts = self.seen, self.counts
        dev = _device_of(seen, "seen")
        if seen.dtype is not torch.int32 or seen.shape != (self.n_rows, _words(self.width)) or not seen.is_contiguous():
            raise ValueError("seen must be a contiguous int32 tensor [%d, %d]" % (self.n_rows, _words(self.width)))
        if counts is not None:
            _on(counts, "counts", dev)
            if counts.dtype is not torch.int32 or counts.shape != (self.n_rows, self.width) or not counts.is_contiguous():
                raise ValueError("counts must be a contiguous int32 tensor [%d, %d]" % (self.n_rows, self.width))
        return dev

    def add(self, ids, lengths=None, *, offsets=None, pad_left: bool = False, generated: bool = False, rows=None) -> None:
        """Enter the ids of whole rows.  ``ids`` int32 or int64: padded rows [n, T] with their ``lengths`` (int32 [n]; all
        columns without) and the padding on the right unless ``pad_left``, or flat ids with ``offsets`` (int64 [n + 1]): the
        encoder's two layouts.  ``generated``: the row produced them itself, so they are counted too.  ``rows`` [n]: the
        history row of each (0, 1, ... by default).  Ids outside the vocabulary are no tokens."""
        dev = self._check()
        _on(ids, "ids", dev)
        if ids.dtype not in _BITS:
            raise ValueError("ids must be int32 or int64")
        h = _cabi.History()
        if offsets is not None:
            if lengths is not None or pad_left:
                raise ValueError("flat ids have offsets, padded rows lengths and a side")
            _on(offsets, "offsets", dev)
            if ids.dim() != 1 or not ids.is_contiguous():
                raise ValueError("flat ids must be a contiguous tensor [total]")
            if offsets.dtype is not torch.int64 or offsets.dim() != 1 or offsets.shape[0] < 1 or not offsets.is_contiguous():
                raise ValueError("offsets must be a contiguous int64 tensor [n + 1]")
            n = offsets.shape[0] - 1
            h.offsets, h.total = (offsets.data_ptr() or _nowhere(offsets, "offsets")), ids.shape[0]
        else:
            if ids.dim() != 2 or (ids.shape[1] > 1 and ids.stride(1) != 1):
                raise ValueError("padded ids must be a tensor [n, T] whose rows are contiguous")
            n, h.columns = ids.shape
            h.id_stride = ids.stride(0)
            if lengths is not None:
                _on(lengths, "lengths", dev)
                if lengths.dtype is not torch.int32 or lengths.shape != (n,) or not lengths.is_contiguous():
                    raise ValueError("lengths must be a contiguous int32 tensor [%d]" % n)
                h.lengths = lengths.data_ptr() or _nowhere(lengths, "lengths")
            h.pad_left = 1 if pad_left else 0
        self._enter(h, ids, n, rows, generated, dev)

    def append(self, tokens, rows=None) -> None:
        """Enter one generated token per row: ``tokens`` [n] int32 or int64; ``rows`` as in ``add``.  A token outside the
        vocabulary (-1, say) is none."""
        dev = self._check()
        n = tokens.shape[0] if isinstance(tokens, torch.Tensor) and tokens.dim() == 1 else 0
        _tokens(tokens, "tokens", n, dev)
        h = _cabi.History()
        h.columns = h.id_stride = 1
        self._enter(h, tokens, n, rows, True, dev)

    def _enter(self, h, ids, n: int, rows, generated: bool, dev: int) -> None:
        if rows is not None:
            h.rows_bits = _tokens(rows, "rows", n, dev)
            h.rows = rows.data_ptr() or _nowhere(rows, "rows")
        elif n != self.n_rows:
            raise ValueError("the history has %d rows, the call %d" % (self.n_rows, n))
        h.seen, h.history_rows, h.width = (self.seen.data_ptr() or _nowhere(self.seen, "seen")), self.n_rows, self.width
        if self.counts is not None:
            h.counts = self.counts.data_ptr() or _nowhere(self.counts, "counts")
        h.ids, h.id_bits, h.n_rows = (ids.data_ptr() or _nowhere(ids, "ids")), _BITS[ids.dtype], n
        _call(_cabi.lib().dnatok_history_add, dev, h, 1 if generated else 0)
        _written(self.seen)
        if generated and self.counts is not None:
            _written(self.counts)


# --------------------------------------------------------------------------- grammar

class Grammar:
    """The masks of an ``Automaton`` for a vocabulary.  ``tokens``: the bytes of every token, as a list (``None`` or empty:
    a token that never follows, such as the specials) or as a pair (flat uint8, int64 offsets); ``end_id``: the token that
    ends a row, allowed in accepting states; ``width``: columns of the masks where the logits have more than the
    vocabulary.  States are int32: 0 and up the automaton's, ``DEAD`` (-1), ``FINISHED`` (-2)."""

    def __init__(self, automaton: Automaton, tokens: Union[Sequence[Optional[bytes]], Tuple[np.ndarray, np.ndarray]], *,
                 end_id: Optional[int] = None, width: Optional[int] = None):
        if isinstance(tokens, tuple) and len(tokens) == 2 and isinstance(tokens[0], np.ndarray):
            flat = whole_numbers(tokens[0], np.uint8, "token bytes").reshape(-1)
            offsets = whole_numbers(tokens[1], np.int64, "token offsets")
        else:
            tokens = list(tokens)
            for v, t in enumerate(tokens):
                if isinstance(t, (int, np.generic)):               # (bytes(5) would be five zeros)
                    raise TypeError("token %d is a number; a token is its bytes, or None" % v)
            tokens = [bytes(t or b"") for t in tokens]
            flat = np.frombuffer(b"".join(tokens), dtype=np.uint8)
            offsets = np.zeros(len(tokens) + 1, dtype=np.int64)
            np.cumsum([len(t) for t in tokens], out=offsets[1:])
        if offsets.ndim != 1 or offsets.shape[0] < 2 or offsets[0] != 0 or offsets[-1] != flat.shape[0] or np.any(np.diff(offsets) < 0):
            raise ValueError("token offsets must start at 0, be non-decreasing and end at len(bytes)")
        n = offsets.shape[0] - 1
        self.width = n if width is None else int(width)
        if self.width < n:
            raise ValueError("width %d is smaller than the vocabulary (%d tokens)" % (self.width, n))
        if self.width > n:
            offsets = np.concatenate([offsets, np.full(self.width - n, offsets[-1], dtype=np.int64)])
        if end_id is not None and not 0 <= int(end_id) < n:
            raise ValueError("end_id %d is outside the vocabulary" % int(end_id))
        self.automaton, self.end_id = automaton, None if end_id is None else int(end_id)
        a, h = automaton, ctypes.c_void_p()
        _cabi.check(_cabi.lib().dnatok_create_grammar(
            _cabi.np_ptr(a.next_state), a.next_state.shape[0], a.next_state.shape[1], _cabi.np_ptr(a.accepting),
            _cabi.np_ptr(a.byte_class), _cabi.np_ptr(flat) if flat.size else None, _cabi.np_ptr(offsets), self.width,
            -1 if self.end_id is None else self.end_id, ctypes.byref(h)))
        self.ptr = h

    def close(self) -> None:
        if getattr(self, "ptr", None):
            _cabi.lib().dnatok_destroy_grammar(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __copy__(self) -> "Grammar":                 # (a grammar does not change, and owns what it would share)
        return self

    def __deepcopy__(self, memo) -> "Grammar":
        return self

    def start(self, n_rows: int, device=None) -> torch.Tensor:
        """The first state of ``n_rows`` rows."""
        return torch.full((int(n_rows),), self.automaton.start, dtype=torch.int32,
                          device=torch.device("cuda" if device is None else device))

    @staticmethod
    def _states(states) -> Tuple[int, int, int]:
        """(how many, the number of their GPU, their address)."""
        dev = _device_of(states, "states")
        if states.dtype is not torch.int32 or states.dim() != 1 or (states.shape[0] > 1 and states.stride(0) != 1):
            raise ValueError("states must be a contiguous int32 tensor [n]")
        return states.shape[0], dev, (states.data_ptr() or _nowhere(states, "states"))

    def _mask(self, states, n: int, dev: int, out):
        words = _words(self.width)
        if out is None:
            return states.new_empty((n, words))
        _on(out, "the mask", dev)
        if out.dtype is not torch.int32 or out.shape != (n, words) or not out.is_contiguous():
            raise ValueError("the mask must be a contiguous int32 tensor [%d, %d]" % (n, words))
        return out

    @staticmethod
    def _new_states(states, n: int, dev: int, out):
        if out is None:
            return states.new_empty((n,))
        _on(out, "out", dev)
        if out.dtype is not torch.int32 or out.shape != (n,) or not out.is_contiguous():
            raise ValueError("out must be a contiguous int32 tensor [%d]" % n)
        return out

    def allowed(self, states, *, out=None) -> torch.Tensor:
        """int32 [n, words]: the tokens that may follow in each state."""
        n, dev, at = self._states(states)
        mask = self._mask(states, n, dev, out)
        _call(_cabi.lib().dnatok_grammar_allowed, dev, self.ptr, at, n, (mask.data_ptr() or _nowhere(mask, "the mask")))
        if out is not None:
            _written(out)
        return mask

    def advance(self, states, tokens, *, out=None) -> torch.Tensor:
        """int32 [n]: the states after ``tokens`` [n] (int32 or int64); a token outside the vocabulary (-1, say) leaves its
        row as it was.  ``out`` may be ``states``, but may not overlap them in another way."""
        n, dev, at = self._states(states)
        bits = _tokens(tokens, "tokens", n, dev)
        new = self._new_states(states, n, dev, out)
        _call(_cabi.lib().dnatok_grammar_step, dev, self.ptr, at, (tokens.data_ptr() or _nowhere(tokens, "tokens")), bits, n,
              (new.data_ptr() or _nowhere(new, "out")), None)
        if out is not None:
            _written(out)
        return new

    def step(self, states, tokens, *, out=None, out_allowed=None) -> Tuple[torch.Tensor, torch.Tensor]:
        """``advance`` and the masks of the new states in one call: (states, allowed).  ``out`` may not overlap ``states``
        or ``tokens``, nor ``out_allowed`` any of them."""
        n, dev, at = self._states(states)
        bits = _tokens(tokens, "tokens", n, dev)
        new = self._new_states(states, n, dev, out)
        mask = self._mask(states, n, dev, out_allowed)
        _call(_cabi.lib().dnatok_grammar_step, dev, self.ptr, at, (tokens.data_ptr() or _nowhere(tokens, "tokens")), bits, n,
              (new.data_ptr() or _nowhere(new, "out")), (mask.data_ptr() or _nowhere(mask, "the mask")))
        if out is not None:
            _written(out)
        if out_allowed is not None:
            _written(out_allowed)
        return new, mask


# --------------------------------------------------------------------------- logits

def _rows_of(t: torch.Tensor, what: str) -> Tuple[int, int, int]:
    """(rows, columns, elements from row to row)."""
    shape, strides = t.shape, t.stride()
    if len(shape) != 2 or shape[1] < 1 or (shape[1] > 1 and strides[1] != 1):
        raise ValueError("%s must be a tensor [n, width] whose rows are contiguous" % what)
    return shape[0], shape[1], strides[0]


def _penalty(name: str, v, n: int, dev: int):
    """(number, address of one value a row, whether it is a penalty)."""
    neutral = 1.0 if name == "repetition" else 0.0
    if isinstance(v, torch.Tensor):
        _on(v, name, dev)
        if v.dtype is not torch.float32 or v.shape != (n,) or (n > 1 and v.stride(0) != 1):
            raise ValueError("%s must be a number or a contiguous float32 tensor [%d]" % (name, n))
        return neutral, (v.data_ptr() or _nowhere(v, name)), True
    v = float(v)
    if neutral:
        if not _LEAST <= v <= _MOST:
            raise ValueError("repetition must be positive and finite (2^-126 to 2^126)")
    elif not abs(v) <= 3.4028234e38:
        raise ValueError("%s must be a finite float32 number" % name)
    return v, None, v != neutral


def _shared(shape) -> bool:
    """Whether an array of one row, or without rows, stands for all of them."""
    return len(shape) == 1 or shape[0] == 1


def _row_array(t, what: str, dtype, n: int, columns: int, dev: int) -> Tuple[int, int]:
    """(address, elements from row to row) of an array [columns], [1, columns] or [n, columns]; 0 elements where one row stands
    for all."""
    _on(t, what, dev)
    shape, strides = t.shape, t.stride()
    if t.dtype is not dtype or len(shape) not in (1, 2) or shape[-1] != columns or (columns > 1 and strides[-1] != 1) \
            or (len(shape) == 2 and shape[0] != 1 and shape[0] != n):
        raise ValueError("%s must be a %s tensor [%d, %d] or [%d] whose rows are contiguous" % (what, str(dtype)[6:], n, columns, columns))
    if len(shape) == 1 or shape[0] == 1:
        return (t.data_ptr() or _nowhere(t, what)), 0
    if strides[0] < columns:
        raise ValueError("rows of %s overlap" % what)
    return (t.data_ptr() or _nowhere(t, what)), strides[0]


def _arguments(logits, history, rows, repetition, frequency, presence, bias, allowed):
    """(the C arguments, the number of the GPU)."""
    dev = _device_of(logits, "logits")
    n, width, stride = _rows_of(logits, "logits")
    dtype = _TYPES.get(logits.dtype)
    if dtype is None:
        raise ValueError("logits must be float32, float16 or bfloat16")
    a = _cabi.Logits()
    a.logits, a.dtype, a.n_rows, a.width, a.stride = (logits.data_ptr() or _nowhere(logits, "logits")), dtype, n, width, stride
    a.repetition, a.d_repetition, once = _penalty("repetition", repetition, n, dev)
    a.frequency, a.d_frequency, often = _penalty("frequency", frequency, n, dev)
    a.presence, a.d_presence, also = _penalty("presence", presence, n, dev)
    often = often or also
    if history is None:
        if once or often:
            raise ValueError("penalties need a history")
        if rows is not None:
            raise ValueError("rows need a history")
    else:
        if history.width != width:
            raise ValueError("the history has %d tokens, the logits %d" % (history.width, width))
        if history._check() != dev:
            raise ValueError("the history is on %s, the logits on %s" % (history.device, logits.device))
        if rows is not None:
            a.rows_bits = _tokens(rows, "rows", n, dev)
            a.rows = rows.data_ptr() or _nowhere(rows, "rows")
        elif history.n_rows != n:
            raise ValueError("the history has %d rows, the logits %d" % (history.n_rows, n))
        if often and history.counts is None:
            raise ValueError("frequency and presence need a history that keeps counts")
        if once or often:
            a.seen, a.history_rows = (history.seen.data_ptr() or _nowhere(history.seen, "seen")), history.n_rows
        if often:
            a.counts = history.counts.data_ptr() or _nowhere(history.counts, "counts")
    if bias is not None:
        a.bias, a.bias_stride = _row_array(bias, "bias", torch.float32, n, width, dev)
    if allowed is not None:
        a.allowed, a.allowed_stride = _row_array(allowed, "allowed", torch.int32, n, _words(width), dev)
    return a, dev


def _output(logits, out, out_dtype):
    dtype = out_dtype or (logits.dtype if out is None else out.dtype)
    if dtype is not logits.dtype and dtype is not torch.float32:
        raise ValueError("the output has the logits' type or is float32")
    if out is None:
        if dtype is logits.dtype and logits.is_contiguous():
            return torch.empty_like(logits)                        # (the quickest of the two calls)
        return logits.new_empty(logits.shape, dtype=dtype)
    _on(out, "out", logits.get_device())
    _rows_of(out, "out")
    if out.dtype is not dtype or out.shape != logits.shape:
        raise ValueError("out must be a %s tensor %r" % (dtype, tuple(logits.shape)))
    return out


def _forward(a, dev: int, out):
    _call(_cabi.lib().dnatok_process_logits, dev, a, (out.data_ptr() or _nowhere(out, "out")), _TYPES[out.dtype], out.stride(0))
    return out


def _backward(a, dev: int, dtype, grad, bias_shape, want_logits: bool):
    """(gradient of logits of ``dtype``, if wanted, gradient of a bias of ``bias_shape``, if that is not None)."""
    if grad.shape[1] > 1 and grad.stride(1) != 1:
        grad = grad.contiguous()
    n, width = grad.shape
    d_grad = grad.data_ptr() or _nowhere(grad, "grad")
    L = _cabi.lib()
    dx = grad.new_empty((n, width), dtype=dtype) if want_logits else None
    db, scratch, need = None, None, 0
    if bias_shape is not None:
        db = grad.new_empty(bias_shape, dtype=torch.float32)
        a.bias_stride = 0 if _shared(bias_shape) else width
        if _shared(bias_shape):
            need = L.dnatok_logits_scratch_bytes(n, width)
            if need:
                scratch = grad.new_empty((need,), dtype=torch.uint8)
    _call(L.dnatok_process_logits_backward, dev, a, d_grad, _TYPES[grad.dtype], grad.stride(0),
          dx.data_ptr() if dx is not None else None, width, db.data_ptr() if db is not None else None,
          scratch.data_ptr() if need else None, need)
    return dx, db


class _Process(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, history, rows, repetition, frequency, presence, allowed, out_dtype):
        a, dev = _arguments(logits, history, rows, repetition, frequency, presence, bias, allowed)
        out = _forward(a, dev, _output(logits, None, out_dtype))
        ctx.dtype = logits.dtype
        ctx.bias_shape = None if bias is None else bias.shape     # (its values have no part in the gradients)
        ctx.number = 1.0 if isinstance(repetition, torch.Tensor) else float(repetition)
        # The logits' signs, and the history, matter to the gradient of penalised logits alone.
        if history is not None and ctx.needs_input_grad[0] and (isinstance(repetition, torch.Tensor) or ctx.number != 1.0):
            ctx.save_for_backward(allowed, logits, history.seen, rows, repetition if isinstance(repetition, torch.Tensor) else None)
        else:
            ctx.save_for_backward(allowed, None, None, None, None)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        # (the tensors may have been stored elsewhere in the meantime: nothing but them holds for their addresses)
        allowed, logits, seen, rows, repetition = ctx.saved_tensors
        a = _cabi.Logits()
        a.dtype, a.repetition = _TYPES[ctx.dtype], ctx.number
        a.n_rows, a.width = grad.shape
        if logits is None:
            a.logits = grad.data_ptr() or _nowhere(grad, "grad")          # not read: no token counts as seen
        else:
            a.logits, a.stride = (logits.data_ptr() or _nowhere(logits, "logits")), logits.stride(0)
            a.seen, a.history_rows = (seen.data_ptr() or _nowhere(seen, "seen")), seen.shape[0]
            if rows is not None:
                a.rows, a.rows_bits = (rows.data_ptr() or _nowhere(rows, "rows")), _BITS[rows.dtype]
            if repetition is not None:
                a.d_repetition = repetition.data_ptr() or _nowhere(repetition, "repetition")
        if allowed is not None:
            a.allowed, a.allowed_stride = (allowed.data_ptr() or _nowhere(allowed, "allowed")), 0 if _shared(allowed.shape) else allowed.stride(0)
        dx, db = _backward(a, grad.get_device(), ctx.dtype, grad, ctx.bias_shape if ctx.needs_input_grad[1] else None, ctx.needs_input_grad[0])
        return dx, db, None, None, None, None, None, None, None


def process_logits(logits, *, history: Optional[TokenHistory] = None, rows=None, repetition: Number = 1.0,
                   frequency: Number = 0.0, presence: Number = 0.0, bias=None, allowed=None, out=None, out_dtype=None):
    """``logits`` [n, width] (float32, float16 or bfloat16; a view such as ``model_output[:, -1]`` is fine) after penalties,
    bias and mask, as a new tensor of its type or of ``out_dtype`` float32, or in ``out``, which may be ``logits`` but may
    not overlap them, or another argument, in any other way.

    * A token the row has seen: ``x > 0 ? x / repetition : x * repetition`` (by the rounded ``1 / repetition``); one it
      generated ``c > 0`` times, then ``- frequency * c - presence``.  Each is a number, or a float32 tensor [n] (repetition
      from 2^-126 to 2^126 there too).  ``rows`` [n] names each row's history row (a row outside the history has none); two
      rows may share one.
    * ``bias`` float32 [width] or [n, width] is added.
    * ``allowed`` int32 [n, words] or [words]: tokens whose bit is 0 become ``-inf`` whatever their logits hold, NaN
      included.  A row without an allowed token is ``-inf`` throughout.

    All of it is computed in 32 bits and then rounded to the output's type.  Differentiable in ``logits`` and ``bias`` (a penalty
    that requires a gradient is refused, and so is forward mode); the mask and, with a repetition penalty, the logits and the
    history must then stay as they are until the backward pass (autograd refuses it otherwise)."""
    if getattr(forward_ad, "_current_level", 0) >= 0:              # a level is open (to ask every tensor takes 0.5 us apiece)
        _no_tangents(logits=logits, repetition=repetition, frequency=frequency, presence=presence, bias=bias, out=out)
    differentiable = False
    if torch.is_grad_enabled():                      # (asked here: inside of an autograd function it is not)
        if repetition.__class__ is not float:
            _no_gradient("repetition", repetition)
        if frequency.__class__ is not float:
            _no_gradient("frequency", frequency)
        if presence.__class__ is not float:
            _no_gradient("presence", presence)
        if out is not None:
            _no_gradient("out=", out)
        differentiable = getattr(logits, "requires_grad", False) or (bias is not None and getattr(bias, "requires_grad", False))
    if differentiable:
        if out is not None:
            raise ValueError("out= has no gradient; leave it out or call under torch.no_grad()")
        return _Process.apply(logits, bias, history, rows, repetition, frequency, presence, allowed, out_dtype)
    a, dev = _arguments(logits, history, rows, repetition, frequency, presence, bias, allowed)
    result = _forward(a, dev, _output(logits, out, out_dtype))
    if out is not None:
        _written(out)
    return result


def process_logits_backward(grad, logits, *, history: Optional[TokenHistory] = None, rows=None, repetition: Number = 1.0,
                            frequency: Number = 0.0, presence: Number = 0.0, bias=None, allowed=None):
    """(gradient of ``logits``, gradient of ``bias`` or None) for ``grad``, the gradient of ``process_logits`` called with the
    same arguments; without autograd."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _no_tangents(grad=grad, logits=logits, repetition=repetition, frequency=frequency, presence=presence, bias=bias)
    with torch.no_grad():
        a, dev = _arguments(logits, history, rows, repetition, frequency, presence, bias, allowed)
        _on(grad, "grad", dev)
        if grad.dim() != 2 or grad.shape != logits.shape or grad.dtype not in (logits.dtype, torch.float32):
            raise ValueError("grad must be a tensor %r of the logits' type or float32" % (tuple(logits.shape),))
        return _backward(a, dev, logits.dtype, grad, None if bias is None else bias.shape, True)
