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
nothing waits for it.  Sets of tokens are int32 words: bit ``v % 32`` of word ``v // 32`` stands for token ``v``.

The calls can be captured into a CUDA graph (use a ``Grammar`` on the device once before).  To capture a gradient while an
eager graph over the same leaf tensors is alive, call ``process_logits_backward``, which needs no autograd graph:
autograd's own accumulation into a leaf waits on the stream of the older graph, which a capture does not allow.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _cabi
from .automaton import Automaton

DEAD, FINISHED = _cabi.STATE_DEAD, _cabi.STATE_FINISHED
_TYPES = {torch.float32: _cabi.F32, torch.float16: _cabi.F16, torch.bfloat16: _cabi.BF16}
_BITS = {torch.int32: 32, torch.int64: 64}

Number = Union[float, int, torch.Tensor]


def _words(width: int) -> int:
    return (width + 31) // 32


def _need_cuda(t, what: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor" % what)
    if t.device.type != "cuda":
        raise RuntimeError("%s must be a CUDA tensor; there is no CPU path" % what)


def _same_device(t, what: str, device) -> None:
    _need_cuda(t, what)
    if t.device != device:
        raise ValueError("%s is on %s, the call on %s" % (what, t.device, device))


def _written(t: torch.Tensor) -> None:
    """A kernel has written into ``t``: a graph that saved it before must not use it."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


class _On:
    """The current stream of a device, with the device current."""
    __slots__ = ("guard", "stream")

    def __init__(self, device):
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)
        self.stream = torch.cuda.current_stream(device).cuda_stream

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return self.stream

    def __exit__(self, *a):
        if self.guard is not None:
            self.guard.__exit__(*a)


def _tokens(t, what: str, n: int, device) -> torch.Tensor:
    """[n] whole numbers, int32 or int64, contiguous."""
    _same_device(t, what, device)
    if t.dtype not in _BITS or tuple(t.shape) != (n,) or (n > 1 and t.stride(0) != 1):
        raise ValueError("%s must be a contiguous int32 or int64 tensor [%d]" % (what, n))
    return t


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
        words = _words(width)
        self.n_rows, self.width = n_rows, width
        if counts:                                   # one array, cleared at once: the words, then the counts
            split = (n_rows * words + 3) // 4 * 4
            both = torch.zeros(split + n_rows * width, dtype=torch.int32, device=device)
            self.seen = both[:n_rows * words].view(n_rows, words)
            self.counts = both[split:].view(n_rows, width)
        else:
            self.seen = torch.zeros((n_rows, words), dtype=torch.int32, device=device)
            self.counts: Optional[torch.Tensor] = None
        self.device = self.seen.device

    def clear(self) -> None:
        self.seen.zero_()
        if self.counts is not None:
            self.counts.zero_()

    def _check(self) -> None:
        for t, what, shape in ((self.seen, "seen", (self.n_rows, _words(self.width))), (self.counts, "counts", (self.n_rows, self.width))):
            if t is None:
                continue
            _same_device(t, what, self.device)
            if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError("%s must be a contiguous int32 tensor %r" % (what, shape))

    def add(self, ids, lengths=None, *, offsets=None, pad_left: bool = False, generated: bool = False, rows=None) -> None:
        """Enter the ids of whole rows.  ``ids`` int32 or int64: padded rows [n, T] with their ``lengths`` (int32 [n]; all
        columns without) and the padding on the right unless ``pad_left``, or flat ids with ``offsets`` (int64 [n + 1]): the
        encoder's two layouts.  ``generated``: the row produced them itself, so they are counted too.  ``rows`` [n]: the
        history row of each (0, 1, ... by default).  Ids outside the vocabulary are no tokens."""
        self._check()
        _same_device(ids, "ids", self.device)
        if ids.dtype not in _BITS:
            raise ValueError("ids must be int32 or int64")
        h = _cabi.History()
        if offsets is not None:
            if lengths is not None or pad_left:
                raise ValueError("flat ids have offsets, padded rows lengths and a side")
            _same_device(offsets, "offsets", self.device)
            if ids.dim() != 1 or not ids.is_contiguous():
                raise ValueError("flat ids must be a contiguous tensor [total]")
            if offsets.dtype != torch.int64 or offsets.dim() != 1 or offsets.shape[0] < 1 or not offsets.is_contiguous():
                raise ValueError("offsets must be a contiguous int64 tensor [n + 1]")
            n = offsets.shape[0] - 1
            h.offsets, h.total = offsets.data_ptr(), ids.shape[0]
        else:
            if ids.dim() != 2 or (ids.shape[1] > 1 and ids.stride(1) != 1):
                raise ValueError("padded ids must be a tensor [n, T] whose rows are contiguous")
            n = ids.shape[0]
            h.columns, h.id_stride = ids.shape[1], ids.stride(0)
            if lengths is not None:
                _same_device(lengths, "lengths", self.device)
                if lengths.dtype != torch.int32 or tuple(lengths.shape) != (n,) or not lengths.is_contiguous():
                    raise ValueError("lengths must be a contiguous int32 tensor [%d]" % n)
                h.lengths = lengths.data_ptr()
            h.pad_left = 1 if pad_left else 0
        self._enter(h, ids, n, rows, generated)

    def append(self, tokens, rows=None) -> None:
        """Enter one generated token per row: ``tokens`` [n] int32 or int64; ``rows`` as in ``add``.  A token outside the
        vocabulary (-1, say) is none."""
        self._check()
        n = tokens.shape[0] if isinstance(tokens, torch.Tensor) and tokens.dim() == 1 else 0
        _tokens(tokens, "tokens", n, self.device)
        h = _cabi.History()
        h.columns = h.id_stride = 1
        self._enter(h, tokens, n, rows, True)

    def _enter(self, h, ids, n: int, rows, generated: bool) -> None:
        if rows is not None:
            h.rows, h.rows_bits = _tokens(rows, "rows", n, self.device).data_ptr(), _BITS[rows.dtype]
        elif n != self.n_rows:
            raise ValueError("the history has %d rows, the call %d" % (self.n_rows, n))
        h.seen, h.history_rows, h.width = self.seen.data_ptr(), self.n_rows, self.width
        if self.counts is not None:
            h.counts = self.counts.data_ptr()
        h.ids, h.id_bits, h.n_rows = ids.data_ptr(), _BITS[ids.dtype], n
        with _On(self.device) as stream:
            _cabi.check(_cabi.lib().dnatok_history_add(ctypes.byref(h), 1 if generated else 0, stream))
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
            flat = np.ascontiguousarray(tokens[0], dtype=np.uint8).reshape(-1)
            offsets = np.ascontiguousarray(tokens[1], dtype=np.int64)
        else:
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

    def start(self, n_rows: int, device=None) -> torch.Tensor:
        """The first state of ``n_rows`` rows."""
        return torch.full((int(n_rows),), self.automaton.start, dtype=torch.int32,
                          device=torch.device("cuda" if device is None else device))

    @staticmethod
    def _states(states) -> int:
        _need_cuda(states, "states")
        if states.dtype != torch.int32 or states.dim() != 1 or (states.shape[0] > 1 and states.stride(0) != 1):
            raise ValueError("states must be a contiguous int32 tensor [n]")
        return states.shape[0]

    def _mask(self, n: int, device, out):
        shape = (n, _words(self.width))
        if out is None:
            return torch.empty(shape, dtype=torch.int32, device=device)
        _same_device(out, "the mask", device)
        if out.dtype != torch.int32 or tuple(out.shape) != shape or not out.is_contiguous():
            raise ValueError("the mask must be a contiguous int32 tensor %r" % (shape,))
        return out

    def allowed(self, states, *, out=None) -> torch.Tensor:
        """int32 [n, words]: the tokens that may follow in each state."""
        n = self._states(states)
        mask = self._mask(n, states.device, out)
        with _On(states.device) as stream:
            _cabi.check(_cabi.lib().dnatok_grammar_allowed(self.ptr, states.data_ptr(), n, mask.data_ptr(), stream))
        if out is not None:
            _written(out)
        return mask

    def advance(self, states, tokens, *, out=None) -> torch.Tensor:
        """int32 [n]: the states after ``tokens`` [n] (int32 or int64); a token outside the vocabulary (-1, say) leaves its
        row as it was.  ``out`` may be ``states``."""
        n = self._states(states)
        _tokens(tokens, "tokens", n, states.device)
        new = self._new_states(n, states.device, out)
        with _On(states.device) as stream:
            _cabi.check(_cabi.lib().dnatok_grammar_step(self.ptr, states.data_ptr(), tokens.data_ptr(), _BITS[tokens.dtype], n,
                                                        new.data_ptr(), None, stream))
        if out is not None:
            _written(out)
        return new

    def step(self, states, tokens, *, out=None, out_allowed=None) -> Tuple[torch.Tensor, torch.Tensor]:
        """``advance`` and the masks of the new states in one call: (states, allowed).  ``out`` may not be ``states``."""
        n = self._states(states)
        _tokens(tokens, "tokens", n, states.device)
        new = self._new_states(n, states.device, out)
        mask = self._mask(n, states.device, out_allowed)
        with _On(states.device) as stream:
            _cabi.check(_cabi.lib().dnatok_grammar_step(self.ptr, states.data_ptr(), tokens.data_ptr(), _BITS[tokens.dtype], n,
                                                        new.data_ptr(), mask.data_ptr(), stream))
        if out is not None:
            _written(out)
        if out_allowed is not None:
            _written(out_allowed)
        return new, mask

    @staticmethod
    def _new_states(n: int, device, out):
        if out is None:
            return torch.empty(n, dtype=torch.int32, device=device)
        _same_device(out, "out", device)
        if out.dtype != torch.int32 or tuple(out.shape) != (n,) or not out.is_contiguous():
            raise ValueError("out must be a contiguous int32 tensor [%d]" % n)
        return out


# --------------------------------------------------------------------------- logits

def _rows_of(t: torch.Tensor, what: str) -> None:
    if t.dim() != 2 or t.shape[1] < 1 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError("%s must be a tensor [n, width] whose rows are contiguous" % what)


def _penalty(a, name: str, v, n: int, device, keep: list) -> bool:
    """Enters one penalty; whether it is one."""
    neutral = 1.0 if name == "repetition" else 0.0
    if isinstance(v, torch.Tensor):
        _same_device(v, name, device)
        if v.dtype != torch.float32 or tuple(v.shape) != (n,) or (n > 1 and v.stride(0) != 1):
            raise ValueError("%s must be a number or a contiguous float32 tensor [%d]" % (name, n))
        if v.requires_grad and torch.is_grad_enabled():
            raise ValueError("%s has no gradient" % name)
        setattr(a, "d_" + name, v.data_ptr())
        setattr(a, name, neutral)
        keep.append(v)
        return True
    v = float(v)
    if name == "repetition" and not 2.0 ** -126 <= v <= 2.0 ** 126:
        raise ValueError("repetition must be positive and finite (2^-126 to 2^126)")
    if v != v or v in (float("inf"), -float("inf")):
        raise ValueError("%s must be finite" % name)
    setattr(a, name, v)
    return v != neutral


def _arguments(logits, history, rows, repetition, frequency, presence, bias, allowed):
    """(the C arguments, tensors whose addresses they hold)."""
    _need_cuda(logits, "logits")
    _rows_of(logits, "logits")
    if logits.dtype not in _TYPES:
        raise ValueError("logits must be float32, float16 or bfloat16")
    n, width = logits.shape
    device = logits.device
    a, keep = _cabi.Logits(), [logits]
    a.logits, a.dtype, a.n_rows, a.width, a.stride = logits.data_ptr(), _TYPES[logits.dtype], n, width, logits.stride(0)
    once = _penalty(a, "repetition", repetition, n, device, keep)
    often = _penalty(a, "frequency", frequency, n, device, keep) | _penalty(a, "presence", presence, n, device, keep)
    if history is None:
        if once or often:
            raise ValueError("penalties need a history")
        if rows is not None:
            raise ValueError("rows need a history")
    else:
        if history.width != width:
            raise ValueError("the history has %d tokens, the logits %d" % (history.width, width))
        history._check()
        if history.device != device:
            raise ValueError("the history is on %s, the logits on %s" % (history.device, device))
        if rows is not None:
            a.rows, a.rows_bits = _tokens(rows, "rows", n, device).data_ptr(), _BITS[rows.dtype]
            keep.append(rows)
        elif history.n_rows != n:
            raise ValueError("the history has %d rows, the logits %d" % (history.n_rows, n))
        if often and history.counts is None:
            raise ValueError("frequency and presence need a history that keeps counts")
        if once or often:
            a.seen, a.history_rows = history.seen.data_ptr(), history.n_rows
            keep.append(history.seen)
        if often:
            a.counts = history.counts.data_ptr()
            keep.append(history.counts)
    if bias is not None:
        _same_device(bias, "bias", device)
        if bias.dtype != torch.float32 or tuple(bias.shape) not in ((width,), (1, width), (n, width)) or (width > 1 and bias.stride(-1) != 1):
            raise ValueError("bias must be a float32 tensor [%d] or [%d, %d] whose rows are contiguous" % (width, n, width))
        shared = bias.dim() == 1 or bias.shape[0] == 1
        if not shared and bias.stride(0) < width:
            raise ValueError("rows of the bias overlap")
        a.bias, a.bias_stride = bias.data_ptr(), 0 if shared else bias.stride(0)
        keep.append(bias)
    if allowed is not None:
        words = _words(width)
        _same_device(allowed, "allowed", device)
        if allowed.dtype != torch.int32 or tuple(allowed.shape) not in ((words,), (1, words), (n, words)) or (words > 1 and allowed.stride(-1) != 1):
            raise ValueError("allowed must be an int32 tensor [%d, %d] or [%d] whose rows are contiguous" % (n, words, words))
        shared = allowed.dim() == 1 or allowed.shape[0] == 1
        if not shared and allowed.stride(0) < words:
            raise ValueError("rows of the mask overlap")
        a.allowed, a.allowed_stride = allowed.data_ptr(), 0 if shared else allowed.stride(0)
        keep.append(allowed)
    return a, keep


def _output(logits, out, out_dtype):
    dtype = out_dtype or (logits.dtype if out is None else out.dtype)
    if dtype not in (logits.dtype, torch.float32):
        raise ValueError("the output has the logits' type or is float32")
    if out is None:
        return torch.empty(logits.shape, dtype=dtype, device=logits.device)
    _same_device(out, "out", logits.device)
    _rows_of(out, "out")
    if out.dtype != dtype or out.shape != logits.shape:
        raise ValueError("out must be a %s tensor %r" % (dtype, tuple(logits.shape)))
    return out


def _forward(a, logits, out):
    with _On(logits.device) as stream:
        _cabi.check(_cabi.lib().dnatok_process_logits(ctypes.byref(a), out.data_ptr(), _TYPES[out.dtype], out.stride(0), stream))
    return out


def _backward(a, logits, grad, bias_shape, want_logits: bool, want_bias: bool):
    if grad.shape[1] > 1 and grad.stride(1) != 1:
        grad = grad.contiguous()
    n, width = grad.shape
    dx = torch.empty((n, width), dtype=logits.dtype, device=grad.device) if want_logits else None
    db = scratch = None
    need = 0
    L = _cabi.lib()
    with _On(grad.device) as stream:
        if want_bias:
            db = torch.empty(bias_shape, dtype=torch.float32, device=grad.device)
            need = L.dnatok_logits_scratch_bytes(n, width) if a.bias_stride == 0 else 0
            if need:
                scratch = torch.empty(need, dtype=torch.uint8, device=grad.device)
        _cabi.check(L.dnatok_process_logits_backward(
            ctypes.byref(a), grad.data_ptr(), _TYPES[grad.dtype], grad.stride(0), dx.data_ptr() if dx is not None else None,
            dx.stride(0) if dx is not None else 0, db.data_ptr() if db is not None else None,
            scratch.data_ptr() if scratch is not None else None, need, stream))
    return dx, db


class _Process(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, history, rows, repetition, frequency, presence, allowed, out_dtype):
        a, _ = _arguments(logits, history, rows, repetition, frequency, presence, bias, allowed)
        out = _forward(a, logits, _output(logits, None, out_dtype))
        ctx.save_for_backward(logits, bias, rows if a.rows else None, allowed, history.seen if a.seen else None,
                              repetition if isinstance(repetition, torch.Tensor) else None)
        ctx.number = a.repetition
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        # (the tensors may have been stored elsewhere in the meantime: nothing but them holds for their addresses)
        logits, bias, rows, allowed, seen, repetition = ctx.saved_tensors
        a = _cabi.Logits()
        a.logits, a.dtype, a.stride = logits.data_ptr(), _TYPES[logits.dtype], logits.stride(0)
        a.n_rows, a.width = logits.shape
        a.repetition = ctx.number
        if repetition is not None:
            a.d_repetition = repetition.data_ptr()
        if seen is not None:
            a.seen, a.history_rows = seen.data_ptr(), seen.shape[0]
        if rows is not None:
            a.rows, a.rows_bits = rows.data_ptr(), _BITS[rows.dtype]
        if allowed is not None:
            a.allowed, a.allowed_stride = allowed.data_ptr(), 0 if allowed.dim() == 1 or allowed.shape[0] == 1 else allowed.stride(0)
        if bias is not None and bias.dim() == 2 and bias.shape[0] != 1:
            a.bias_stride = bias.stride(0)
        dx, db = _backward(a, logits, grad, bias.shape if bias is not None else None, ctx.needs_input_grad[0],
                           ctx.needs_input_grad[1])
        return dx, db, None, None, None, None, None, None, None


def process_logits(logits, *, history: Optional[TokenHistory] = None, rows=None, repetition: Number = 1.0,
                   frequency: Number = 0.0, presence: Number = 0.0, bias=None, allowed=None, out=None, out_dtype=None):
    """``logits`` [n, width] (float32, float16 or bfloat16; a view such as ``model_output[:, -1]`` is fine) after penalties,
    bias and mask, as a new tensor of its type or of ``out_dtype`` float32, or in ``out`` (which may be ``logits``).

    * A token the row has seen: ``x > 0 ? x / repetition : x * repetition``; one it generated ``c > 0`` times, then
      ``- frequency * c - presence``.  Each is a number, or a float32 tensor [n] (repetition from 2^-126 to 2^126 there too).
      ``rows`` [n] names each row's history row (a row outside the history has none); two rows may share one.
    * ``bias`` float32 [width] or [n, width] is added.
    * ``allowed`` int32 [n, words] or [words]: tokens whose bit is 0 become ``-inf`` whatever their logits hold, NaN
      included.  A row without an allowed token is ``-inf`` throughout.

    All of it is computed in 32 bits and rounded once.  Differentiable in ``logits`` and ``bias``; the history and the mask
    must then stay as they are until the backward pass (autograd refuses it otherwise)."""
    if torch.is_grad_enabled() and ((isinstance(logits, torch.Tensor) and logits.requires_grad)
                                    or (isinstance(bias, torch.Tensor) and bias.requires_grad)):
        if out is not None:
            raise ValueError("out= has no gradient; leave it out or call under torch.no_grad()")
        return _Process.apply(logits, bias, history, rows, repetition, frequency, presence, allowed, out_dtype)
    a, _ = _arguments(logits, history, rows, repetition, frequency, presence, bias, allowed)
    result = _forward(a, logits, _output(logits, out, out_dtype))
    if out is not None:
        _written(out)
    return result


def process_logits_backward(grad, logits, *, history: Optional[TokenHistory] = None, rows=None, repetition: Number = 1.0,
                            frequency: Number = 0.0, presence: Number = 0.0, bias=None, allowed=None):
    """(gradient of ``logits``, gradient of ``bias`` or None) for ``grad``, the gradient of ``process_logits`` called with the
    same arguments; without autograd."""
    with torch.no_grad():
        a, _ = _arguments(logits, history, rows, repetition, frequency, presence, bias, allowed)
        _same_device(grad, "grad", logits.device)
        if grad.dim() != 2 or grad.shape != logits.shape or grad.dtype not in (logits.dtype, torch.float32):
            raise ValueError("grad must be a tensor %r of the logits' type or float32" % (tuple(logits.shape),))
        return _backward(a, logits, grad, bias.shape if bias is not None else None, True, bias is not None)
