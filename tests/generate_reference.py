"""Plain 64-bit implementations of the operators around logits, and the bounds their kernels are held to."""
import numpy as np
import torch

U32 = 2.0 ** -24                                                  # half a step of each type, relative to the value
U = {torch.float32: U32, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}    # half a step below the normals
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def pack(ok):
    """bool [n, width] -> int32 words [n, ceil(width / 32)]."""
    ok = np.asarray(ok, dtype=bool)
    n, width = ok.shape
    full = np.zeros((n, (width + 31) // 32 * 32), dtype=bool)
    full[:, :width] = ok
    return np.packbits(full, axis=1, bitorder="little").view("<i4").reshape(n, -1) if n else np.zeros((0, (width + 31) // 32), np.int32)


def unpack(words, width):
    words = np.ascontiguousarray(words, dtype=np.int32)
    return np.unpackbits(words.view(np.uint8), axis=1, bitorder="little")[:, :width].astype(bool)


def logits(x, seen=None, counts=None, r=1.0, f=0.0, p=0.0, bias=None, ok=None):
    """(result, bound on the error of its 32-bit evaluation before the last rounding).  Six roundings at most, none of them
    of a value larger than the sum of the terms: 6 * 2^-24 of that sum, and a hundredth for the products of errors."""
    x = np.asarray(x, dtype=np.float64)
    col = lambda v: np.asarray(v, dtype=np.float64).reshape(-1, 1)  # noqa: E731
    r, f, p = col(r), col(f), col(p)
    with np.errstate(all="ignore"):
        y = x.copy()
        if seen is not None:
            y = np.where(seen, np.where(x > 0, x / r, x * r), x)
        size = np.abs(y)
        if counts is not None:
            c = np.asarray(counts, dtype=np.float64)
            y = np.where(c > 0, y - f * c - p, y)
            size = size + np.where(c > 0, np.abs(f * c) + np.abs(p), 0)
        if bias is not None:
            y = y + bias
            size = size + np.abs(bias)
        if ok is not None:
            y = np.where(ok, y, -np.inf)
    return y, 1.01 * 6 * U32 * size


def gradients(x, grad, seen=None, r=1.0, ok=None):
    """(gradient of the logits, gradient of a bias of every row)."""
    x, g = np.asarray(x, dtype=np.float64), np.asarray(grad, dtype=np.float64)
    r = np.asarray(r, dtype=np.float64).reshape(-1, 1)
    if ok is not None:
        g = np.where(ok, g, 0.0)
    return (g if seen is None else np.where(seen, np.where(x > 0, g / r, g * r), g)), g


def host(t):
    return t.detach().double().cpu().numpy()


def close(got, want, bound, dtype):
    """Every value within the bound and its own rounding; infinities and NaN in the same places."""
    got = host(got)
    with np.errstate(all="ignore"):
        limit = bound + 1.01 * U[dtype] * np.abs(want) + TINY[dtype]
        same = (got == want) | (np.isnan(got) & np.isnan(want)) | (np.isfinite(want) & (np.abs(got - want) <= limit))
        # what lies within its error of the largest value of the type may have been rounded to infinity
        top = float(torch.finfo(dtype).max)
        same |= np.isinf(got) & (np.sign(got) == np.sign(want)) & (np.abs(want) + limit >= top)
    bad = np.argwhere(~same)
    assert bad.size == 0, "%d of %d values, first at %s: got %r, want %r" % (
        len(bad), got.size, bad[0], got[tuple(bad[0])], np.broadcast_to(want, got.shape)[tuple(bad[0])])


def history(n_rows, width, rows_of_ids, generated, targets=None):
    seen, counts = np.zeros((n_rows, width), dtype=bool), np.zeros((n_rows, width), dtype=np.int64)
    for i, ids in enumerate(rows_of_ids):
        h = i if targets is None else int(targets[i])
        if not 0 <= h < n_rows:
            continue
        for v in np.asarray(ids).tolist():
            if 0 <= v < width:
                seen[h, v] = True
                counts[h, v] += generated
    return seen, counts


def walk(automaton, state, text):
    if state < 0 or state >= automaton.n_states or not text:
        return -1
    for b in text:
        state = int(automaton.next_state[state, automaton.byte_class[b]])
        if state < 0:
            return -1
    return state


def may_end(automaton, state):
    return state == -2 or (0 <= state < automaton.n_states and bool(automaton.accepting[state]))


def allowed(automaton, tokens, end_id, states, width=None):
    out = np.zeros((len(states), width or len(tokens)), dtype=bool)
    known = {}
    for i, s in enumerate(np.asarray(states).tolist()):
        if s not in known:
            row = np.array([walk(automaton, s, t) >= 0 for t in tokens])
            if end_id is not None:
                row[end_id] = may_end(automaton, s)
            known[s] = row
        out[i, :len(tokens)] = known[s]
    return out


def advance(automaton, tokens, end_id, states, chosen, width=None):
    out = []
    for s, v in zip(np.asarray(states).tolist(), np.asarray(chosen).tolist()):
        if not 0 <= v < (width or len(tokens)):
            out.append(s)
        elif v == end_id:
            out.append(-2 if may_end(automaton, s) else -1)
        else:
            out.append(walk(automaton, s, tokens[v]) if v < len(tokens) else -1)
    return np.array(out, dtype=np.int32)
