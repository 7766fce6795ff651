"""Finite automata over bases, as host tables: what a grammar mask lets a row become.

``Automaton.from_pattern("ATG(NNN)*TRA")`` accepts the sequences that a regular expression of IUPAC letters describes,
``Automaton.avoiding(["GAATTC", "GANTC"])`` all sequences without those motifs, and ``a & b`` what both accept.  Any other
deterministic automaton over bytes can be given as its table.
"""
from __future__ import annotations

from typing import Iterable, List, Optional, Tuple

import numpy as np

BASES = "ACGT"
IUPAC = {"A": "A", "C": "C", "G": "G", "T": "T", "U": "T", "R": "AG", "Y": "CT", "S": "CG", "W": "AT", "K": "GT", "M": "AC",
         "B": "CGT", "D": "AGT", "H": "ACT", "V": "ACG", "N": "ACGT"}
_COMPLEMENT = str.maketrans("ACGTURYSWKMBDHVN", "TGCAAYRSWMKVHDBN")
OTHER = 4                      # the class of every byte that is not a base
MAX_STATES = 1 << 22


def base_classes(lowercase: bool = True) -> np.ndarray:
    """uint8[256]: A, C, G, T = 0..3 (soft-masked lower-case letters too, unless ``lowercase`` is false), others 4."""
    table = np.full(256, OTHER, dtype=np.uint8)
    for i, c in enumerate(BASES):
        table[ord(c)] = i
        if lowercase:
            table[ord(c.lower())] = i
    return table


def whole_numbers(values, dtype, what: str) -> np.ndarray:
    """A contiguous array of ``dtype`` with these values; one that the type does not hold is refused, not wrapped or cut."""
    given = np.asarray(values)
    try:
        with np.errstate(invalid="ignore"):
            a = np.ascontiguousarray(given, dtype=dtype)
    except (OverflowError, TypeError, ValueError):
        a = None
    if a is None or not np.array_equal(a, given):
        raise ValueError("%s must hold whole numbers of %s" % (what, np.dtype(dtype).name))
    return a


class Automaton:
    """``next_state`` int [states, classes] (-1: no way on), ``accepting`` [states], ``byte_class`` uint8[256] (which column
    a byte takes; bases and others by default), ``start`` the first state.  From every state the row may go on as long as
    a token leads to a state; the end token is allowed in accepting states."""

    def __init__(self, next_state, accepting, *, byte_class=None, start: int = 0):
        self.next_state = whole_numbers(next_state, np.int32, "next_state")
        self.accepting = np.ascontiguousarray(np.asarray(accepting) != 0, dtype=np.uint8)
        self.byte_class = whole_numbers(base_classes() if byte_class is None else byte_class, np.uint8, "byte_class")
        if self.next_state.ndim != 2 or not self.next_state.shape[0] or not self.next_state.shape[1]:
            raise ValueError("next_state must be [states, classes]")
        n, classes = self.next_state.shape
        if self.accepting.shape != (n,):
            raise ValueError("accepting must have one value per state")
        if self.byte_class.shape != (256,) or int(self.byte_class.max()) >= classes:
            raise ValueError("byte_class must name a class below %d for each of 256 bytes" % classes)
        if int(self.next_state.min()) < -1 or int(self.next_state.max()) >= n:
            raise ValueError("next_state leads outside the automaton")
        if not 0 <= start < n:
            raise ValueError("start is not a state")
        self.start = int(start)

    @property
    def n_states(self) -> int:
        return self.next_state.shape[0]

    # ------------------------------------------------------------------ host walk
    def walk(self, text, state: Optional[int] = None) -> int:
        """The state after ``text`` (str or bytes), -1 where there is no way on."""
        s = self.start if state is None else int(state)
        for b in (text.encode("latin-1") if isinstance(text, str) else bytes(text)):
            if s < 0:
                return -1
            s = int(self.next_state[s, self.byte_class[b]])
        return s

    def accepts(self, text) -> bool:
        s = self.walk(text)
        return s >= 0 and bool(self.accepting[s])

    # ------------------------------------------------------------------ construction
    @classmethod
    def from_pattern(cls, pattern: str, *, lowercase: bool = True) -> "Automaton":
        """The sequences that match the whole pattern: IUPAC letters (``N`` or ``.``: any base), sets ``[AC]``, groups
        ``( )``, alternatives ``|`` and the repeats ``* + ? {m} {m,} {m,n}``.  Bytes that are no base never match."""
        edges, empty, first, last = _Pattern(pattern).build()
        return cls._subsets(edges, empty, {first}, last, lowercase=lowercase)

    @classmethod
    def avoiding(cls, motifs: Iterable[str], *, reverse_complement: bool = False, lowercase: bool = True) -> "Automaton":
        """The sequences in which none of the motifs (IUPAC letters) occurs, nor the reverse complement of one where asked
        for.  A byte that is no base belongs to no motif and is allowed; a row may end anywhere."""
        every: List[str] = []
        for m in ([motifs] if isinstance(motifs, str) else motifs):
            m = m.upper()
            if not m or any(c not in IUPAC for c in m):
                raise ValueError("a motif is one or more IUPAC letters: got %r" % (m,))
            every.append(m)
            if reverse_complement:
                every.append(m.translate(_COMPLEMENT)[::-1])
        edges: List[List[Tuple[int, int]]] = [[(0b1111, 0)]]       # node 0 goes on with every base: a motif may begin anywhere
        bad = set()
        for m in dict.fromkeys(every):
            at = 0
            for c in m:
                edges.append([])
                edges[at].append((_mask(c), len(edges) - 1))
                at = len(edges) - 1
            bad.add(at)
        return cls._subsets(edges, [[] for _ in edges], {0}, bad, lowercase=lowercase, avoid=True)

    @classmethod
    def _subsets(cls, edges, empty, first, last, *, lowercase: bool, avoid: bool = False) -> "Automaton":
        """Subset construction; ``avoid``: sets that hold one of ``last`` are no states, and a byte that is no base leads
        back to the first set.  States from which nothing can be accepted are left out."""
        last = last if isinstance(last, set) else {last}

        def closure(nodes) -> frozenset:
            todo, got = list(nodes), set(nodes)
            while todo:
                for t in empty[todo.pop()]:
                    if t not in got:
                        got.add(t)
                        todo.append(t)
            return frozenset(got)

        begin = closure(first)
        number, queue, rows = {begin: 0}, [begin], []
        for s in queue:
            row = []
            for c in range(4):
                to = {t for n in s for m, t in edges[n] if m >> c & 1}
                if not to or (avoid and to & last):
                    row.append(-1)
                    continue
                to = closure(to)
                if to not in number:
                    if len(number) >= MAX_STATES:
                        raise ValueError("the automaton has more than %d states" % MAX_STATES)
                    number[to] = len(number)
                    queue.append(to)
                row.append(number[to])
            row.append(0 if avoid else -1)
            rows.append(row)
        accepting = np.array([True if avoid else bool(s & last) for s in queue])
        nxt = np.array(rows, dtype=np.int32)
        return cls(_without_dead_ends(nxt, accepting), accepting, byte_class=base_classes(lowercase))

    def __and__(self, other: "Automaton") -> "Automaton":
        if not isinstance(other, Automaton):
            return NotImplemented
        pairs = np.stack([self.byte_class, other.byte_class], axis=1)
        columns, byte_class = np.unique(pairs, axis=0, return_inverse=True)
        if len(columns) > 256:
            raise ValueError("more than 256 classes of bytes")
        begin = (self.start, other.start)
        number, queue, rows = {begin: 0}, [begin], []
        for a, b in queue:
            row = []
            for x, y in columns.tolist():
                to = (int(self.next_state[a, x]), int(other.next_state[b, y]))
                if to[0] < 0 or to[1] < 0:
                    row.append(-1)
                    continue
                if to not in number:
                    if len(number) >= MAX_STATES:
                        raise ValueError("the automaton has more than %d states" % MAX_STATES)
                    number[to] = len(number)
                    queue.append(to)
                row.append(number[to])
            rows.append(row)
        accepting = np.array([bool(self.accepting[a] and other.accepting[b]) for a, b in queue])
        return Automaton(_without_dead_ends(np.array(rows, dtype=np.int32), accepting), accepting,
                         byte_class=byte_class.reshape(-1).astype(np.uint8))


def _without_dead_ends(nxt: np.ndarray, accepting: np.ndarray) -> np.ndarray:
    """The table with -1 in place of every state that no accepting state can be reached from."""
    n, classes = nxt.shape
    src = np.repeat(np.arange(n), classes)
    dst = nxt.reshape(-1)
    keep = dst >= 0
    src, dst = src[keep], dst[keep]
    order = np.argsort(dst, kind="stable")
    src = src[order]
    begin = np.searchsorted(dst[order], np.arange(n + 1))
    alive = accepting.copy()
    todo = np.flatnonzero(alive).tolist()
    while todo:
        t = todo.pop()
        for s in src[begin[t]:begin[t + 1]].tolist():
            if not alive[s]:
                alive[s] = True
                todo.append(s)
    return np.where((nxt >= 0) & alive[np.maximum(nxt, 0)], nxt, -1).astype(np.int32)


def _mask(letter: str) -> int:
    return sum(1 << BASES.index(b) for b in IUPAC[letter])


class _Pattern:
    """A pattern's nodes: ``edges[n]`` (set of bases, node) and ``empty[n]`` (node)."""

    def __init__(self, text: str):
        self.text, self.at = text.upper(), 0
        self.edges: List[List[Tuple[int, int]]] = []
        self.empty: List[List[int]] = []

    def node(self) -> int:
        if len(self.edges) >= MAX_STATES:
            raise ValueError("the pattern has more than %d positions" % MAX_STATES)
        self.edges.append([])
        self.empty.append([])
        return len(self.edges) - 1

    def fail(self, what: str):
        raise ValueError("pattern %r, position %d: %s" % (self.text, self.at, what))

    def peek(self) -> str:
        return self.text[self.at] if self.at < len(self.text) else ""

    def build(self):
        tree = self.alternatives()
        if self.at < len(self.text):
            self.fail("unexpected %r" % self.peek())
        first, last = self.lay(tree)
        return self.edges, self.empty, first, last

    # a tree of ("set", bases), ("seq", parts), ("or", parts), ("repeat", part, least, most)
    def alternatives(self):
        parts = [self.sequence()]
        while self.peek() == "|":
            self.at += 1
            parts.append(self.sequence())
        return parts[0] if len(parts) == 1 else ("or", parts)

    def sequence(self):
        parts = []
        while self.peek() not in ("", "|", ")"):
            parts.append(self.repeated())
        return ("seq", parts)

    def repeated(self):
        part = self.single()
        while self.peek() and self.peek() in "*+?{":
            c = self.peek()
            self.at += 1
            if c == "{":
                end = self.text.find("}", self.at)
                body = self.text[self.at:end].split(",") if end >= 0 else []
                if len(body) not in (1, 2) or not all(b.isdigit() for b in body[:1]) or not all(b == "" or b.isdigit() for b in body[1:]):
                    self.fail("a repeat is {m}, {m,} or {m,n}")
                self.at = end + 1
                least = int(body[0])
                most = least if len(body) == 1 else int(body[1]) if body[1] else None
                if most is not None and most < least:
                    self.fail("a repeat's bounds are in order")
            else:
                least, most = {"*": (0, None), "+": (1, None), "?": (0, 1)}[c]
            part = ("repeat", part, least, most)
        return part

    def single(self):
        c = self.peek()
        self.at += 1
        if c == "(":
            part = self.alternatives()
            if self.peek() != ")":
                self.fail("a group is not closed")
            self.at += 1
            return part
        if c == "[":
            end = self.text.find("]", self.at)
            letters = self.text[self.at:end] if end >= 0 else ""
            if not letters or any(x not in IUPAC for x in letters):
                self.fail("a set is [ ] around IUPAC letters")
            self.at = end + 1
            m = 0
            for x in letters:
                m |= _mask(x)
            return ("set", m)
        if c == ".":
            return ("set", 0b1111)
        if c not in IUPAC:
            self.at -= 1
            self.fail("unexpected %r" % c)
        return ("set", _mask(c))

    def lay(self, tree) -> Tuple[int, int]:
        kind = tree[0]
        if kind == "set":
            a, b = self.node(), self.node()
            self.edges[a].append((tree[1], b))
            return a, b
        if kind == "seq":
            first = last = self.node()
            for part in tree[1]:
                a, b = self.lay(part)
                self.empty[last].append(a)
                last = b
            return first, last
        if kind == "or":
            first, last = self.node(), self.node()
            for part in tree[1]:
                a, b = self.lay(part)
                self.empty[first].append(a)
                self.empty[b].append(last)
            return first, last
        _, part, least, most = tree
        first = last = self.node()
        for _ in range(least):
            a, b = self.lay(part)
            self.empty[last].append(a)
            last = b
        end = self.node()
        if most is None:
            hub = self.node()
            a, b = self.lay(part)
            self.empty[last].append(hub)
            self.empty[hub] += [a, end]
            self.empty[b].append(hub)
            return first, end
        for _ in range(most - least):
            a, b = self.lay(part)
            self.empty[last] += [a, end]
            last = b
        self.empty[last].append(end)
        return first, end
