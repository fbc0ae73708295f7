"""The generation cache of the MQA decoder on the GPU: the reference's Rows /
Reading / Cache (packages/wpt-model/src/wpt_model/cache.py:54-174) for exact
layers, whose carried value is every token's key and value side by side
(carry.Entries, carry.py:66-71), and for window layers, whose carried value
is the last window - 1 tokens' (carry.Tail, carry.py:30-63).

A window layer's entries live in a ring of R rows per batch row (R a power
of 2 of at least window - 1 + the widest reading), token p at row p mod R: a
reading writes its tokens over ones more than R - 1 tokens back, which no
query of it or of a later reading sees, so the ring holds the reference's
tail (the window - 1 rows before each row's length, tail(layer) gathers it)
with no copy per step, and undo, which only restores the lengths, cuts it
back as carry.Tail.undo does (rows past a length are written again before
any query reads them).

A sparse layer carries nothing (it reads the exact layer's table before it)
and has no table: its entry in `tables` is None.

Each exact layer's entries live in one (B, capacity, 2c) table, keys first, token p
of row b at row p.  A reading appends each row's own new entries at its own
length (wptv_kv_append) and returns nothing to copy: the attention reads the
table in place up to each query's position.  Undo restores the lengths from
before the undoable reading plus kept; the entries past a row's length are
never read, and are written again when the row reaches them.

A beam search's rows take over each other's states with reorder, in place.  A
weighted cache also keeps the attention weight that each exact layer's rows have
received (`weights`, FP32 (exact layers, B, capacity)): the decoder adds each
reading's, an undoable one's when its kept tokens are known.  evict then brings
every row down to its first, its last and its heaviest entries, moved together
in place: from then on token p is no longer at row p of the exact layers' tables
(whose attention has no use for the position), and `evicted` counts each row's
entries taken out, so that the window layers' rings still place token
lengths + evicted.

The lengths stay on the device; `bound` is a host-side upper bound of every
row's length (raised by each reading's width, never lowered by undo) so that
growing the tables needs no host synchronization.  The tables grow to
max(need, 2 x capacity) as the reference's do, by a copy; a HIP graph of a
step is captured with the capacity reserved beforehand.
"""

import torch

from . import _lib, kernels
from ._lib import check, ptr


def _lengths(lengths, before, counts, undo):
    """wptv_cache_lengths on the lengths' device: before = lengths (when
    given), lengths += counts; or, undo, lengths = before + counts."""
    if counts.device != lengths.device or counts.shape != lengths.shape or counts.dtype not in _lib.INDEX_DTYPES:
        raise ValueError(f"counts must be ({lengths.shape[0]},) int64 or int32 on {lengths.device}")
    counts = counts.contiguous()
    check(_lib.lib().wptv_cache_lengths(ptr(lengths), ptr(before), ptr(counts), _lib.INDEX_DTYPES[counts.dtype],
                                        lengths.shape[0], int(undo), _lib.stream(lengths.device)), "cache_lengths")


class Cache:
    """rings: the layers whose table is a ring of ring_rows rows (window
    layers); bare: the layers with no table (sparse layers); every other
    layer's table grows with the text.  weighted: the growing tables' rows
    carry the attention weight they have received, and may be evicted, but for
    the last `recent` (what the sparse layers read of them by position)."""

    def __init__(self, rows, layers, width, dtype, device, capacity=256, rings=(), ring_rows=256, bare=(),
                 weighted=False, recent=0):
        if ring_rows <= 0 or ring_rows & (ring_rows - 1):
            raise ValueError(f"a ring holds a power of 2 of rows, not {ring_rows}")
        self.lengths = torch.zeros(rows, dtype=torch.long, device=device)
        self.before = torch.zeros_like(self.lengths)  # the lengths before the last undoable reading
        self.rings = frozenset(rings)
        self.tables = [None if i in bare else
                       torch.zeros(rows, ring_rows if i in self.rings else capacity, width, dtype=dtype, device=device)
                       for i in range(layers)]
        self.pending = False
        self.bound = 0
        self.routes = None
        self.weights = self.evicted = None
        self.recent = recent
        self._read = []  # a weighted cache's undoable reading: (weights' row, layer, q, positions, lse, scale, counts)
        self._captured = False  # whether that reading was made under stream capture
        self._reading = []  # the same of a reading that has not finished
        if weighted:
            if not self.growing:
                raise ValueError("a weighted cache has at least one table that grows with the text")
            self.weights = torch.zeros(len(self.growing), rows, capacity, dtype=torch.float32, device=device)
            self.evicted = torch.zeros_like(self.lengths)

    @property
    def growing(self):
        """The layers whose table grows with the text."""
        return [i for i, t in enumerate(self.tables) if t is not None and i not in self.rings]

    @property
    def rows(self):
        return self.lengths.shape[0]

    @property
    def capacity(self):
        grown = [t.shape[1] for i, t in enumerate(self.tables) if t is not None and i not in self.rings]
        return grown[0] if grown else None

    @property
    def ring_rows(self):
        rings = [self.tables[i].shape[1] for i in sorted(self.rings)]
        return rings[0] if rings else None

    def reserve(self, need):
        """Growing tables of at least `need` rows (grown to max(need, 2 x
        capacity)); the rings keep their size."""
        if self.capacity is None or need <= self.capacity:
            return
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"the cache needs {need} rows but holds {self.capacity}: reserve them before "
                               "capturing a step")
        grown = max(need, 2 * self.capacity)
        self.tables = [t if t is None or i in self.rings else torch.cat([t, t.new_zeros(t.shape[0], grown - t.shape[1],
                                                                           t.shape[2])], 1)
                       for i, t in enumerate(self.tables)]
        if self.weights is not None:
            self.weights = torch.cat([self.weights, self.weights.new_zeros(*self.weights.shape[:2],
                                                                           grown - self.weights.shape[2])], 2)

    def starts(self):
        """The position of each row's next token in its text: its length, and
        the entries evicted before."""
        return self.lengths if self.evicted is None else self.lengths + self.evicted

    def tail(self, layer, steps):
        """A window layer's carried tail (B, steps, width): the entries of the
        steps tokens before each row's length, zeros before the text (the
        reference's Reading.before, cache.py:97-108)."""
        if layer not in self.rings:
            raise ValueError(f"layer {layer} keeps every entry, not a tail")
        ring = self.tables[layer]
        R = ring.shape[1]
        if steps > R:
            raise ValueError(f"the ring holds {R} rows, fewer than {steps}")
        positions = self.starts()[:, None] - steps + torch.arange(steps, device=ring.device)
        rows = ring.gather(1, (positions % R)[..., None].expand(-1, -1, ring.shape[2]))
        return rows.masked_fill((positions < 0)[..., None], 0)

    def finish(self, counts, undoable, width):
        """The rows have read their tokens (the reference's Reading.finish).
        The lengths change in place, so that a captured step replays on the
        cache's current state."""
        _lengths(self.lengths, self.before if undoable else None, counts, undo=False)
        self.pending = bool(undoable)
        self.bound += width
        self._read, self._reading = self._reading, []
        self._captured = bool(self._read) and torch.cuda.is_current_stream_capturing()

    def undo(self, kept):
        """Back to the lengths before the last undoable reading, plus kept."""
        if not self.pending:
            raise ValueError("no undoable extend to undo")
        if self.weights is not None and not self._read:
            raise ValueError("the weights of the reading to undo are not here: a captured undoable reading of a weighted "
                             "cache is captured together with its undo")
        self._together()
        _lengths(self.lengths, self.before, kept, undo=True)
        self.settle(kept)
        self.pending = False

    def undo_on_device(self):
        """The lengths and the lengths before the last undoable reading, for a
        kernel that applies the undo itself (the sampler's commit); the
        reading counts as undone from here on."""
        if not self.pending:
            raise ValueError("no undoable extend to undo")
        if self.weights is not None:
            raise ValueError("a weighted cache adds the kept tokens' weights in undo()")
        self.pending = False
        return self.lengths, self.before

    def weigh(self, layer, q, positions, lse, scale, counts, undoable):
        """Adds the weights that a growing layer's rows got from a reading of
        counts tokens (q (B, T, H, c) at positions, lse the attention's); an
        undoable reading's when undo tells how many tokens were kept."""
        reading = (self.growing.index(layer), layer, q, positions, lse, scale, counts)
        if undoable:
            self._reading.append(reading)
        else:
            self._add(reading, counts, self.lengths)

    def _add(self, reading, counts, start):
        at, layer, q, positions, lse, scale, _ = reading
        kernels.add_attention_weights(q, self.tables[layer][..., :q.shape[-1]], positions, lse, scale, self.weights[at],
                                      counts=counts, start=start)

    def _together(self):
        """Refuses to add an undoable reading's weights in a capture that it was
        not made in, where every replay would add them again, or a captured
        reading's outside its capture, where they were never computed."""
        if self._read and self._captured != torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a captured undoable reading of a weighted cache is captured together with its undo"
                               if self._captured else
                               "an undoable reading of this weighted cache is pending: undo it before capturing a step")

    def settle(self, kept=None):
        """Adds the weights of an undoable reading of which kept tokens stay
        (None: all of them, when another reading follows it).  What a reading
        that failed before its end has left is dropped: none of its tokens is in
        the cache."""
        self._together()
        self._reading = []
        for reading in self._read:
            self._add(reading, reading[-1] if kept is None else kept, self.before)
        self._read = []

    def select(self, index):
        """A new cache of the rows index names (a row may come several times),
        copied (the reference's Cache.select, cache.py:157-166)."""
        if self.pending:
            raise ValueError("an undoable extend is pending: undo it before copying rows")
        index = torch.as_tensor(index, dtype=torch.long, device=self.lengths.device)
        copy = object.__new__(Cache)
        copy.lengths = self.lengths[index]
        copy.before = torch.zeros_like(copy.lengths)
        copy.tables = [None if t is None else t[index] for t in self.tables]
        copy.rings, copy.recent = self.rings, self.recent
        copy.pending, copy.bound, copy.routes = False, self.bound, None
        copy.weights = None if self.weights is None else self.weights[:, index]
        copy.evicted = None if self.evicted is None else self.evicted[index]
        copy._read, copy._captured, copy._reading = [], False, []
        return copy

    def reorder(self, parents):
        """Beam search's step: row i W + w takes over row i W + parents[i, w], for
        parents (texts, W) int64 and every row at once, in place (select copies
        into a new cache): only what the sources hold is moved."""
        if self.pending:
            raise ValueError("an undoable extend is pending: undo it before moving rows")
        if parents.dim() != 2 or parents.shape[0] * parents.shape[1] != self.rows:
            raise ValueError(f"parents must be (texts, beams) of the cache's {self.rows} rows; got {tuple(parents.shape)}")
        tables = [self.tables[i] for i in self.growing]
        if self.weights is not None:
            tables += [w[..., None] for w in self.weights]
        if tables:  # not bounded by `bound`: replays of a captured reading do not raise it
            kernels.reorder_rows(tables, parents, self.lengths)
        if self.rings:
            kernels.reorder_rows([self.tables[i] for i in sorted(self.rings)], parents, self.starts())
        states = [self.lengths] if self.evicted is None else [self.lengths, self.evicted]
        kernels.reorder_rows([x.view(-1, 1, 1) for x in states], parents)

    def evict(self, keep, first=4, recent=128):
        """Brings every row of a weighted cache down to at most keep entries a
        layer: its first `first`, its last `recent`, and the others that have
        received the most attention weight, in their order, in place.  Returns
        the rows kept, (exact layers, B, keep) int64, -1 past a row's count."""
        if self.weights is None:
            raise ValueError("only a weighted cache evicts: it keeps the attention weight its rows have received")
        if self.pending:
            raise ValueError("an undoable extend is pending: undo it before evicting rows")
        if recent < self.recent:
            raise ValueError(f"the sparse layers read the last {self.recent} tokens: recent = {recent} does not hold them")
        kept, counts = kernels.choose_kept(self.weights, self.lengths, keep, first, recent)
        kernels.keep_rows([self.tables[i] for i in self.growing], kept, counts)
        kernels.keep_rows([w[..., None] for w in self.weights], kept, counts)
        self.evicted += self.lengths - counts
        self.lengths.copy_(counts)
        self.bound = min(self.bound, int(keep))
        return kept
