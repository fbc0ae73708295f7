"""Beam search on the GPU decoder: each text goes on as the `beams` continuations
of the largest summed log-probability (no counterpart in the reference, whose
Writer samples).

How a step runs here, with no host synchronization:
    read       one extend of every beam's last token, the logits as the head
               writes them
    select     sampling.beam_step: the next beams over beams and vocabulary
    reorder    the cache's rows take over their parents' states in place
               (MQADecoder.reorder)
    evict      with `keep`, a weighted cache is brought back to keep entries an
               exact layer whenever it may hold an eighth more (MQADecoder.evict):
               the host knows the longest row's bound, so that a text is evicted
               from when the longest beside it is
Each beam's text is read back along its parents when it is asked for.
"""

import torch

from . import sampling
from .writer import cut

CHUNK = 1024  # tokens of a prompt read at once
CHECK = 8     # steps between two looks at whether every beam has ended


class BeamWriter:
    """Writes `beams` continuations of each of `prompts` (lists of ints, each
    at least one token) with an MQADecoder.  stops: the tokens that end a
    beam (at most 16); keep, first, recent: the entries an exact layer's cache
    is bounded to (MQADecoder.evict; None: every entry is kept)."""

    def __init__(self, model, prompts, beams, *, stops=(), keep=None, first=4, recent=None):
        prompts = [list(p) for p in prompts]
        if not prompts or not all(prompts):
            raise ValueError("beam search writes for at least one prompt, each of at least one token")
        if not 1 <= beams <= 64:
            raise ValueError(f"a text is written by 1 to 64 beams; got {beams}")
        stops = tuple(int(s) for s in stops)
        if len(stops) > 16:
            raise ValueError(f"a beam ends at one of at most 16 tokens; got {len(stops)}")
        vocab = model.config.vocab
        if any(not 0 <= t < vocab for p in prompts for t in p) or any(not 0 <= t < vocab for t in stops):
            raise IndexError(f"token ids must lie in [0, {vocab})")
        self.model, self.beams, self.stops = model, int(beams), stops
        self.bounds = None if keep is None else model.evict_rows(keep, first, recent)
        self.device = next(model.parameters()).device
        n = len(prompts)
        self.cache = model.new_cache(n, weighted=keep is not None)
        counts = torch.tensor([len(p) - 1 for p in prompts])
        ids = torch.zeros(n, max(1, int(counts.max())), dtype=torch.long)
        for i, p in enumerate(prompts):
            ids[i, :len(p) - 1] = torch.tensor(p[:-1], dtype=torch.long)
        ids = ids.to(self.device)
        for start in range(0, int(counts.max()), CHUNK):  # every prompt but its last token, once a text
            part = ids[:, start:start + CHUNK]
            model.extend(part, self.cache, (counts - start).clamp(0, part.shape[1]), logits=True)
            self._evict()
        self.cache = self.cache.select([i for i in range(n) for _ in range(self.beams)])
        self.last = torch.tensor([[p[-1]] for p in prompts for _ in range(self.beams)], dtype=torch.long,
                                 device=self.device)
        # a text starts as one beam: the other places hold none
        self.totals = torch.full((n, self.beams), float("-inf"), device=self.device)
        self.totals[:, 0] = 0
        self.ended = torch.zeros(n, self.beams, dtype=torch.bool, device=self.device)
        self._steps = []  # (parents, tokens) of each step

    def _evict(self):
        if self.bounds is not None and self.cache.bound > self.bounds[0] + self.bounds[0] // 8:
            self.model.evict(self.cache, *self.bounds)

    @torch.no_grad()
    def step(self):
        """One more token for every beam that has not ended."""
        n, W = self.totals.shape
        scores = self.model.extend(self.last, self.cache, logits=True)[0].view(n, W, -1)
        self.totals, parents, tokens, self.ended = sampling.beam_step(
            scores, self.totals, self.ended if self.stops else None, self.stops)
        self.model.reorder(self.cache, parents)
        self.last = tokens.view(n * W, 1)
        self._steps.append((parents, tokens))
        self._evict()

    def write(self, limit):
        """Up to limit more tokens a beam, fewer when every beam has ended:
        texts()."""
        for i in range(limit):
            if self.stops and i % CHECK == 0 and bool((self.ended | (self.totals == float("-inf"))).all()):
                break
            self.step()
        return self.texts()

    @torch.no_grad()
    def texts(self):
        """For each text its beams, best first, as (the tokens written, through
        the first stop token; their summed log-probability).  A place that
        holds no beam is left out."""
        n, W = self.totals.shape
        beam = torch.arange(W, device=self.device).expand(n, W)
        written = []
        for parents, tokens in reversed(self._steps):
            written.append(tokens.gather(1, beam))
            beam = parents.gather(1, beam)
        lists = torch.stack(written[::-1], -1).tolist() if written else [[[] for _ in range(W)] for _ in range(n)]
        totals = self.totals.tolist()
        return [[(cut(lists[i][w], self.stops, len(self._steps)), totals[i][w]) for w in range(W)
                 if totals[i][w] > float("-inf")] for i in range(n)]
