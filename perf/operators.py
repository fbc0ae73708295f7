"""Beam search's operators and the cache's eviction, as measurable cases: the
selection of the next beams over beams and vocabulary, the reordering of the
cache's rows after it, the accumulation of the attention weight every cached
row has received, and the choice and the move of the rows a bounded cache
keeps.

listed() names twelve cases, draw(rng) gives more of the same ranges,
prepare(case, seed) makes what a program holds before the call, run(state) is
one pass: the framework's calls where `own` is true, the same operators by
elementary torch operations where it is false.  exact(case, seed) is the
operators' definition in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
STOP = 2  # the token that ends a beam
FIRST, RECENT = 4, 128  # the rows an eviction keeps whatever their weight: a text's first and its last


def listed():
    return [
        # one text written by 4 beams of the small decoder's vocabulary: launches are all there is
        {"name": "beam_one_text", "kind": "beam", "dtype": "fp32", "n": 1, "W": 4, "V": 8192},
        # a batch of texts, 8 beams each, on the large decoder's logits as its head writes them
        {"name": "beam_batch", "kind": "beam", "dtype": "bf16", "n": 32, "W": 8, "V": 32768},
        # many texts, an odd count of beams and a vocabulary whose rows are not aligned
        {"name": "beam_odd_vocab", "kind": "beam", "dtype": "fp32", "n": 64, "W": 5, "V": 50257},
        # the small decoder's four layers, one text of 4 beams
        {"name": "reorder_one_text", "kind": "reorder", "dtype": "bf16", "layers": 4, "n": 1, "W": 4, "N": 300, "width": 128,
         "moved": 3, "sources": 2},
        # the large decoder's 24 layers, 8 texts of 4 beams and up to 1500 tokens
        {"name": "reorder_batch", "kind": "reorder", "dtype": "bf16", "layers": 24, "n": 8, "W": 4, "N": 1500, "width": 256,
         "moved": 3, "sources": 2},
        # one token of one text: the weights of a decode step without drafts
        {"name": "weights_one_token", "kind": "weights", "dtype": "bf16", "B": 1, "T": 1, "H": 16, "c": 128, "N": 4096},
        # the headline verify step: 32 texts of 4096 tokens, the pending token and 4 drafts
        {"name": "weights_verify", "kind": "weights", "dtype": "bf16", "B": 32, "T": 5, "H": 16, "c": 128, "N": 4100},
        # two prompts of 4096 tokens read in one pass
        {"name": "weights_prompt", "kind": "weights", "dtype": "bf16", "B": 2, "T": 4096, "H": 16, "c": 128, "N": 4096},
        # the small decoder in FP32, ragged lengths
        {"name": "weights_fp32", "kind": "weights", "dtype": "fp32", "B": 6, "T": 7, "H": 4, "c": 64, "N": 3001},
        # one short text of the small decoder, a few rows over its budget
        {"name": "evict_one_text", "kind": "evict", "dtype": "bf16", "layers": 4, "B": 1, "N": 320, "keep": 256, "width": 128},
        # the large decoder's 24 layers: 16 texts of 4096 tokens brought down to 2048 rows
        {"name": "evict_batch", "kind": "evict", "dtype": "bf16", "layers": 24, "B": 16, "N": 4096, "keep": 2048, "width": 256},
        # FP32 tables of an odd size, some texts below the budget
        {"name": "evict_fp32", "kind": "evict", "dtype": "fp32", "layers": 6, "B": 5, "N": 1777, "keep": 901, "width": 128},
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["beam", "reorder", "weights", "evict"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "beam":
        W, V = _log(rng, 1, 16), _log(rng, 500, 131072)
        n = min(_log(rng, 1, 64), max(1, 16_000_000 // (W * V)))
        return {"kind": kind, "dtype": dtype, "n": n, "W": W, "V": V}
    if kind == "reorder":
        W, layers, width = rng.randint(2, 16), rng.randint(1, 24), rng.choice([64, 128, 256])
        n, N = _log(rng, 1, 12), _log(rng, 20, 6000)
        n = max(1, min(n, 140_000_000 // (layers * W * N * width)))
        N = min(N, 140_000_000 // (layers * W * n * width))
        moved = rng.randint(1, W)
        return {"kind": kind, "dtype": dtype, "layers": layers, "n": n, "W": W, "N": N, "width": width, "moved": moved,
                "sources": rng.randint(1, moved)}
    if kind == "weights":
        H, c = rng.choice([4, 8, 12, 16, 32]), rng.choice([64, 128])
        if rng.random() < 0.3:  # a prompt, or a chunk of one
            T = _log(rng, 64, 2048)
            N = T + rng.choice([0, 0, _log(rng, 1, 2048)])
            B = max(1, min(_log(rng, 1, 4), 250_000_000 // (T * H * N)))
            return {"kind": kind, "dtype": dtype, "B": B, "T": T, "H": H, "c": c, "N": N}
        T, N = rng.randint(1, 9), _log(rng, 30, 16000)
        B = max(1, min(_log(rng, 1, 64), 400_000 // N))
        return {"kind": kind, "dtype": dtype, "B": B, "T": T, "H": H, "c": c, "N": N}
    layers, width, N = rng.randint(1, 24), rng.choice([64, 128, 256]), _log(rng, 200, 16000)
    B = max(1, min(_log(rng, 1, 16), 300_000_000 // (layers * N * width)))
    return {"kind": kind, "dtype": dtype, "layers": layers, "B": B, "N": N, "keep": rng.randint(FIRST + RECENT + 1, N - 1),
            "width": width}


def _lengths(low, high, count, generator, device):
    """count lengths between low and high, evenly spread, in a seeded order;
    their sum does not depend on the seed."""
    even = torch.linspace(low, high, count, dtype=torch.float64).round().long() if count > 1 else torch.tensor([high])
    return even.to(device)[torch.randperm(count, generator=generator, device=device)]


def _span(case):
    """The shortest and the longest text of a case whose rows have lengths."""
    if case["kind"] == "reorder":
        return max(1, case["N"] // 2), case["N"]
    return max(case["keep"] // 2, FIRST + RECENT), case["N"]


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=device)

    if kind == "beam":
        n, W, V = case["n"], case["W"], case["V"]
        scores = 2.5 * normal(n, W, V)
        banned = uniform(n, 1, V) < 0.02  # tokens a text may not write
        banned[:, :, STOP] = False
        scores.masked_fill_(banned, -math.inf)
        if W > 2:  # a beam that may write nothing more
            scores[n // 2, W - 2] = -math.inf
        totals = -(40 * uniform(n, W)).sort(-1).values - 3
        ended = uniform(n, W) < 0.1
        ended[:, 0] = False
        return {"case": case, "scores": scores.to(dtype), "totals": totals, "ended": ended}
    if kind == "reorder":
        L, n, W, N, width = (case[k] for k in ("layers", "n", "W", "N", "width"))
        stacked = normal(L, n * W, N, width).to(dtype)
        parents = torch.arange(W, device=device).repeat(n, 1)
        for t in range(n):  # `moved` beams of each text take the states of `sources` others
            order = torch.randperm(W, generator=g, device=device)
            movers, held = order[:case["moved"]], order[torch.arange(case["sources"], device=device) - case["sources"]]
            take = held[torch.arange(case["moved"], device=device) % case["sources"]]
            parents[t, movers] = torch.where(take == movers, (movers + 1) % W, take)
        lengths = _lengths(*_span(case), n, g, device).repeat_interleave(W)
        return {"case": case, "stacked": stacked, "tables": stacked.unbind(0), "parents": parents, "lengths": lengths}
    if kind == "weights":
        B, T, H, c, N = (case[k] for k in ("B", "T", "H", "c", "N"))
        # normed queries and keys, the keys with a common part that makes some rows heavy
        q = torch.nn.functional.normalize(normal(B, T, H, c), dim=-1) * c ** 0.5
        table = normal(B, N, 2 * c)
        table[..., :c] += 2 * uniform(B, N, 1) * normal(B, 1, c) * (uniform(B, N, 1) < 0.1)
        table[..., :c] = torch.nn.functional.normalize(table[..., :c], dim=-1) * c ** 0.5
        q, table = q.to(dtype), table.to(dtype)
        start = _lengths(max(0, (N - T) // 2), N - T, B, g, device)
        positions = start[:, None] + torch.arange(T, device=device)
        counts = torch.full((B,), T, device=device)
        if B > 1 and T > 1:  # one padded row
            counts[-1] = (T + 1) // 2
        k = table[..., :c]
        scores = (q.float().reshape(B, T * H, c) @ k.float().transpose(1, 2).contiguous()).view(B, T, H, N) * c ** -0.5
        scores.masked_fill_((torch.arange(N, device=device) > positions[..., None])[:, :, None], -math.inf)
        lse = scores.logsumexp(-1)
        weights = 4 * uniform(B, N) ** 4
        return {"case": case, "q": q, "k": k, "positions": positions, "lse": lse, "start": start, "counts": counts,
                "weights": weights}
    L, B, N, width = (case[k] for k in ("layers", "B", "N", "width"))
    stacked = normal(L, B, N, width).to(dtype)
    weights = 1 / (1e-3 + uniform(L, B, N)) * (uniform(L, B, N) < 0.9)  # a few heavy rows, some that were never read
    lengths = _lengths(*_span(case), B, g, device)
    return {"case": case, "stacked": stacked, "tables": stacked.unbind(0), "weights": weights, "lengths": lengths}


# ---- the plain forms ---------------------------------------------------------


def _beam_plain(scores, totals, ended, K):
    """Ranked in 64 bits, so that equal and nearly equal values fall the same way."""
    n, W, V = scores.shape
    x = scores.double()
    top = x.amax(-1, keepdim=True)
    alive = torch.isfinite(top) & torch.isfinite(totals.double())[..., None]
    total = (x - top).exp().sum(-1, keepdim=True)
    value = totals.double()[..., None] + (x - (top + total.log()))
    value = torch.where(alive & ~ended[..., None] & ~torch.isnan(value), value, -math.inf)
    value[:, :, STOP] = torch.where(ended, totals.double(), value[:, :, STOP])
    best, at = value.view(n, W * V).sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    parents, tokens = at // V, at % V
    return best.float(), parents, tokens, ended.gather(1, parents) | (tokens == STOP)


def _reorder_plain(stacked, parents, lengths):
    n, W = parents.shape
    source = (torch.arange(n, device=parents.device)[:, None] * W + parents).view(-1)
    live = torch.arange(stacked.shape[2], device=parents.device) < lengths[source][:, None]
    stacked.copy_(torch.where(live[None, :, :, None], stacked[:, source], stacked))
    return stacked


def _weights_plain(q, k, positions, lse, scale, weights, counts, start):
    B, T, H, c = q.shape
    N = k.shape[1]
    rows = torch.arange(N, device=q.device)
    scores = (q.float().reshape(B, T * H, c) @ k.float().transpose(1, 2).contiguous()).view(B, T, H, N) * scale
    counted = torch.arange(T, device=q.device) < counts[:, None]
    seen = (rows <= positions[..., None]) & counted[..., None]
    got = torch.where(seen[:, :, None], (scores - lse[..., None]).exp(), 0).sum((1, 2))
    last = torch.where(counted, positions, -1).amax(1, keepdim=True)
    before = torch.where(rows < start[:, None], weights, 0)
    weights.copy_(torch.where(rows <= last, before + got, weights))
    return weights


def _evict_plain(stacked, weights, lengths, keep):
    L, B, N, width = stacked.shape
    rows = torch.arange(N, device=weights.device)
    inside = rows < lengths[:, None]
    held = inside & ((rows < FIRST) | (rows >= lengths[:, None] - RECENT) | (lengths[:, None] <= keep))
    order = torch.where(inside & ~held, weights, -math.inf).sort(dim=-1, descending=True, stable=True).indices
    rank = order.argsort(-1)
    kept = torch.where(held | (inside & (rank < keep - FIRST - RECENT)), rows, N).sort(-1).values[..., :keep]
    live = (kept < N)[..., None]
    moved = stacked.gather(2, kept.clamp(max=N - 1)[..., None].expand(-1, -1, -1, width))
    stacked[:, :, :keep] = torch.where(live, moved, stacked[:, :, :keep])
    return torch.where(kept < N, kept, -1), lengths.clamp(max=keep), stacked


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from wpt_amd import kernels, sampling
    if kind == "beam":
        if own:
            return sampling.beam_step(state["scores"], state["totals"], state["ended"], stops=(STOP,))
        return _beam_plain(state["scores"], state["totals"], state["ended"], case["W"])
    if kind == "reorder":
        if own:
            kernels.reorder_rows(state["tables"], state["parents"], state["lengths"])
            return state["stacked"]
        return _reorder_plain(state["stacked"], state["parents"], state["lengths"])
    if kind == "weights":
        scale = case["c"] ** -0.5
        if own:
            return kernels.add_attention_weights(state["q"], state["k"], state["positions"], state["lse"], scale,
                                                 state["weights"], counts=state["counts"], start=state["start"])
        return _weights_plain(state["q"], state["k"], state["positions"], state["lse"], scale, state["weights"],
                              state["counts"], state["start"])
    # the weights stay in their places, so that every pass chooses and moves alike
    if own:
        kept, counts = kernels.choose_kept(state["weights"], state["lengths"], case["keep"], first=FIRST, recent=RECENT)
        kernels.keep_rows(state["tables"], kept, counts)
        return kept, counts, state["stacked"]
    return _evict_plain(state["stacked"], state["weights"], state["lengths"], case["keep"])


def work(case):
    kind, size = case["kind"], 2 if case["dtype"] == "bf16" else 4
    if kind == "beam":
        n, W, V = case["n"], case["W"], case["V"]
        return {"bytes": n * W * (V * size + 4 + 1 + 4 + 8 + 8 + 1), "flops": 4 * n * W * V}
    if kind == "reorder":
        low, high = _span(case)
        rows = (low + high) / 2 if case["n"] > 1 else high
        moving = case["moved"] + case["sources"]  # written, and read
        return {"bytes": case["layers"] * case["n"] * rows * moving * case["width"] * size, "flops": 0}
    if kind == "weights":
        B, T, H, c, N = (case[k] for k in ("B", "T", "H", "c", "N"))
        low = max(0, (N - T) // 2)
        start = (low + N - T) / 2 if B > 1 else N - T
        pairs = B * H * T * (start + (T + 1) / 2)
        moved = (start + T) * (c * size + 8) + T * H * (c * size + 4)
        return {"bytes": B * moved, "flops": pairs * (2 * c + 3)}
    L, B, keep = case["layers"], case["B"], case["keep"]
    low, high = _span(case)
    lengths = [round(low + (high - low) * i / (B - 1)) for i in range(B)] if B > 1 else [high]
    over = sum(1 for x in lengths if x > keep)
    return {"bytes": L * (over * (keep - FIRST) * 2 * case["width"] * size + sum(lengths) * 4 + B * keep * 8),
            "flops": 0}


# ---- 64 bits -------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "beam":
        x, totals, ended = state["scores"].double(), state["totals"].double(), state["ended"]
        n, W, V = x.shape
        logs = torch.nan_to_num(torch.log_softmax(x, -1), nan=-math.inf, neginf=-math.inf)
        for t in range(n):
            for w in range(W):
                if ended[t, w]:
                    logs[t, w] = -math.inf
                    logs[t, w, STOP] = 0
        value = (logs + totals[..., None]).reshape(n, W * V)
        return torch.topk(value, W, -1).values, None, None, None
    if kind == "reorder":
        tables, old = state["stacked"], state["stacked"].clone()
        n, W = state["parents"].shape
        for t, row in enumerate(state["parents"].tolist()):
            for w, parent in enumerate(row):
                m = int(state["lengths"][t * W + parent])
                tables[:, t * W + w, :m] = old[:, t * W + parent, :m]
        return tables
    if kind == "weights":
        out = state["weights"].double()
        for b in range(case["B"]):
            m = int(state["counts"][b])
            first = int(state["start"][b])
            out[b, first:first + m] = 0
            k = state["k"][b].double()
            for t0 in range(0, m, 512):
                t1 = min(m, t0 + 512)
                s = torch.tensordot(state["q"][b, t0:t1].double(), k, ([2], [1])) * case["c"] ** -0.5
                s = (s - state["lse"][b, t0:t1, :, None].double()).exp()
                for i, p in enumerate(state["positions"][b, t0:t1].tolist()):
                    s[i, :, p + 1:] = 0
                out[b] += s.sum((0, 1))
        return out
    tables, keep = state["stacked"], case["keep"]
    for layer in range(case["layers"]):
        for b, m in enumerate(state["lengths"].tolist()):
            if m > keep:
                middle = state["weights"][layer, b, FIRST:m - RECENT].double()
                best = torch.sort(-middle, stable=True).indices[:keep - FIRST - RECENT].sort().values + FIRST
                ends = [torch.arange(FIRST, device=best.device), torch.arange(m - RECENT, m, device=best.device)]
                tables[layer, b, :keep] = tables[layer, b, torch.cat([ends[0], best, ends[1]])]
    return None, None, tables
