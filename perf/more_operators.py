"""The mixture of experts and the log-probabilities of written tokens, as
measurable cases: a router's choice of experts with their gates, a whole
mixture-of-experts layer for the tokens of a verify step (the router, the
experts' gate/up products with SwiGLU, their down products, the gated sum),
and the log-probability, the entropy and the likeliest alternatives of given
tokens from a head's logits.

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


def listed():
    return [
        # the small decoder's width, one token: launches are all there is
        {"name": "route_one_token", "kind": "route", "dtype": "bf16", "B": 1, "T": 1, "D": 256, "E": 8, "k": 2, "bias": False},
        # the headline verify step's rows: 32 texts, the pending token and 4 drafts, some texts with fewer; a
        # load-balanced router's bias
        {"name": "route_verify", "kind": "route", "dtype": "bf16", "B": 32, "T": 5, "D": 2048, "E": 64, "k": 8, "bias": True},
        # one token of a small decoder
        {"name": "moe_small", "kind": "moe", "dtype": "bf16", "B": 1, "T": 1, "D": 256, "E": 8, "k": 2, "F": 704,
         "bias": False},
        # one token of a large decoder with the feed-forward block cut into fine experts: a decode step without drafts
        {"name": "moe_one_token", "kind": "moe", "dtype": "bf16", "B": 1, "T": 1, "D": 2048, "E": 64, "k": 8, "F": 704,
         "bias": False},
        # its verify step: 32 texts of up to 5 rows, every expert read, about 20 rows an expert
        {"name": "moe_verify", "kind": "moe", "dtype": "bf16", "B": 32, "T": 5, "D": 2048, "E": 64, "k": 8, "F": 704,
         "bias": True},
        # few wide experts, each the large decoder's whole feed-forward block, 16 texts of one token
        {"name": "moe_wide_experts", "kind": "moe", "dtype": "bf16", "B": 16, "T": 1, "D": 2048, "E": 8, "k": 2, "F": 5632,
         "bias": False},
        # FP32, odd counts and widths
        {"name": "moe_fp32", "kind": "moe", "dtype": "fp32", "B": 6, "T": 7, "D": 776, "E": 11, "k": 3, "F": 500,
         "bias": True},
        # the most rows of a verify step (512) over many experts, about 32 rows an expert
        {"name": "moe_largest", "kind": "moe", "dtype": "bf16", "B": 64, "T": 8, "D": 2048, "E": 128, "k": 8, "F": 704,
         "bias": False},
        # the token that one text of the small decoder just wrote, with 5 alternatives
        {"name": "logprobs_one_token", "kind": "logprobs", "dtype": "fp32", "B": 1, "T": 1, "V": 8192, "top": 5,
         "temperature": 1.0},
        # a verify step's tokens from the bf16 logits as the head writes them, with 20 alternatives
        {"name": "logprobs_verify", "kind": "logprobs", "dtype": "bf16", "B": 32, "T": 5, "V": 32768, "top": 20,
         "temperature": 0.8},
        # FP32 logits over an odd vocabulary, whose rows are not aligned
        {"name": "logprobs_odd_vocab", "kind": "logprobs", "dtype": "fp32", "B": 3, "T": 67, "V": 50257, "top": 8,
         "temperature": 1.0},
        # scoring given texts: every token of two prompts, no alternatives
        {"name": "logprobs_prompt", "kind": "logprobs", "dtype": "bf16", "B": 2, "T": 1024, "V": 32768, "top": 0,
         "temperature": 1.0},
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["route", "moe", "moe", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "logprobs":
        V = _log(rng, 500, 131072)
        rows = min(_log(rng, 1, 2048), max(1, 60_000_000 // V) if dtype == "bf16" else max(1, 30_000_000 // V))
        T = min(rows, _log(rng, 1, 64))
        return {"kind": kind, "dtype": dtype, "B": rows // T, "T": T, "V": V, "top": rng.choice([0, 0, 1, rng.randint(2, 32)]),
                "temperature": rng.choice([1.0, 1.0, rng.uniform(0.3, 1.5)])}
    B, T = _log(rng, 1, 64), rng.randint(1, 8)
    E = _log(rng, 2, 128)
    k = rng.randint(1, min(8, E))
    D = 8 * _log(rng, 8, 512)
    case = {"kind": kind, "dtype": dtype, "B": B, "T": T, "D": D, "E": E, "k": k}
    if kind == "moe":
        most = 500_000_000 // (3 * E * D) // (2 if dtype == "fp32" else 1)
        case["F"] = min(_log(rng, 32, 5632), most)
        products = 1_300_000_000 if dtype == "fp32" else 5_900_000_000  # FP32 products cost more than bf16 ones
        case["B"] = min(B, max(1, products // (D * case["F"] * k * T)))
    case["bias"] = rng.random() < 0.5
    return case


def _inputs(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    B, T = case["B"], case["T"]

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device=device).normal_(0, std, generator=g)

    if case["kind"] == "logprobs":
        scores = 2.5 * normal(B, T, case["V"])
        scores.masked_fill_(torch.rand(B, 1, case["V"], generator=g, device=device) < 0.02, -math.inf)  # banned tokens
        scores = scores.to(dtype)
        # tokens drawn from the distribution, as a Writer draws them
        race = torch.empty(B, T, case["V"], device=device).exponential_(generator=g)
        tokens = (scores.float() / case["temperature"] - race.log()).argmax(-1)
        return {"case": case, "scores": scores, "tokens": tokens}
    D, E = case["D"], case["E"]
    # rows as RMSNorm leaves them, with a part that all share, so that some experts get more rows than others
    x = normal(B, T, D) + 0.3 * normal(D)
    x = (x * x.square().mean(-1, keepdim=True).rsqrt()).to(dtype)
    state = {"case": case, "x": x, "router": normal(E, D, std=D ** -0.5),
             "bias": normal(E, std=0.3) if case["bias"] else None}
    # each text's tokens in this reading, the others padding; their sum does not depend on the seed
    counts = torch.linspace(T, max(1, T // 2), B, dtype=torch.float64).round().long()
    state["counts"] = counts.to(device)[torch.randperm(B, generator=g, device=device)]
    if case["kind"] == "moe":
        state["gate_up"] = normal(E, 2 * case["F"], D, std=D ** -0.5, dtype=dtype)
        state["down"] = normal(E, D, case["F"], std=case["F"] ** -0.5, dtype=dtype)
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if own and case["kind"] == "moe":  # laid out once, kept instead of the matrices
        from wpt_amd import experts
        state["weights"] = experts.ExpertWeights(state.pop("gate_up"), state.pop("down"))
    return state


# ---- the plain forms ---------------------------------------------------------


def _route_plain(x, router, k, bias, counts):
    """Ranked in 64 bits, so that nearly equal logits fall the same way."""
    B, T, D = x.shape
    logits = x.double().view(B * T, D) @ router.double().T
    value = logits if bias is None else logits + bias.double()
    order = value.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    logits = logits.gather(1, order)
    weight = (logits - logits.amax(-1, keepdim=True)).exp()
    gates = (weight / weight.sum(-1, keepdim=True)).float()
    read = (torch.arange(T, device=x.device) < counts[:, None]).view(B * T, 1)
    chosen = torch.where(read, order, -1).to(torch.int32)
    return chosen.view(B, T, k), torch.where(read, gates, 0).view(B, T, k)


def _moe_plain(x, router, gate_up, down, k, bias, counts):
    B, T, D = x.shape
    chosen, gates = _route_plain(x, router, k, bias, counts)
    rows, flat, gate = x.float().view(B * T, D), chosen.view(B * T, k), gates.view(B * T, k)
    y = torch.zeros_like(rows)
    for e in range(gate_up.shape[0]):
        token, slot = (flat == e).nonzero(as_tuple=True)
        if token.numel():
            g, u = (rows[token] @ gate_up[e].float().T).chunk(2, -1)
            act = g / (1 + (-g).exp()) * u
            y[token] += (act @ down[e].float().T) * gate[token, slot, None]
    return y.to(x.dtype).view(B, T, D), chosen, gates


def _logprobs_plain(scores, tokens, top, temperature):
    x = scores.float() / temperature
    high = x.amax(-1, keepdim=True)
    weight = (x - high).exp()
    total = weight.sum(-1, keepdim=True)
    logs = (x - high) - total.log()
    entropy = -torch.where(weight > 0, weight / total * logs, 0).sum(-1)
    ids = scores.float().sort(dim=-1, descending=True, stable=True).indices[..., :top] if top else tokens[..., None][..., :0]
    return logs.gather(-1, tokens[..., None])[..., 0], entropy, ids, logs.gather(-1, ids)


def run(state):
    case = state["case"]
    if own:
        from wpt_amd import experts, sampling
    if case["kind"] == "route":
        route = experts.route if own else _route_plain
        return route(state["x"], state["router"], case["k"], state["bias"], state["counts"])
    if case["kind"] == "moe":
        if own:
            return experts.mixture(state["x"], state["router"], state["weights"], case["k"], state["bias"], state["counts"])
        return _moe_plain(state["x"], state["router"], state["gate_up"], state["down"], case["k"], state["bias"],
                          state["counts"])
    log_probs = sampling.log_probs if own else _logprobs_plain
    return log_probs(state["scores"], state["tokens"], case["top"], case["temperature"])


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    M = case["B"] * case["T"]
    if case["kind"] == "logprobs":
        return {"bytes": M * (case["V"] * size + 8 + 4 + 4 + case["top"] * 12), "flops": 4 * M * case["V"]}
    D, E, k = case["D"], case["E"], case["k"]
    T = case["T"]
    M = sum(round(T + (max(1, T // 2) - T) * i / max(1, case["B"] - 1)) for i in range(case["B"]))  # the rows read
    routing = M * D * size + E * D * 4 + M * k * 8
    if case["kind"] == "route":
        return {"bytes": routing, "flops": 2 * M * E * D}
    hit = E * (1 - (1 - k / E) ** M)  # the experts that some row chooses
    return {"bytes": routing + hit * 3 * D * case["F"] * size + M * D * size,
            "flops": 2 * M * E * D + 6 * M * k * D * case["F"]}


# ---- 64 bits -------------------------------------------------------------------


def exact(case, seed):
    state = _inputs(case, seed)
    if case["kind"] == "logprobs":
        logs = torch.log_softmax(state["scores"].double() / case["temperature"], -1)
        entropy = -torch.nan_to_num(logs.exp() * logs, nan=0.0).sum(-1)  # a banned token's 0 times -inf
        best = torch.topk(logs, case["top"], -1).values
        return torch.take_along_dim(logs, state["tokens"][..., None], -1).squeeze(-1), entropy, None, best
    x, B, T, k = state["x"].double(), case["B"], case["T"], case["k"]
    logits = torch.tensordot(x, state["router"].double(), ([2], [1]))
    value = logits if state["bias"] is None else logits + state["bias"].double()
    chosen = torch.topk(value, k, -1).indices
    gates = torch.softmax(torch.take_along_dim(logits, chosen, -1), -1)
    for b, count in enumerate(state["counts"].tolist()):
        gates[b, count:] = 0
    if case["kind"] == "route":
        return None, gates
    share = torch.zeros_like(logits).scatter_(-1, chosen, gates)  # each token's gate of each expert
    y = torch.zeros_like(x)
    for e in range(case["E"]):
        rows = share[..., e] > 0
        h = torch.tensordot(x[rows], state["gate_up"][e].double(), ([1], [1]))
        g, u = h[:, :case["F"]], h[:, case["F"]:]
        act = g * torch.sigmoid(g) * u
        y[rows] += share[..., e][rows][:, None] * torch.tensordot(act, state["down"][e].double(), ([1], [1]))
    return y, None, gates
