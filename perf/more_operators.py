"""Operators of the half of a decoder layer behind the attention, as cases to be measured.

* ``norm``:    the attention's output added to the residual stream, its RMSNorm,
  and the normalised values in 8 bits with a scale for every 128
  (``feedforward.residual_rms_norm``).
* ``route``:   each token's experts from the router's logits: scores, the bias for
  balance, groups, the top k and their weights (``feedforward.route_experts``).
* ``experts``: the routed experts' gated MLP in 8 bits, summed by those weights
  (``feedforward.expert_mlp`` over ``feedforward.ExpertWeights``).

Where ``own`` is false, ``run`` computes each in elementary torch operations: in
64 bits what is rounded to few bits or compared afterwards (norms, scores), else
in 32, rounded once at the end or where the operator's definition rounds. Sizes
are those of the layer cases beside this file (a model of 7,168 dims, latent
queries of 1,536) and generic ones. Codes come back as e4m3 tensors, whose values
are what the bits stand for, beside the scales that they are to be multiplied by.
"""

import math

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-6
BLOCK = 128  # values that share a scale: of a row, and rows by columns of a weight
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # One decode step of 16 users: a call of launch latency.
        {"name": "norm_decode_16", "kind": "norm", "tokens": 16, "dim": 7168, "residual": True,
         "quantize": True, "dtype": "bf16"},
        # A long prompt's tokens before a projection in 8 bits.
        {"name": "norm_prompt_8k", "kind": "norm", "tokens": 8192, "dim": 7168, "residual": True,
         "quantize": True, "dtype": "bf16"},
        # Latent queries: normalised alone, an odd count of narrow rows.
        {"name": "norm_latent_1023", "kind": "norm", "tokens": 1023, "dim": 1536,
         "residual": False, "quantize": False, "dtype": "bf16"},
        # One decode step's routing: 8 of 256 experts, from 4 of 8 groups.
        {"name": "route_decode_16", "kind": "route", "tokens": 16, "experts": 256, "k": 8,
         "groups": 8, "top_groups": 4, "scoring": "sigmoid", "bias": True, "renormalize": True,
         "dtype": "fp32"},
        # A batch of long prompts.
        {"name": "route_prompt_16k", "kind": "route", "tokens": 16384, "experts": 256, "k": 8,
         "groups": 8, "top_groups": 4, "scoring": "sigmoid", "bias": True, "renormalize": True,
         "dtype": "fp32"},
        # Softmax scores as they are, from 16-bit logits, an odd count of tokens.
        {"name": "route_softmax_4099", "kind": "route", "tokens": 4099, "experts": 160, "k": 6,
         "groups": 8, "top_groups": 3, "scoring": "softmax", "bias": False,
         "renormalize": False, "dtype": "bf16"},
        # One token's 8 experts: their weights are read, little else is done.
        {"name": "experts_1", "kind": "experts", "tokens": 1, "dim": 7168, "inner": 2048,
         "experts": 32, "total": 32, "k": 8},
        # A decode step of 64 users: some 16 rows an expert.
        {"name": "experts_64", "kind": "experts", "tokens": 64, "dim": 7168, "inner": 2048,
         "experts": 32, "total": 32, "k": 8},
        # One rank's quarter of a smaller model's experts, an odd count of tokens.
        {"name": "experts_slice_777", "kind": "experts", "tokens": 777, "dim": 2048,
         "inner": 1408, "experts": 24, "total": 96, "k": 6},
        # A prompt's tokens: some 2,048 rows an expert, matrix products.
        {"name": "experts_8192", "kind": "experts", "tokens": 8192, "dim": 7168, "inner": 2048,
         "experts": 32, "total": 32, "k": 8},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choice(["norm", "route", "experts", "experts"])
    if kind == "norm":
        dim = rng.choice([512, 1536, 2048, 4096, 7168, BLOCK * rng.randint(1, 64)])
        return {"kind": "norm", "tokens": _log(rng, 1, 8192), "dim": dim,
                "residual": rng.random() < 0.7, "quantize": rng.random() < 0.7,
                "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if kind == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * rng.choice([2, 8, 15, 20, 32, 48])
        top_groups = groups if groups == 1 else rng.randint(1, groups)
        return {"kind": "route", "tokens": _log(rng, 1, 16384), "experts": experts,
                "k": rng.randint(1, min(8, top_groups * (experts // groups))), "groups": groups,
                "top_groups": top_groups, "scoring": rng.choice(["sigmoid", "softmax"]),
                "bias": rng.random() < 0.5, "renormalize": rng.random() < 0.6,
                "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"])}
    dim = rng.choice([1024, 2048, 4096, 7168, BLOCK * rng.randint(4, 40)])
    inner = rng.choice([512, 768, 1408, 2048, BLOCK * rng.randint(1, 16)])
    experts = rng.choice([1, 8, 16, 24, 32])
    total = experts * rng.choice([1, 1, 2, 4])
    return {"kind": "experts", "tokens": _log(rng, 1, 6000), "dim": dim, "inner": inner,
            "experts": experts, "total": total, "k": rng.randint(1, min(8, total))}


# ------------------------------------------------------------------ inputs --
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=dtype)


def _power_of_two(amax):
    """The scale of values up to ``amax`` (32 bits): the power of two at or above amax / 448."""
    bits = (amax.clamp_min(1e-4) * (1.0 / 448.0)).view(torch.int32)
    return ((bits + 0x7FFFFF) & 0x7F800000).view(torch.float32)


def _codes(values):
    """Rows in 8 bits: e4m3 codes and a power-of-two scale for every 128 values."""
    parts = values.float().unflatten(-1, (-1, BLOCK))
    scale = _power_of_two(parts.abs().amax(-1))
    codes = (parts / scale[..., None]).clamp(-448, 448).to(E4M3)
    return codes.flatten(-2), scale.to(E8M0)


def _weight_codes(gen, experts, rows, columns):
    """A weight for each expert, e4m3 with a scale for every 128 rows by 128 columns."""
    values = _randn(gen, experts, rows // BLOCK, BLOCK, columns // BLOCK, BLOCK)
    values *= columns ** -0.5
    scale = _power_of_two(values.abs().amax((2, 4)).float())
    codes = torch.empty_like(values, dtype=E4M3)
    for e in range(experts):
        codes[e] = (values[e].float() / scale[e, :, None, :, None]).clamp(-448, 448).to(E4M3)
    return codes.view(experts, rows, columns), scale.to(E8M0)


def prepare(case, seed):
    gen, kind = _generator(seed), case["kind"]
    state = {"case": dict(case)}
    if kind == "norm":
        # A residual stream of a few outlying dims, what the attention adds to it.
        tokens, dim, dtype = case["tokens"], case["dim"], DTYPES[case["dtype"]]
        loud = 1 + 20 * (torch.rand(dim, generator=gen, device=DEVICE) < 0.01)
        stream = _randn(gen, tokens, dim, dtype=torch.float32) * loud
        state.update(x=_randn(gen, tokens, dim, dtype=torch.float32).to(dtype),
                     weight=1 + 0.1 * _randn(gen, dim, dtype=torch.float32))
        if case["residual"]:
            state["residual"] = stream.to(dtype)
        else:
            state.update(x=stream.to(dtype), residual=None)
    elif kind == "route":
        # Logits of tokens that prefer some experts, a bias that evens them out in part.
        tokens, experts = case["tokens"], case["experts"]
        liked = _randn(gen, experts, dtype=torch.float32)
        logits = _randn(gen, tokens, experts, dtype=torch.float32) + 0.5 * liked
        state.update(logits=logits.to(DTYPES[case["dtype"]]),
                     bias=-0.05 * liked if case["bias"] else None,
                     scale=2.5 if case["renormalize"] else 16.0)
    else:
        # Normalised tokens in 8 bits, their experts (some better liked) and weights, and
        # this rank's experts: those from `first` on, in the middle of all.
        tokens, dim, inner = case["tokens"], case["dim"], case["inner"]
        experts, total, k = case["experts"], case["total"], case["k"]
        first = (total - experts) // 2
        x, x_scale = _codes(_randn(gen, tokens, dim))
        scores = _randn(gen, tokens, total, dtype=torch.float32)
        scores = torch.sigmoid(scores + 0.3 * _randn(gen, total, dtype=torch.float32))
        top, ids = scores.topk(k)
        gate_up, gate_up_scale = _weight_codes(gen, experts, 2 * inner, dim)
        down, down_scale = _weight_codes(gen, experts, dim, inner)
        # (What the plain form pads each expert's rows to.)
        rows = torch.bincount(ids.flatten(), minlength=total)[first:first + experts]
        state.update(x=x, x_scale=x_scale, ids=ids.to(torch.int32), first=first,
                     weights=2.5 * top / top.sum(1, keepdim=True), most=int(rows.max()),
                     parts=(gate_up, gate_up_scale, down, down_scale))
        if own:
            # The weights as the kernels read them, laid out once when a model is loaded.
            from cxldsagr_amd import feedforward

            state["packed"] = feedforward.ExpertWeights(*state["parts"], first=first,
                                                        total=total)
    return state


# -------------------------------------------------------------- plain form --
def _norm_plain(state):
    x, residual, case = state["x"], state["residual"], state["case"]
    total = x.float()
    if residual is not None:
        total = total + residual.float()
    wide = total.double()
    normed = wide * torch.rsqrt((wide * wide).mean(-1, keepdim=True) + EPS)
    values = (normed * state["weight"].double()).to(x.dtype)
    out = {"values": values}
    if residual is not None:
        out["residual"] = total.to(x.dtype)
    if case["quantize"]:
        out["codes"], out["scales"] = _codes(values)
    return out


def _route_plain(state):
    case, logits = state["case"], state["logits"].double()
    tokens, experts, groups = case["tokens"], case["experts"], case["groups"]
    if case["scoring"] == "sigmoid":
        scores = torch.sigmoid(logits).float()
    else:
        scores = torch.exp(logits - logits.amax(1, keepdim=True))
        scores = (scores / scores.sum(1, keepdim=True)).float()
    ranked = scores if state["bias"] is None else scores + state["bias"]
    if case["top_groups"] < groups:
        each = ranked.view(tokens, groups, experts // groups)
        best = each.sort(dim=-1, descending=True)[0]
        size = best[..., 0] if state["bias"] is None or experts == groups else best[..., 0] + best[..., 1]
        order = size.sort(dim=-1, descending=True, stable=True)[1]
        kept = torch.zeros_like(size, dtype=torch.bool)
        kept.scatter_(1, order[:, :case["top_groups"]], True)
        ranked = each.masked_fill(~kept[..., None], -math.inf).view(tokens, experts)
    ids = ranked.sort(dim=-1, descending=True, stable=True)[1][:, :case["k"]]
    weights = scores.gather(1, ids)
    if case["renormalize"]:
        weights = weights / (weights.sum(1, keepdim=True) + 1e-20)
    return [weights * state["scale"], ids.to(torch.int32)]


def _dequantised(codes, scale):
    """Weights ``[n, rows, columns]`` of 8 bits and a scale per 128 by 128, in 32 bits."""
    n, rows, columns = codes.shape
    parts = codes.float().view(n, rows // BLOCK, BLOCK, columns // BLOCK, BLOCK)
    return (parts * scale.float()[:, :, None, :, None]).view(n, rows, columns)


def _experts_plain(state):
    case = state["case"]
    tokens, dim, inner, k = case["tokens"], case["dim"], case["inner"], case["k"]
    experts, most = case["experts"], state["most"]
    gate_up, gate_up_scale, down, down_scale = state["parts"]
    # (Token, choice) pairs by expert, each at its place in a padded batch of rows.
    mine = state["ids"].flatten().long() - state["first"]
    mine = torch.where((mine >= 0) & (mine < experts), mine, experts)
    taken, order = mine.sort(stable=True)
    starts = torch.searchsorted(taken, torch.arange(experts + 1, device=DEVICE))
    place = torch.arange(tokens * k, device=DEVICE) - starts[taken]
    place = torch.where(taken < experts, taken * most + place, experts * most)
    rows = torch.zeros(experts * most + 1, dtype=torch.long, device=DEVICE)
    rows[place] = order // k
    x = (state["x"].float().view(tokens, -1, BLOCK) * state["x_scale"].float()[..., None])
    x = x.view(tokens, dim)[rows[:-1]].view(experts, most, dim)
    both = torch.matmul(x, _dequantised(gate_up, gate_up_scale).transpose(1, 2))
    gate, up = both.split(inner, -1)
    hidden, scale = _codes(gate / (1 + torch.exp(-gate)) * up)
    hidden = (hidden.float().unflatten(-1, (-1, BLOCK)) * scale.float()[..., None]).flatten(-2)
    out = torch.matmul(hidden, _dequantised(down, down_scale).transpose(1, 2)).view(-1, dim)
    at = torch.empty_like(place)
    at[order] = place
    out = torch.cat([out, out.new_zeros(1, dim)])[at].view(tokens, k, dim)
    return (out * state["weights"][..., None]).sum(1).to(torch.bfloat16)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from cxldsagr_amd import feedforward

        if kind == "norm":
            got = feedforward.residual_rms_norm(state["x"], state["weight"], state["residual"],
                                                eps=EPS, quantize=case["quantize"])
            out = {"values": got.values}
            if state["residual"] is not None:
                out["residual"] = got.residual
            if case["quantize"]:
                out["codes"], out["scales"] = got.codes, got.scales
            return out
        if kind == "route":
            return list(feedforward.route_experts(
                state["logits"], case["k"], bias=state["bias"], scoring=case["scoring"],
                groups=case["groups"], top_groups=case["top_groups"],
                renormalize=case["renormalize"], scale=state["scale"]))
        return feedforward.expert_mlp(state["x"], state["x_scale"], state["packed"],
                                      state["ids"], state["weights"])
    if kind == "norm":
        return _norm_plain(state)
    if kind == "route":
        return _route_plain(state)
    return _experts_plain(state)


# -------------------------------------------------------------------- work --
def work(case):
    """What the operator has to read, write and compute."""
    kind, tokens = case["kind"], case["tokens"]
    if kind == "norm":
        size, values = DTYPES[case["dtype"]].itemsize, tokens * case["dim"]
        moved = values * size * (4 if case["residual"] else 2) + 4 * case["dim"]
        if case["quantize"]:
            moved += values + values // BLOCK
        return {"bytes": moved, "flops": 5 * values}
    if kind == "route":
        size = DTYPES[case["dtype"]].itemsize
        return {"bytes": tokens * (case["experts"] * size + case["k"] * 8) + 4 * case["experts"],
                "flops": 20 * tokens * case["experts"]}
    dim, inner, k = case["dim"], case["inner"], case["k"]
    pairs = tokens * k * case["experts"] / case["total"]
    # Experts that at least one token takes, on average.
    used = case["experts"] * (1 - (1 - k / case["total"]) ** tokens)
    return {"bytes": used * 3 * dim * inner * (1 + 1 / BLOCK ** 2)
            + tokens * (dim * (1 + 1 / BLOCK) + 8 * k + 2 * dim),
            "flops": 6 * pairs * dim * inner}


# ------------------------------------------------------------ 64-bit values --
def _e4m3_64(values):
    """The nearest values that e4m3 holds: steps of an eighth of the power of two at or
    below, 2^-9 at the least, up to 448."""
    step = torch.exp2(torch.floor(torch.log2(values.abs().clamp_min(2.0 ** -6))) - 3)
    return ((values / step).round() * step).clamp(-448, 448)


def _scale64(values):
    """Per 128 values: the scale, whose rule is one of 32 bits (the largest times 1/448, up
    to a power of two)."""
    top = values.view(len(values), -1, BLOCK).abs().amax(-1).float().clamp_min(1e-4)
    part, power = torch.frexp(top * (1.0 / 448.0))
    return torch.ldexp(torch.ones_like(top), power - (part == 0.5).to(power.dtype)).double()


def _quantised64(values):
    scale = _scale64(values)
    wide = scale.repeat_interleave(BLOCK, 1)
    return _e4m3_64(values / wide), scale, wide


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "norm":
        total = state["x"].double()
        out = {}
        if state["residual"] is not None:
            # (The sum is one of 32 bits.)
            total = (total + state["residual"].double()).float().double()
            out["residual"] = total
        mean = torch.linalg.vector_norm(total, dim=1, keepdim=True).square() / case["dim"]
        normed = total / (mean + EPS).sqrt() * state["weight"].double()
        out["values"] = normed
        if case["quantize"]:
            out["codes"], out["scales"], _ = _quantised64(normed.to(state["x"].dtype).double())
        return out
    if kind == "route":
        logits, tokens = state["logits"].double(), case["tokens"]
        scores = 1 / (1 + torch.exp(-logits)) if case["scoring"] == "sigmoid" else torch.softmax(logits, 1)
        # Experts are ranked by scores of 32 bits: as whole numbers, an expert's index last.
        ranked = scores.float() if state["bias"] is None else scores.float() + state["bias"]
        bits = (ranked + 0.0).view(torch.int32).long()
        rank = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
        experts, groups = case["experts"], case["groups"]
        index = torch.arange(experts, device=DEVICE)
        if case["top_groups"] < groups:
            each = ranked.view(tokens, groups, -1)
            first, at = each.max(-1, keepdim=True)
            size = first[..., 0]
            if state["bias"] is not None and experts > groups:
                size = size + each.scatter(-1, at, -math.inf).amax(-1)
            beats = (size[:, None, :] > size[:, :, None]) | (
                (size[:, None, :] == size[:, :, None])
                & (torch.arange(groups, device=DEVICE)[None, :] < torch.arange(groups, device=DEVICE)[:, None]))
            kept = (beats.sum(-1) < case["top_groups"]).repeat_interleave(experts // groups, 1)
            rank = torch.where(kept, rank, -2 ** 40)
        ids = (rank * 1024 + (1023 - index)).topk(case["k"], dim=1)[1]
        weights = scores.gather(1, ids)
        if case["renormalize"]:
            weights = weights / weights.sum(1, keepdim=True)
        return [weights * state["scale"], ids]
    dim, inner = case["dim"], case["inner"]
    codes = state["x"].double() * state["x_scale"].double().repeat_interleave(BLOCK, 1)
    out = torch.zeros(case["tokens"], dim, dtype=torch.float64, device=DEVICE)

    def matrix(which, e):
        wide = state["parts"][which + 1][e].double()
        wide = wide.repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)
        return state["parts"][which][e].double() * wide

    for e in range(case["experts"]):
        token, choice = (state["ids"] == e + state["first"]).nonzero(as_tuple=True)
        if not len(token):
            continue
        both = codes[token] @ matrix(0, e).t()
        gate, up = both[:, :inner], both[:, inner:]
        hidden, _, wide = _quantised64(gate * torch.sigmoid(gate) * up)
        rows = (hidden * wide) @ matrix(2, e).t()
        out.index_add_(0, token, rows * state["weights"][token, choice].double()[:, None])
    return out
