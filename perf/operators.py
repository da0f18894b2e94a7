"""Operators of the dense attention path around the DSA layer, as cases to be measured.

* ``rope``:   rotary positions of queries and keys (``projections.apply_rope_pair``).
* ``cache``:  new tokens normalised, rotated and quantised into the fp8 paged
  cache as they are written, and a sequence's records read back as bf16
  (``attention.write_kv_fp8``, ``attention.read_kv_fp8``).
* ``prompt``: causal attention over packed sequences with grouped heads
  (``attention.prompt_attention``), the queries' own tokens alone, after a
  history, or single tokens.
* ``prefix``: MLA attention of branches that share a long prefix in the fp8
  paged cache, each with its own suffix (``attention.shared_prefix_mla``).

Where ``own`` is false, ``run`` computes each in elementary torch operations in
32 bits (rotation angles in 64), rounded once at the end or where the
operator's definition rounds. Sizes are those of the layer cases beside this
file: 128 or fewer heads of 192 = 128 + 64 dims, records of 512 + 64 dims in
656 bytes, pages of 64 tokens, histories up to 65,536.
"""

import math

import torch

own = False

DEVICE = "cuda:0"
LATENT, ROPE, PAGE, RECORD = 512, 64, 64, 656
MAX_POSITION = 163840
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # One decode step's queries of 16 users: a call of launch latency.
        {"name": "rope_decode_16", "kind": "rope", "tokens": 16, "heads": 128, "kv_heads": 1,
         "dim": 64, "offset": 0, "rotated": 64, "layout": "interleaved", "dtype": "bf16"},
        # A long prompt's queries and keys: the rope part of 128 heads.
        {"name": "rope_prompt_8k", "kind": "rope", "tokens": 8192, "heads": 128, "kv_heads": 1,
         "dim": 64, "offset": 0, "rotated": 64, "layout": "interleaved", "dtype": "bf16"},
        # The indexer's layout: the first 64 of 128 dims, half layout, odd count.
        {"name": "rope_index_1023", "kind": "rope", "tokens": 1023, "heads": 64, "kv_heads": 1,
         "dim": 128, "offset": 0, "rotated": 64, "layout": "half", "dtype": "fp32"},
        # 128 candidate tokens appended and read back.
        {"name": "cache_128", "kind": "cache", "history": 0, "tokens": 128},
        # A prompt's chunk after 20,011 tokens: its records written, all read.
        {"name": "cache_20011_1021", "kind": "cache", "history": 20011, "tokens": 1021},
        # A user's whole history.
        {"name": "cache_64k", "kind": "cache", "history": 0, "tokens": 65536},
        # A prompt of 2,048 tokens, all heads of one layer.
        {"name": "prompt_2048", "kind": "prompt", "sequences": 1, "tokens": 2048, "history": 0,
         "heads": 128, "kv_heads": 128, "qk": 192, "v": 128, "dtype": "bf16"},
        # Seven prompts of different lengths in one batch, grouped heads.
        {"name": "prompt_7x_4001", "kind": "prompt", "sequences": 7, "tokens": 4001, "history": 0,
         "heads": 32, "kv_heads": 8, "qk": 128, "v": 128, "dtype": "bf16"},
        # Single tokens of 8 users after histories of different lengths.
        {"name": "prompt_single_8", "kind": "prompt", "sequences": 8, "tokens": 8,
         "history": 40000, "heads": 64, "kv_heads": 8, "qk": 128, "v": 128, "dtype": "fp16"},
        # A request's 64 candidates scored as branches of a 64K history.
        {"name": "prefix_64k_64", "kind": "prefix", "prefix": 65536, "branches": 64, "queries": 1,
         "suffix": 64, "heads": 128},
        # One branch: a single token over a long history.
        {"name": "prefix_32k_1", "kind": "prefix", "prefix": 32768, "branches": 1, "queries": 1,
         "suffix": 128, "heads": 128},
        # Branches of a few new tokens on one half of a tensor-parallel pair.
        {"name": "prefix_4099_13x4_h64", "kind": "prefix", "prefix": 4099, "branches": 13,
         "queries": 4, "suffix": 200, "heads": 64},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choice(["rope", "cache", "prompt", "prompt", "prefix", "prefix"])
    if kind == "rope":
        dim = rng.choice([64, 128, 192])
        rotated = rng.choice([r for r in (32, 64, 128) if r <= dim])
        heads = rng.choice([1, 8, 16, 64, 128])
        return {"kind": "rope", "tokens": _log(rng, 1, min(16384, 2 ** 26 // (heads * dim))),
                "heads": heads, "kv_heads": rng.choice([1, 8]), "dim": dim,
                "offset": rng.choice([0, dim - rotated]), "rotated": rotated,
                "layout": rng.choice(["interleaved", "half"]),
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind == "cache":
        return {"kind": "cache", "history": rng.choice([0, _log(rng, 50, 40000)]),
                "tokens": _log(rng, 1, 24000)}
    if kind == "prompt":
        qk, v = rng.choice([(192, 128), (192, 128), (128, 128), (64, 64)])
        kv_heads, group = rng.choice([1, 2, 8, 16]), rng.choice([1, 2, 5, 8])
        if rng.random() < 0.3:
            sequences = rng.randint(1, 24)
            tokens, history = sequences, _log(rng, sequences, 60000)
        else:
            tokens = _log(rng, 16, 4096)
            sequences = rng.randint(1, max(1, min(9, tokens // 8)))
            history = rng.choice([0, 0, _log(rng, 16, 16384)])
        # The scores of the padded batch, in 32 bits, stay within 4 GiB.
        while tokens > 8 * sequences and (sequences * kv_heads * group * (2 * tokens // sequences)
                                          * (2 * (tokens + history) // sequences)) > 2 ** 30:
            tokens //= 2
        return {"kind": "prompt", "sequences": sequences, "tokens": tokens, "history": history,
                "heads": kv_heads * group, "kv_heads": kv_heads, "qk": qk, "v": v,
                "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    branches = _log(rng, 1, 64)
    queries = rng.choice([1, 1, 1, rng.randint(2, 6)])
    prefix = _log(rng, 100, min(65536, 65536 * 64 // (branches * queries)))
    return {"kind": "prefix", "prefix": rng.choice([prefix, prefix, prefix, 0]),
            "branches": branches, "queries": queries, "suffix": _log(rng, max(queries, 4), 512),
            "heads": rng.choice([64, 128, 128])}


# ------------------------------------------------------------------ inputs --
def _ragged(total, parts, least=1):
    """``parts`` different lengths of at least ``least`` that sum to ``total``."""
    weights = [0.25 + (0.6180339887 * (i + 1)) % 1 for i in range(parts)]
    spare = total - least * parts
    lengths = [least + int(spare * w / sum(weights)) for w in weights]
    lengths[-1] += total - sum(lengths)
    return lengths


def _prompt_lengths(case):
    """Per sequence: its query count and its key count."""
    n = case["sequences"]
    queries = _ragged(case["tokens"], n)
    history = _ragged(case["history"], n, 0)
    return queries, [a + b for a, b in zip(queries, history)]


def _branch_lengths(case):
    """Per branch: its query count and its suffix's length."""
    n, most, suffix = case["branches"], case["queries"], case["suffix"]
    queries = [1 + (3 * i) % most for i in range(n)]
    lengths = [max(q, 1 + (i * 7919 + suffix - 1) % suffix) for i, q in enumerate(queries)]
    return queries, lengths


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen, device=DEVICE).to(dtype)


def _frequencies(rotated):
    """Rotary frequencies stretched for long contexts: below 1 turn in the
    first 4,096 positions by 40, above 32 turns not, in between in part."""
    freq = 10000.0 ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / rotated)
    turns = freq * 4096 / (2 * math.pi)
    keep = (torch.log(turns) / math.log(32.0)).clamp(0, 1)
    return (freq * keep + freq / 40 * (1 - keep)).float().to(DEVICE)


def _cu(lengths):
    return torch.tensor([0] + lengths).cumsum(0).to(device=DEVICE, dtype=torch.int32)


def _quantised(latent, rope):
    """Records of 656 bytes: 512 e4m3 codes, 4 fp32 scales, 64 bf16 values.
    The scale of 128 values is the power of two at or above amax / 448."""
    tiles = latent.float().view(-1, 4, 128)
    amax = tiles.abs().amax(-1).clamp_min(1e-4)
    bits = (amax * (1.0 / 448.0)).view(torch.int32)
    scale = ((bits + 0x7FFFFF) & 0x7F800000).view(torch.float32)
    codes = (tiles / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    parts = [codes.view(-1, LATENT).view(torch.uint8), scale.contiguous().view(torch.uint8),
             rope.to(torch.bfloat16).contiguous().view(torch.uint8)]
    return torch.cat(parts, dim=1)


def _dequantised(records):
    """The values that records stand for, fp32 ``[n, 576]``."""
    codes = records[:, :LATENT].contiguous().view(torch.float8_e4m3fn).float().view(-1, 4, 128)
    scale = records[:, LATENT:LATENT + 16].contiguous().view(torch.float32)
    rope = records[:, LATENT + 16:].contiguous().view(torch.bfloat16).float()
    return torch.cat([(codes * scale[..., None]).view(-1, LATENT), rope], dim=1)


def _slots(table, count):
    place = torch.arange(count, device=DEVICE)
    return table[place // PAGE].long() * PAGE + place % PAGE


def prepare(case, seed):
    gen, kind = _generator(seed), case["kind"]
    state = {"case": dict(case)}
    if kind == "rope":
        # The rope part of wider heads (or the whole of them), at positions
        # anywhere in the context.
        tokens, dtype = case["tokens"], DTYPES[case["dtype"]]
        start = int(torch.randint(MAX_POSITION - tokens, (1,), generator=gen, device=DEVICE))
        wide = case["dim"] + (128 if case["dim"] == 64 else 0)
        state.update(
            q=_randn(gen, tokens, case["heads"], wide, dtype=dtype)[..., wide - case["dim"]:],
            k=_randn(gen, tokens, case["kv_heads"], case["dim"], dtype=dtype),
            positions=torch.arange(start, start + tokens, device=DEVICE, dtype=torch.int32),
            frequencies=_frequencies(case["rotated"]), magnitude=0.1 * math.log(40.0) + 1.0)
    elif kind == "cache":
        # New tokens after a history already in the cache, pages in any order
        # among those of other users.
        history, tokens = case["history"], case["tokens"]
        pages = (history + tokens + PAGE - 1) // PAGE
        table = torch.randperm(pages + pages // 4 + 1, generator=gen, device=DEVICE)[:pages]
        slots = _slots(table, history + tokens)
        cache = torch.zeros(pages + pages // 4 + 1, PAGE, RECORD, dtype=torch.uint8, device=DEVICE)
        if history:
            rows = _randn(gen, history, LATENT + ROPE)
            cache.view(-1, RECORD)[slots[:history]] = _quantised(rows[:, :LATENT], rows[:, LATENT:])
        state.update(
            cache=cache, slots=slots, new=slots[history:].clone(),
            kv=_randn(gen, tokens, LATENT + ROPE),
            weight=1 + 0.1 * torch.randn(LATENT, generator=gen, device=DEVICE),
            positions=torch.arange(history, history + tokens, device=DEVICE, dtype=torch.int32),
            frequencies=_frequencies(ROPE))
    elif kind == "prompt":
        # Keys and values as a layer has them: values in the second part of
        # the rows that hold the keys' position-free part before them.
        queries, keys = _prompt_lengths(case)
        dtype = DTYPES[case["dtype"]]
        total = sum(keys)
        up = _randn(gen, total, case["kv_heads"], 128 + case["v"], dtype=dtype)
        state.update(
            q=_randn(gen, sum(queries), case["heads"], case["qk"], dtype=dtype),
            k=_randn(gen, total, case["kv_heads"], case["qk"], dtype=dtype), v=up[..., 128:],
            cu_q=_cu(queries), cu_k=_cu(keys), max_q=max(queries), max_k=max(keys),
            scale=case["qk"] ** -0.5)
    else:
        queries, lengths = _branch_lengths(case)
        prefix, branches = case["prefix"], case["branches"]
        width = (max(lengths) + PAGE - 1) // PAGE
        own_pages = branches * width
        first = (prefix + PAGE - 1) // PAGE
        order = torch.randperm(first + own_pages, generator=gen, device=DEVICE).to(torch.int32)
        rows = _randn(gen, (first + own_pages) * PAGE, LATENT + ROPE)
        cache = _quantised(rows[:, :LATENT], rows[:, LATENT:]).view(-1, PAGE, RECORD)
        state.update(
            q=_randn(gen, sum(queries), case["heads"], LATENT + ROPE), cache=cache,
            prefix_table=order[:first].contiguous(),
            suffix_tables=order[first:].view(branches, width).contiguous(),
            suffix_tokens=torch.tensor(lengths, device=DEVICE, dtype=torch.int32),
            cu_q=_cu(queries) if case["queries"] > 1 else None, max_q=max(queries),
            scale=(128 + 64) ** -0.5)
    return state


# -------------------------------------------------------------- plain form --
def _rotated(x, cos, sin, case):
    """``x [..., dim]`` (32 bits) with its rotary part turned by ``cos, sin``."""
    a, b = case["offset"], case["offset"] + case["rotated"]
    part = x[..., a:b]
    if case["layout"] == "interleaved":
        one, two = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([one * cos - two * sin, two * cos + one * sin], -1).flatten(-2)
    else:
        one, two = part.chunk(2, -1)
        turned = torch.cat([one * cos - two * sin, two * cos + one * sin], -1)
    return torch.cat([x[..., :a], turned, x[..., b:]], -1)


def _cos_sin(positions, frequencies, magnitude):
    angles = positions.double()[:, None] * frequencies.double()[None, :]
    return (angles.cos() * magnitude).float(), (angles.sin() * magnitude).float()


def _rope_plain(state):
    cos, sin = _cos_sin(state["positions"], state["frequencies"], state["magnitude"])
    cos, sin = cos[:, None], sin[:, None]
    return [_rotated(x.float(), cos, sin, state["case"]).to(x.dtype)
            for x in (state["q"], state["k"])]


def _cache_plain(state):
    kv = state["kv"].float()
    latent, rope = kv[:, :LATENT], kv[:, LATENT:]
    norm = torch.rsqrt((latent * latent).mean(-1, keepdim=True) + EPS)
    latent = (latent * norm * state["weight"]).to(torch.bfloat16)
    cos, sin = _cos_sin(state["positions"], state["frequencies"], 1.0)
    part = {"offset": 0, "rotated": ROPE, "layout": "interleaved"}
    rope = _rotated(rope, cos, sin, part).to(torch.bfloat16)
    records = state["cache"].view(-1, RECORD)
    records[state["new"]] = _quantised(latent, rope)
    return _dequantised(records[state["slots"]]).to(torch.bfloat16)


def _packed_places(cu, most):
    """Rows of a packed tensor as a padded batch, and which of them are real."""
    place = torch.arange(most, device=DEVICE)[None, :]
    starts, ends = cu[:-1, None].long(), cu[1:, None].long()
    real = starts + place < ends
    return torch.where(real, starts + place, torch.zeros_like(starts)), real


def _prompt_plain(state):
    rows_q, real_q = _packed_places(state["cu_q"], state["max_q"])
    rows_k, real_k = _packed_places(state["cu_k"], state["max_k"])
    heads, kv_heads = state["q"].shape[1], state["k"].shape[1]
    group = heads // kv_heads
    q = state["q"].float()[rows_q].transpose(1, 2)  # [B, H, q, qk]
    batch, _, most, width = q.shape
    q = q.reshape(batch, kv_heads, group * most, width)
    k = state["k"].float()[rows_k].permute(0, 2, 3, 1)
    v = state["v"].float()[rows_k].transpose(1, 2)
    scores = torch.matmul(q, k.contiguous()).view(batch, kv_heads, group, most, -1)
    scores *= state["scale"]
    shift = (real_k.sum(1) - real_q.sum(1))[:, None, None]
    sees = (torch.arange(state["max_k"], device=DEVICE)[None, None, :]
            <= torch.arange(most, device=DEVICE)[None, :, None] + shift)
    sees = (sees & real_k[:, None, :] & real_q[:, :, None])[:, None, None]
    scores.masked_fill_(~sees, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(batch, kv_heads, group * most, -1), v.contiguous())
    out = out.view(batch, kv_heads, group, most, -1) / total.clamp_min(1e-30)
    out = out.reshape(batch, heads, most, -1).transpose(1, 2)
    return out[real_q].to(state["q"].dtype)


def _token_views(state):
    """Per query token: its branch and how much of its suffix it sees."""
    tokens = state["q"].shape[0]
    if state["cu_q"] is None:
        branch = torch.arange(tokens, device=DEVICE)
        return branch, state["suffix_tokens"].long()
    cu = state["cu_q"].long()
    place = torch.arange(tokens, device=DEVICE)
    branch = torch.searchsorted(cu[1:].contiguous(), place, right=True)
    return branch, state["suffix_tokens"].long()[branch] - (cu[1:][branch] - 1 - place)


def _prefix_plain(state):
    records, prefix = state["cache"].view(-1, RECORD), state["case"]["prefix"]
    q = state["q"].float()
    tokens, heads, width = q.shape
    shared = _dequantised(records[_slots(state["prefix_table"], prefix)])
    branch, sees = _token_views(state)
    tables = state["suffix_tables"]
    most = tables.shape[1] * PAGE
    place = torch.arange(most, device=DEVICE)
    rows = tables[:, place // PAGE].long() * PAGE + place % PAGE
    tails = _dequantised(records[rows.flatten()]).view(len(tables), most, width)[branch]
    ahead = torch.matmul(q.view(-1, width), shared.t().contiguous()).view(tokens, heads, prefix)
    behind = torch.matmul(q, tails.transpose(1, 2).contiguous())
    behind.masked_fill_((place[None, :] >= sees[:, None])[:, None], -math.inf)
    scores = torch.cat([ahead, behind], -1)
    scores *= state["scale"]
    p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p[..., :prefix].reshape(tokens * heads, prefix), shared[:, :LATENT].contiguous())
    out = out.view(tokens, heads, LATENT)
    out = out + torch.matmul(p[..., prefix:].contiguous(), tails[..., :LATENT].contiguous())
    return (out / total).to(state["q"].dtype)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from cxldsagr_amd import attention, projections

        if kind == "rope":
            return list(projections.apply_rope_pair(
                state["q"], state["k"], state["positions"], state["frequencies"],
                offset=case["offset"], interleaved=case["layout"] == "interleaved",
                magnitude=state["magnitude"]))
        if kind == "cache":
            attention.write_kv_fp8(
                state["kv"], state["cache"], state["new"], norm_weight=state["weight"], eps=EPS,
                positions=state["positions"], frequencies=state["frequencies"])
            return attention.read_kv_fp8(state["cache"], state["slots"])
        if kind == "prompt":
            return attention.prompt_attention(state["q"], state["k"], state["v"], state["scale"],
                                              state["cu_q"], state["cu_k"],
                                              max_k=state["max_k"])
        return attention.shared_prefix_mla(
            state["q"], state["cache"], state["prefix_table"], case["prefix"],
            state["suffix_tables"], state["suffix_tokens"], state["scale"], cu_q=state["cu_q"])
    if kind == "rope":
        return _rope_plain(state)
    if kind == "cache":
        return _cache_plain(state)
    if kind == "prompt":
        return _prompt_plain(state)
    return _prefix_plain(state)


# -------------------------------------------------------------------- work --
def work(case):
    """What the operator has to read, write and compute."""
    kind = case["kind"]
    if kind == "rope":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 2 * values * size + 4 * case["tokens"],
                "flops": 3 * values * case["rotated"] // case["dim"]}
    if kind == "cache":
        tokens, read = case["tokens"], case["history"] + case["tokens"]
        wide = 2 * (LATENT + ROPE)
        return {"bytes": tokens * (wide + RECORD + 12) + read * (RECORD + wide + 8),
                "flops": tokens * 6 * (LATENT + ROPE) + read * LATENT}
    if kind == "prompt":
        queries, keys = _prompt_lengths(case)
        pairs = sum(q * (k - q) + q * (q + 1) // 2 for q, k in zip(queries, keys))
        wide = case["qk"] + case["v"]
        return {"bytes": 2 * wide * (case["heads"] * sum(queries) + case["kv_heads"] * sum(keys)),
                "flops": 2 * pairs * case["heads"] * wide}
    queries, lengths = _branch_lengths(case)
    tokens, heads = sum(queries), case["heads"]
    own_pairs = sum(q * (n - q) + q * (q + 1) // 2 for q, n in zip(queries, lengths))
    pairs = tokens * case["prefix"] + own_pairs
    return {"bytes": (case["prefix"] + sum(lengths)) * RECORD
            + tokens * heads * 2 * (LATENT + ROPE + LATENT),
            "flops": 2 * pairs * heads * (LATENT + ROPE + LATENT)}


# ------------------------------------------------------------ 64-bit values --
def _turn64(x, positions, frequencies, magnitude, offset, layout):
    """Each pair (a, b) as the complex number a + ib, times magnitude e^(i angle)."""
    half = len(frequencies)
    out = x.double().clone()
    angle = positions.double()[:, None] * frequencies.double()
    factor = torch.polar(torch.full_like(angle, magnitude), angle)
    factor = factor.view(len(angle), *[1] * (x.ndim - 2), half)
    step = torch.arange(half, device=x.device)
    if layout == "interleaved":
        first, second = offset + 2 * step, offset + 2 * step + 1
    else:
        first, second = offset + step, offset + half + step
    turned = torch.complex(out[..., first], out[..., second]) * factor
    out[..., first], out[..., second] = turned.real, turned.imag
    return out


def _values64(records):
    """What records stand for, from the bits of their codes."""
    code = records[:, :LATENT].long()
    power, part = (code >> 3) & 15, (code & 7).double()
    size = torch.where(power == 0, part / 8 * 2.0 ** -6,
                       (1 + part / 8) * torch.exp2((power - 7).double()))
    size = torch.where(code >= 128, -size, size)
    scale = records[:, LATENT:LATENT + 16].contiguous().view(torch.float32).double()
    rope = records[:, LATENT + 16:].contiguous().view(torch.bfloat16).double()
    return torch.cat([size * scale.repeat_interleave(128, dim=1), rope], 1)


def _attend64(q, k, v, scale, sees):
    """Softmax attention of ``q [h, n, d]`` over ``k [h or 1, m, d]``, ``v``."""
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    s = s.masked_fill(~sees, -math.inf)
    return torch.matmul(torch.softmax(s, -1), v)


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "rope":
        return [_turn64(x, state["positions"], state["frequencies"], state["magnitude"],
                        case["offset"], case["layout"]) for x in (state["q"], state["k"])]
    if kind == "cache":
        latent, rope = state["kv"].double().split([LATENT, ROPE], 1)
        latent = latent / (latent.square().sum(1, keepdim=True) / LATENT + EPS).sqrt()
        latent = (latent * state["weight"].double()).bfloat16()
        rope = _turn64(rope, state["positions"], state["frequencies"], 1.0, 0, "interleaved")
        values = latent.double().view(-1, 4, 128)
        # The scale's rule is one of 32 bits: amax times 1/448, up to a power of two.
        amax = values.abs().amax(-1, keepdim=True).float().clamp_min(1e-4) * (1.0 / 448.0)
        part, power = torch.frexp(amax)
        scale = torch.ldexp(torch.ones_like(amax), power - (part == 0.5).to(power.dtype)).double()
        # e4m3: steps of 1/8 of the power of two at or below, 2^-9 at the least.
        units = values / scale
        size = units.abs().clamp_min(2.0 ** -6)
        step = torch.exp2(torch.floor(torch.log2(size)) - 3)
        new = torch.cat([((units / step).round() * step * scale).view(-1, LATENT),
                         rope.bfloat16().double()], 1)
        old = state["slots"][:case["history"]]
        return torch.cat([_values64(state["cache"].view(-1, RECORD)[old]), new])
    if kind == "prompt":
        queries, keys = _prompt_lengths(case)
        group, done_q, done_k, out = case["heads"] // case["kv_heads"], 0, 0, []
        for n, m in zip(queries, keys):
            q = state["q"][done_q:done_q + n].double().transpose(0, 1)
            k = state["k"][done_k:done_k + m].double().transpose(0, 1)
            v = state["v"][done_k:done_k + m].double().transpose(0, 1)
            sees = torch.ones(n, m, dtype=torch.bool, device=DEVICE).tril(m - n)
            per_head = [_attend64(q[h], k[h // group], v[h // group], state["scale"], sees)
                        for h in range(case["heads"])]
            out.append(torch.stack(per_head, 1))
            done_q, done_k = done_q + n, done_k + m
        return torch.cat(out)
    queries, lengths = _branch_lengths(case)
    records, out, done = state["cache"].view(-1, RECORD), [], 0
    shared = _values64(records[_slots(state["prefix_table"], case["prefix"])])
    for b, (n, m) in enumerate(zip(queries, lengths)):
        keys = torch.cat([shared, _values64(records[_slots(state["suffix_tables"][b], m)])])
        for i in range(n):
            seen = len(shared) + m - n + 1 + i
            everything = torch.ones(1, seen, dtype=torch.bool, device=DEVICE)
            out.append(_attend64(state["q"][done + i].double(), keys[:seen],
                                 keys[:seen, :LATENT], state["scale"], everything))
        done += n
    return torch.stack(out)
