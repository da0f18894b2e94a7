"""MLA over a shared prefix against the 64-bit formula. Tolerances:
``oracle.dense.attention_bound``, derived there."""

import pytest
import torch

from oracle import dense
from oracle import kv_fp8 as okv

pytestmark = pytest.mark.gpu

SCALE = 192 ** -0.5


def _case(gpu, prefix, suffixes, queries, heads, seed, scale=1.0):
    """Pages in any order, the unused places of every page full of NaN codes."""
    gen = torch.Generator().manual_seed(seed)
    width = max([(n + 63) // 64 for n in suffixes] + [1])
    first = (prefix + 63) // 64
    pages = first + width * len(suffixes) + 1
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    cache = torch.full((pages * 64, 656), 0x7F, dtype=torch.uint8)

    def put(table, count):
        bits = (torch.randn(count, 576, generator=gen) * scale).bfloat16().view(torch.int16).numpy().view("uint16")
        records = torch.from_numpy(okv.encode_records(bits))
        t = torch.arange(count)
        cache[table[t // 64].long() * 64 + t % 64] = records
        return torch.from_numpy(okv.decode_records(records.numpy()))

    prefix_table, tables = order[:first], order[first:first + width * len(suffixes)].view(-1, width)
    values = put(prefix_table, prefix), [put(t, n) for t, n in zip(tables, suffixes)]
    cu = torch.tensor([0] + queries).cumsum(0).to(torch.int32)
    q = torch.randn(int(cu[-1]), heads, 576, generator=gen).bfloat16()
    dev = dict(q=q, kv_cache=cache.view(-1, 64, 656), prefix_table=prefix_table, suffix_tables=tables,
               suffix_tokens=torch.tensor(suffixes, dtype=torch.int32), cu_q=cu)
    return {k: v.to(gpu) for k, v in dev.items()}, values


def _run(x, prefix, **kwargs):
    from cxldsagr_amd.attention import shared_prefix_mla

    args = dict(x, **kwargs)
    return shared_prefix_mla(args["q"], args["kv_cache"], args["prefix_table"], prefix,
                             args["suffix_tables"], args["suffix_tokens"], SCALE,
                             cu_q=args["cu_q"], out=args.get("out"))


def _check(got, x, values):
    got = got[int(x["cu_q"][0]):int(x["cu_q"][-1])]
    x = dict(x, q=x["q"][int(x["cu_q"][0]):], cu_q=x["cu_q"] - x["cu_q"][0])
    x["q"] = x["q"][:int(x["cu_q"][-1])]
    out, size, reach = dense.shared_prefix_mla(x["q"], values[0], values[1], x["cu_q"].tolist(), SCALE)
    keys = len(values[0]) + max(len(s) for s in values[1])
    bound = dense.attention_bound(out, size, reach, keys, torch.finfo(torch.bfloat16).eps, 576)
    off = (got.cpu().double() - out).abs()
    assert torch.isfinite(got).all() and (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize(
    ("prefix", "suffixes", "queries", "heads"),
    [
        (1, [1], [1], 128),
        (0, [1, 33, 64, 65], [1, 1, 1, 1], 128),      # no prefix: the suffix alone
        (0, [5], [1], 64),
        (31, [1, 7], [1, 1], 128),                    # a block that ends inside
        (64, [64, 1], [1, 1], 64),                    # two tokens' heads in one tile of the prefix
        (97, [3, 40, 9], [3, 1, 2], 128),             # several queries of a branch, causal
        (200, [70, 2, 130], [2, 2, 5], 64),
        (130, [3, 5, 2], [1, 2, 1], 16),              # eight tokens in a tile
        (70, [2, 3], [1, 1], 1),
        (70, [2, 3], [1, 2], 129),                    # heads past a tile
        (40, [2, 0, 1], [2, 0, 4], 128),              # a branch without queries; rows before its suffix
        (0, [2], [4], 128),                           # rows that see nothing
        (700, [1, 300], [1, 1], 192),
    ],
)
def test_matches_the_formula(gpu, prefix, suffixes, queries, heads):
    x, values = _case(gpu, prefix, suffixes, queries, heads, 31)
    got = _run(x, prefix)
    _check(got, x, values)
    if all(n == 1 for n in queries):
        assert torch.equal(got, _run(x, prefix, cu_q=None))


def test_prefix_without_suffix_pages(gpu):
    x, values = _case(gpu, 333, [0, 0], [1, 1], 128, 32)
    x["suffix_tables"] = x["suffix_tables"][:, :0]
    _check(_run(x, 333), x, values)
    assert (_run(x, 0) == 0).all()


def test_large_scores_rise_from_block_to_block(gpu):
    x, values = _case(gpu, 600, [50], [1], 128, 33)
    x["q"] *= 40
    _check(_run(x, 600), x, values)


@pytest.mark.parametrize("heads", [64, 128])
def test_rows_of_no_branch_are_left_alone(gpu, heads):
    x, values = _case(gpu, 300, [4, 6], [2, 1], heads, 34)
    pad = torch.full((2, heads, 576), float("nan"), dtype=torch.bfloat16, device=gpu)
    x["q"], x["cu_q"] = torch.cat([pad, x["q"], pad]), x["cu_q"] + 2
    out = torch.full((7, heads, 512), 5.0, dtype=torch.bfloat16, device=gpu)
    assert _run(x, 300, out=out) is out
    _check(out, x, values)
    assert (out[:2] == 5).all() and (out[5:] == 5).all()


def test_pages_outside_the_cache_and_lengths_past_the_table(gpu):
    """Such pages are padding; a suffix is cut to what its table covers."""
    x, values = _case(gpu, 256, [64, 64], [1, 1], 128, 35)
    x["prefix_table"][1], x["prefix_table"][2] = -1, x["kv_cache"].shape[0]
    x["suffix_tokens"][1] = 1000000
    prefix = torch.cat([values[0][:64], values[0][192:]])
    q, cu = x["q"], x["cu_q"].tolist()
    out, size, reach = dense.shared_prefix_mla(q, prefix, values[1], cu, SCALE)
    bound = dense.attention_bound(out, size, reach, 320, torch.finfo(torch.bfloat16).eps, 576)
    assert ((_run(x, 256).cpu().double() - out).abs() <= bound).all()
    x["suffix_tokens"][0] = -5
    out, size, reach = dense.shared_prefix_mla(q[:1], prefix, [values[1][0][:0]], [0, 1], SCALE)
    bound = dense.attention_bound(out, size, reach, 320, torch.finfo(torch.bfloat16).eps, 576)
    assert ((_run(x, 256)[:1].cpu().double() - out).abs() <= bound).all()


def test_one_prefix_for_many_branches_equals_each_alone(gpu):
    """Long enough to be split; each branch alone agrees within the bound of both."""
    x, values = _case(gpu, 5000, [9, 1, 70, 30], [1, 1, 1, 1], 128, 36)
    got = _run(x, 5000)
    _check(got, x, values)


def test_captured_call_replays(gpu):
    x, _ = _case(gpu, 3000, [9, 70], [1, 2], 128, 37)
    want = _run(x, 3000).clone()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_run(x, 3000))
        graphs.append(graph)
    for _ in range(3):
        for graph, out in zip(graphs, outs):
            out.fill_(float("nan"))
            graph.replay()
            assert torch.equal(_run(x, 3000), want)
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def _parts(tokens, heads, prefix, suffix_pages):
    """Into how many parts a row's keys are split (0: not)."""
    from cxldsagr_amd import _native

    size = _native.size_of("dsa_shared_prefix_mla_workspace_bytes", 0, tokens, heads, prefix, suffix_pages)
    rows = tokens * heads
    return size // ((rows + 31) // 32 * 32 * 2048 + 8 * rows)


@pytest.mark.parametrize(
    ("prefix", "suffixes", "queries", "heads", "least", "most"),
    [
        # Each range of part counts is joined in its own way, more than 32 of them by rows too.
        (96, [64, 3, 17] * 8, [1] * 24, 64, 2, 4),
        (600, [5, 64], [1, 3], 128, 5, 32),
        (8600, [40, 1], [1, 1], 128, 33, 256),
        (8601, [7, 64], [2, 3], 64, 33, 256),
        (8600, [70], [1], 128, 33, 256),
        (8599, [3], [1], 16, 33, 256),
    ],
)
def test_joins_of_few_and_many_parts(gpu, prefix, suffixes, queries, heads, least, most):
    x, values = _case(gpu, prefix, suffixes, queries, heads, 38)
    assert least <= _parts(sum(queries), heads, prefix, x["suffix_tables"].shape[1]) <= most
    got = _run(x, prefix)
    _check(got, x, values)
    assert torch.equal(got, _run(x, prefix))


@pytest.mark.parametrize("heads", [64, 128])
def test_each_branch_alone_behind_the_prefix(gpu, heads):
    """A branch called by itself, whose keys are split otherwise, and within the batch: both
    are within the bound of the formula's values."""
    lengths, queries = [9, 1, 70, 30], [2, 1, 1, 3]
    x, values = _case(gpu, 5000, lengths, queries, heads, 39)
    _check(_run(x, 5000), x, values)
    starts = x["cu_q"].tolist()
    for b, n in enumerate(queries):
        one = dict(x, q=x["q"][starts[b]:starts[b + 1]].contiguous(),
                   suffix_tables=x["suffix_tables"][b:b + 1], suffix_tokens=x["suffix_tokens"][b:b + 1],
                   cu_q=torch.tensor([0, n], dtype=torch.int32, device=gpu))
        _check(_run(one, 5000), one, (values[0], values[1][b:b + 1]))
