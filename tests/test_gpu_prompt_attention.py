"""Prompt attention against the 64-bit formula, at the sizes and masks where it can go
wrong. Tolerances: ``oracle.dense.attention_bound``, derived there."""

import math

import pytest
import torch

from oracle import dense

pytestmark = pytest.mark.gpu

DIMS = [(192, 128), (128, 128), (64, 64)]


def _cu(lengths, device, first=0):
    return torch.tensor([first] + lengths, device=device).cumsum(0).to(torch.int32)


def _inputs(gpu, queries, keys, heads, kv_heads, dims, dtype, seed, first=0, behind=0):
    gen = torch.Generator().manual_seed(seed)
    tq, tk = first + sum(queries) + behind, first + sum(keys) + behind
    # K and V in one buffer, as an up-projection leaves them: strided heads.
    q = torch.randn(tq, heads, dims[0] + 8, generator=gen).to(dtype).to(gpu)[..., :dims[0]]
    kv = torch.randn(tk, kv_heads, sum(dims), generator=gen).to(dtype).to(gpu)
    return q, kv[..., :dims[0]], kv[..., dims[0]:], _cu(queries, gpu, first), _cu(keys, gpu, first)


def _check(got, q, k, v, scale, cu_q, cu_k, causal=True):
    out, size, reach = dense.prompt_attention(q, k, v, scale, cu_q.tolist(), cu_k.tolist(), causal)
    keys = int((cu_k[1:] - cu_k[:-1]).max())
    tiny = v.float().nan_to_num().abs().max().item() if q.dtype == torch.float16 else 0.0
    bound = dense.attention_bound(out, size, reach, keys, torch.finfo(q.dtype).eps, q.shape[2], tiny)
    lo, hi = int(cu_q[0]), int(cu_q[-1])
    off = (got.cpu().double() - out).abs()[lo:hi]
    assert torch.isfinite(got[lo:hi]).all()
    assert (off <= bound[lo:hi]).all(), (off / bound[lo:hi]).max()


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize(
    ("queries", "keys", "heads", "kv_heads"),
    [
        ([1], [1], 1, 1),
        ([65], [65], 2, 1),                    # one row more than a wave's tile
        ([257], [257], 1, 1),                  # one more than a work-group's
        ([3, 1, 70], [3, 130, 200], 5, 1),     # five heads to a KV head, histories
        ([0, 33, 0, 20], [17, 33, 0, 63], 8, 8),  # sequences without queries, or without anything
        ([9, 40], [4, 0], 2, 2),               # more queries than keys: rows that see none
        ([1, 1, 1], [1, 64, 511], 16, 2),      # single tokens
    ],
)
def test_matches_the_formula(gpu, dims, dtype, queries, keys, heads, kv_heads):
    from cxldsagr_amd.attention import prompt_attention

    x = _inputs(gpu, queries, keys, heads, kv_heads, dims, dtype, 11)
    got = prompt_attention(*x[:3], dims[0] ** -0.5, *x[3:])
    _check(got, *x[:3], dims[0] ** -0.5, *x[3:])


@pytest.mark.parametrize("keys", [255, 256, 257, 2049])
@pytest.mark.parametrize("queries", [1, 3])
def test_few_queries_over_split_keys(gpu, keys, queries):
    """Keys split over work-groups and joined; some splits see nothing of some rows."""
    from cxldsagr_amd import _native
    from cxldsagr_amd.attention import prompt_attention

    x = _inputs(gpu, [queries, queries], [keys, 5], 4, 2, (128, 128), torch.bfloat16, 12)
    assert _native.size_of("dsa_prompt_attention_workspace_bytes", 0, 2 * queries, 4, 2, 128, 2,
                           keys + 5, keys) > 0 or keys <= 257  # (so few are not worth a join)
    got = prompt_attention(*x[:3], 0.1, *x[3:], max_k=keys)
    _check(got, *x[:3], 0.1, *x[3:])
    # max_k only says how keys are split.
    _check(prompt_attention(*x[:3], 0.1, *x[3:], max_k=1), *x[:3], 0.1, *x[3:])


def test_without_the_causal_mask(gpu):
    from cxldsagr_amd.attention import prompt_attention

    x = _inputs(gpu, [70, 5], [30, 100], 4, 2, (64, 64), torch.float16, 13)
    got = prompt_attention(*x[:3], 0.2, *x[3:], causal=False)
    _check(got, *x[:3], 0.2, *x[3:], causal=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_that_rise_from_block_to_block(gpu, dtype):
    """Each block of keys raises its rows' maxima beyond what is left unscaled; the last
    rows' scores fall again by far more than a probability's range."""
    from cxldsagr_amd.attention import prompt_attention

    q, k, v, cu_q, cu_k = _inputs(gpu, [40], [300], 2, 1, (64, 64), dtype, 14)
    q, k = q * 0.05, k * 0.05
    q[..., 0] = 4
    climb = torch.arange(300, device=gpu) // 16
    k[..., 0] = (20.0 * climb * (1 - 2 * (torch.arange(300, device=gpu) > 280)))[:, None].to(dtype)
    got = prompt_attention(q, k, v, 1.0, cu_q, cu_k)
    _check(got, q, k, v, 1.0, cu_q, cu_k)


@pytest.mark.parametrize("keys", [90, 1000])
def test_rows_outside_the_sequences(gpu, keys):
    """Rows before the first and behind the last sequence are left as they were, and their
    keys (NaN here) are not read into anything."""
    from cxldsagr_amd.attention import prompt_attention

    q, k, v, cu_q, cu_k = _inputs(gpu, [4, 2], [keys, 2], 2, 1, (128, 128), torch.bfloat16, 15,
                                  first=3, behind=5)
    for t in (q, k, v):
        t[:3] = float("nan")
        t[-5:] = float("nan")
    out = torch.full((q.shape[0], 2, 128), 7.0, dtype=torch.bfloat16, device=gpu)
    assert prompt_attention(q, k, v, 0.1, cu_q, cu_k, out=out) is out
    _check(out, q, k, v, 0.1, cu_q, cu_k)
    assert (out[:3] == 7).all() and (out[-5:] == 7).all()


def test_a_sequence_gives_the_same_alone_as_in_a_batch(gpu):
    from cxldsagr_amd.attention import prompt_attention

    q, k, v, cu_q, cu_k = _inputs(gpu, [300, 41, 600], [300, 41, 600], 32, 8, (192, 128),
                                  torch.bfloat16, 16)
    # Enough row tiles that neither call splits keys.
    both = prompt_attention(q, k, v, 0.07, cu_q, max_k=0)
    one = torch.tensor([0, 41], dtype=torch.int32, device=gpu)
    alone = prompt_attention(q[300:341], k[300:341], v[300:341], 0.07, one, max_k=0)
    assert torch.equal(both[300:341].view(torch.int16), alone.view(torch.int16))


def test_layouts_that_need_a_copy(gpu):
    from cxldsagr_amd.attention import prompt_attention

    q, k, v, cu_q, cu_k = _inputs(gpu, [20], [50], 4, 2, (64, 64), torch.bfloat16, 17)
    want = prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), 0.2, cu_q, cu_k)
    odd = torch.zeros(50 * 2 * 64 + 1, dtype=torch.bfloat16, device=gpu)
    k_odd = odd[1:].view(50, 2, 64)
    k_odd.copy_(k)
    v_turned = v.transpose(1, 2).contiguous().transpose(1, 2)
    got = prompt_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k_odd, v_turned, 0.2,
                           cu_q, cu_k)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))


def test_one_kv_head_broadcast_over_heads(gpu):
    """A stride of zero: expanded keys and values."""
    from cxldsagr_amd.attention import prompt_attention

    q, k, v, cu_q, cu_k = _inputs(gpu, [20], [50], 4, 1, (64, 64), torch.bfloat16, 18)
    got = prompt_attention(q, k.expand(50, 4, 64), v.expand(50, 4, 64), 0.2, cu_q, cu_k)
    _check(got, q, k, v, 0.2, cu_q, cu_k)


def test_infinities_and_nan_in_seen_keys_spread_as_in_the_formula(gpu):
    from cxldsagr_amd.attention import prompt_attention

    q, k, v, cu_q, cu_k = _inputs(gpu, [1, 1], [600, 600], 2, 1, (64, 64), torch.bfloat16, 19)
    k[590] = float("nan")       # of the first sequence, in a split of its own
    v[700, :, 3] = float("inf")
    got = prompt_attention(q, k, v, 0.1, cu_q, cu_k).float()
    assert got[0].isnan().all()
    assert got[1, :, 3].isposinf().all() and got[1, :, 4:].isfinite().all()


def test_captured_call_replays_and_other_streams(gpu):
    from cxldsagr_amd.attention import prompt_attention

    q, k, v, cu_q, cu_k = _inputs(gpu, [2, 3], [700, 900], 8, 2, (128, 128), torch.bfloat16, 20)

    def call():
        return prompt_attention(q, k, v, 0.1, cu_q, cu_k)

    want = call().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = call()
    again = call()  # at the same time, with a workspace of its own
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(beside, want) and torch.equal(again, want)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    for _ in range(3):
        for graph, out in zip(graphs, outs):
            out.fill_(float("nan"))
            graph.replay()
            assert torch.equal(call(), want)
            torch.cuda.synchronize()
            assert torch.equal(out, want)


@pytest.mark.parametrize("drop", [15.7, 20.3, 25.3])
@pytest.mark.parametrize(("queries", "keys"), [(1, 3000), (40, 900)])
def test_many_low_scores_behind_one_peak(gpu, queries, keys, drop):
    """fp16: the first key's probability is 1 and its value 0, every other's 2^-drop and 1,
    which are then all of the result: small probabilities must not be lost, nor counted
    otherwise in the sum than in the product. They are held against a maximum of at least 2^7, so
    what the bound allows for subnormal ones is 2^7 less than for a maximum of 1."""
    from cxldsagr_amd.attention import prompt_attention

    q = torch.zeros(queries, 2, 64, dtype=torch.float16, device=gpu)
    k = torch.zeros(keys, 1, 64, dtype=torch.float16, device=gpu)
    v = torch.ones_like(k)
    q[..., 0] = 1
    k[1:, :, 0] = -drop * math.log(2)
    v[0] = 0
    cu_q, cu_k = _cu([queries], gpu), _cu([keys], gpu)
    out, size, reach = dense.prompt_attention(q, k, v, 1.0, cu_q.tolist(), cu_k.tolist())
    bound = dense.attention_bound(out, size, reach, keys, torch.finfo(q.dtype).eps, 64, 2.0 ** -7)
    off = (prompt_attention(q, k, v, 1.0, cu_q, cu_k, max_k=keys).cpu().double() - out).abs()
    assert (off <= bound).all(), (off / out).max()
    # The peak last: what was summed before is scaled by 2^-drop in 32 bits.
    k, v = k.flip(0), v.flip(0)
    out, size, reach = dense.prompt_attention(q[:1], k, v, 1.0, [0, 1], [0, keys])
    bound = dense.attention_bound(out, size, reach, keys, torch.finfo(q.dtype).eps, 64, 2.0 ** -7)
    got = prompt_attention(q[:1], k, v, 1.0, _cu([1], gpu), cu_k, max_k=keys)
    assert ((got.cpu().double() - out).abs() <= bound).all()


@pytest.mark.parametrize("power", [20, 24, 26])
def test_fp16_scores_far_from_zero(gpu, power):
    """Scores of up to 2^power in log2 units, whose 32-bit steps are then up to 4: the
    probabilities, which are only as near to 1 as such steps let them be, stay within fp16."""
    from cxldsagr_amd.attention import prompt_attention

    gen = torch.Generator().manual_seed(21)
    q = torch.zeros(3, 1, 64, dtype=torch.float16, device=gpu)
    k = torch.zeros(400, 1, 64, dtype=torch.float16, device=gpu)
    v = torch.randn(400, 1, 64, generator=gen).half().to(gpu)
    q[..., 0] = 2.0 ** (power - 14)
    k[..., 0] = 2.0 ** 13 * (1 + 2.0 ** -10 * torch.randint(16, (400, 1), generator=gen)).to(gpu)
    cu_q, cu_k = _cu([3], gpu), _cu([400], gpu)
    got = prompt_attention(q, k, v, 1.0, cu_q, cu_k)
    assert got.isfinite().all()
    # The keys of the largest score share the result equally, the others are at least 2^9 below
    # it; what is off is fp32 sums and one rounding to fp16.
    for i in range(3):
        seen = k[:398 + i, 0, 0]
        want = v[:398 + i, 0][seen == seen.max()].double().mean(0)
        assert ((got[i, 0].double() - want).abs() <= 2.0 ** -10 * (want.abs() + 1)).all()


def _parts(queries, heads, kv_heads, v_dim, keys):
    """Into how many ranges one sequence's keys are split (0: not)."""
    from cxldsagr_amd import _native

    size = _native.size_of("dsa_prompt_attention_workspace_bytes", 0, queries, heads, kv_heads, v_dim, 1,
                           keys, keys)
    return size // (queries * heads * (4 * v_dim + 8))


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize(
    ("queries", "keys", "least", "most"),
    [
        (1, 700, 2, 4),         # each range of part counts is joined in its own way
        (1, 2049, 5, 32),
        (1, 33001, 33, 256),
        (2, 33000, 33, 256),
        (17, 703, 2, 4),        # more rows than one wave has
        (17, 9001, 33, 256),
    ],
)
def test_joins_of_few_and_many_parts(gpu, dims, dtype, queries, keys, least, most):
    from cxldsagr_amd.attention import prompt_attention

    assert least <= _parts(queries, 4, 2, dims[1], keys) <= most
    q, k, v, cu_q, cu_k = _inputs(gpu, [queries], [keys], 4, 2, dims, dtype, 22)
    # The largest scores in different parts for different rows, and one part that hardly counts.
    k[keys // 3:keys // 2] *= 2
    k[-100:-60] *= 0.125
    got = prompt_attention(q, k, v, dims[0] ** -0.5, cu_q, cu_k, max_k=keys)
    _check(got, q, k, v, dims[0] ** -0.5, cu_q, cu_k)
    again = prompt_attention(q, k, v, dims[0] ** -0.5, cu_q, cu_k, max_k=keys)
    assert torch.equal(got, again)


@pytest.mark.parametrize("keys", [511, 512, 513, 767, 768, 769])
@pytest.mark.parametrize("queries", [1, 3])
def test_lengths_around_two_and_three_parts(gpu, keys, queries):
    from cxldsagr_amd.attention import prompt_attention

    q, k, v, cu_q, cu_k = _inputs(gpu, [queries], [keys], 4, 2, (128, 128), torch.bfloat16, 23)
    assert _parts(queries, 4, 2, 128, keys) >= 2
    got = prompt_attention(q, k, v, 0.1, cu_q, cu_k, max_k=keys)
    _check(got, q, k, v, 0.1, cu_q, cu_k)
