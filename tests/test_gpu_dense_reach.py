"""The dense operators where their calls reach furthest: addresses past 32 bits, batches of
many and uneven sequences, two calls at once. Formulas and tolerances as in the tests of
each operator."""

import numpy as np
import pytest
import torch

from oracle import kv_fp8 as okv
from test_gpu_prompt_attention import _check as check_prompt, _inputs
from test_gpu_shared_prefix import _case, _check as check_prefix, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize(
    ("queries", "keys", "heads", "kv_heads"),
    [
        ([7] * 65 + [40], [9] * 65 + [300], 4, 4),              # more sequences than lanes
        ([1 + 9 * (i % 5) for i in range(64)], [60 + 7 * i for i in range(64)], 2, 1),
        ([300, 1, 700, 0, 129], [300, 40, 700, 5, 900], 8, 2),  # several tiles, by rank
        ([500, 20], [40, 2000], 3, 3),                          # a first sequence's rows see nothing
        ([1] * 40, [2000] + [3] * 39, 2, 1),                    # one long one among short ones
    ],
)
def test_batches_of_uneven_sequences(gpu, queries, keys, heads, kv_heads):
    """Their longest known, and not."""
    from cxldsagr_amd.attention import prompt_attention

    x = _inputs(gpu, queries, keys, heads, kv_heads, (64, 64), torch.bfloat16, 61)
    for longest in (None, max(keys)):
        check_prompt(prompt_attention(*x[:3], 0.125, *x[3:], max_k=longest), *x[:3], 0.125, *x[3:])


def test_batches_of_uneven_sequences_without_the_causal_mask(gpu):
    from cxldsagr_amd.attention import prompt_attention

    x = _inputs(gpu, [300, 1, 700], [150, 40, 701], 4, 2, (128, 128), torch.float16, 62)
    got = prompt_attention(*x[:3], 0.1, *x[3:], causal=False)
    check_prompt(got, *x[:3], 0.1, *x[3:], causal=False)


def test_keys_and_queries_past_32_bits(gpu):
    """Token strides that put the last tokens more than 4 GiB behind the first."""
    from cxldsagr_amd.attention import prompt_attention
    from cxldsagr_amd.projections import apply_rope_pair

    tokens, stride = 17000, 1 << 17
    buffer = torch.empty(tokens * stride, dtype=torch.bfloat16, device=gpu)
    x = buffer.view(tokens, stride)
    gen = torch.Generator().manual_seed(63)
    x[:, :192] = torch.randn(tokens, 192, generator=gen).bfloat16().to(gpu)
    q, k, v = (x[:, 64 * i:64 * (i + 1)].unsqueeze(1) for i in range(3))
    starts = torch.tensor([0, 5, tokens - 4, tokens], dtype=torch.int32, device=gpu)
    assert (tokens - 4) * stride * 2 > 1 << 32
    for a in (q, k, v):
        a[5:tokens - 4] = 0  # (the sequence in the middle is not looked at)
    got = prompt_attention(q, k, v, 0.125, starts)
    want = prompt_attention(*(t.contiguous() for t in (q, k, v)), 0.125, starts)
    assert torch.equal(got, want)
    ends = torch.tensor([*range(5), *range(tokens - 4, tokens)], device=gpu)
    starts = torch.tensor([0, 5, 9], dtype=torch.int32, device=gpu)
    check_prompt(got[ends], q[ends], k[ends], v[ends], 0.125, starts, starts)

    positions = torch.arange(tokens, device=gpu)
    frequencies = torch.rand(32, generator=gen).to(gpu)
    rotated, _ = apply_rope_pair(q, None, positions, frequencies)
    apply_rope_pair(q, None, positions, frequencies, q_out=q)
    assert torch.equal(q, rotated)
    last = x[-1:, 64:128].unsqueeze(1)
    one, _ = apply_rope_pair(last, None, positions[-1:], frequencies)
    assert torch.equal(apply_rope_pair(k, None, positions, frequencies)[0][-1:], one)


def test_cache_records_past_32_bits(gpu):
    """Records more than 4 GiB into a cache are written, read and attended to."""
    from cxldsagr_amd.attention import read_kv_fp8, shared_prefix_mla, write_kv_fp8

    pages = (1 << 32) // (64 * 656) + 20
    cache = torch.empty(pages, 64, 656, dtype=torch.uint8, device=gpu)
    table = torch.tensor([pages - 1, 0, pages - 9, 3], dtype=torch.int32)
    gen = torch.Generator().manual_seed(64)
    kv = torch.randn(256, 576, generator=gen).bfloat16().to(gpu)
    t = torch.arange(256)
    slots = (table[t // 64].long() * 64 + t % 64).to(gpu)
    write_kv_fp8(kv, cache, slots)
    small = torch.empty(4, 64, 656, dtype=torch.uint8, device=gpu)
    write_kv_fp8(kv, small, t.to(gpu))
    assert torch.equal(cache[table.long()], small)
    assert torch.equal(read_kv_fp8(cache, slots), read_kv_fp8(small, t.to(gpu)))
    q = torch.randn(2, 128, 576, generator=gen).bfloat16().to(gpu)
    tables = [table.to(gpu), torch.arange(4, dtype=torch.int32, device=gpu)]
    lengths = torch.tensor([30, 64], dtype=torch.int32, device=gpu)
    far, near = (shared_prefix_mla(q, c, p[:2], 100, p[2:].view(2, 1), lengths, 0.07)
                 for c, p in zip((cache, small), tables))
    assert torch.equal(far, near)


@pytest.mark.parametrize("tokens", [4097, 4104])
def test_many_records_written_at_once(gpu, tokens):
    """Enough that a wave takes several, an odd count too: as written in small calls."""
    from cxldsagr_amd.attention import write_kv_fp8
    from cxldsagr_amd.projections import rotary_frequencies

    gen = torch.Generator().manual_seed(65)
    kv = torch.randn(tokens, 576, generator=gen).bfloat16().to(gpu)
    slots = torch.randperm(65 * 64, generator=gen)[:tokens].to(gpu)
    slots[11] = -1
    slots[tokens - 1] = 65 * 64 + 5
    positions = torch.arange(tokens, device=gpu)
    weight = torch.rand(512, generator=gen).to(gpu)
    caches = [torch.full((65, 64, 656), 0xAB, dtype=torch.uint8, device=gpu) for _ in range(2)]
    status = torch.zeros(2, dtype=torch.int32, device=gpu)
    for interleaved in (True, False):
        kwargs = dict(norm_weight=weight, frequencies=rotary_frequencies().to(gpu), interleaved=interleaved)
        write_kv_fp8(kv, caches[0], slots, positions=positions, status=status[:1], **kwargs)
        for part in torch.arange(tokens, device=gpu).split(500):
            write_kv_fp8(kv[part], caches[1], slots[part], positions=positions[part], status=status[1:],
                         **kwargs)
        assert torch.equal(*caches)
    assert status.tolist() == [1, 1]
    plain = torch.full((65, 64, 656), 0xAB, dtype=torch.uint8, device=gpu)
    write_kv_fp8(kv, plain, slots)
    bits = kv.cpu().view(torch.int16).numpy().view(np.uint16)
    records = okv.encode_records(bits)
    held = ((slots >= 0) & (slots < 65 * 64)).cpu().numpy()
    assert np.array_equal(plain.view(-1, 656).cpu().numpy()[slots.cpu().numpy()[held]], records[held])


@pytest.mark.parametrize(
    ("prefix", "suffixes", "queries", "heads"),
    [
        (2500, [70, 3], [2, 1], 48),      # heads that straddle groups of 32 rows, keys split
        (2500, [9, 200], [1, 1], 1),
        (2500, [9, 200], [1, 3], 200),    # suffix items of 128 and 72 heads
        (2500, [300, 40], [1, 1], 256),   # two joint tiles a token
        (0, [2500, 900], [1, 2], 64),     # long suffixes alone
    ],
)
def test_split_prefixes_of_odd_head_counts(gpu, prefix, suffixes, queries, heads):
    x, values = _case(gpu, prefix, suffixes, queries, heads, 66)
    check_prefix(_run(x, prefix), x, values)


def test_two_prefix_calls_at_once(gpu):
    x, _ = _case(gpu, 3000, [9, 70], [1, 2], 48, 67)
    want = _run(x, 3000).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            beside = _run(x, 3000)
        again = _run(x, 3000)
        torch.cuda.synchronize()
        assert torch.equal(beside, want) and torch.equal(again, want)


@pytest.mark.parametrize("dims", [(192, 128), (128, 128), (64, 64)])
@pytest.mark.parametrize(
    ("queries", "keys", "heads", "kv_heads"),
    [
        ([100], [3000], 2, 2),
        ([70, 40], [2500, 100], 5, 1),  # the shorter one's rows are in the first split only
    ],
)
def test_chunks_whose_keys_are_split(gpu, dims, queries, keys, heads, kv_heads):
    """More rows than a wave, few enough to be split over keys and joined."""
    from cxldsagr_amd import _native
    from cxldsagr_amd.attention import prompt_attention

    x = _inputs(gpu, queries, keys, heads, kv_heads, dims, torch.bfloat16, 68)
    assert _native.size_of("dsa_prompt_attention_workspace_bytes", 0, sum(queries), heads, kv_heads, dims[1],
                           len(queries), sum(keys), max(keys)) > 0
    for causal in (True, False):
        got = prompt_attention(*x[:3], 0.1, *x[3:], max_k=max(keys), causal=causal)
        check_prompt(got, *x[:3], 0.1, *x[3:], causal=causal)
