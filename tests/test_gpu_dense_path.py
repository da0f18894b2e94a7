"""The dense operators together: a layer's prompt from its projections, and its candidates.

Rotate queries, write the new tokens' records through norm and rotation, read them back,
project them up and attend (the form for prompts); the same attention in the absorbed form
over the cache; and branches over that prompt as a shared prefix. One layer's algebra in
64 bits from the records that the cache holds is what all are held to."""

import pytest
import torch

from oracle import dense

pytestmark = pytest.mark.gpu


def test_prompt_read_back_absorbed_and_shared_forms_agree(gpu):
    from cxldsagr_amd.attention import (prompt_attention, read_kv_fp8, shared_prefix_mla,
                                        sparse_mla_fp8_paged, write_kv_fp8)
    from cxldsagr_amd.projections import apply_rope_pair, rotary_frequencies

    gen = torch.Generator().manual_seed(61)
    tokens, heads = 150, 64
    frequencies = rotary_frequencies().to(gpu)
    positions = torch.arange(tokens, device=gpu)
    kv = torch.randn(tokens, 576, generator=gen).bfloat16().to(gpu)
    weight = torch.ones(512, device=gpu)
    table = torch.tensor([2, 0, 3], dtype=torch.int32, device=gpu)
    slots = table[positions // 64].long() * 64 + positions % 64
    cache = torch.zeros(6, 64, 656, dtype=torch.uint8, device=gpu)
    write_kv_fp8(kv, cache, slots, norm_weight=weight, positions=positions, frequencies=frequencies)
    records = read_kv_fp8(cache, slots)

    # Up-projections of a head: keys' position-free part and values, 128 dims each.
    w_k, w_v = (torch.randn(heads, 512, 128, generator=gen).mul(512 ** -0.5).bfloat16().to(gpu) for _ in range(2))
    q = torch.randn(tokens, heads, 192, generator=gen).bfloat16().to(gpu)
    _, _ = apply_rope_pair(q, None, positions, frequencies, offset=128, interleaved=True, q_out=q)
    scale, cu = 192 ** -0.5, torch.tensor([0, tokens], dtype=torch.int32, device=gpu)

    up = torch.matmul(records[:, :512].float(), torch.cat([w_k, w_v], 2).float().transpose(0, 1).reshape(512, -1))
    up = up.view(tokens, heads, 256).bfloat16()
    k = torch.cat([up[..., :128], records[:, None, 512:].expand(-1, heads, -1)], -1)
    prompt = prompt_attention(q, k, up[..., 128:], scale, cu)
    out, size, reach = dense.prompt_attention(q, k, up[..., 128:], scale, cu.tolist(), cu.tolist())
    eps = torch.finfo(torch.bfloat16).eps
    assert ((prompt.cpu().double() - out).abs() <= dense.attention_bound(out, size, reach, tokens, eps, 192)).all()

    # Absorbed: queries through w_k, over the latent; every earlier token selected.
    absorbed = torch.empty(tokens, heads, 576, dtype=torch.bfloat16, device=gpu)
    absorbed[..., :512] = torch.matmul(q[..., :128].float().transpose(0, 1), w_k.float().transpose(1, 2).contiguous()).transpose(0, 1)
    absorbed[..., 512:] = q[..., 128:]
    ids = torch.arange(tokens, device=gpu).expand(tokens, -1)
    ids = torch.where(ids <= positions[:, None], ids, -1).int()
    sparse = sparse_mla_fp8_paged(absorbed, cache, table, ids, scale, n_tokens=tokens)
    # The last 22 tokens as one branch's queries behind the first 128 as the prefix.
    shared = shared_prefix_mla(absorbed[128:], cache, table, 128, table[None, 2:],
                               torch.tensor([22], dtype=torch.int32, device=gpu), scale,
                               cu_q=torch.tensor([0, 22], dtype=torch.int32, device=gpu))
    values = records.cpu().double()
    out, size, reach = dense.shared_prefix_mla(absorbed[128:], values[:128], [values[128:]], [0, 22], scale)
    bound = dense.attention_bound(out, size, reach, tokens, eps, 576)
    assert ((shared.cpu().double() - out).abs() <= bound).all()
    # The sparse operator rounds at the same places: within both bounds of each other.
    assert ((shared - sparse[128:]).abs().cpu().double() <= 2 * bound + eps * bound).all()


def test_candidates_of_a_request(gpu):
    """Branches written in one call to their own pages, scored over one prefix: each as if
    it were alone behind it."""
    from cxldsagr_amd.attention import read_kv_fp8, shared_prefix_mla, write_kv_fp8
    from cxldsagr_amd.projections import rotary_frequencies

    gen = torch.Generator().manual_seed(62)
    prefix, branches, heads = 200, 5, 128
    order = torch.randperm(10, generator=gen).to(torch.int32).to(gpu)
    table, own = order[:4], order[4:9].view(5, 1)
    cache = torch.zeros(10, 64, 656, dtype=torch.uint8, device=gpu)
    place = torch.arange(prefix, device=gpu)
    slots = table[place // 64].long() * 64 + place % 64
    write_kv_fp8(torch.randn(prefix, 576, generator=gen).bfloat16().to(gpu), cache, slots)
    lengths = torch.tensor([1, 2, 3, 1, 64], dtype=torch.int32, device=gpu)
    rows = [own[b, 0].long() * 64 + torch.arange(int(n), device=gpu) for b, n in enumerate(lengths)]
    tail = torch.cat(rows)
    write_kv_fp8(torch.randn(len(tail), 576, generator=gen).bfloat16().to(gpu), cache, tail,
                 positions=torch.cat([prefix + torch.arange(int(n), device=gpu) for n in lengths]),
                 frequencies=rotary_frequencies().to(gpu))
    q = torch.randn(branches, heads, 576, generator=gen).bfloat16().to(gpu)
    got = shared_prefix_mla(q, cache, table, prefix, own, lengths, 0.07)
    values, suffixes = read_kv_fp8(cache, slots).cpu(), [read_kv_fp8(cache, r).cpu() for r in rows]
    out, size, reach = dense.shared_prefix_mla(q, values, suffixes, list(range(branches + 1)), 0.07)
    bound = dense.attention_bound(out, size, reach, 264, torch.finfo(torch.bfloat16).eps, 576)
    assert ((got.cpu().double() - out).abs() <= bound).all()
