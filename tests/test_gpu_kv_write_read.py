"""Writing any slots of the fp8 paged cache through norm and rotation, and reading back."""

import numpy as np
import pytest
import torch

from oracle import dense
from oracle import kv_fp8 as okv

pytestmark = pytest.mark.gpu


def _bits(t):
    return t.contiguous().cpu().view(torch.int16).numpy().view(np.uint16)


def _cache(pages, gpu, fill=0xAB):
    return torch.full((pages, 64, 656), fill, dtype=torch.uint8, device=gpu)


@pytest.mark.parametrize("tokens", [1, 3, 64, 131])
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_plain_write_is_the_packed_record(gpu, tokens, wide):
    from cxldsagr_amd.attention import read_kv_fp8, write_kv_fp8

    gen = torch.Generator().manual_seed(51)
    buffer = torch.randn(tokens, 2120, generator=gen).bfloat16().to(gpu)
    kv = buffer[:, 1536:2112]  # as a fused projection leaves it
    kv[0, :128] = 0
    slots = torch.randperm(4 * 64, generator=gen)[:tokens].to(wide).to(gpu)
    cache = _cache(4, gpu)
    assert write_kv_fp8(kv, cache, slots) is cache
    records = okv.encode_records(_bits(kv))
    flat = cache.view(-1, 656).cpu().numpy()
    assert np.array_equal(flat[slots.cpu().numpy()], records)
    others = np.setdiff1d(np.arange(256), slots.cpu().numpy())
    assert (flat[others] == 0xAB).all()
    back = read_kv_fp8(cache, slots)
    assert np.array_equal(_bits(back), _bits(torch.from_numpy(okv.decode_records(records)).bfloat16()))


@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_and_rotation(gpu, interleaved):
    """The RoPE part as the rotary operator rounds it, bit for bit. The latent: the norm's
    value, off by its bf16 rounding (2^-8) and 2^-18 of fp32, then the e4m3 rounding of
    at most 2^-4, or 2^-10 of the scale where the code is subnormal; the scale is the power
    of two at or above amax / 448 of such values."""
    from cxldsagr_amd.attention import read_kv_fp8, write_kv_fp8
    from cxldsagr_amd.projections import apply_rope_pair, rotary_frequencies

    gen = torch.Generator().manual_seed(52)
    tokens = 97
    kv = (torch.randn(tokens, 576, generator=gen) * torch.logspace(-3, 3, tokens)[:, None]).bfloat16().to(gpu)
    weight = (1 + 0.3 * torch.randn(512, generator=gen)).to(gpu)
    positions = torch.randint(163840, (tokens,), generator=gen).to(gpu)
    frequencies = rotary_frequencies().to(gpu)
    slots = torch.randperm(128, generator=gen)[:tokens].to(gpu)
    cache = _cache(2, gpu)
    write_kv_fp8(kv, cache, slots, norm_weight=weight, eps=1e-5, positions=positions,
                 frequencies=frequencies, interleaved=interleaved, magnitude=0.9)
    got = read_kv_fp8(cache, slots)
    rope, _ = apply_rope_pair(kv[:, None, 512:], None, positions, frequencies, interleaved=interleaved,
                              magnitude=0.9)
    assert torch.equal(got[:, 512:], rope[:, 0])
    want = dense.rms_norm(kv[:, :512], weight, 1e-5)
    scale = cache.view(-1, 656)[slots][:, 512:528].contiguous().view(torch.float32).cpu().double()
    amax = want.view(tokens, 4, 128).abs().amax(-1) / 448
    wobble = 2.0 ** -8 + 2.0 ** -18 + 2.0 ** -23
    assert (amax * (1 - wobble) <= scale).all() and (scale < 2 * amax * (1 + wobble)).all()
    value = want.abs() * (1 + 2.0 ** -8 + 2.0 ** -18)
    bound = (2.0 ** -8 + 2.0 ** -18) * want.abs() + torch.maximum(
        2.0 ** -4 * value, scale.repeat_interleave(128, 1) * 2.0 ** -10)
    assert ((got[:, :512].cpu().double() - want).abs() <= bound).all()


def test_norm_of_exact_values(gpu):
    """Rows of +-c have norm 1: the record of +-weight (eps 0)."""
    from cxldsagr_amd.attention import write_kv_fp8

    gen = torch.Generator().manual_seed(53)
    sign = torch.randint(2, (5, 512), generator=gen) * 2.0 - 1
    kv = torch.zeros(5, 576)
    kv[:, :512] = sign * 2.0 ** torch.tensor([-3, 0, 1, 4, 7])[:, None]
    weight = torch.randn(512, generator=gen).bfloat16()
    cache = _cache(1, gpu)
    write_kv_fp8(kv.bfloat16().to(gpu), cache, torch.arange(5, device=gpu), norm_weight=weight.float().to(gpu),
                 eps=0.0)
    kv[:, :512] = sign * weight.float()
    assert np.array_equal(cache.view(-1, 656)[:5].cpu().numpy(), okv.encode_records(_bits(kv.bfloat16())))


def test_padding_and_slots_past_the_cache(gpu):
    from cxldsagr_amd.attention import read_kv_fp8, write_kv_fp8

    kv = torch.randn(4, 576, generator=torch.Generator().manual_seed(54)).bfloat16().to(gpu)
    cache = _cache(1, gpu)
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    slots = torch.tensor([-1, 7, -(2 ** 40), 63], device=gpu)
    write_kv_fp8(kv, cache, slots, status=status)
    assert status.item() == 0
    flat = cache.view(-1, 656).cpu().numpy()
    assert np.array_equal(flat[[7, 63]], okv.encode_records(_bits(kv[[1, 3]])))
    assert (np.delete(flat, [7, 63], 0) == 0xAB).all()
    before = cache.clone()
    write_kv_fp8(kv, cache, torch.tensor([64, -1, 2 ** 40, -1], device=gpu), status=status)
    assert status.item() == 1 and torch.equal(cache, before)
    status.zero_()
    out = torch.full((5, 576), 9.0, dtype=torch.bfloat16, device=gpu)
    got = read_kv_fp8(cache, torch.tensor([7, -1, 7, 63, -9], device=gpu), out=out, status=status)
    assert got is out and status.item() == 0
    assert torch.equal(got[0], got[2]) and (got[[1, 4]] == 0).all() and got[3].abs().sum() > 0
    got = read_kv_fp8(cache, torch.tensor([64, 2 ** 33], device=gpu), status=status)
    assert status.item() == 1 and (got == 0).all()


def test_rows_with_infinities_and_nan_as_packed(gpu):
    from cxldsagr_amd.attention import pack_kv_fp8, write_kv_fp8

    kv = torch.randn(3, 576, generator=torch.Generator().manual_seed(55)).bfloat16().to(gpu)
    kv[0, 5], kv[1, 200], kv[2, 570] = float("inf"), float("nan"), float("nan")
    want, got = _cache(1, gpu, 0), _cache(1, gpu, 0)
    pack_kv_fp8(kv, want, torch.zeros(1, dtype=torch.int32, device=gpu))
    write_kv_fp8(kv, got, torch.arange(3, device=gpu))
    assert torch.equal(got, want)


def test_captured_write_and_read_replay(gpu):
    from cxldsagr_amd.attention import read_kv_fp8, write_kv_fp8

    kv = torch.randn(70, 576, generator=torch.Generator().manual_seed(56)).bfloat16().to(gpu)
    slots = torch.arange(69, -1, -1, device=gpu)
    cache = _cache(2, gpu)
    write_kv_fp8(kv, cache, slots)
    want = read_kv_fp8(cache, slots).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        write_kv_fp8(kv, cache, slots)
        out = read_kv_fp8(cache, slots)
    for _ in range(3):
        cache.zero_()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
