"""Rotary pairs against the 64-bit formula. Tolerance: cos and sin are off by at most
2^-20 m in all (derived for 32-bit functions of an angle in turns rounded to 32 bits: the
rounding moves it by 2 pi 2^-25, their evaluation by 4 units of 2^-24, the magnitude's product
by one more; formed in 64 bits and rounded once they are off by 2^-24 m), so a result by
2^-20 m (|a| + |b|) and the fp32 products and sum by 2^-22 m (|a| + |b|); then it is rounded
once, by at most half a step."""

import math

import pytest
import torch

from oracle import dense

pytestmark = pytest.mark.gpu


def _frequencies(rotated, gpu):
    from cxldsagr_amd.projections import rotary_frequencies

    return rotary_frequencies(rotated).to(gpu)


def _check(got, x, positions, frequencies, offset, interleaved, magnitude, inverse=False):
    args = (positions, frequencies, offset, interleaved, magnitude, inverse)
    want = dense.rope(x, *args)
    half = len(frequencies)
    part = x.detach().cpu().double()[..., offset:offset + 2 * half].abs()
    if interleaved:
        both = (part[..., 0::2] + part[..., 1::2]).repeat_interleave(2, -1)
    else:
        both = (part[..., :half] + part[..., half:]).repeat(1, 1, 2)
    bound = torch.zeros_like(want)
    inner = (2.0 ** -20 + 2.0 ** -22) * abs(magnitude) * both
    turned = want[..., offset:offset + 2 * half].abs()
    bound[..., offset:offset + 2 * half] = inner + torch.finfo(x.dtype).eps / 2 * (turned + inner) + 2.0 ** -25
    off = (got.cpu().double() - want).abs()
    assert (off <= bound).all(), (off - bound).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize(
    ("tokens", "heads", "kv_heads", "dim", "offset", "rotated"),
    [
        (1, 1, 1, 64, 0, 64),
        (17, 128, 1, 192, 128, 64),   # a head's last part
        (3, 64, 8, 128, 0, 64),       # its first part
        (5, 3, 2, 96, 16, 48),        # in the middle
        (7, 2, 1, 30, 3, 6),          # no vectors: odd offset, few pairs
        (300, 1, 1, 64, 0, 64),       # many tokens to a work-group
        (2, 200, 5, 128, 64, 64),     # a token over several work-groups
        (2, 1, 0, 256, 0, 256),
    ],
)
def test_matches_the_formula(gpu, dtype, interleaved, tokens, heads, kv_heads, dim, offset, rotated):
    from cxldsagr_amd.projections import apply_rope_pair

    gen = torch.Generator().manual_seed(41)
    q = torch.randn(tokens, heads, dim, generator=gen).to(dtype).to(gpu)
    k = torch.randn(tokens, kv_heads, dim, generator=gen).to(dtype).to(gpu)
    positions = torch.randint(163840, (tokens,), generator=gen).to(gpu)
    positions[0] = 163839
    frequencies = _frequencies(rotated, gpu)
    kwargs = dict(offset=offset, interleaved=interleaved, magnitude=1.37)
    a, b = apply_rope_pair(q, k, positions, frequencies, **kwargs)
    for got, x in ((a, q), (b, k)):
        _check(got, x, positions, frequencies, offset, interleaved, 1.37)
        rest = [i for i in range(dim) if not offset <= i < offset + rotated]
        assert torch.equal(got[..., rest], x[..., rest])
    c, none = apply_rope_pair(q, None, positions.int(), frequencies, **kwargs)
    assert none is None and torch.equal(a, c)


@pytest.mark.parametrize("interleaved", [False, True])
def test_strided_in_place_and_into_wider_heads(gpu, interleaved):
    from cxldsagr_amd.projections import apply_rope_pair

    gen = torch.Generator().manual_seed(42)
    wide = torch.randn(9, 4, 192, generator=gen).bfloat16().to(gpu)
    k = torch.randn(9, 1, 64, generator=gen).bfloat16().to(gpu)
    positions = torch.arange(1000, 1009, device=gpu)
    frequencies = _frequencies(64, gpu)
    want, k_want = apply_rope_pair(wide[..., 128:].contiguous(), k, positions, frequencies,
                                   interleaved=interleaved)
    absorbed = torch.full((9, 4, 576), 3.0, dtype=torch.bfloat16, device=gpu)
    got, _ = apply_rope_pair(wide[..., 128:], k, positions, frequencies, interleaved=interleaved,
                             q_out=absorbed[..., 512:])
    assert got.data_ptr() == absorbed[..., 512:].data_ptr()
    assert torch.equal(absorbed[..., 512:], want) and (absorbed[..., :512] == 3).all()
    # Strides that allow no vectors.
    odd = torch.zeros(9, 4, 195, dtype=torch.bfloat16, device=gpu)
    odd[..., 1:193] = wide
    got, _ = apply_rope_pair(odd[..., 129:193], None, positions, frequencies, interleaved=interleaved)
    assert torch.equal(got, want)
    keep = wide[..., :128].clone()
    got, k_got = apply_rope_pair(wide, k.new_zeros(9, 0, 192), positions, frequencies, offset=128,
                                 interleaved=interleaved, q_out=wide)
    assert got is wide and torch.equal(wide[..., 128:], want) and torch.equal(wide[..., :128], keep)
    got, k_got = apply_rope_pair(want.clone(), k, positions, frequencies, interleaved=interleaved, k_out=k)
    assert k_got is k and torch.equal(k, k_want)


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_gradient(gpu, interleaved):
    """The gradient of sum(g * rope(x)) is the inverse rotation of g: against the formula's
    and against differences."""
    from cxldsagr_amd.projections import apply_rope_pair

    gen = torch.Generator().manual_seed(43)
    x, g = (torch.randn(4, 2, 32, generator=gen).to(gpu) for _ in range(2))
    positions, frequencies = torch.tensor([0, 1, 77, 100000], device=gpu), _frequencies(16, gpu)
    kwargs = dict(offset=8, interleaved=interleaved, magnitude=1.2)
    grad, _ = apply_rope_pair(g, None, positions, frequencies, inverse=True, **kwargs)
    _check(grad, g, positions, frequencies, 8, interleaved, 1.2, inverse=True)
    # The map is linear: a difference of step 1 along each of three directions.
    for seed in range(3):
        step = torch.randn(4, 2, 32, generator=gen).to(gpu)
        rise = (apply_rope_pair(x + step, None, positions, frequencies, **kwargs)[0].double()
                - apply_rope_pair(x, None, positions, frequencies, **kwargs)[0].double())
        # Unrotated dims have gradient g times 1; fp32 results of size ~5 on 256 terms.
        assert (rise * g).sum().item() == pytest.approx((grad.double() * step).sum().item(),
                                                        abs=256 * 5 * 5 * 2.0 ** -20)


def test_far_positions_of_64_bits(gpu):
    from cxldsagr_amd.projections import apply_rope_pair

    x = torch.randn(3, 1, 64, generator=torch.Generator().manual_seed(44)).to(gpu)
    positions = torch.tensor([0, 2 ** 24 + 1, 2 ** 31 + 5], device=gpu)
    got, _ = apply_rope_pair(x, None, positions, _frequencies(64, gpu))
    _check(got, x, positions, _frequencies(64, gpu), 0, False, 1.0)


def test_agrees_with_the_index_producers_table(gpu):
    """The same rotation as ``rotary_table``'s, at positions whose fp32 angles are good."""
    from cxldsagr_amd import projections

    x = torch.randn(64, 2, 64, generator=torch.Generator().manual_seed(45)).to(gpu)
    positions, frequencies = torch.arange(64, device=gpu), _frequencies(64, gpu)
    table = projections.rotary_table(positions.float(), frequencies)
    cos, sin = table[:, None, :32], table[:, None, 32:]
    a, b = x.chunk(2, -1)
    want = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    got, _ = projections.apply_rope_pair(x, None, positions, frequencies)
    # An fp32 angle up to 63 is off by 2^-19 at most.
    torch.testing.assert_close(got, want, rtol=0, atol=2.0 ** -18 * 8)


def test_captured_call_replays(gpu):
    from cxldsagr_amd.projections import apply_rope_pair

    q = torch.randn(33, 4, 64, generator=torch.Generator().manual_seed(46)).bfloat16().to(gpu)
    positions, frequencies = torch.arange(33, device=gpu), _frequencies(64, gpu)
    want, _ = apply_rope_pair(q, None, positions, frequencies)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = apply_rope_pair(q, None, positions, frequencies)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_and_nan_as_in_the_formula(gpu, dtype):
    from cxldsagr_amd.projections import apply_rope_pair

    gen = torch.Generator().manual_seed(47)
    q = torch.randn(9, 4, 64, generator=gen).to(dtype)
    q[1, 0, 3], q[2, 1, 40], q[3, 2, 7], q[0, 3, 5] = float("inf"), -float("inf"), float("nan"), float("inf")
    q[4, 0, 8], q[4, 0, 9] = float("inf"), float("inf")
    positions = torch.arange(9) * 1001
    frequencies = _frequencies(64, gpu)
    for interleaved in (True, False):
        got, _ = apply_rope_pair(q.to(gpu), None, positions.to(gpu), frequencies, interleaved=interleaved)
        want = dense.rope(q, positions, frequencies.cpu(), 0, interleaved, 1.0)
        got = got.cpu().double()
        assert torch.equal(got.isnan(), want.isnan())
        infinite = want.isinf()
        assert torch.equal(got.isinf(), infinite) and torch.equal(got[infinite], want[infinite])


def _near(got, x, positions, frequencies, offset, interleaved, magnitude, inverse=False):
    """cos and sin come from 64-bit angles and a 64-bit magnitude and are rounded once: off by
    2^-24 of themselves and, for the series, less than 2^-31 m. The two products and the sum
    round once each in fp32, the result once to its type (fp32: the sum's rounding). Each is at
    most half a step."""
    want = dense.rope(x, positions, frequencies, offset, interleaved, magnitude, inverse)
    half = len(frequencies)
    part = x.detach().cpu().double()[..., offset:offset + 2 * half].abs()
    if interleaved:
        both = (part[..., 0::2] + part[..., 1::2]).repeat_interleave(2, -1)
    else:
        both = (part[..., :half] + part[..., half:]).repeat(1, 1, 2)
    turned = want[..., offset:offset + 2 * half].abs()
    inner = (2 * 2.0 ** -24 + 2.0 ** -31 + 2.0 ** -47) * abs(magnitude) * both
    inner += 2.0 ** -24 * (turned + inner)
    if x.dtype != torch.float32:  # (fp16 has steps of 2^-24 below 2^-14)
        inner += torch.finfo(x.dtype).eps / 2 * (turned + inner) + 2.0 ** -25
    off = (got.cpu().double() - want)[..., offset:offset + 2 * half].abs()
    assert (off <= inner).all(), (off - inner).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_as_near_as_the_roundings_allow(gpu, dtype, interleaved, inverse):
    from cxldsagr_amd.projections import apply_rope_pair

    gen = torch.Generator().manual_seed(48)
    magnitude = 0.1 * math.log(40.0) + 1.0  # (not a value of 32 bits)
    frequencies = _frequencies(64, gpu)
    positions = torch.randint(163840, (200,), generator=gen).to(gpu)
    positions[:3] = torch.tensor([0, 1, 163839])
    kwargs = dict(offset=128, interleaved=interleaved, magnitude=magnitude, inverse=inverse)
    x = torch.randn(200, 8, 192, generator=gen).to(dtype).to(gpu)
    odd = torch.zeros(200, 8, 193, dtype=dtype, device=gpu)[..., 1:].copy_(x)  # (no vectors)
    for part in (x, odd):
        got, _ = apply_rope_pair(part, None, positions, frequencies, **kwargs)
        _near(got, x, positions, frequencies, 128, interleaved, magnitude, inverse)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_cos_and_sin_are_rounded_once(gpu, interleaved, inverse):
    """Pairs (1, 0) and (0, 1) give them as they are: off by half a step of fp32, 2^-24 of
    themselves, and less than 2^-31 of the magnitude for the series."""
    from cxldsagr_amd.projections import apply_rope_pair

    gen = torch.Generator().manual_seed(49)
    magnitude = 0.1 * math.log(40.0) + 1.0
    frequencies = _frequencies(64, gpu)
    positions = torch.randint(163840, (300,), generator=gen).to(gpu)
    x = torch.zeros(300, 2, 64, device=gpu)
    second = torch.arange(1, 64, 2) if interleaved else torch.arange(32, 64)
    x[:, 0] = 1
    x[:, 0, second] = 0
    x[:, 1, second] = 1
    got, _ = apply_rope_pair(x, None, positions, frequencies, interleaved=interleaved, magnitude=magnitude,
                             inverse=inverse)
    want = dense.rope(x, positions, frequencies, 0, interleaved, magnitude, inverse)
    off = (got.cpu().double() - want).abs()
    assert (off <= 2.0 ** -24 * want.abs() + 2.0 ** -31 * magnitude).all(), (off / want.abs()).max()
