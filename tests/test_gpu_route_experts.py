"""``feedforward.route_experts`` against the definition in 64 bits: the same experts in the
same order, weights within their roundings (a score's 2^-24, k of the sum, the quotient's
and the product's; the hardware's division is exact to half a step)."""

import pytest
import torch

from oracle import feedforward as off

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def check(gpu, logits, k, bias=None, **how):
    from cxldsagr_amd.feedforward import route_experts

    weights, ids = route_experts(logits.to(gpu), k, bias=None if bias is None else bias.to(gpu), **how)
    want, want_ids = off.route(logits, k, bias=bias, **how)
    assert torch.equal(ids.cpu(), want_ids)
    assert weights.dtype == torch.float32
    bound = (k + 4) * 2.0 ** -24 * want.abs() + 2.0 ** -148
    got = weights.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    assert ((got - want).abs() <= bound)[~want.isnan()].all()


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize(
    ("tokens", "experts", "k", "groups", "top_groups", "biased", "dtype"),
    [(1, 1, 1, 1, 1, False, "fp32"), (5, 8, 2, 1, 1, False, "bf16"), (37, 64, 6, 1, 1, False, "fp32"),
     (33, 256, 8, 8, 4, True, "fp32"), (33, 256, 8, 8, 4, False, "fp32"), (19, 160, 6, 8, 3, False, "bf16"),
     (7, 160, 6, 8, 3, True, "fp16"), (9, 60, 4, 4, 4, True, "fp32"), (5, 384, 8, 1, 1, True, "fp32"),
     (3, 1024, 64, 1, 1, True, "fp32"), (3, 1023, 8, 31, 5, True, "fp32"), (4, 64, 3, 64, 3, True, "fp32"),
     (4, 1024, 16, 64, 2, False, "fp32"), (6, 45, 5, 3, 1, True, "fp32"), (5, 7, 7, 7, 7, True, "fp32"),
     (2, 990, 9, 33, 7, True, "fp32"), (3, 200, 5, 40, 2, True, "bf16")],
)
def test_experts_and_weights(gpu, scoring, tokens, experts, k, groups, top_groups, biased, dtype):
    gen = torch.Generator().manual_seed(experts + k)
    logits = torch.randn(tokens, experts, generator=gen).mul(2).to(TYPES[dtype])
    bias = 0.1 * torch.randn(experts, generator=gen) if biased else None
    for renormalize in (True, False):
        check(gpu, logits, k, bias, scoring=scoring, groups=groups, top_groups=top_groups, renormalize=renormalize,
              scale=2.5)


@pytest.mark.parametrize("groups, top_groups", [(1, 1), (8, 3), (16, 2)])
def test_ties_go_to_the_lower_index(gpu, groups, top_groups):
    gen = torch.Generator().manual_seed(11)
    logits = torch.randint(-2, 3, (50, 64), generator=gen).float()
    logits[0] = 0.0
    logits[1] = 40.0  # sigmoid is 1 in 32 bits from 17 on
    logits[1, ::2] = 17.5
    logits[2] = -200.0  # and 0 below -104
    logits[2, 5] = -300.0
    for bias in (None, torch.randint(-1, 2, (64,), generator=gen).float()):
        for scoring in ("sigmoid", "softmax"):
            check(gpu, logits, 6, bias, scoring=scoring, groups=groups, top_groups=top_groups)


def test_infinities_nan_and_masked_experts(gpu):
    gen = torch.Generator().manual_seed(12)
    logits, inf = torch.randn(8, 32, generator=gen), float("inf")
    logits[0, 3:] = -inf  # fewer live experts than choices
    logits[1, 7] = inf
    logits[2, 9] = float("nan")
    logits[3] = torch.finfo(torch.float32).min
    logits[4] = -inf
    masked = torch.zeros(32)
    masked[::3] = -inf  # experts out of service
    for bias in (None, masked):
        check(gpu, logits, 5, bias)
        check(gpu, logits, 5, bias, groups=4, top_groups=2)
        check(gpu, logits[[0, 3, 5, 6, 7]], 5, bias, scoring="softmax", renormalize=False)
    check(gpu, logits[[1, 2, 4]], 5, scoring="softmax")  # NaN rows


@pytest.mark.parametrize("experts", [64, 63])
def test_rows_that_are_not_contiguous_and_none(gpu, experts):
    from cxldsagr_amd.feedforward import route_experts

    wide = torch.randn(9, 70, generator=torch.Generator().manual_seed(13)).to(gpu)
    got = route_experts(wide[:, 3:3 + experts], 4)
    want = route_experts(wide[:, 3:3 + experts].contiguous(), 4)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    turned = route_experts(wide.t()[:9, :9], 4)
    want = route_experts(wide.t()[:9, :9].contiguous(), 4)
    assert torch.equal(turned[1], want[1])
    weights, ids = route_experts(wide[:0, :experts], 4)
    assert weights.shape == ids.shape == (0, 4)


@pytest.mark.parametrize("tokens", [4001, 20000])
def test_many_tokens_are_each_as_alone(gpu, tokens):
    from cxldsagr_amd.feedforward import route_experts

    gen = torch.Generator().manual_seed(14)
    logits = torch.randn(tokens, 256, generator=gen).to(gpu)
    bias = (0.1 * torch.randn(256, generator=gen)).to(gpu)
    how = dict(bias=bias, groups=8, top_groups=4, scale=2.5)
    weights, ids = route_experts(logits, 8, **how)
    for t in (0, 1, 17, tokens // 2, tokens - 2):
        one = route_experts(logits[t:t + 1], 8, **how)
        assert torch.equal(one[0][0], weights[t]) and torch.equal(one[1][0], ids[t])
    part = slice(tokens - 33, tokens)
    want, want_ids = off.route(logits[part], 8, bias=bias, groups=8, top_groups=4, scale=2.5)
    assert torch.equal(ids[part].cpu(), want_ids)
    assert ((weights[part].cpu().double() - want).abs() <= 12 * 2.0 ** -24 * want).all()


@pytest.mark.parametrize("experts, stride, tokens", [(1024, 1024, 2_100_001), (100, 70_003, 31_000)])
def test_offsets_that_pass_32_bits(gpu, experts, stride, tokens):
    from cxldsagr_amd.feedforward import route_experts

    assert tokens * stride > 2 ** 31
    gen = torch.Generator(device=gpu).manual_seed(15)
    logits = torch.empty(tokens, stride, device=gpu, dtype=torch.bfloat16)[:, :experts]
    logits.normal_(generator=gen)
    weights, ids = route_experts(logits, 6)
    for part in (slice(tokens - 7, tokens), slice(0, 7)):
        want = route_experts(logits[part].contiguous(), 6)
        assert torch.equal(weights[part], want[0]) and torch.equal(ids[part], want[1])


@pytest.mark.parametrize("tokens", [37, 5000])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("k", [1, 6, 64])
def test_weights_are_rounded_once(gpu, k, scoring, tokens):
    """From the scores of 32 bits (weights without a sum and a scale) the formula in 64 bits:
    half a step, 2^-24 of the value, and what the 64 bits lose, below 2^-40."""
    from cxldsagr_amd.feedforward import route_experts

    gen = torch.Generator().manual_seed(16 + k)
    logits = torch.randn(tokens, 128, generator=gen).mul(3).to(gpu)
    scores, ids = route_experts(logits, k, scoring=scoring, renormalize=False)
    wide = scores.double()
    for renormalize, want in ((True, wide / (wide.sum(1, keepdim=True) + 1e-20) * 2.3), (False, wide * 2.3)):
        weights, same = route_experts(logits, k, scoring=scoring, renormalize=renormalize, scale=2.3)
        assert torch.equal(same, ids)
        assert ((weights.double() - want).abs() <= (2.0 ** -24 + 2.0 ** -40) * want + 2.0 ** -150).all()
