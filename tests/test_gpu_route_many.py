"""``feedforward.route_experts`` where there are many tokens, four of which share a wave: each form
of it (4, 8 and 16 experts a lane at most, whole lanes and partial ones), against the definition
in 64 bits on the first and last tokens and some between.

The weights' error: a score's 2^-24, the sum's scores' 2^-24 and the weight's own."""

import pytest
import torch

from oracle import feedforward as off

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize(
    ("experts", "groups", "top_groups", "k", "dtype"),
    [(64, 1, 1, 4, "fp32"), (50, 1, 1, 8, "bf16"), (64, 16, 5, 6, "fp16"),  # 4 a lane
     (128, 8, 3, 6, "fp32"), (128, 1, 1, 64, "bf16"), (100, 1, 1, 6, "fp32"),  # 5 to 8
     (160, 8, 3, 6, "bf16"), (150, 1, 1, 6, "fp32"), (180, 2, 1, 8, "fp16"), (192, 1, 1, 8, "fp32"),  # 9 to 12
     (256, 8, 4, 8, "fp32"), (256, 1, 1, 8, "fp16"), (240, 8, 2, 8, "bf16"), (176, 16, 4, 8, "fp32")],  # to 16
)
def test_many_tokens(gpu, experts, groups, top_groups, k, dtype, scoring, biased):
    from cxldsagr_amd.feedforward import route_experts

    tokens, inf = 256 * 16 + 21, float("inf")  # (the last work-group's 16 are not all there)
    gen = torch.Generator().manual_seed(experts + k)
    logits = torch.randn(tokens, experts, generator=gen).mul(2)
    for at in (0, tokens - 12):
        logits[at] = 0.0
        logits[at + 1] = torch.randint(-1, 2, (experts,), generator=gen).float()
        logits[at + 2, experts // 3:] = -inf
        logits[at + 3] = -inf
        logits[at + 4, experts // 2] = float("nan")
        logits[at + 5, experts - 1] = inf
        logits[at + 6] = 40.0
        logits[at + 6, ::2] = 17.5
    logits = logits.to(TYPES[dtype])
    bias = None
    if biased:
        bias = 0.1 * torch.randn(experts, generator=gen)
        bias[::7] = -inf  # experts out of service
    some = torch.tensor([*range(18), 33, 1000, 2047, 2048, 4093, *range(tokens - 23, tokens)])
    for renormalize in (True, False):
        how = dict(scoring=scoring, groups=groups, top_groups=top_groups, renormalize=renormalize, scale=2.5)
        weights, ids = route_experts(logits.to(gpu), k, bias=None if bias is None else bias.to(gpu), **how)
        want, want_ids = off.route(logits[some], k, bias=bias, **how)
        assert torch.equal(ids.cpu()[some], want_ids)
        got = weights.cpu()[some].double()
        assert torch.equal(got.isnan(), want.isnan())
        assert ((got - want).abs() <= (3 + 2.0 ** -20) * 2.0 ** -24 * want.abs() + 2.0 ** -148)[~want.isnan()].all()
        # Each as in a call of its own, where a wave takes one token.
        alone = route_experts(logits[some].to(gpu), k, bias=None if bias is None else bias.to(gpu), **how)
        assert torch.equal(alone[1], ids[some.to(gpu)])
        assert torch.equal(alone[0].nan_to_num(7.0), weights[some.to(gpu)].nan_to_num(7.0))
