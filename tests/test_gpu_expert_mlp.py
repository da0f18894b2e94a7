"""``feedforward.expert_mlp`` against the formula in 64 bits, within the bound that the oracle
derives from the kernel's roundings element by element, plus the result's own."""

import pytest
import torch

from oracle import feedforward as off

pytestmark = pytest.mark.gpu

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def tokens_in_codes(gen, tokens, dim):
    x = torch.randn(tokens, dim, generator=gen)
    scale = torch.exp2(torch.randint(-3, 2, (tokens, dim // 128), generator=gen).float())
    return (x * 60).to(F8), (scale / 64).to(E8)


def matrix(gen, experts, rows, columns):
    codes = torch.randn(experts, rows, columns, generator=gen) * 60
    if columns > 8192:
        # One of 64 columns, any in a block: a sum of as many terms as a shallow one's.
        at = torch.randint(0, 64, (1, 1, columns // 64, 1), generator=gen)
        codes = torch.where(torch.arange(64) == at, codes.view(experts, rows, -1, 64), 0).view(experts, rows, columns)
    codes = codes.to(F8)
    scale = torch.exp2(torch.randint(-2, 2, (experts, rows // 128, columns // 128), generator=gen).float())
    terms = columns if columns <= 8192 else columns // 64
    return codes, scale / 64 * 2.0 ** -round(torch.tensor(terms).double().log2().item() / 2)


class Model:
    def __init__(self, gpu, dim, inner, experts, first=0, total=None, seed=0):
        from cxldsagr_amd.feedforward import ExpertWeights

        gen = torch.Generator().manual_seed(seed + dim + inner)
        self.parts = (*matrix(gen, experts, 2 * inner, dim), *matrix(gen, experts, dim, inner))
        self.own = ExpertWeights(*(t.to(gpu) for t in self.parts), first=first, total=total)
        self.first, self.gen, self.gpu, self.dim = first, gen, gpu, dim
        self.inner, self.part = inner, experts / (self.own.total)

    def tokens(self, tokens, choices, low, high):
        x, scale = tokens_in_codes(self.gen, tokens, self.dim)
        ids = torch.randint(low, high, (tokens, choices), generator=self.gen, dtype=torch.int32)
        return x, scale, ids, torch.randn(tokens, choices, generator=self.gen)

    def run(self, x, scale, ids, weights, **how):
        from cxldsagr_amd.feedforward import expert_mlp

        return expert_mlp(x.to(self.gpu), scale.to(self.gpu), self.own, ids.to(self.gpu), weights.to(self.gpu), **how)

    def check(self, x, scale, ids, weights, dtype=torch.bfloat16):
        got = self.run(x, scale, ids, weights, dtype=dtype)
        assert got.dtype == dtype and got.shape == x.shape
        # (Up to 2^20 values of h, or 16 rows an expert, up's products are in 16 bits.)
        want, bound = off.expert_mlp(x, scale, *self.parts, ids, weights, self.first,
                                     cut_up=ids.numel() * self.part * self.inner > 2 ** 20 and ids.numel() >= 17 * self.own.total)
        bound = bound + torch.finfo(dtype).eps / 2 * (want.abs() + bound) + 2.0 ** -25
        far = (got.cpu().double() - want).abs()
        assert (far <= bound).all(), (far / bound).max()
        # The bound is one of roundings: most of it is the codes of silu(gate) * up.
        assert bound.mean() < 0.2 * want.abs().mean().clamp_min(1e-3)
        return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_types(gpu, dtype):
    model = Model(gpu, 256, 128, 3)
    model.check(*model.tokens(5, 2, 0, 3), dtype=dtype)


@pytest.mark.parametrize(
    ("tokens", "choices", "dim", "inner", "experts"),
    [(1, 1, 128, 128, 1), (1, 8, 512, 256, 8), (2, 3, 384, 384, 5), (17, 4, 640, 128, 16), (31, 2, 256, 640, 4),
     (33, 1, 896, 256, 1), (64, 8, 256, 256, 6), (129, 3, 384, 128, 2), (257, 2, 1152, 384, 3), (300, 6, 256, 128, 40),
     (1, 64, 256, 128, 70)],
)
def test_sizes(gpu, tokens, choices, dim, inner, experts):
    model = Model(gpu, dim, inner, experts, seed=tokens)
    model.check(*model.tokens(tokens, choices, 0, experts))


@pytest.mark.parametrize("rows", [15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 513])
@pytest.mark.parametrize("experts", [3, 2])
def test_rows_around_a_tile(gpu, rows, experts):
    """One expert with so many rows, one with a single one, one with none or none more."""
    model = Model(gpu, 256, 128, experts)
    x, scale, ids, weights = model.tokens(rows + 1, 1, experts - 2, experts - 1)
    ids[rows // 2] = experts - 1
    model.check(x, scale, ids, weights)


@pytest.mark.parametrize("rows", [1, 3, 16, 17, 31, 33, 47, 49, 63, 65, 96, 127, 129, 257, 300, 513])
def test_rows_around_a_tile_of_long_calls(gpu, rows):
    """More than 2^20 values of h: each expert with a row more or less than the next."""
    inner, dim = (4096, 128) if rows > 1 else (16128, 256)
    experts = max(2, -(-(2 ** 20 + 1) // (rows * inner)) + 1)
    model = Model(gpu, dim, inner, experts)
    ids = torch.repeat_interleave(torch.arange(experts), torch.tensor([rows - 1, rows + 1] * experts)[:experts])
    x, scale, _, weights = model.tokens(len(ids), 1, 0, experts)
    ids = ids[torch.randperm(len(ids), generator=model.gen)].int()[:, None]
    assert ids.numel() * inner > 2 ** 20
    model.check(x, scale, ids, weights)


@pytest.mark.parametrize("tokens, experts, inner", [(1, 1, 4096), (2, 1, 2048), (40, 8, 1024)])
def test_hidden_codes_of_few_values(gpu, tokens, experts, inner):
    """Codes of h as the results of a down that picks them: those of 64 bits, but for one in
    20,000 (silu's 2^-21 of a value, within a step of 1/8 to 1/16 of it, is half of that)."""
    from cxldsagr_amd.feedforward import ExpertWeights

    dim = inner
    model = Model(gpu, dim, inner, experts)
    model.parts = (*model.parts[:2], torch.eye(inner).expand(experts, inner, inner).contiguous().to(F8),
                   torch.ones(experts, inner // 128, inner // 128))
    model.own = ExpertWeights(*(t.to(gpu) for t in model.parts))
    x, scale, ids, weights = model.tokens(tokens, 1, 0, experts)
    got = model.run(x, scale, ids, torch.ones_like(weights), dtype=torch.float32).cpu().double()
    rows = off.wide(x) * off.wide(scale).repeat_interleave(128, 1)
    both = torch.stack([rows[t] @ off.weight_values(*(p[ids[t]] for p in model.parts[:2]))[0].t() for t in range(tokens)])
    want, _ = off.quantized(off.silu(both[:, :inner]) * both[:, inner:])
    assert int((got != want).sum()) <= 2 + want.numel() // 20000


@pytest.mark.parametrize(
    ("tokens", "choices", "dim", "inner", "experts", "total"),
    [(60, 1, 16128, 128, 1, 1), (2, 2, 16128, 128, 2, 6), (1, 8, 128, 16128, 1, 1), (70, 1, 128, 16128, 1, 1),
     (1, 64, 128, 1024, 3, 90), (3, 5, 256, 384, 4, 40), (6, 2, 384, 256, 8, 16), (7, 2, 384, 256, 8, 16),
     (40, 1, 32768, 128, 1, 1)],
)
def test_deep_products_and_pairs_by_themselves(gpu, tokens, choices, dim, inner, experts, total):
    """Depths whose scales or codes do not fit where those of others do; few tokens of many
    experts, some of them other ranks'."""
    model = Model(gpu, dim, inner, experts, first=(total - experts) // 2, total=total, seed=choices)
    model.check(*model.tokens(tokens, choices, 0, total))


@pytest.mark.parametrize("seed", [9, 11, 12, 13])
def test_small_sums_of_large_products(gpu, seed):
    """Results far smaller than the products in them, as exact as 32 bits can show them."""
    model = Model(gpu, 128, 128, 1, first=2, total=11, seed=seed)
    model.check(*model.tokens(339, 4, 2, 3), dtype=torch.float32)
    model.check(*model.tokens(339, 4, 0, 11), dtype=torch.float32)


def test_choices_of_other_ranks_none_and_twice(gpu):
    """Slices of the experts sum to the whole; what is not here adds nothing."""
    model = Model(gpu, 256, 128, 4, first=10, total=24)
    x, scale, ids, weights = model.tokens(40, 4, 6, 18)
    ids[0], ids[1], ids[2], ids[3] = -1, 12, 2 ** 31 - 1, -2 ** 31
    weights[2] = float("nan")  # of choices that are not here
    got = model.check(x, scale, ids, weights.nan_to_num())
    assert not got[0].any() and not got[2].any() and not got[3].any()
    assert torch.equal(model.run(x, scale, ids, weights), got)
    one = model.run(x[:3], scale[:3], ids[:3], weights[:3])
    assert not one[0].any() and not one[2].any()
    want, bound = off.expert_mlp(x[1:2], scale[1:2], *model.parts, ids[1:2], weights[1:2], model.first)
    assert ((one[1].cpu().double() - want[0]).abs() <= bound[0] + 2.0 ** -8 * (want[0].abs() + bound[0])).all()
    nothing = model.run(x, scale, torch.full_like(ids, 9), weights)
    assert nothing.shape == x.shape and not nothing.any()
    assert model.run(x[:0], scale[:0], ids[:0], weights[:0]).shape == (0, 256)


@pytest.mark.parametrize("tokens, total", [(9, 2), (200, 2), (9, 60), (4200, 2)])
def test_a_row_s_infinities_and_nan_stay_in_it(gpu, tokens, total):
    model = Model(gpu, 256, 128, 2, total=total)
    x, scale, ids, weights = model.tokens(tokens, 2, 0, 2)
    clean = model.run(x, scale, ids, weights)
    scale.view(torch.uint8)[2, 1] = 255  # NaN
    x.view(torch.uint8)[4, 7] = 127  # NaN
    weights[6, 0] = float("inf")
    scale.view(torch.uint8)[7] = 254  # 2^127: products overflow
    got = model.run(x, scale, ids, weights)
    keep = [t for t in range(tokens) if t not in (2, 4, 6, 7)]
    assert torch.equal(got[keep], clean[keep])
    assert got[2].isnan().all() and got[4].isnan().all()
    assert not got[6].isfinite().any() and not got[7].isfinite().any()


@pytest.mark.parametrize("tokens", [6, 4200])
@pytest.mark.parametrize("power", [-40, -20, 20, 40])
def test_scales_far_from_one(gpu, power, tokens):
    """Exponents of tokens and weights that cancel in part; results far below and above 1."""
    model = Model(gpu, 256, 128, 2)
    x, scale, ids, weights = model.tokens(tokens, 2, 0, 2)
    scale = (scale.float() * 2.0 ** power).to(E8)
    model.parts = (*model.parts[:2], model.parts[2], model.parts[3] * 2.0 ** (power // 2))
    from cxldsagr_amd.feedforward import ExpertWeights

    model.own = ExpertWeights(*(t.to(gpu) for t in model.parts))
    got = model.run(x, scale, ids, weights, dtype=torch.float32)[:6]
    want, bound = off.expert_mlp(x[:6], scale[:6], *model.parts, ids[:6], weights[:6], cut_up=tokens > 6)
    bound = bound + 2.0 ** -24 * (want.abs() + bound) + 2.0 ** -149
    assert ((got.cpu().double() - want).abs() <= bound).all()


def test_inputs_that_are_not_contiguous_and_an_output_given(gpu):
    from cxldsagr_amd.feedforward import expert_mlp

    model = Model(gpu, 256, 128, 3)
    x, scale, ids, weights = (t.to(gpu) for t in model.tokens(12, 4, 0, 3))
    want = model.run(x, scale, ids, weights)
    wide = torch.zeros(12, 300, dtype=torch.uint8, device=gpu)
    wide[:, 5:261] = x.view(torch.uint8)
    out = torch.full((13, 256), 7.0, dtype=torch.bfloat16, device=gpu)
    got = expert_mlp(wide.view(F8)[:, 5:261], scale.view(torch.uint8).t().contiguous().t().view(E8), model.own,
                     ids.t().contiguous().t(), weights.repeat_interleave(2, 1)[:, ::2], out=out[:12])
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(out[:12], want) and (out[12] == 7).all()


@pytest.mark.parametrize("tokens", [2, 60])
def test_scales_at_any_address(gpu, tokens):
    model = Model(gpu, 512, 128, 1)
    x, scale, ids, weights = (t.to(gpu) for t in model.tokens(tokens, 1, 0, 1))
    flat = torch.zeros(tokens * 4 + 1, dtype=torch.uint8, device=gpu)
    flat[1:] = scale.view(torch.uint8).flatten()
    got = model.run(x, flat[1:].view(E8).view(tokens, 4), ids, weights)
    assert torch.equal(got, model.run(x, scale, ids, weights))


def test_many_rows_are_each_as_in_small_calls(gpu):
    """A large batch against the formula on some of its tokens."""
    model = Model(gpu, 512, 256, 4)
    x, scale, ids, weights = model.tokens(3000, 3, 0, 4)
    got = model.run(x, scale, ids, weights)
    some = torch.tensor([0, 1, 511, 1500, 2047, 2998, 2999])
    want, bound = off.expert_mlp(x[some], scale[some], *model.parts, ids[some], weights[some])
    bound = bound + 2.0 ** -8 * (want.abs() + bound)
    assert ((got[some.to(gpu)].cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("tokens, dim, inner", [(8300, 16128, 128), (4161, 32768, 256)])
def test_many_rows_of_deep_products(gpu, tokens, dim, inner):
    """Depths whose rows' scales do not fit beside the largest tile, on some of the rows."""
    model = Model(gpu, dim, inner, 1)
    x, scale, ids, weights = model.tokens(tokens, 1, 0, 1)
    got = model.run(x, scale, ids, weights)
    some = torch.tensor([0, 1, 31, 32, 63, 64, 127, 128, tokens // 2, tokens - 65, tokens - 2, tokens - 1])
    want, bound = off.expert_mlp(x[some], scale[some], *model.parts, ids[some], weights[some])
    bound = bound + 2.0 ** -8 * (want.abs() + bound)
    assert ((got[some.to(gpu)].cpu().double() - want).abs() <= bound).all()


def test_offsets_that_pass_32_bits(gpu):
    """Inputs, weights, hidden codes and results of more than 2^31 elements each: the last
    and the first tokens as in a call of their own."""
    from cxldsagr_amd.feedforward import ExpertWeights, expert_mlp

    tokens, dim, inner, experts = 300_001, 7168, 4096, 40
    gen = torch.Generator(device=gpu).manual_seed(51)

    def codes(*shape):  # (magnitudes below 1, no NaN)
        return torch.randint(0, 256, shape, generator=gen, device=gpu, dtype=torch.uint8).bitwise_and_(0xBF).view(F8)

    def scales(*shape):
        return torch.randint(118, 122, shape, generator=gen, device=gpu, dtype=torch.uint8).view(E8)

    own = ExpertWeights(codes(experts, 2 * inner, dim), scales(experts, inner // 64, dim // 128),
                        codes(experts, dim, inner), scales(experts, dim // 128, inner // 128))
    x, scale = codes(tokens, dim), scales(tokens, dim // 128)
    ids = torch.randint(0, experts, (tokens, 2), generator=gen, device=gpu, dtype=torch.int32)
    ids[-3000:, 0] = experts - 1  # the last rows and the last weights of all
    weights = torch.rand(tokens, 2, generator=gen, device=gpu)
    assert min(x.numel(), own.gate_up.numel(), 2 * tokens * inner, 2 * tokens * dim) > 2 ** 31
    got = expert_mlp(x, scale, own, ids, weights)
    for part in (slice(tokens - 3000, tokens), slice(0, 3000)):
        want = expert_mlp(x[part], scale[part], own, ids[part], weights[part])
        assert want.abs().amax(1).min() > 0 and torch.equal(got[part], want)


def test_the_most_tokens(gpu):
    """2^22 tokens, the last of which is joined by a launch of its own; few have a choice here."""
    from cxldsagr_amd.feedforward import expert_mlp

    tokens, dim = 1 << 22, 6272  # four work-groups a token
    model = Model(gpu, dim, 128, 1)
    some = torch.tensor([0, 77, tokens - 3, tokens - 2, tokens - 1])
    few, few_scale, few_ids, few_weights = model.tokens(len(some), 1, 0, 1)
    x = torch.zeros(tokens, dim, dtype=torch.uint8, device=gpu)
    scale = torch.zeros(tokens, dim // 128, dtype=torch.uint8, device=gpu)
    ids = torch.full((tokens, 1), -1, dtype=torch.int32, device=gpu)
    weights = torch.zeros(tokens, 1, device=gpu)
    out = torch.empty(tokens, dim, dtype=torch.bfloat16, device=gpu).fill_(7.0)
    for to, of in ((x, few.view(torch.uint8)), (scale, few_scale.view(torch.uint8)), (ids, few_ids), (weights, few_weights)):
        to[some.to(gpu)] = of.to(gpu)
    expert_mlp(x.view(F8), scale.view(E8), model.own, ids, weights, out=out)
    want, bound = off.expert_mlp(few, few_scale, *model.parts, few_ids, few_weights)
    bound = bound + 2.0 ** -8 * (want.abs() + bound) + 2.0 ** -25
    assert ((out[some.to(gpu)].cpu().double() - want).abs() <= bound).all()
    out[some.to(gpu)] = 0
    assert not any(bool(part.any()) for part in out.split(1 << 18))
    del x, scale, ids, weights, out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("choices, inner", [(8, 2048), (3, 384), (64, 128)])
def test_pairs_of_other_ranks_are_not_read(gpu, choices, inner):
    """A slice of many experts, pairs by themselves, over a workspace and a result of NaN: as over
    zeros; tokens without a choice here are zeros."""
    from cxldsagr_amd import _native

    experts, total, dim, tokens = 8, 64 * choices, 384, 9
    model = Model(gpu, dim, inner, experts, first=16, total=total)
    x, scale, ids, weights = (t.to(gpu) for t in model.tokens(tokens, choices, 0, total))
    ids[0], ids[1], ids[2, 0], ids[3] = 5, 17, 23, -1  # none, all, at least one, none
    want = model.check(x, scale, ids, weights)
    assert want[1].any() and want[2].any() and not want[0].any() and not want[3].any()
    own = model.own
    needed = _native.size_of("dsa_expert_mlp_workspace_bytes", 0, tokens, choices, dim, inner, experts, total)
    assert needed == tokens * choices * inner * 4  # (the pairs' hidden values alone)
    for fill in (0, 255):
        workspace = torch.full((needed,), fill, dtype=torch.uint8, device=gpu)
        out = torch.full((tokens, dim), float("nan"), dtype=torch.bfloat16, device=gpu)
        _native.call("dsa_expert_mlp_fp8", x.data_ptr(), scale.data_ptr(), tokens, dim, inner, own.gate_up.data_ptr(),
                     own.gate_up_scale.data_ptr(), own.down.data_ptr(), own.down_scale.data_ptr(), experts, own.first,
                     total, ids.data_ptr(), weights.data_ptr(), choices, out.data_ptr(), 0, workspace.data_ptr(), needed,
                     torch.cuda.current_stream().cuda_stream)
        assert torch.equal(out, want)
