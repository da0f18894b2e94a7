"""``feedforward.residual_rms_norm`` against the formula in 64 bits.

The kernel sums and normalises in 64 bits and rounds the result to 32 and then to the
type: off by at most half a step of the type and half a step of fp32, 2^-24, relative
(fp32: half a step, and the 64-bit sums' 2^-45 or so)."""

import pytest
import torch

from oracle import feedforward as off

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def rows(gen, tokens, dim, dtype):
    loud = 1 + 30 * (torch.rand(dim, generator=gen) < 0.02)
    return (torch.randn(tokens, dim, generator=gen) * loud).to(dtype)


def near(got, want, dtype):
    eps = torch.finfo(dtype).eps / 2
    bound = (eps + (2.0 ** -24 if dtype != torch.float32 else 2.0 ** -40)) * want.abs()
    tiny = torch.finfo(dtype).smallest_normal * eps * 2  # a subnormal's step
    assert ((got.cpu().double() - want).abs() <= bound + tiny).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize(
    ("tokens", "dim", "residual", "quantize"),
    [(1, 1, False, False), (3, 7, True, False), (5, 128, True, True), (1, 7168, True, True), (17, 1536, False, True),
     (9, 4096, True, True), (4, 4104, True, False), (3, 8320, True, True), (2, 16384, True, True),
     (2, 16383, True, False), (1025, 384, True, True)],
)
def test_values_codes_and_sum(gpu, dtype, tokens, dim, residual, quantize):
    from cxldsagr_amd.feedforward import residual_rms_norm
    from cxldsagr_amd.indexer import quantize_index

    dtype = TYPES[dtype]
    gen = torch.Generator().manual_seed(dim + tokens)
    x, weight = rows(gen, tokens, dim, dtype), torch.randn(dim, generator=gen)
    r = rows(gen, tokens, dim, dtype) if residual else None
    for w in (weight, weight.to(dtype)):
        got = residual_rms_norm(x.to(gpu), w.to(gpu), None if r is None else r.to(gpu), eps=1e-5, quantize=quantize)
        y, t = off.rms_norm(x, w, r, 1e-5)
        near(got.values, y, dtype)
        if residual:
            assert torch.equal(got.residual.cpu(), t.to(dtype))
        else:
            assert got.residual is None
        if not quantize:
            assert got.codes is None and got.scales is None
            continue
        # The quantiser's own codes of these values, bit for bit.
        codes, scales = quantize_index(got.values.view(tokens, dim // 128, 128))
        assert torch.equal(got.codes.view(torch.uint8), codes.view(tokens, dim).view(torch.uint8))
        assert torch.equal(got.scales.float(), scales.view(tokens, -1))
        only = residual_rms_norm(x.to(gpu), w.to(gpu), None if r is None else r.to(gpu), eps=1e-5, values=False,
                                 quantize=True)
        assert only.values is None and torch.equal(only.codes.view(torch.uint8), got.codes.view(torch.uint8))


@pytest.mark.parametrize("shift, pad", [(0, 0), (1, 3), (8, 8), (0, 4)])
@pytest.mark.parametrize("quantize", [False, True])
def test_strides_and_alignment(gpu, shift, pad, quantize):
    from cxldsagr_amd.feedforward import residual_rms_norm

    gen = torch.Generator().manual_seed(5)
    wide = rows(gen, 6, 512 + shift + pad, torch.bfloat16).to(gpu)
    other = rows(gen, 6, 512 + 8, torch.bfloat16).to(gpu)
    weight = torch.randn(513, generator=gen).to(gpu)[1:]
    x, r = wide[:, shift:shift + 512], other[:, 8:]
    got = residual_rms_norm(x, weight, r, quantize=quantize)
    want = residual_rms_norm(x.contiguous(), weight.clone(), r.contiguous(), quantize=quantize)
    assert torch.equal(got.values, want.values) and torch.equal(got.residual, want.residual)
    if quantize:
        assert torch.equal(got.codes.view(torch.uint8), want.codes.view(torch.uint8))
    # Columns as rows, and one row for all.
    across = residual_rms_norm(x.t()[:, :6], torch.ones(6, device=gpu))
    assert torch.equal(across.values, residual_rms_norm(x.t().contiguous(), torch.ones(6, device=gpu)).values)
    one = residual_rms_norm(x[:1].expand(4, -1), weight)
    assert torch.equal(one.values, one.values[:1].expand(4, -1))


@pytest.mark.parametrize("dim", [512, 509])
def test_sum_in_place_and_no_rows(gpu, dim):
    from cxldsagr_amd.feedforward import residual_rms_norm

    gen = torch.Generator().manual_seed(6)
    x, r = (rows(gen, 33, dim, torch.bfloat16).to(gpu) for _ in range(2))
    weight = torch.ones(dim, device=gpu)
    want = residual_rms_norm(x, weight, r)
    kept = r.clone()
    got = residual_rms_norm(x, weight, kept, residual_out=kept)
    assert got.residual is kept
    assert torch.equal(kept, want.residual) and torch.equal(got.values, want.values)
    none = residual_rms_norm(x[:0], weight, r[:0], quantize=dim == 512)
    assert none.values.shape == (0, dim) and none.residual.shape == (0, dim)


def test_zeros_infinities_and_nan_stay_in_their_rows(gpu):
    from cxldsagr_amd.feedforward import residual_rms_norm

    x = rows(torch.Generator().manual_seed(7), 6, 256, torch.bfloat16)
    clean = residual_rms_norm(x.to(gpu), torch.ones(256, device=gpu), quantize=True)
    x[1], x[2, 5], x[3, 200], x[4] = 0, float("inf"), float("nan"), 1e38
    got = residual_rms_norm(x.to(gpu), torch.ones(256, device=gpu), quantize=True)
    for row in (0, 5):
        assert torch.equal(got.values[row], clean.values[row])
        assert torch.equal(got.codes[row].view(torch.uint8), clean.codes[row].view(torch.uint8))
    assert not got.values[1].any() and not got.codes[1].float().any()
    assert got.values[2, 5].isnan() and not got.values[2, :5].any()  # inf / inf, x / inf
    assert got.values[3].isnan().all() and got.codes[3].float().isnan().all()
    # 64-bit squares: 1e38 does not overflow the mean.
    assert torch.equal(got.values[4].float(), torch.ones(256, device=gpu))


@pytest.mark.parametrize("dim", [16384, 16383])
def test_offsets_that_pass_32_bits(gpu, dim):
    from cxldsagr_amd.feedforward import residual_rms_norm

    tokens, quantize = 132_000, dim % 128 == 0
    assert tokens * dim > 2 ** 31
    gen = torch.Generator(device=gpu).manual_seed(8)
    x, r = (torch.randn(tokens, dim, generator=gen, device=gpu, dtype=torch.bfloat16) for _ in range(2))
    weight = torch.randn(dim, generator=gen, device=gpu)
    got = residual_rms_norm(x, weight, r, quantize=quantize)
    for part in (slice(tokens - 5, tokens), slice(0, 5)):
        want = residual_rms_norm(x[part], weight, r[part], quantize=quantize)
        assert torch.equal(got.values[part], want.values) and torch.equal(got.residual[part], want.residual)
        if quantize:
            for a, b in ((got.codes, want.codes), (got.scales, want.scales)):
                assert torch.equal(a[part].view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype, bits", [("bf16", 8), ("fp16", 11)])
@pytest.mark.parametrize("dim", [7168, 7161])
def test_values_are_rounded_to_32_bits_and_then_to_the_type(gpu, dtype, bits, dim):
    """As a cast of the 64-bit value does: every value, and not all are those of one rounding.
    (The kernel's 46 bits fall on another side of a border of 32 in one of 2^22 values, which
    shows in 16 bits where that is next to a tie, one in 2^13 or fewer of these.)"""
    from cxldsagr_amd.feedforward import residual_rms_norm

    gen = torch.Generator(device=gpu).manual_seed(31)
    tokens, dtype = 1024, TYPES[dtype]
    x, r = (torch.randn(tokens, dim, generator=gen, device=gpu).to(dtype) for _ in range(2))
    weight = 1 + 0.1 * torch.randn(dim, generator=gen, device=gpu)
    got = residual_rms_norm(x, weight, r)
    t = (x.float() + r.float()).double()
    want = t / (t.square().mean(1, keepdim=True) + 1e-6).sqrt() * weight.double()
    assert torch.equal(got.values, want.float().to(dtype))
    part, power = torch.frexp(want)
    once = torch.ldexp((part * 2.0 ** bits).round(), power - bits)  # (ties to even, as round)
    normal = want.abs() >= torch.finfo(dtype).smallest_normal
    assert int((once != got.values.double())[normal].sum()) > 0
