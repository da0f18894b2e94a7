"""The oracle of the operators behind the attention, on closed forms and library routines."""

import math

import pytest
import torch

from oracle import feedforward as off


def test_norm_of_a_constant_row():
    y, t = off.rms_norm(torch.full((2, 8), 3.0), torch.arange(8.0), torch.full((2, 8), 1.0), eps=0.0)
    assert torch.equal(t, torch.full((2, 8), 4.0, dtype=torch.float64))
    assert torch.allclose(y, torch.arange(8.0, dtype=torch.float64).expand(2, 8), atol=1e-15)


def test_e4m3_is_the_library_cast():
    values = torch.cat([torch.linspace(-448, 448, 20011), torch.linspace(-0.02, 0.02, 4001)])
    got, step, border = off.e4m3(values.double())
    assert torch.equal(got, values.to(torch.float8_e4m3fn).double())
    # A value moved by less than its border keeps its code, by a little more loses it.
    inside = (values.double() + 0.98 * border).abs() <= 448
    assert torch.equal(off.e4m3(values.double() + 0.98 * border)[0][inside], got[inside])


@pytest.mark.parametrize("amax, scale", [(448.0, 1.0), (449.0, 2.0), (0.0, 2.0 ** -22), (224.0, 0.5),
                                         (1e30, 2.0 ** 91)])
def test_scale(amax, scale):
    assert off.scale_of(amax) == scale


def test_quantized_rows_are_the_quantiser_s():
    from oracle import quantize

    rows = torch.randn(5, 256, generator=torch.Generator().manual_seed(1)).bfloat16()
    codes, scales = quantize.quantize_index(rows.float().view(5, 2, 128).numpy())
    want = torch.from_numpy(codes).view(torch.float8_e4m3fn).double() * torch.from_numpy(scales).double()
    assert torch.equal(off.quantized(rows.double())[0], want.reshape(5, 256))
    assert not off.quantized(rows.double())[1].any()


def test_moved_covers_what_a_change_moves():
    gen = torch.Generator().manual_seed(2)
    rows = torch.randn(40, 128, generator=gen).double()
    # Some blocks whose largest value lies at a scale's border.
    rows[:10, 0] = 3.5 * (1 + 1e-4 * torch.randn(10, generator=gen).double())
    slack = 1e-3 * rows.abs()
    value, moved = off.quantized(rows, slack)
    for _ in range(20):
        other = off.quantized(rows + slack * (2 * torch.rand(rows.shape, generator=gen) - 1))[0]
        assert ((other - value).abs() <= moved).all()


def test_route_by_hand():
    logits = torch.tensor([[0.0, 1.0, 1.0, -1.0], [2.0, 0.0, 0.0, 5.0]])
    weights, ids = off.route(logits, 2)
    assert ids.tolist() == [[1, 2], [3, 0]]
    assert torch.allclose(weights.sum(1), torch.ones(2, dtype=torch.float64))
    weights, ids = off.route(logits, 2, scoring="softmax", renormalize=False, scale=2.0)
    assert weights[1, 0].item() == pytest.approx(2 * math.exp(5) / (math.exp(5) + math.exp(2) + 2))
    # The bias ranks, and does not weigh; of groups the one with the two best sums.
    _, ids = off.route(logits, 1, bias=torch.tensor([5.0, 0.0, 0.0, 0.0]))
    assert ids.tolist() == [[0], [0]]
    _, ids = off.route(logits, 1, bias=torch.zeros(4), groups=2, top_groups=1)
    assert ids.tolist() == [[1], [3]]  # 0.5 + 0.73 against 0.73 + 0.27; 0.88 + 0.5 against 0.5 + 0.99
    _, ids = off.route(torch.tensor([[0.0, float("nan"), 9.0, float("-inf")]]), 4)
    assert ids.tolist() == [[1, 2, 0, 3]]


def test_experts_of_unit_weights():
    # gate = up = x's first 128 values, down the identity: x * silu(x), in codes.
    eye = torch.eye(128).to(torch.float8_e4m3fn)
    one = torch.ones(1, 1, 1)
    x = torch.randn(3, 128, generator=torch.Generator().manual_seed(3)).to(torch.float8_e4m3fn)
    out, bound = off.expert_mlp(x, torch.full((3, 1), 2.0), torch.cat([eye, eye])[None],
                                torch.ones(1, 2, 1), eye[None], one, torch.tensor([[4], [4], [5]]),
                                torch.tensor([[1.0], [0.5], [1.0]]), first=4)
    rows = 2 * x.double()
    want = off.quantized(rows * rows * torch.sigmoid(rows))[0]
    assert torch.allclose(out[0], want[0], atol=1e-12) and torch.allclose(out[1], want[1] / 2, atol=1e-12)
    assert not out[2].any() and not bound[2].any()


def test_what_the_unit_cuts_off():
    row = torch.zeros(1, 24, dtype=torch.float64)
    row[0, 0], row[0, 1], row[0, 2] = 1.75, 15 * 2.0 ** -13, -1.75 * 2.0 ** -13
    row[0, 8], row[0, 9], row[0, 23] = -1.0, 2.0 ** -7, 2.0 ** -20
    weight = torch.ones(3, 24, dtype=torch.float64)
    weight[1] = -1.5
    weight[2, 9] = 2.0 ** -8  # the product 2^-15 beside 1
    # 15 units of 2^-13 stay, of 1.75 one does, of 2.625 two do; alone all is whole.
    want = torch.tensor([[-0.75 * 2.0 ** -13, (0.625 - 0.5) * 2.0 ** -13, (0.25 - 0.75) * 2.0 ** -13]], dtype=torch.float64)
    assert torch.equal(off.cut_off(row, weight), want)
    assert not off.cut_off(torch.zeros(1, 24, dtype=torch.float64), weight).any()
    assert torch.equal(off.cut_off(row, weight, torch.zeros_like(row)), want.abs())
    # The first eight may be off: what each may lose of 1.75 (2 with what it may be off by).
    moved = torch.zeros_like(row)
    moved[0, 0] = 0.25
    got = off.cut_off(row, weight[:1], moved)
    assert torch.equal(got, torch.tensor([[(2.0 + 1.75) * 2.0 ** -13]], dtype=torch.float64))
