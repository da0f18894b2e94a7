"""The 64-bit oracle of the dense operators on closed forms (CPU)."""

import math

import pytest
import torch

from oracle import dense


def test_attention_closed_forms():
    k = torch.tensor([[0.0], [0.0], [math.log(3.0)]], dtype=torch.float64)
    v = torch.tensor([[1.0], [2.0], [-6.0]], dtype=torch.float64)
    q = torch.ones(3, 1, dtype=torch.float64)
    sees = torch.tensor([[1, 1, 0], [1, 1, 1], [0, 0, 0]], dtype=torch.bool)
    out, size, reach = dense.attend(q, k, v, 1.0, sees)
    # Weights (1, 1) / 2 and (1, 1, 3) / 5; the row that sees nothing is zero.
    torch.testing.assert_close(out[:, 0], torch.tensor([1.5, -3.0, 0.0], dtype=torch.float64))
    torch.testing.assert_close(size[:, 0], torch.tensor([1.5, 4.2, 0.0], dtype=torch.float64))
    assert reach[1] == pytest.approx(math.log(3.0)) and reach[2] == 0


def test_packed_sequences_see_their_own_keys_up_to_their_place():
    torch.manual_seed(3)
    q, k, v = torch.randn(3, 2, 4), torch.randn(6, 1, 4), torch.randn(6, 1, 2)
    # One query after 3 keys (it sees 4), then two queries of one key (the first sees none).
    out, _, _ = dense.prompt_attention(q, k, v, 0.5, [0, 1, 3], [0, 4, 5])
    p = torch.softmax(k[:4, 0].double() @ q[0, 1].double() * 0.5, 0)
    torch.testing.assert_close(out[0, 1], p @ v[:4, 0].double())
    assert torch.equal(out[1], torch.zeros(2, 2, dtype=torch.float64))
    torch.testing.assert_close(out[2], v[4].double().expand(2, 2))


def test_branches_see_the_prefix_and_their_own_suffix():
    torch.manual_seed(4)
    prefix, suffixes = torch.randn(3, 576), [torch.randn(2, 576), torch.randn(1, 576)]
    q = torch.randn(3, 1, 576)
    out, _, _ = dense.shared_prefix_mla(q, prefix, suffixes, [0, 2, 3], 0.1)
    keys = torch.cat([prefix, suffixes[0][:1]]).double()
    p = torch.softmax(keys @ q[0, 0].double() * 0.1, 0)
    torch.testing.assert_close(out[0, 0], p @ keys[:, :512])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_is_a_rotation_and_inverse_undoes_it(interleaved):
    x = torch.zeros(2, 1, 6)
    x[:, :, 2], x[:, :, 0] = 1.0, 7.0
    positions, frequencies = torch.tensor([0, 3]), torch.tensor([math.pi / 6, 0.1])
    y = dense.rope(x, positions, frequencies, 2, interleaved, 2.0)
    other = 3 if interleaved else 4
    # A quarter turn takes the pair's first value into its second, twice as long.
    assert y[1, 0, 2].abs() < 1e-6 and y[1, 0, other] == pytest.approx(2.0, rel=1e-6)
    assert y[0, 0, 2] == 2.0 and y[1, 0, 0] == 7.0
    back = dense.rope(y, positions, frequencies, 2, interleaved, 0.5, inverse=True)
    torch.testing.assert_close(back, x.double())


def test_rms_norm_of_equal_values_is_the_weight():
    got = dense.rms_norm(torch.full((1, 4), -3.0), torch.arange(4.0), 0.0)
    torch.testing.assert_close(got[0], -torch.arange(4.0).double())


def test_bound_covers_a_rounded_computation_and_not_a_planted_mistake():
    torch.manual_seed(5)
    q, k, v = (torch.randn(n, d).bfloat16() for n, d in ((5, 64), (300, 64), (300, 8)))
    sees = torch.ones(5, 300, dtype=torch.bool)
    out, size, reach = dense.attend(q.double(), k.double(), v.double(), 0.125, sees)
    p = torch.exp(q.float() @ k.float().T * 0.125).bfloat16().float()
    got = ((p @ v.float()) / p.sum(1, keepdim=True)).bfloat16().double()
    bound = dense.attention_bound(out, size, reach, 300, torch.finfo(torch.bfloat16).eps, 64)
    assert ((got - out).abs() <= bound).all()
    p[:, 7] = 0  # a key left out
    wrong = ((p @ v.float()) / p.sum(1, keepdim=True)).double()
    assert not ((wrong * 1.05 - out).abs() <= bound).all()
