"""What the operators behind the attention refuse, with no GPU: wrong types, shapes and sizes
raise before anything is launched, and so does the C ABI under them."""

import ctypes

import pytest
import torch

from cxldsagr_amd import _native
from cxldsagr_amd.feedforward import ExpertWeights, expert_mlp, residual_rms_norm, route_experts

B16, F8, E8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu


def z(*shape, dtype=B16):
    return torch.zeros(*shape, dtype=torch.uint8).view(dtype) if dtype in (F8, E8) else torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize(
    ("change", "message"),
    [
        (dict(x=z(256)), "Expected x"),
        (dict(weight=z(128)), "Expected x"),
        (dict(x=z(2, 256, dtype=torch.float64)), "bf16, fp16 or fp32"),
        (dict(weight=z(256, dtype=torch.float16)), "weight must be"),
        (dict(x=z(2, 0), weight=z(0)), "dims"),
        (dict(x=z(2, 16385), weight=z(16385)), "dims"),
        (dict(x=z(2, 200), weight=z(200), quantize=True), "whole blocks"),
        (dict(eps=-1.0), "eps"),
        (dict(eps=float("nan")), "eps"),
        (dict(residual=z(1, 256)), "residual must"),
        (dict(residual=z(2, 256, dtype=torch.float32)), "residual must"),
        (dict(residual_out=z(2, 256)), "without a residual"),
        (dict(residual=z(2, 256), residual_out=z(4, 256)[::2]), "residual_out must"),
        (dict(residual=z(2, 256), residual_out=z(2, 256, dtype=torch.float32)), "residual_out must"),
        (dict(values=False), "nothing to return"),
        (dict(x=z(2, 256).requires_grad_()), "no backward"),
        (dict(weight=z(256).requires_grad_()), "no backward"),
    ],
)
def test_norm(change, message):
    args = dict(x=z(2, 256), weight=z(256))
    args.update(change)
    with pytest.raises(ValueError, match=message):
        residual_rms_norm(**args)


@pytest.mark.parametrize(
    ("change", "message"),
    [
        (dict(logits=z(8)), "Expected logits"),
        (dict(logits=z(2, 0)), "Expected logits"),
        (dict(logits=z(2, 1025)), "Expected logits"),
        (dict(logits=z(2, 16, dtype=torch.float64)), "logits must"),
        (dict(scoring="relu"), "scoring"),
        (dict(groups=3), "groups"),
        (dict(groups=0), "groups"),
        (dict(groups=4, top_groups=5), "groups"),
        (dict(groups=4, top_groups=0), "groups"),
        (dict(logits=z(2, 130), groups=65), "groups"),
        (dict(k=0), "k must"),
        (dict(k=17), "k must"),
        (dict(k=2.0), "k must"),
        (dict(logits=z(2, 256), k=65), "k must"),
        (dict(groups=4, top_groups=1, k=5), "k must"),
        (dict(scale=float("inf")), "scale"),
        (dict(bias=z(16)), "bias"),
        (dict(bias=z(8, dtype=torch.float32)), "bias"),
        (dict(logits=z(2, 16).requires_grad_()), "no backward"),
    ],
)
def test_route(change, message):
    args = dict(logits=z(2, 16), k=2)
    args.update(change)
    with pytest.raises(ValueError, match=message):
        route_experts(**args)


def _parts(**change):
    parts = dict(gate_up=z(2, 256, 256, dtype=F8), gate_up_scale=torch.ones(2, 2, 2),
                 down=z(2, 256, 128, dtype=F8), down_scale=torch.ones(2, 2, 1))
    parts.update(change)
    return parts


@pytest.mark.parametrize(
    ("change", "message"),
    [
        (dict(gate_up=z(2, 256, dtype=F8)), "Expected gate_up"),
        (dict(gate_up=z(3, 256, 256, dtype=F8)), "Expected gate_up"),
        (dict(gate_up=z(2, 128, 256, dtype=F8)), "Expected gate_up"),
        (dict(gate_up=z(2, 256, 256)), "e4m3"),
        (dict(down=z(2, 256, 256, dtype=F8)[..., ::2]), "contiguous"),
        (dict(gate_up=z(2, 256, 64, dtype=F8), down=z(2, 64, 128, dtype=F8)), "whole blocks"),
        (dict(gate_up=z(0, 256, 256, dtype=F8), down=z(0, 256, 128, dtype=F8)), "experts must"),
        (dict(gate_up_scale=torch.ones(2, 2)), "gate_up_scale must be"),
        (dict(down_scale=torch.ones(2, 1, 2)), "down_scale must be"),
        (dict(down_scale=torch.full((2, 2, 1), 3.0)), "powers of two"),
        (dict(down_scale=torch.zeros(2, 2, 1)), "powers of two"),
        (dict(down_scale=torch.full((2, 2, 1), -2.0)), "powers of two"),
        (dict(down_scale=torch.full((2, 2, 1), float("inf"))), "powers of two"),
        (dict(down_scale=z(2, 2, 1)), "e8m0 or FP32"),
        (dict(first=-1), "first"),
        (dict(first=4, total=5), "total"),
        (dict(total=(1 << 30) + 1), "total"),
    ],
)
def test_weights(change, message):
    with pytest.raises(ValueError, match=message):
        ExpertWeights(**_parts(**change))


def test_weights_from_either_scale_type():
    a = ExpertWeights(**_parts())
    b = ExpertWeights(**_parts(gate_up_scale=torch.ones(2, 2, 2).to(E8)))
    assert torch.equal(a.gate_up_scale.view(torch.uint8), b.gate_up_scale.view(torch.uint8))
    assert int(a.gate_up_scale.view(torch.uint8)[0, 0, 0]) == 127
    assert (a.experts, a.dim, a.inner, a.first, a.total) == (2, 256, 128, 0, 2)


@pytest.mark.parametrize("x, residual, out", [
    (slice(8, 12), slice(0, 4), slice(1, 5)),  # rows of the residual, one on
    (slice(0, 4), slice(8, 12), slice(3, 7)),  # x's last row
])
def test_a_sum_that_overlaps_is_refused(x, residual, out):
    rows = torch.zeros(12, 256)
    with pytest.raises(ValueError, match="overlap"):
        residual_rms_norm(rows[x], torch.ones(256), rows[residual], residual_out=rows[out])


def test_a_sum_over_a_row_for_all_is_refused():
    rows = torch.zeros(4, 256)
    with pytest.raises(ValueError, match="overlap"):
        residual_rms_norm(torch.zeros(4, 256), torch.ones(256), rows[:1].expand(4, 256), residual_out=rows)


def test_sums_in_place_or_beside_are_not():
    rows = torch.zeros(12, 256)
    for x, residual, out in [(slice(0, 4), slice(4, 8), slice(8, 12)), (slice(0, 4), slice(4, 8), slice(4, 8)),
                             (slice(0, 4), slice(4, 8), slice(0, 4)), (slice(0, 4), slice(0, 4), slice(0, 4))]:
        # (As far as a CPU's tensors get.)
        with pytest.raises((ValueError, RuntimeError), match="(?i)gpu|gfx950|device"):
            residual_rms_norm(rows[x], torch.ones(256), rows[residual], residual_out=rows[out])


def test_given_scales_are_not_kept():
    scale = torch.ones(2, 2, 2).to(E8)
    own = ExpertWeights(**_parts(gate_up_scale=scale))
    scale.view(torch.uint8).fill_(3)
    assert int(own.gate_up_scale.view(torch.uint8).min()) == 127


def test_tiles_hold_what_the_layout_says():
    codes = torch.randint(0, 256, (2, 512, 384), generator=torch.Generator().manual_seed(4), dtype=torch.uint8)
    parts = _parts(gate_up=codes.view(F8), gate_up_scale=torch.ones(2, 4, 3),
                   down=codes[:, :384, :256].contiguous().view(F8), down_scale=torch.ones(2, 3, 2))
    # (A view that does not begin at a multiple of 16 bytes.)
    flat = torch.empty(parts["gate_up"].numel() + 3, dtype=torch.uint8)
    flat[3:] = codes.flatten()
    parts["gate_up"] = flat[3:].view(codes.shape).view(F8)
    own = ExpertWeights(**parts)
    got = own.gate_up.view(2, 32, 3, 2, 4, 16, 16)
    for tile, k, plane, g, r in [(0, 0, 0, 0, 0), (1, 2, 1, 3, 15), (30, 1, 0, 2, 7), (31, 2, 1, 1, 5), (14, 0, 1, 0, 9)]:
        # Tiles of gate and up in turn; two of each make 32 neighbouring columns.
        row = (tile % 2) * 256 + tile // 4 * 32 + r // 4 * 8 + tile // 2 % 2 * 4 + r % 4
        at = 128 * k + 64 * plane + 16 * g
        assert torch.equal(got[1, tile, k, plane, g, r], codes[1, row, at:at + 16])
    got = own.down.view(2, 24, 2, 2, 4, 16, 16)
    for tile, k, plane, g, r in [(0, 0, 0, 0, 0), (1, 1, 1, 3, 15), (23, 1, 0, 2, 7), (14, 0, 1, 0, 9)]:
        row = tile // 4 * 64 + r // 4 * 16 + tile % 4 * 4 + r % 4
        at = 128 * k + 64 * plane + 16 * g
        assert torch.equal(got[1, tile, k, plane, g, r], codes[1, row, at:at + 16])


@pytest.mark.parametrize(
    ("change", "message"),
    [
        (dict(experts=None), "ExpertWeights"),
        (dict(x=z(3, 128, dtype=F8)), "x must"),
        (dict(x=z(3, 256)), "x must"),
        (dict(x_scale=z(3, 1, dtype=E8)), "x_scale"),
        (dict(x_scale=torch.ones(3, 2)), "x_scale"),
        (dict(ids=torch.zeros(3, 2, dtype=torch.int64)), "ids"),
        (dict(ids=torch.zeros(2, 2, dtype=torch.int32)), "ids"),
        (dict(ids=torch.zeros(3, 65, dtype=torch.int32), weights=torch.zeros(3, 65)), "ids"),
        (dict(ids=torch.zeros(3, 0, dtype=torch.int32), weights=torch.zeros(3, 0)), "ids"),
        (dict(weights=torch.zeros(3, 1)), "weights"),
        (dict(weights=z(3, 2)), "weights"),
        (dict(out=z(3, 128)), "out must"),
        (dict(out=z(3, 256, dtype=torch.float32)), "out must"),
        (dict(dtype=torch.float64), "dtype must"),
        (dict(weights=torch.zeros(3, 2).requires_grad_()), "no backward"),
    ],
)
def test_experts(change, message):
    args = dict(x=z(3, 256, dtype=F8), x_scale=z(3, 2, dtype=E8), experts=ExpertWeights(**_parts()),
                ids=torch.zeros(3, 2, dtype=torch.int32), weights=torch.zeros(3, 2))
    args.update(change)
    with pytest.raises(ValueError, match=message):
        expert_mlp(**args)


def test_cpu_tensors_are_refused():
    with pytest.raises(NotImplementedError):
        residual_rms_norm(z(2, 256), z(256))
    with pytest.raises(NotImplementedError):
        route_experts(z(2, 16), 2)
    with pytest.raises(NotImplementedError):
        expert_mlp(z(3, 256, dtype=F8), z(3, 2, dtype=E8), ExpertWeights(**_parts()),
                   torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2))


@pytest.mark.parametrize(
    ("args", "message"),
    [
        ((0, 8, 0, 0, 3, 16, 0, 4, 8, 1e-6, 0, 0, 0, 0), "element type"),
        ((0, 8, 0, 0, 0, 16, 1, 4, 8, 1e-6, 0, 0, 0, 0), "weight is fp32"),
        ((0, 8, 0, 0, 0, 16, 0, -1, 8, 1e-6, 0, 0, 0, 0), "norm shape"),
        ((0, 8, 0, 0, 0, 16, 0, 4, 16385, 1e-6, 0, 0, 0, 0), "norm shape"),
        ((0, 8, 0, 0, 0, 16, 0, 4, 8, -1.0, 0, 0, 0, 0), "eps"),
        ((16, 8, 0, 0, 0, 16, 0, 4, 8, 1e-6, 0, 0, 16, 0), "come together"),
        ((16, 8, 0, 0, 0, 16, 0, 4, 8, 1e-6, 0, 16, 0, 0), "without a residual"),
        ((0, 8, 0, 0, 0, 16, 0, 4, 8, 1e-6, 16, 0, 0, 0), "null pointer"),
        ((16, 200, 0, 0, 0, 16, 0, 4, 200, 1e-6, 0, 0, 16, 16), "whole blocks"),
        ((16, 129, 0, 0, 0, 16, 0, 4, 128, 1e-6, 0, 0, 16, 16), "whole blocks"),
    ],
)
def test_c_norm(args, message):
    with pytest.raises(ValueError, match=message):
        _native.call("dsa_residual_rms_norm", *args, None)


@pytest.mark.parametrize(
    ("args", "message"),
    [
        ((0, 8, 5, 4, 8, 2, 0, 0, 1, 1, 1, 1.0, 0, 0), "element type"),
        ((0, 8, 0, 4, 1025, 2, 0, 0, 1, 1, 1, 1.0, 0, 0), "experts must"),
        ((0, 8, 0, 4, 8, 2, 0, 0, 3, 1, 1, 1.0, 0, 0), "groups must"),
        ((0, 8, 0, 4, 8, 5, 0, 0, 2, 1, 1, 1.0, 0, 0), "k must"),
        ((0, 8, 0, 4, 8, 2, 0, 0, 1, 1, 1, float("inf"), 0, 0), "scale"),
        ((0, 8, 0, 1 << 31, 8, 2, 0, 0, 1, 1, 1, 1.0, 16, 16), "too many tokens"),
        ((0, 8, 0, (1 << 26) - 1, 8, 2, 0, 0, 1, 1, 1, 1.0, 16, 16), "too many tokens"),
        ((0, 8, 0, 1 << 62, 8, 2, 0, 0, 1, 1, 1, 1.0, 16, 16), "too many tokens"),
        ((0, 8, 0, 4, 8, 2, 0, 0, 1, 1, 1, 1.0, 16, 16), "null pointer"),
    ],
)
def test_c_route(args, message):
    with pytest.raises(ValueError, match=message):
        _native.call("dsa_route_experts", *args, None)


def test_c_experts():
    size = ctypes.c_int64()
    query = "dsa_expert_mlp_workspace_bytes"
    _native.call(query, 0, 8, 256, 128, 4, 4, ctypes.byref(size))
    for args, message in [((4, 8, 100, 128, 4, 4), "whole blocks"), ((4, 8, 256, 0, 4, 4), "whole blocks"),
                          ((4, 8, 256, 128, 0, 4), "experts must"), ((4, 8, 256, 128, 4, 3), "experts must"),
                          ((4, 8, 256, 128, 4, 1 << 31), "experts must"),
                          ((4, 65, 256, 128, 4, 4), "choices"), ((4, 0, 256, 128, 4, 4), "choices"),
                          ((-1, 8, 256, 128, 4, 4), "tokens"), (((1 << 22) + 1, 8, 256, 128, 4, 4), "tokens")]:
        with pytest.raises(ValueError, match=message):
            _native.call(query, *args, ctypes.byref(size))
    with pytest.raises(ValueError, match="null pointer"):
        _native.call(query, 4, 8, 256, 128, 4, 4, None)
    good = dict(x=16, x_scale=16, tokens=4, dim=256, inner=128, gate_up=16, gate_up_scale=16, down=16, down_scale=16,
                experts=4, first=0, total=4, ids=16, weights=16, choices=8, out=16, dtype=0, workspace=16, bytes=1 << 30)
    for change, message in [(dict(x=0), "null pointer"), (dict(down=24), "aligned"), (dict(bytes=64), "workspace of"),
                            (dict(dtype=3), "element type"), (dict(first=-1), "first"), (dict(dim=192), "whole blocks"),
                            (dict(tokens=1 << 22, dim=32768, inner=32768, choices=64, bytes=1 << 62), "too many tokens")]:
        with pytest.raises(ValueError, match=message):
            _native.call("dsa_expert_mlp_fp8", *{**good, **change}.values(), None)
    # No tokens: nothing is read.
    _native.call("dsa_expert_mlp_fp8", *{**good, "tokens": 0, "x": 0, "out": 0}.values(), None)


@pytest.mark.parametrize("name", ["x", "x_scale", "weights"])
def test_experts_refuse_what_wants_gradients(name):
    args = dict(x=z(3, 256, dtype=F8), x_scale=z(3, 2, dtype=E8), experts=ExpertWeights(**_parts()),
                ids=torch.zeros(3, 2, dtype=torch.int32), weights=torch.zeros(3, 2))
    args[name].requires_grad_()
    with pytest.raises(ValueError, match="no backward"):
        expert_mlp(**args)
    with torch.no_grad(), pytest.raises(NotImplementedError):  # (as far as a CPU's tensors get)
        expert_mlp(**args)


@pytest.mark.parametrize("name", sorted(_parts()))
def test_weights_that_want_gradients_are_refused(name):
    parts = _parts()
    parts[name].requires_grad_()
    with pytest.raises(ValueError, match="no backward"):
        ExpertWeights(**parts)
    with torch.no_grad():
        assert ExpertWeights(**parts).experts == 2


def test_an_output_over_an_input_is_refused():
    own = ExpertWeights(**_parts())
    whole = torch.zeros(8192, dtype=torch.uint8)

    def at(offset, dtype, *shape):
        size = torch.empty(shape, dtype=dtype).numel() * dtype.itemsize
        return whole[offset:offset + size].view(dtype).view(shape)

    out = at(2048, B16, 3, 256)  # 1,536 bytes
    free = dict(x=at(0, F8, 3, 256), x_scale=at(1024, E8, 3, 2), ids=at(1100, torch.int32, 3, 2),
                weights=at(1200, torch.float32, 3, 2))
    over = dict(x=[at(2048, F8, 3, 256), at(2048 + 1520, F8, 3, 256), at(2048 - 752, F8, 3, 256)],
                x_scale=[at(2048 + 1535, E8, 3, 2), at(2043, E8, 3, 2)], ids=[at(2028, torch.int32, 3, 2)],
                weights=[at(2048 + 1532, torch.float32, 3, 2)])
    for name, tensors in over.items():
        for tensor in tensors:
            with pytest.raises(ValueError, match="overlap"):
                expert_mlp(**{**free, name: tensor}, experts=own, out=out)
    # Neighbours are not, nor what is copied first, nor a call without tokens.
    for change in (dict(x=at(2048 - 768, F8, 3, 256)), dict(x=at(2048 + 1536, F8, 3, 256)),
                   dict(ids=at(2048, torch.int32, 2, 3).t())):
        with pytest.raises(NotImplementedError):  # (as far as a CPU's tensors get)
            expert_mlp(**{**free, **change}, experts=own, out=out)
    none = {name: t[:0] for name, t in {**free, "x": over["x"][0]}.items()}
    with pytest.raises(NotImplementedError):
        expert_mlp(**none, experts=own, out=out[:0])


def test_sizes_of_too_many_tokens_are_refused_with_the_query():
    size = ctypes.c_int64()
    query = "dsa_expert_mlp_workspace_bytes"
    for args in [(1 << 22, 64, 32768, 32768, 4, 4), (1 << 22, 64, 7168, 128, 256, 256), (1 << 22, 64, 128, 7168, 256, 256)]:
        with pytest.raises(ValueError, match="too many tokens"):
            _native.call(query, *args, ctypes.byref(size))
    # The most tokens, of a choice and of eight.
    for args in [(1 << 22, 1, 32768, 128, 1, 1), (1 << 22, 8, 7168, 2048, 256, 256)]:
        _native.call(query, *args, ctypes.byref(size))
        assert size.value > (1 << 22) * args[1] * (args[2] * 2 + args[3])


@pytest.mark.parametrize(("args", "alone"), [
    ((1, 8, 7168, 2048, 32, 32), True), ((2, 8, 7168, 2048, 32, 32), False), ((1, 8, 7168, 2048, 256, 256), True),
    ((24, 8, 7168, 2048, 256, 256), False), ((8, 8, 7168, 2048, 32, 256), True), ((24, 8, 7168, 2048, 32, 256), False),
    ((6, 8, 1024, 512, 64, 64), True), ((12, 8, 1024, 512, 64, 64), False),
])
def test_pairs_are_taken_by_themselves_where_that_is_sooner(args, alone):
    """The workspace is then the pairs' hidden values."""
    size = ctypes.c_int64()
    _native.call("dsa_expert_mlp_workspace_bytes", *args, ctypes.byref(size))
    assert (size.value == args[0] * args[1] * args[3] * 4) == alone
