"""The operators behind the attention together, as a layer calls them; captured; on streams."""

import pytest
import torch

from oracle import feedforward as off

pytestmark = pytest.mark.gpu


class Layer:
    """A layer's half: norm, router, experts in two slices as on two ranks, next norm."""

    def __init__(self, gpu, dim=512, inner=256, experts=16, seed=21):
        from cxldsagr_amd.feedforward import ExpertWeights

        gen = torch.Generator().manual_seed(seed)
        f8 = torch.float8_e4m3fn
        half = experts // 2
        self.gate = torch.randn(experts, dim, generator=gen).mul(dim ** -0.5)
        self.bias = 0.1 * torch.randn(experts, generator=gen)
        self.weight = 1 + 0.1 * torch.randn(dim, generator=gen)
        self.parts = ((torch.randn(experts, 2 * inner, dim, generator=gen) * 60).to(f8),
                      torch.full((experts, 2 * inner // 128, dim // 128), 2.0 ** -10),
                      (torch.randn(experts, dim, inner, generator=gen) * 60).to(f8),
                      torch.full((experts, dim // 128, inner // 128), 2.0 ** -10))
        self.slices = [ExpertWeights(*(t[s].contiguous().to(gpu) for t in self.parts), first=s.start, total=experts)
                       for s in (slice(0, half), slice(half, experts))]
        self.gate_gpu, self.bias_gpu, self.weight_gpu = (t.to(gpu) for t in (self.gate, self.bias, self.weight))

    def step(self, attention, stream):
        from cxldsagr_amd import ops

        normed = ops.residual_rms_norm(attention, self.weight_gpu, stream, quantize=True)
        logits = torch.nn.functional.linear(normed.values.float(), self.gate_gpu)
        weights, ids = ops.route_experts(logits, 4, bias=self.bias_gpu, groups=4, top_groups=2, scale=2.5)
        halves = [ops.expert_mlp(normed.codes, normed.scales, s, ids, weights, dtype=torch.float32) for s in self.slices]
        moved = (halves[0] + halves[1]).bfloat16()
        after = ops.residual_rms_norm(moved, self.weight_gpu, normed.residual)
        return normed, logits, weights, ids, moved, after

    def inputs(self, gpu, tokens, seed):
        gen = torch.Generator().manual_seed(seed)
        return [torch.randn(tokens, 512, generator=gen).bfloat16().to(gpu) for _ in range(2)]


@pytest.mark.parametrize("tokens", [1, 7, 130])
def test_a_layer_s_half(gpu, tokens):
    layer = Layer(gpu)
    attention, stream = layer.inputs(gpu, tokens, 22)
    normed, logits, weights, ids, moved, after = layer.step(attention, stream)
    y, t = off.rms_norm(attention, layer.weight, stream)
    assert ((normed.values.cpu().double() - y).abs() <= (2.0 ** -8 + 2.0 ** -24) * y.abs()).all()
    want, want_ids = off.route(logits, 4, bias=layer.bias, groups=4, top_groups=2, scale=2.5)
    assert torch.equal(ids.cpu(), want_ids)
    assert ((weights.cpu().double() - want).abs() <= 8 * 2.0 ** -24 * want).all()
    out, bound = off.expert_mlp(normed.codes, normed.scales, *layer.parts, ids, weights)
    bound = bound + 2.0 ** -23 * (out.abs() + bound) + 2.0 ** -8 * (out.abs() + bound)
    assert ((moved.cpu().double() - out).abs() <= bound).all()
    y, t = off.rms_norm(moved, layer.weight, normed.residual)
    assert torch.equal(after.residual.cpu(), t.bfloat16())
    assert ((after.values.cpu().double() - y).abs() <= (2.0 ** -8 + 2.0 ** -24) * y.abs()).all()


@pytest.mark.parametrize("tokens", [3, 200])
def test_captured_and_replayed(gpu, tokens):
    """One graph replayed on other inputs, with eager work and another graph of the same
    layer between: every replay is the eager result."""
    layer = Layer(gpu)
    eager = [layer.step(*layer.inputs(gpu, tokens, seed)) for seed in (31, 32, 33)]
    held = [t.clone() for t in layer.inputs(gpu, tokens, 30)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = layer.step(*held)
        graphs.append((graph, outputs))
    for turn, seed in enumerate((31, 32, 33, 31)):
        for to, new in zip(held, layer.inputs(gpu, tokens, seed)):
            to.copy_(new)
        for graph, outputs in graphs if turn % 2 else graphs[::-1]:
            graph.replay()
            torch.cuda.synchronize()
            want = eager[(seed - 31) % 3]
            assert torch.equal(outputs[3], want[3]) and torch.equal(outputs[4], want[4])
            assert torch.equal(outputs[5].values, want[5].values)
            layer.step(*layer.inputs(gpu, tokens + 1, 34 + turn))


def test_calls_at_once_on_two_streams(gpu):
    layer = Layer(gpu)
    inputs = [layer.inputs(gpu, tokens, 40 + tokens) for tokens in (5, 300)]
    want = [layer.step(*pair)[5].values for pair in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        for s, pair in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append(layer.step(*pair)[5].values)
    torch.cuda.synchronize()
    for i, values in enumerate(got):
        assert torch.equal(values, want[i % 2])
