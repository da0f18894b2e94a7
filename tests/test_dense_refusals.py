"""What the dense operators refuse, with no GPU: wrong types, shapes, layouts and sizes
raise before anything is launched, and so does the C ABI under them."""

import ctypes

import pytest
import torch

from cxldsagr_amd import _native
from cxldsagr_amd.attention import (prompt_attention, read_kv_fp8, shared_prefix_mla,
                                    write_kv_fp8)
from cxldsagr_amd.projections import apply_rope_pair

B16, I32 = torch.bfloat16, torch.int32


def z(*shape, dtype=B16):
    return torch.zeros(*shape, dtype=dtype)


def cu(*values):
    return torch.tensor(values, dtype=I32)


def _prompt(**change):
    args = dict(q=z(3, 4, 128), k=z(5, 2, 128), v=z(5, 2, 128), scale=0.1, cu_q=cu(0, 3), cu_k=cu(0, 5))
    args.update(change)
    return prompt_attention(**args)


@pytest.mark.parametrize(
    ("change", "message"),
    [
        (dict(q=z(3, 128)), "Expected q"),
        (dict(v=z(4, 2, 128)), "do not agree"),
        (dict(q=z(3, 4, 64)), "do not agree"),
        (dict(q=z(3, 3, 128)), "multiple of k's"),
        (dict(k=z(5, 0, 128), v=z(5, 0, 128)), "multiple of k's"),
        (dict(q=z(3, 4, 96), k=z(5, 2, 96)), "must be one of"),
        (dict(v=z(5, 2, 64)), "must be one of"),
        (dict(q=z(3, 4, 128, dtype=torch.float32)), "share bf16 or fp16"),
        (dict(k=z(5, 2, 128, dtype=torch.float16)), "share bf16 or fp16"),
        (dict(scale=0.0), "positive and finite"),
        (dict(scale=-1.0), "positive and finite"),
        (dict(scale=float("nan")), "positive and finite"),
        (dict(cu_q=cu(0, 3).long()), "cu_q must be int32"),
        (dict(cu_q=[0, 3]), "cu_q must be int32"),
        (dict(cu_k=cu(0, 2, 5)), "same sequences"),
        (dict(max_k=-1), "max_k"),
        (dict(max_k=2.0), "max_k"),
        (dict(q=z(3, 4, 128).requires_grad_()), "no backward"),
    ],
)
def test_prompt_attention(change, message):
    with pytest.raises(ValueError, match=message):
        _prompt(**change)


def _shared(**change):
    args = dict(q=z(2, 8, 576), kv_cache=z(4, 64, 656, dtype=torch.uint8), prefix_table=cu(0, 1),
                prefix_tokens=100, suffix_tables=cu(2, 3).view(2, 1), suffix_tokens=cu(1, 1), scale=0.1)
    args.update(change)
    return shared_prefix_mla(**args)


@pytest.mark.parametrize(
    ("change", "message"),
    [
        (dict(q=z(2, 8, 512)), "Expected q"),
        (dict(q=z(2, 0, 576)), "Expected q"),
        (dict(value_dim=256), "Expected q"),
        (dict(q=z(2, 8, 576, dtype=torch.float16)), "BF16"),
        (dict(scale=float("inf")), "positive and finite"),
        (dict(kv_cache=z(4, 64, 576)), "kv_cache must be"),
        (dict(prefix_table=cu(0, 1).long()), "page_table must be"),
        (dict(prefix_tokens=129), "covered by the prefix table"),
        (dict(prefix_tokens=-1), "covered by the prefix table"),
        (dict(prefix_tokens=torch.tensor(5)), "covered by the prefix table"),
        (dict(suffix_tables=cu(2, 3)), "suffix_tables must be"),
        (dict(suffix_tokens=cu(1)), "suffix_tokens must be"),
        (dict(suffix_tokens=cu(1, 1).long()), "suffix_tokens must be"),
        (dict(cu_q=cu(0, 2)), "branches \\+ 1"),
        (dict(q=z(3, 8, 576)), "one query"),
        (dict(q=z(2, 8, 576).requires_grad_()), "no backward"),
    ],
)
def test_shared_prefix(change, message):
    with pytest.raises(ValueError, match=message):
        _shared(**change)


def _write(**change):
    args = dict(kv=z(2, 576), kv_cache=z(1, 64, 656, dtype=torch.uint8), slots=cu(0, 1))
    args.update(change)
    return write_kv_fp8(**args)


@pytest.mark.parametrize(
    ("change", "message"),
    [
        (dict(kv=z(2, 512)), "kv must be"),
        (dict(kv=z(2, 576, dtype=torch.float32)), "kv must be"),
        (dict(kv_cache=z(1, 64, 656)), "kv_cache must be"),
        (dict(kv_cache=z(1, 128, 656, dtype=torch.uint8)[:, ::2]), "contiguous"),
        (dict(slots=cu(0)), "slots must be"),
        (dict(slots=torch.zeros(2)), "slots must be"),
        (dict(eps=-1.0), "eps"),
        (dict(magnitude=float("inf")), "magnitude"),
        (dict(norm_weight=z(512)), "norm_weight"),
        (dict(norm_weight=torch.ones(576)), "norm_weight"),
        (dict(positions=cu(0, 1)), "positions and frequencies"),
        (dict(frequencies=torch.ones(32)), "positions and frequencies"),
        (dict(positions=torch.zeros(2), frequencies=torch.ones(32)), "positions must be"),
        (dict(positions=cu(0, 1), frequencies=torch.ones(64)), "frequencies must be"),
        (dict(status=torch.zeros(1)), "status"),
        (dict(status=torch.zeros(0, dtype=I32)), "status"),
    ],
)
def test_write(change, message):
    with pytest.raises(ValueError, match=message):
        _write(**change)


def test_read():
    cache = z(1, 64, 656, dtype=torch.uint8)
    for slots in (cu(0).view(1, 1), torch.zeros(2), [0]):
        with pytest.raises(ValueError, match="slots must be"):
            read_kv_fp8(cache, slots)
    with pytest.raises(ValueError, match="kv_cache must be"):
        read_kv_fp8(z(64, 656, dtype=torch.uint8), cu(0))
    with pytest.raises(ValueError, match="out must be"):
        read_kv_fp8(cache, cu(0), out=z(2, 576))


@pytest.mark.parametrize(
    ("change", "message"),
    [
        (dict(q=z(2, 64)), "q must be"),
        (dict(q=z(2, 4, 64, dtype=torch.float64)), "q must be"),
        (dict(k=z(3, 1, 64)), "k must be"),
        (dict(k=z(2, 1, 64, dtype=torch.float16)), "k must be"),
        (dict(k=None, k_out=z(2, 1, 64)), "k_out without k"),
        (dict(positions=torch.zeros(2)), "positions must be"),
        (dict(positions=cu(0)), "positions must be"),
        (dict(frequencies=torch.ones(32, dtype=torch.float64)), "frequencies must be"),
        (dict(frequencies=torch.ones(33)), "within the head"),
        (dict(frequencies=torch.ones(0)), "within the head"),
        (dict(offset=2), "within the head"),
        (dict(offset=-2), "within the head"),
        (dict(q=z(2, 4, 65), k=None), "even rest"),
        (dict(magnitude=float("nan")), "magnitude"),
        (dict(q=z(2, 4, 64).requires_grad_()), "inverse=True"),
    ],
)
def test_rope(change, message):
    args = dict(q=z(2, 4, 64), k=z(2, 1, 64), positions=cu(0, 1), frequencies=torch.ones(32))
    args.update(change)
    with pytest.raises(ValueError, match=message):
        apply_rope_pair(**args)


def test_well_formed_calls_need_the_gpu():
    for call in (_prompt, _shared, _write):
        with pytest.raises(NotImplementedError, match="gfx950"):
            call()
    with pytest.raises(NotImplementedError, match="gfx950"):
        read_kv_fp8(z(1, 64, 656, dtype=torch.uint8), cu(0))
    with pytest.raises(NotImplementedError, match="gfx950"):
        apply_rope_pair(z(2, 4, 64), None, cu(0, 1), torch.ones(32))


# ------------------------------------------------------------------- C ABI --
# (Addresses that are never read: every refusal comes before the launch.)
P = 1 << 20


def _c_prompt(**change):
    args = dict(q=P, q_token=512, q_head=128, k=P, k_token=256, k_head=128, v=P, v_token=256, v_head=128,
                dtype=0, heads=4, kv_heads=2, qk=128, v_dim=128, cu_q=P, cu_k=P, sequences=1, q_tokens=3,
                k_tokens=5, max_k=5, scale=0.1, causal=1, out=P, workspace=None, bytes=0, stream=None)
    args.update(change)
    _native.call("dsa_prompt_attention", *args.values())


@pytest.mark.parametrize(
    ("change", "message"),
    [
        (dict(dtype=2), "bf16 or fp16"),
        (dict(qk=64), "head dims"),
        (dict(heads=3), "multiple of kv_heads"),
        (dict(kv_heads=0), "multiple of kv_heads"),
        (dict(q_tokens=-1), "counts"),
        (dict(k_tokens=1 << 31), "counts"),
        (dict(scale=0.0), "scale"),
        (dict(sequences=0), "need a sequence"),
        (dict(q=None), "null pointer"),
        (dict(v=None), "null pointer"),
        (dict(cu_k=None), "null pointer"),
        (dict(k_token=252), "strides"),
        (dict(k_token=1 << 25), "strides"),
        (dict(v_head=-128), "strides"),
        (dict(q=P + 8), "aligned"),
        (dict(out=P + 8), "aligned"),
        (dict(max_k=4096, k_tokens=4096), "workspace"),
        (dict(max_k=4096, k_tokens=4096, workspace=P + 4, bytes=1 << 30), "workspace"),
    ],
)
def test_prompt_attention_abi(change, message):
    with pytest.raises(ValueError, match=message):
        _c_prompt(**change)


def _c_shared(**change):
    args = dict(q=P, tokens=2, heads=128, cache=P, pages=4, table=P, prefix=64, tables=P, suffix_pages=1,
                suffix_tokens=P, cu_q=None, branches=2, scale=0.1, out=P, workspace=P, bytes=1 << 40,
                stream=None)
    args.update(change)
    _native.call("dsa_shared_prefix_mla_fp8", *args.values())


@pytest.mark.parametrize(
    ("change", "message"),
    [
        (dict(heads=0), "shape"),
        (dict(tokens=-1), "shape"),
        (dict(prefix=-1), "fit int32"),
        (dict(suffix_pages=1 << 31), "fit int32"),
        (dict(scale=float("inf")), "scale"),
        (dict(branches=3), "one query"),
        (dict(branches=0, cu_q=P), "one query"),
        (dict(pages=0), "cache rows"),
        (dict(pages=1 << 31), "cache rows"),
        (dict(table=None), "null pointer"),
        (dict(tables=None), "null pointer"),
        (dict(suffix_tokens=None), "null pointer"),
        (dict(cache=P + 8), "aligned"),
        (dict(heads=64, workspace=None, bytes=0), "workspace"),
        (dict(heads=64, bytes=100), "workspace"),
    ],
)
def test_shared_prefix_abi(change, message):
    with pytest.raises(ValueError, match=message):
        _c_shared(**change)


def test_rope_and_cache_abi():
    def rope(**change):
        args = dict(q=P, a=256, b=64, qo=P, c=256, d=64, heads=4, k=None, e=0, f=0, ko=None, g=0, h=0,
                    k_heads=0, dtype=0, tokens=2, dim=64, offset=0, rotated=64, positions=P, wide=0,
                    frequencies=P, magnitude=1.0, interleaved=0, inverse=0, stream=None)
        args.update(change)
        _native.call("dsa_rope_pair", *args.values())

    for change, message in ((dict(dtype=3), "element type"), (dict(rotated=63), "even"),
                            (dict(offset=2), "within"), (dict(dim=0), "shape"), (dict(tokens=-1), "shape"),
                            (dict(magnitude=float("nan")), "magnitude"), (dict(k_heads=1), "null"),
                            (dict(positions=None), "null")):
        with pytest.raises(ValueError, match=message):
            rope(**change)

    def write(**change):
        args = dict(kv=P, stride=576, tokens=2, slots=P, wide=0, weight=None, eps=0.0, positions=None, wide_p=0,
                    frequencies=None, magnitude=1.0, interleaved=1, pages=1, cache=P, status=None, stream=None)
        args.update(change)
        _native.call("dsa_kv_write_fp8", *args.values())

    for change, message in ((dict(stride=580), "stride"), (dict(tokens=-1), "shape"), (dict(eps=-1.0), "eps"),
                            (dict(kv=None), "null"), (dict(positions=P), "null"), (dict(kv=P + 2), "aligned"),
                            (dict(weight=P + 4), "aligned")):
        with pytest.raises(ValueError, match=message):
            write(**change)
    for args, message in (((P, 1, P, 0, -1, P, None, None), "shape"), ((None, 1, P, 0, 1, P, None, None), "null"),
                          ((P, 1, P, 0, 1, P + 8, None, None), "aligned")):
        with pytest.raises(ValueError, match=message):
            _native.call("dsa_kv_read_fp8", *args)


def test_workspace_queries():
    size = ctypes.c_int64()
    # Whole tiles for every CU: no split. One token over many keys: split.
    _native.call("dsa_prompt_attention_workspace_bytes", 4096, 128, 128, 128, 1, 4096, 4096, ctypes.byref(size))
    assert size.value == 0
    _native.call("dsa_prompt_attention_workspace_bytes", 1, 8, 1, 128, 1, 65536, 65536, ctypes.byref(size))
    assert size.value > 0
    _native.call("dsa_shared_prefix_mla_workspace_bytes", 1, 128, 65536, 1, ctypes.byref(size))
    assert size.value > 0
    for name, args in (("dsa_prompt_attention_workspace_bytes", (-1, 1, 1, 64, 1, 1, 1)),
                       ("dsa_shared_prefix_mla_workspace_bytes", (1, 0, 1, 1))):
        with pytest.raises(ValueError, match="shape"):
            _native.call(name, *args, ctypes.byref(size))


def test_prompt_keys_whose_stages_would_pass_int32():
    for count in (0x7FFFFFFF - 31, 0x7FFFFFFF):
        with pytest.raises(ValueError, match="counts"):
            _c_prompt(k_tokens=count)
        with pytest.raises(ValueError, match="counts"):
            _c_prompt(q_tokens=count)


def test_rope_refuses_expanded_outputs(monkeypatch):
    from cxldsagr_amd import _native

    # (The outputs' checks come after the device's.)
    monkeypatch.setattr(_native, "require_gfx950", lambda *args: None)
    for out in (z(1, 4, 64).expand(2, 4, 64), z(2, 1, 64).expand(2, 4, 64)):
        with pytest.raises(ValueError, match="expanded"):
            apply_rope_pair(z(2, 4, 64), None, cu(0, 1), torch.ones(32), q_out=out)


@pytest.mark.parametrize("heads", [64, 128])
@pytest.mark.parametrize("prefix", [0, 1000])
@pytest.mark.parametrize("suffix_pages", [0, 1])
def test_a_workspace_for_no_tokens_is_empty(heads, prefix, suffix_pages):
    """Calls without tokens are allowed, and so is asking for their workspace first."""
    size = ctypes.c_int64(-1)
    _native.call("dsa_shared_prefix_mla_workspace_bytes", 0, heads, prefix, suffix_pages, ctypes.byref(size))
    assert size.value == 0
    size = ctypes.c_int64(-1)
    _native.call("dsa_prompt_attention_workspace_bytes", 0, heads, heads, 128, 1, prefix, prefix,
                 ctypes.byref(size))
    assert size.value == 0


def test_a_longest_sequence_past_the_keys_is_cut_to_them():
    """(Key splits of so many stages would pass the 32 bits in which a work-group finds its own.)"""
    for k_tokens in (5, 5000):
        sizes = []
        for longest in (k_tokens, k_tokens + 1, 1 << 31, 3 << 40, (1 << 63) - 1):
            size = ctypes.c_int64()
            _native.call("dsa_prompt_attention_workspace_bytes", 1, 8, 8, 128, 1, k_tokens, longest,
                         ctypes.byref(size))
            sizes.append(size.value)
        assert sizes == sizes[:1] * 5


@pytest.mark.parametrize(
    ("name", "args", "message"),
    [
        ("dsa_shared_prefix_mla_workspace_bytes", (1 << 57, 128, 1000, 1), "too many"),
        ("dsa_shared_prefix_mla_workspace_bytes", (1 << 50, 1 << 14, 1000, 1), "too many"),
        ("dsa_shared_prefix_mla_workspace_bytes", (1 << 24, 128, 1000, 1), "too many"),
        ("dsa_shared_prefix_mla_workspace_bytes", (1, 1 << 17, 1000, 1), "shape"),
        ("dsa_shared_prefix_mla_workspace_bytes", (1, 128, (1 << 63) - 1, 1), "fit int32"),
        ("dsa_shared_prefix_mla_workspace_bytes", (1, 128, 1000, 1 << 62), "fit int32"),
        ("dsa_prompt_attention_workspace_bytes", (1, 32, 32, 128, 1 << 59, 1 << 62, 1 << 62), "counts"),
        ("dsa_prompt_attention_workspace_bytes", (1 << 25, 128, 8, 128, 1, 64, 64), "too many"),
        ("dsa_prompt_attention_workspace_bytes", (1, 1 << 17, 1, 128, 1, 64, 64), "multiple of kv_heads"),
    ],
)
def test_sizes_past_what_a_call_takes_have_no_workspace(name, args, message):
    """Refused as the call refuses them, before any arithmetic on them."""
    with pytest.raises(ValueError, match=message):
        _native.call(name, *args, ctypes.byref(ctypes.c_int64()))


def test_row_counts_that_wrap_are_refused_before_the_plan():
    for change in (dict(tokens=1 << 57), dict(tokens=1 << 50, heads=1 << 14), dict(tokens=1 << 24)):
        with pytest.raises(ValueError, match="too many query rows"):
            _c_shared(**{**change, "branches": change["tokens"] if change["tokens"] < 1 << 31 else 1, "cu_q": P})


def test_launches_past_32_bits_of_work_items():
    """Refused with a message, before anything is launched."""
    # 2^25 rows in two parts: the join's work-items.
    with pytest.raises(ValueError, match="too many query rows"):
        _c_shared(tokens=1 << 19, branches=1 << 19, heads=64)
    with pytest.raises(ValueError, match="too many query rows"):
        _c_prompt(sequences=1 << 21, heads=32, kv_heads=32, q_token=4096)
    with pytest.raises(ValueError, match="too many tokens"):  # (33 dims: single pairs)
        _native.call("dsa_rope_pair", P, 8448, 66, P, 8448, 66, 128, None, 0, 0, None, 0, 0, 0, 0, 1 << 24, 66,
                     0, 66, P, 0, P, 1.0, 0, 0, None)
    with pytest.raises(ValueError, match="too many tokens"):
        _native.call("dsa_kv_write_fp8", P, 576, 1 << 27, P, 0, None, 0.0, None, 0, None, 1.0, 1, 1, P, None, None)
    with pytest.raises(ValueError, match="too many tokens"):
        _native.call("dsa_kv_read_fp8", P, 1, P, 0, 1 << 27, P, None, None)
