"""The hot-path operators in one flat namespace, with the reference's names
and argument order (what a caller of the reference's operator modules
imports):

* quantize_index   - operators/deepseek_v32/indexer/quantization.py:63
* logits           - operators/deepseek_v32/indexer/echo.py:299 (prefetch must be None)
* exact_topk       - operators/deepseek_v32/indexer/selection.py:62
* sparse_mla       - operators/deepseek_v32/attention/device_only/mla.py:90
* sparse_mla_from_pool - operators/deepseek_v32/attention/offload/mla.py:12
* gather_host_records  - operators/common/kv_transfer.py:21
* copy_host_records_async - operators/common/kv_transfer.py (contiguous span copy)

plus the operators of the fp8 paged KV record (656 bytes per token), which
the reference does not have: sparse_mla_fp8_paged and pack_kv_fp8, and those of
the dense path around it: apply_rope_pair (rotary.py:47), write_kv_fp8 and
read_kv_fp8 (records to and from any slots of the cache), prompt_attention
(packed sequences, grouped heads) and shared_prefix_mla (branches over one
prefix); and of the half of a layer behind the attention: residual_rms_norm,
route_experts and expert_mlp over ExpertWeights.
"""

from .attention import (pack_kv_fp8, prompt_attention, read_kv_fp8, shared_prefix_mla, sparse_mla,
                        sparse_mla_fp8_paged, sparse_mla_from_pool, write_kv_fp8)
from .feedforward import ExpertWeights, expert_mlp, residual_rms_norm, route_experts
from .indexer import exact_topk, logits, quantize_index
from .kv_transfer import copy_host_records_async, gather_host_records
from .projections import apply_rope_pair

__all__ = [
    "quantize_index",
    "logits",
    "exact_topk",
    "sparse_mla",
    "sparse_mla_from_pool",
    "sparse_mla_fp8_paged",
    "pack_kv_fp8",
    "gather_host_records",
    "copy_host_records_async",
    "apply_rope_pair",
    "write_kv_fp8",
    "read_kv_fp8",
    "prompt_attention",
    "shared_prefix_mla",
    "residual_rms_norm",
    "route_experts",
    "ExpertWeights",
    "expert_mlp",
]
