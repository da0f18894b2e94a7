"""Sparse MLA prefill on MI355X over bf16 records or the fp8 paged KV cache.

Drop-in for the reference's attention operators (same names, argument order,
padding semantics and validation messages):

* ``sparse_mla``           - ``operators/deepseek_v32/attention/device_only/mla.py:90-115``
  with ``_validate`` (``attention/_validation.py:8-24``) and the input
  preparation of ``mla.py:70-87`` (contiguity, 16-byte alignment, int64 ids
  masked before narrowing). The selection is not padded to 128: the kernel
  accepts any count.
* ``sparse_mla_from_pool`` - ``operators/deepseek_v32/attention/offload/mla.py:12-20``.
* ``sparse_mla_fp8_paged`` - the same attention over the 656-byte fp8 paged
  record (512 e4m3 + 4 fp32 tile scales + 64 bf16 RoPE, 64 tokens per page),
  which has no reference counterpart.
* ``pack_kv_fp8``          - writes bf16 ``[T, 576]`` records into that cache
  (quantise-on-append); ``write_kv_fp8`` does so for any slots of it, through
  the latent's norm and the RoPE part's rotation, and ``read_kv_fp8`` reads
  records back.
* ``prompt_attention``     - dense causal attention of packed sequences with
  grouped heads (the non-absorbed form of a prompt).
* ``shared_prefix_mla``    - dense MLA of branches that share a prefix in the
  fp8 paged cache.

Kernels: ``csrc/sparse_mla.hip``, ``csrc/quantize.hip``,
``csrc/prompt_attention.hip`` and ``csrc/shared_prefix.hip``.
"""

import math

import torch

from cxldsagr_amd import _native

QK_DIM = 576
V_DIM = 512
PAGE_TOKENS = 64
RECORD_BYTES = 656


def _validate(q, kv, indices, scale, value_dim):
    """Mirror of ``attention/_validation.py:8-24``."""
    if q.ndim != 3 or kv.ndim != 2 or indices.ndim != 2:
        raise ValueError("Expected q [Q,H,D], kv [N,D], and indices [Q,K]")
    if q.shape[0] != indices.shape[0] or q.shape[-1] != kv.shape[-1]:
        raise ValueError("Query, cache, and selection dimensions do not agree")
    if not isinstance(value_dim, int) or not 1 <= value_dim <= q.shape[-1]:
        raise ValueError("value_dim must be an integer in [1, query dimension]")
    if value_dim > 512 or q.shape[-1] - value_dim > 128:
        raise ValueError("Supported dimensions are value_dim <= 512 and position dimension <= 128")
    if q.device != kv.device or q.device != indices.device:
        raise ValueError("q, kv, and indices must be on the same device")
    if q.dtype != kv.dtype or not q.is_floating_point():
        raise ValueError("q and kv must share a floating-point dtype")
    if indices.dtype not in (torch.int32, torch.int64):
        raise ValueError("indices must be int32 or int64")
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")


def _check_layout(q, value_dim, what):
    _native.require_gfx950(q.device, what)
    if q.dtype != torch.bfloat16:
        raise ValueError("DSA sparse MLA requires BF16 queries and KV records")
    if q.shape[1] % 64 or q.shape[1] == 0 or q.shape[2] != QK_DIM or value_dim != V_DIM:
        raise ValueError("DeepSeek sparse MLA requires H a multiple of 64, QK dimension 576 and V=512")


def _aligned(tensor):
    tensor = tensor.contiguous()
    if tensor.data_ptr() % 16:
        tensor = tensor.clone()
    return tensor


def _narrow_ids(indices, limit):
    if indices.dtype == torch.int64:
        # Mask before narrowing so large invalid ids cannot wrap into valid ones.
        valid = (indices >= 0) & (indices < limit)
        indices = indices.masked_fill(~valid, -1).to(torch.int32)
    return indices.contiguous()


def _workspace(q, selected):
    """The kernel's workspace for this call (None when it needs none), from
    torch's allocator on the current stream, on which the kernels read it."""
    needed = _native.size_of("dsa_sparse_mla_workspace_bytes", q.device.index, q.shape[0],
                             q.shape[1], selected)
    return torch.empty(needed, dtype=torch.uint8, device=q.device) if needed else None


def sparse_mla(q, kv, indices, scale, value_dim=512):
    """Return BF16 ``[Q,H,512]`` sparse attention over bf16 ``kv [N,576]`` records.

    Negative and out-of-range ids are padding; duplicates participate
    independently; all-padding rows return zero. H may be any multiple of 64.
    """
    _validate(q, kv, indices, scale, value_dim)
    _check_layout(q, value_dim, "DSA sparse MLA")
    if kv.shape[0] > torch.iinfo(torch.int32).max:
        raise ValueError("sparse MLA requires the KV row count to fit int32")
    if not q.shape[0] or not kv.shape[0] or not indices.shape[1]:
        return torch.zeros((*q.shape[:2], value_dim), dtype=q.dtype, device=q.device)
    # The kernel writes every output element (all-padding rows as zeros).
    out = torch.empty((*q.shape[:2], value_dim), dtype=q.dtype, device=q.device)
    q, kv = _aligned(q), _aligned(kv)
    ids = _narrow_ids(indices, kv.shape[0])
    with _native.on_device(q.device):
        workspace = _workspace(q, ids.shape[1])
        _native.call(
            "dsa_sparse_mla_bf16_ws",
            _native.ptr(q), q.shape[0], q.shape[1],
            _native.ptr(kv), kv.shape[0],
            _native.ptr(ids), ids.shape[1],
            float(scale),
            _native.ptr(out),
            _native.ptr(workspace), workspace.numel() if workspace is not None else 0,
            _native.stream_of(q.device),
        )
    return out


def sparse_mla_from_pool(q, records, physical_indices, scale, value_dim=512):
    """Consume recalled HBM records using physical pool ids (``offload/mla.py:12-20``).

    Every non-padding id must already name its selected record in ``records``;
    the caller keeps the selected slots resident until stream completion.
    """
    return sparse_mla(q, records, physical_indices, scale, value_dim)


def _check_paged(cache, page_table, device):
    if (
        not isinstance(cache, torch.Tensor)
        or cache.dtype != torch.uint8
        or cache.ndim != 3
        or cache.shape[1:] != (PAGE_TOKENS, RECORD_BYTES)
        or cache.device != device
    ):
        raise ValueError("kv_cache must be uint8 [pages, 64, 656] on the query device")
    if (
        not isinstance(page_table, torch.Tensor)
        or page_table.dtype != torch.int32
        or page_table.ndim != 1
        or page_table.device != device
    ):
        raise ValueError("page_table must be int32 [logical_pages] on the query device")


def sparse_mla_fp8_paged(q, kv_cache, page_table, indices, scale, value_dim=512, *,
                         n_tokens=None, _out=None):
    """Sparse MLA over the fp8 paged cache; same semantics as ``sparse_mla`` on the
    dequantised records.

    ``kv_cache`` is uint8 ``[pages, 64, 656]``; logical token ``t`` lives at
    page ``page_table[t // 64]``, slot ``t % 64``. Ids outside ``[0, n_tokens)``
    (default: every token the page table covers) are padding. ``_out``
    (contiguous, ``q``'s dtype and device, ``[Q, H, value_dim]``) receives the
    result instead of a new tensor.
    """
    if q.ndim != 3 or indices.ndim != 2 or q.shape[0] != indices.shape[0]:
        raise ValueError("Expected q [Q,H,D] and indices [Q,K] with matching Q")
    if indices.dtype not in (torch.int32, torch.int64) or indices.device != q.device:
        raise ValueError("indices must be int32 or int64 on the query device")
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    _check_layout(q, value_dim, "DSA fp8 paged sparse MLA")
    _check_paged(kv_cache, page_table, q.device)
    if n_tokens is None:
        n_tokens = page_table.numel() * PAGE_TOKENS
    if type(n_tokens) is not int or not 0 <= n_tokens <= page_table.numel() * PAGE_TOKENS:
        raise ValueError("n_tokens must be covered by the page table")
    shape = (*q.shape[:2], value_dim)
    if _out is None:
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
    elif (not isinstance(_out, torch.Tensor) or tuple(_out.shape) != shape or _out.dtype != q.dtype
          or _out.device != q.device or not _out.is_contiguous()
          or _out.data_ptr() % 8):
        raise ValueError("_out must be a contiguous, 8-byte aligned [Q, H, value_dim] tensor "
                         "of q's dtype on q's device")
    else:
        out = _out
    if not q.shape[0] or not n_tokens or not indices.shape[1]:
        return out.zero_()
    q = _aligned(q)
    cache = _aligned(kv_cache)
    table = page_table.contiguous()
    ids = _narrow_ids(indices, n_tokens)
    with _native.on_device(q.device):
        workspace = _workspace(q, ids.shape[1])
        _native.call(
            "dsa_sparse_mla_fp8_paged_ws",
            _native.ptr(q), q.shape[0], q.shape[1],
            _native.ptr(cache), cache.shape[0],
            _native.ptr(table), n_tokens,
            _native.ptr(ids), ids.shape[1],
            float(scale),
            _native.ptr(out),
            _native.ptr(workspace), workspace.numel() if workspace is not None else 0,
            _native.stream_of(q.device),
        )
    return out


def pack_kv_fp8(kv, kv_cache, page_table, token_offset=0, status=None):
    """Quantise bf16 ``kv [T, 576]`` into the fp8 paged cache at tokens
    ``token_offset .. token_offset + T`` (A1 rule per 128-value latent tile,
    UE8M0 scales, RoPE copied). ``status`` (int32 [1], optional) gets bit 0 set
    if a page number lies outside the cache.
    """
    if kv.ndim != 2 or kv.shape[1] != QK_DIM or kv.dtype != torch.bfloat16:
        raise ValueError("kv must be bf16 [tokens, 576]")
    _native.require_gfx950(kv.device, "fp8 KV pack")
    _check_paged(kv_cache, page_table, kv.device)
    if not kv_cache.is_contiguous():
        raise ValueError("kv_cache must be contiguous")
    tokens = kv.shape[0]
    if type(token_offset) is not int or token_offset < 0:
        raise ValueError("token_offset must be a nonnegative integer")
    if token_offset + tokens > page_table.numel() * PAGE_TOKENS:
        raise ValueError("tokens exceed the pages covered by the page table")
    if status is not None and (status.dtype != torch.int32 or status.device != kv.device):
        raise ValueError("status must be int32 on the cache device")
    if tokens == 0:
        return kv_cache
    kv = _aligned(kv)
    if kv_cache.data_ptr() % 16:
        raise ValueError("kv_cache must be 16-byte aligned")
    with _native.on_device(kv.device):
        _native.call(
            "dsa_kv_pack_fp8",
            _native.ptr(kv), tokens, token_offset,
            _native.ptr(page_table.contiguous()), kv_cache.shape[0],
            _native.ptr(kv_cache),
            _native.ptr(status),
            _native.stream_of(kv.device),
        )
    return kv_cache


def _check_slots(slots, tokens, device):
    if (not isinstance(slots, torch.Tensor) or slots.dtype not in (torch.int32, torch.int64)
            or slots.shape != (tokens,) or slots.device != device):
        raise ValueError("slots must be int32 or int64 [tokens] on the cache device")
    return slots if slots.is_contiguous() else slots.contiguous()


def _check_cache(cache, device):
    if (not isinstance(cache, torch.Tensor) or cache.dtype != torch.uint8 or cache.ndim != 3
            or cache.shape[1:] != (PAGE_TOKENS, RECORD_BYTES) or cache.device != device):
        raise ValueError("kv_cache must be uint8 [pages, 64, 656] on the records' device")
    if not cache.is_contiguous() or cache.data_ptr() % 16:
        raise ValueError("kv_cache must be contiguous and 16-byte aligned")


def _check_status(status, device):
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1
                               or status.device != device):
        raise ValueError("status must be int32 on the cache device")


def write_kv_fp8(kv, kv_cache, slots, *, norm_weight=None, eps=1e-6, positions=None,
                 frequencies=None, interleaved=True, magnitude=1.0, status=None):
    """Write bf16 ``kv [T, 576]`` (512 latent + 64 RoPE values; any row stride)
    into ``slots`` of the fp8 paged cache, as ``pack_kv_fp8`` writes records.

    ``slots`` int32 / int64 ``[T]``: token ``t``'s place ``page * 64 + offset``,
    any order, of any sequences, distinct; negative: not written. With
    ``norm_weight`` (f32 ``[512]``) the latent goes through RMSNorm first, with
    ``positions`` (int32 / int64 ``[T]``) and ``frequencies`` (f32 ``[32]``, as
    ``projections.rotary_frequencies``) the RoPE part is rotated
    (``projections.apply_rope_pair``); both round to bf16 as separate operators
    would, so the record is that of norm, rotation and ``pack_kv_fp8`` in turn.
    ``status`` (int32 [1], optional) gets bit 0 set if a slot lies past the cache
    (that token is not written). Returns ``kv_cache``.
    """
    if kv.ndim != 2 or kv.shape[1] != QK_DIM or kv.dtype != torch.bfloat16:
        raise ValueError("kv must be bf16 [tokens, 576]")
    tokens, device = kv.shape[0], kv.device
    _check_cache(kv_cache, device)
    slots = _check_slots(slots, tokens, device)
    _check_status(status, device)
    if not math.isfinite(eps) or eps < 0 or not math.isfinite(magnitude):
        raise ValueError("eps must be finite and nonnegative, magnitude finite")
    if norm_weight is not None:
        if (norm_weight.dtype != torch.float32 or norm_weight.shape != (V_DIM,)
                or norm_weight.device != device):
            raise ValueError("norm_weight must be FP32 [512] on the cache device")
        norm_weight = _aligned(norm_weight)
    if (positions is None) != (frequencies is None):
        raise ValueError("a rotation needs positions and frequencies")
    if positions is not None:
        if (positions.dtype not in (torch.int32, torch.int64) or positions.shape != (tokens,)
                or positions.device != device):
            raise ValueError("positions must be int32 or int64 [tokens] on the cache device")
        if (frequencies.dtype != torch.float32
                or frequencies.shape != ((QK_DIM - V_DIM) // 2,) or frequencies.device != device):
            raise ValueError("frequencies must be FP32 [32] on the cache device")
        positions, frequencies = positions.contiguous(), frequencies.contiguous()
    _native.require_gfx950(device, "fp8 KV write")
    if tokens == 0:
        return kv_cache
    stride, unit = kv.stride()
    if unit != 1 or stride % 8 or stride < 0 or kv.data_ptr() % 16:
        kv = kv.clone(memory_format=torch.contiguous_format)
        stride = QK_DIM
    with _native.on_device(device):
        _native.call(
            "dsa_kv_write_fp8", kv.data_ptr(), stride, tokens, slots.data_ptr(),
            slots.dtype == torch.int64, _native.ptr(norm_weight), eps, _native.ptr(positions),
            positions is not None and positions.dtype == torch.int64, _native.ptr(frequencies),
            magnitude, bool(interleaved), kv_cache.shape[0], kv_cache.data_ptr(),
            _native.ptr(status), _native.raw_stream(device))
    return kv_cache


def read_kv_fp8(kv_cache, slots, *, out=None, status=None):
    """Records of the fp8 paged cache back as bf16 ``[T, 576]`` (what they stand
    for, exactly), e.g. a history to be projected up to a prompt's keys and values.

    ``slots`` int32 / int64 ``[T]`` as in ``write_kv_fp8``, repeats allowed; a
    negative slot gives zeros, one past the cache too, and sets bit 0 of
    ``status`` (int32 [1], optional). ``out``: contiguous bf16 ``[T, 576]`` to
    write to instead of a new tensor.
    """
    if not isinstance(kv_cache, torch.Tensor):
        raise ValueError("kv_cache must be uint8 [pages, 64, 656] on the records' device")
    device = kv_cache.device
    _check_cache(kv_cache, device)
    tokens = slots.shape[0] if isinstance(slots, torch.Tensor) and slots.ndim == 1 else -1
    slots = _check_slots(slots, tokens, device)
    _check_status(status, device)
    if out is None:
        out = kv_cache.new_empty((tokens, QK_DIM), dtype=torch.bfloat16)
    elif (not isinstance(out, torch.Tensor) or tuple(out.shape) != (tokens, QK_DIM)
          or out.dtype != torch.bfloat16 or out.device != device or not out.is_contiguous()
          or out.data_ptr() % 16):
        raise ValueError("out must be a contiguous, 16-byte aligned bf16 [T, 576] tensor on the "
                         "cache device")
    _native.require_gfx950(device, "fp8 KV read")
    if tokens == 0:
        return out
    with _native.on_device(device):
        _native.call("dsa_kv_read_fp8", kv_cache.data_ptr(), kv_cache.shape[0], slots.data_ptr(),
                     slots.dtype == torch.int64, tokens, out.data_ptr(), _native.ptr(status),
                     _native.raw_stream(device))
    return out


PROMPT_HEAD_DIMS = ((192, 128), (128, 128), (64, 64))


def _check_starts(starts, device, what):
    if (not isinstance(starts, torch.Tensor) or starts.dtype != torch.int32 or starts.ndim != 1
            or starts.numel() < 1 or starts.device != device):
        raise ValueError(f"{what} must be int32 [sequences + 1] on the query device")
    return starts if starts.is_contiguous() else starts.contiguous()


def _heads_layout(tensor):
    """``tensor`` [tokens, heads, dim] as the kernels read it: the last dim
    contiguous, the other strides multiples of 16 bytes, aligned; else a copy."""
    token, head, dim = tensor.stride()
    address = tensor.data_ptr()
    if (dim != 1 or token % 8 or head % 8 or not 0 <= token < 1 << 25 or not 0 <= head < 1 << 25
            or address % 16):
        tensor = tensor.clone(memory_format=torch.contiguous_format)
        return tensor, tensor.data_ptr(), *tensor.stride()[:2]
    return tensor, address, token, head


def prompt_attention(q, k, v, scale, cu_q, cu_k=None, *, causal=True, max_k=None, out=None):
    """Causal attention over packed sequences with grouped heads.

    ``q`` ``[Tq, H, d_qk]``, ``k`` ``[Tk, H_kv, d_qk]``, ``v`` ``[Tk, H_kv, d_v]``
    in bf16 or fp16 (any token and head strides), ``(d_qk, d_v)`` one of
    ``(192, 128)``, ``(128, 128)``, ``(64, 64)``; head ``h`` reads KV head
    ``h // (H // H_kv)``. Sequence ``b`` holds queries ``cu_q[b]:cu_q[b + 1]`` and
    keys ``cu_k[b]:cu_k[b + 1]`` (int32 ``[sequences + 1]`` on the device,
    ascending; ``cu_k`` defaults to ``cu_q``). Query ``i`` of ``n_q`` sees keys
    ``j <= i + n_k - n_q``: a prompt, a chunk after a history, single tokens
    (``causal=False``: every key). A query that sees no key gives zeros.

    Returns ``[Tq, H, d_v]`` in ``q``'s type, or writes it to ``out``
    (contiguous); queries outside the sequences (before ``cu_q[0]``, from
    ``cu_q[-1]`` on) are left as they were in ``out``, and in a new tensor hold
    anything. ``max_k``: the longest sequence's keys where the caller knows it,
    by which few queries' keys are split over the GPU; it does not change what
    is computed. Forward only. A key that some query of its sequence does not
    see must have finite values.

    Scores (up to 2^25 in magnitude once scaled), the softmax's maxima and all
    sums are in 32 bits; probabilities are rounded to ``q``'s type before the
    product with ``v`` and before they are summed. One cut into row tiles and
    key ranges, chosen from the totals, serves all sequences of a call: single
    tokens over long histories are faster in a call of their own than beside
    prompts (2,048 tokens and one over 40,000 keys, 32 heads on 8: 672 us, apart
    55 + 35).
    """
    if q.ndim != 3 or k.ndim != 3 or v.ndim != 3:
        raise ValueError("Expected q [Tq,H,Dqk], k [Tk,Hkv,Dqk], and v [Tk,Hkv,Dv]")
    q_tokens, heads, qk_dim = q.shape
    k_tokens, kv_heads, v_dim = v.shape
    if k.shape != (k_tokens, kv_heads, qk_dim):
        raise ValueError("Query, key, and value dimensions do not agree")
    if not heads or not kv_heads or heads % kv_heads:
        raise ValueError("q's heads must be a positive multiple of k's")
    if (qk_dim, v_dim) not in PROMPT_HEAD_DIMS:
        raise ValueError(f"(Dqk, Dv) must be one of {PROMPT_HEAD_DIMS}")
    dtype, device = q.dtype, q.device
    if dtype not in (torch.bfloat16, torch.float16) or k.dtype != dtype or v.dtype != dtype:
        raise ValueError("q, k, and v must share bf16 or fp16")
    if k.device != device or v.device != device:
        raise ValueError("q, k, and v must be on the same device")
    if not math.isfinite(scale) or scale <= 0:
        raise ValueError("scale must be positive and finite")
    if max_k is not None and (type(max_k) is not int or max_k < 0):
        raise ValueError("max_k must be a nonnegative integer")
    if (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        raise ValueError("prompt attention has no backward pass")
    cu_q = _check_starts(cu_q, device, "cu_q")
    cu_k = cu_q if cu_k is None else _check_starts(cu_k, device, "cu_k")
    sequences = cu_q.numel() - 1
    if cu_k.numel() != sequences + 1:
        raise ValueError("cu_q and cu_k must describe the same sequences")
    _native.require_gfx950(device, "prompt attention")
    shape = (q_tokens, heads, v_dim)
    if out is None:
        out = (torch.empty_like(q, memory_format=torch.contiguous_format) if v_dim == qk_dim
               else q.new_empty(shape))
    elif (not isinstance(out, torch.Tensor) or out.shape != shape or out.dtype != dtype
          or out.device != device or not out.is_contiguous() or out.data_ptr() % 16):
        raise ValueError("out must be a contiguous, 16-byte aligned [Tq, H, Dv] tensor of q's "
                         "dtype on q's device")
    if not q_tokens or not sequences:
        return out
    max_k = -1 if max_k is None else min(max_k, k_tokens)
    # (The tensors are kept until the call: they may be copies.)
    q, *q_at = _heads_layout(q)
    k, *k_at = _heads_layout(k)
    v, *v_at = _heads_layout(v)
    with _native.on_device(device):
        needed = _native.size_of("dsa_prompt_attention_workspace_bytes", device.index, q_tokens,
                                 heads, kv_heads, v_dim, sequences, k_tokens, max_k)
        workspace = q.new_empty(needed, dtype=torch.uint8) if needed else None
        _native.call(
            "dsa_prompt_attention", *q_at, *k_at, *v_at, _native.DTYPE_CODES[dtype], heads,
            kv_heads, qk_dim, v_dim, cu_q.data_ptr(), cu_k.data_ptr(), sequences, q_tokens,
            k_tokens, max_k, scale, bool(causal), out.data_ptr(), _native.ptr(workspace), needed,
            _native.raw_stream(device))
    return out


def shared_prefix_mla(q, kv_cache, prefix_table, prefix_tokens, suffix_tables, suffix_tokens,
                      scale, *, cu_q=None, value_dim=512, out=None):
    """MLA attention of branches (a request's candidates) that share a prefix.

    ``q`` bf16 ``[T, H, 576]``; records as in ``sparse_mla_fp8_paged``, in
    ``kv_cache`` uint8 ``[pages, 64, 656]``: the shared prefix's
    ``prefix_tokens`` (an int) on the pages of ``prefix_table`` (int32
    ``[>= ceil(prefix_tokens / 64)]``), branch ``b``'s own ``suffix_tokens[b]``
    (int32 ``[B]`` on the device; what the table does not cover is cut off) on
    the pages of ``suffix_tables[b]`` (int32 ``[B, pages]``, from a fresh page
    on). Branch ``b`` has queries ``cu_q[b]:cu_q[b + 1]`` (int32 ``[B + 1]``,
    ascending; default: one query per branch), the last tokens of its suffix:
    query ``i`` of ``n`` sees the prefix and the first
    ``suffix_tokens[b] - n + 1 + i`` tokens of the suffix. The prefix is read
    once for all branches; any H.

    Returns bf16 ``[T, H, 512]``, or writes it to ``out`` (contiguous), where
    queries of no branch are left as they were (in a new tensor they hold
    anything). A query that sees no key gives zeros; tokens on a page outside
    the cache are padding. Scores, maxima and sums are in 32 bits; probabilities
    are rounded to bf16 before the product with the latent and before they are
    summed.
    """
    if q.ndim != 3 or value_dim != V_DIM:
        raise ValueError("Expected q [T,H,576] with H >= 1 and value_dim 512")
    tokens, heads, dim = q.shape
    if dim != QK_DIM or not heads:
        raise ValueError("Expected q [T,H,576] with H >= 1 and value_dim 512")
    device = q.device
    if q.dtype != torch.bfloat16:
        raise ValueError("shared prefix MLA requires BF16 queries")
    if not math.isfinite(scale) or scale <= 0:
        raise ValueError("scale must be positive and finite")
    _check_paged(kv_cache, prefix_table, device)
    if (type(prefix_tokens) is not int
            or not 0 <= prefix_tokens <= prefix_table.numel() * PAGE_TOKENS):
        raise ValueError("prefix_tokens must be covered by the prefix table")
    if (not isinstance(suffix_tables, torch.Tensor) or suffix_tables.dtype != torch.int32
            or suffix_tables.ndim != 2 or suffix_tables.device != device):
        raise ValueError("suffix_tables must be int32 [branches, pages] on the query device")
    branches, suffix_pages = suffix_tables.shape
    if (not isinstance(suffix_tokens, torch.Tensor) or suffix_tokens.dtype != torch.int32
            or suffix_tokens.shape != (branches,) or suffix_tokens.device != device):
        raise ValueError("suffix_tokens must be int32 [branches] on the query device")
    if cu_q is not None:
        cu_q = _check_starts(cu_q, device, "cu_q")
        if cu_q.numel() != branches + 1:
            raise ValueError("cu_q must be int32 [branches + 1]")
    elif branches != tokens:
        raise ValueError("without cu_q every branch has one query")
    if q.requires_grad and torch.is_grad_enabled():
        raise ValueError("shared prefix MLA has no backward pass")
    _native.require_gfx950(device, "shared prefix MLA")
    shape = (tokens, heads, value_dim)
    if out is None:
        out = q.new_empty(shape)
    elif (not isinstance(out, torch.Tensor) or out.shape != shape or out.dtype != q.dtype
          or out.device != device or not out.is_contiguous() or out.data_ptr() % 16):
        raise ValueError("out must be a contiguous, 16-byte aligned [T, H, 512] tensor of q's "
                         "dtype on q's device")
    if not tokens or not branches:
        return out
    pages = kv_cache.shape[0]
    if not pages:
        raise ValueError("kv_cache must hold a page")
    q, cache = _aligned(q), _aligned(kv_cache)
    prefix_table, suffix_tables = prefix_table.contiguous(), suffix_tables.contiguous()
    suffix_tokens = suffix_tokens.contiguous()
    with _native.on_device(device):
        needed = _native.size_of("dsa_shared_prefix_mla_workspace_bytes", device.index, tokens,
                                 heads, prefix_tokens, suffix_pages)
        workspace = q.new_empty(needed, dtype=torch.uint8) if needed else None
        _native.call(
            "dsa_shared_prefix_mla_fp8",
            q.data_ptr(), tokens, heads, cache.data_ptr(), pages,
            prefix_table.data_ptr(), prefix_tokens, suffix_tables.data_ptr(),
            suffix_pages, suffix_tokens.data_ptr(), _native.ptr(cu_q), branches,
            float(scale), out.data_ptr(), _native.ptr(workspace), needed,
            _native.raw_stream(device),
        )
    return out
