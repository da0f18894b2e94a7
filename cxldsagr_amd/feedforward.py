"""The half of a decoder layer behind the attention on MI355X, forward only:

* ``residual_rms_norm`` - the attention's output added to the residual stream,
  its RMSNorm, and the normalised values in e4m3 with a scale for every 128.
* ``route_experts``     - each token's experts and their weights from the
  router's logits.
* ``expert_mlp``        - the routed experts' gated MLP in e4m3 over
  ``ExpertWeights``, summed by those weights.

A layer's step: ``normed = residual_rms_norm(attention, weight, residual,
quantize=True)``, the router's logits from ``normed.values`` (a plain product),
``route_experts``, ``expert_mlp(normed.codes, normed.scales, ...)``, whose result
goes into the next layer's ``residual_rms_norm`` with ``normed.residual``. The
codes are also what ``indexer.quantize_index`` gives for rows viewed as blocks of
128. Scales are powers of two, held as ``torch.float8_e8m0fnu``.

Kernels: ``csrc/norm.hip``, ``csrc/route.hip`` and ``csrc/experts.hip``.
"""

import math
from typing import NamedTuple, Optional

import torch

from cxldsagr_amd import _native

SCALE_BLOCK = 128
MAX_NORM_DIM = 16384
MAX_EXPERTS = 1024
MAX_GROUPS = 64
MAX_CHOICES = 64
CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu


class Normed(NamedTuple):
    """What ``residual_rms_norm`` returns; None for what was not asked for."""

    values: Optional[torch.Tensor]  # [T, D], x's type
    codes: Optional[torch.Tensor]  # e4m3 [T, D]
    scales: Optional[torch.Tensor]  # e8m0 [T, D / 128]
    residual: Optional[torch.Tensor]  # [T, D], x's type: x + residual


_CODES = _native.DTYPE_CODES
# (Two thirds of what new_empty takes.)
_empty = torch.empty_strided


def _rows(tensor, aligned=False):
    """``tensor`` [T, D] with contiguous rows (any row stride; ``aligned``: to 16 bytes), or
    a copy, and its address and row stride."""
    stride, unit = tensor.stride()
    address = tensor.data_ptr()
    if unit != 1 or stride < 0 or (aligned and (address % 16 or stride * tensor.element_size() % 16)):
        tensor = tensor.clone(memory_format=torch.contiguous_format)
        return tensor, tensor.data_ptr(), tensor.shape[1]
    return tensor, address, stride


def _apart(out, tensor):
    """Whether contiguous rows ``out`` share no memory with the rows ``tensor``, or are the
    same rows."""
    begin, other = out.data_ptr(), tensor.data_ptr()
    rows, dim = tensor.shape
    stride, size = tensor.stride(0), tensor.element_size()
    if begin == other and (stride == dim or rows == 1):
        return True
    # (As far as its unit stride goes; other rows are copied before anything is written.)
    return (tensor.stride(1) != 1 or begin >= other + ((rows - 1) * stride + dim) * size
            or other >= begin + rows * dim * size)


def _over(out, tensor):
    """Whether contiguous ``out`` shares memory with ``tensor``, if that is contiguous too
    (else it is copied before anything is written)."""
    begin, other = out.data_ptr(), tensor.data_ptr()
    return (begin < other + tensor.numel() * tensor.element_size()
            and other < begin + out.numel() * out.element_size() and tensor.is_contiguous())


def residual_rms_norm(x, weight, residual=None, *, eps=1e-6, values=True, quantize=False,
                      residual_out=None):
    """``t = x + residual`` and ``t * weight / sqrt(mean(t^2) + eps)`` of every row.

    ``x`` (and ``residual``) ``[T, D]`` in bf16, fp16 or fp32, any row stride, D up to
    16384; ``weight`` ``[D]`` in fp32 or ``x``'s type. The sum is one of 32 bits, rounded
    to ``x``'s type where it is returned; the norm is formed from the sum before that, to 46
    bits or more, and rounded to 32 bits and then to ``x``'s type, as a cast from 64 bits
    does (one rounding would give another value in one of some 130,000 in bf16, 17,000 in
    fp16). With ``quantize`` (D in whole blocks of 128) the rounded
    values come as e4m3 codes too, with a power-of-two scale for every 128 of a row (the
    rule of ``indexer.quantize_index``); ``values=False`` leaves them as codes only.

    Returns ``Normed(values, codes, scales, residual)``; ``residual`` is ``t``, in a new
    tensor or in ``residual_out`` (contiguous; it may be ``residual`` or ``x`` itself, else
    it must not overlap them). Forward only.
    """
    shape, dtype, device = x.shape, x.dtype, x.device
    if len(shape) != 2 or weight.shape != shape[1:]:
        raise ValueError("Expected x [T, D] and weight [D]")
    tokens, dim = shape
    code, weight_code = _CODES.get(dtype), _CODES.get(weight.dtype)
    if code is None:
        raise ValueError("x must be bf16, fp16 or fp32")
    if weight_code != code and weight_code != 2:
        raise ValueError("weight must be fp32 or of x's type")
    if not 1 <= dim <= MAX_NORM_DIM:
        raise ValueError(f"x must have 1 to {MAX_NORM_DIM} dims")
    if quantize and dim % SCALE_BLOCK:
        raise ValueError("quantised rows must be whole blocks of 128 values")
    if not math.isfinite(eps) or eps < 0:
        raise ValueError("eps must be finite and nonnegative")
    if weight.device != device:
        raise ValueError("x and weight must be on the same device")
    if residual is not None:
        if residual.shape != shape or residual.dtype != dtype or residual.device != device:
            raise ValueError("residual must have x's shape, type and device")
    elif residual_out is not None:
        raise ValueError("residual_out without a residual")
    elif not values and not quantize:
        raise ValueError("nothing to return: ask for values, codes or a residual's sum")
    if residual_out is not None and (
            residual_out.shape != shape or residual_out.dtype != dtype
            or residual_out.device != device or not residual_out.is_contiguous()
            or residual_out.data_ptr() % 16):
        raise ValueError("residual_out must be a contiguous, 16-byte aligned tensor of x's shape, "
                         "type and device")
    if residual_out is not None and tokens and not (_apart(residual_out, x)
                                                    and _apart(residual_out, residual)):
        raise ValueError("residual_out must be residual or x itself, or overlap neither")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        raise ValueError("residual RMS norm has no backward pass")
    _native.require_gfx950(device, "residual RMS norm")
    # (Codes are written by lanes of 8 values; the tensors are kept until the call: they may
    # be copies.)
    x, x_at, x_stride = _rows(x, quantize)
    residual_at = residual_stride = 0
    if residual is not None:
        residual, residual_at, residual_stride = _rows(residual, quantize)
        if residual_out is None:
            residual_out = _empty(shape, (dim, 1), dtype=dtype, device=device)
    if not weight.is_contiguous() or (quantize and weight.data_ptr() % 16):
        weight = weight.clone(memory_format=torch.contiguous_format)
    out = _empty(shape, (dim, 1), dtype=dtype, device=device) if values else None
    codes = scales = None
    if quantize:
        codes = _empty(shape, (dim, 1), dtype=CODES, device=device)
        blocks = dim // SCALE_BLOCK
        scales = _empty((tokens, blocks), (blocks, 1), dtype=SCALES, device=device)
    if tokens:
        with _native.on_device(device):
            _native.call(
                "dsa_residual_rms_norm", x_at, x_stride, residual_at, residual_stride, code,
                weight.data_ptr(), weight_code, tokens, dim, eps,
                out.data_ptr() if values else 0, _native.ptr(residual_out),
                codes.data_ptr() if quantize else 0, scales.data_ptr() if quantize else 0,
                _native.raw_stream(device))
    return Normed(out, codes, scales, residual_out)


def route_experts(logits, k, *, bias=None, scoring="sigmoid", groups=1, top_groups=None,
                  renormalize=True, scale=1.0):
    """Each token's ``k`` experts and their weights from the router's logits.

    ``logits`` ``[T, E]`` in fp32, bf16 or fp16 (any row stride), E up to 1024. Scores
    ``s`` are ``sigmoid(logits)`` or, with ``scoring="softmax"``, their softmax, rounded
    to 32 bits. Experts are ranked by ``s + bias`` (``bias`` fp32 ``[E]``, for an even
    load; it does not enter the weights). With ``groups`` of equal size (up to 64) only
    the experts of the ``top_groups`` best are eligible, a group counting as its best
    expert, with a bias as the sum of its two best. Ties go to the lower index, a NaN
    ranks above all.

    Returns ``(weights fp32 [T, k], ids int32 [T, k])``, best first (``k`` up to 64):
    ``s * scale``, with ``renormalize`` ``s / (sum of the k + 1e-20) * scale``, formed from
    ``s`` in 64 bits and rounded once. Forward only.
    """
    shape, device = logits.shape, logits.device
    if len(shape) != 2 or not 1 <= shape[1] <= MAX_EXPERTS:
        raise ValueError(f"Expected logits [T, E] of 1 to {MAX_EXPERTS} experts")
    tokens, experts = shape
    code = _CODES.get(logits.dtype)
    if code is None:
        raise ValueError("logits must be fp32, bf16 or fp16")
    if scoring not in ("sigmoid", "softmax"):
        raise ValueError("scoring must be 'sigmoid' or 'softmax'")
    if top_groups is None:
        top_groups = groups
    if (type(groups) is not int or type(top_groups) is not int or not 1 <= groups <= MAX_GROUPS
            or experts % groups or not 1 <= top_groups <= groups):
        raise ValueError(f"groups (1 to {MAX_GROUPS}) must divide the experts, top_groups be 1 to "
                         "groups")
    if type(k) is not int or not 1 <= k <= MAX_CHOICES or k > top_groups * (experts // groups):
        raise ValueError(f"k must be 1 to {MAX_CHOICES} and within the experts of top_groups groups")
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != shape[1:] or bias.device != device:
            raise ValueError("bias must be FP32 [E] on the logits' device")
        if not bias.is_contiguous():
            bias = bias.contiguous()
    if torch.is_grad_enabled() and (logits.requires_grad or (bias is not None and bias.requires_grad)):
        raise ValueError("routing to experts has no backward pass")
    _native.require_gfx950(device, "routing to experts")
    logits, logits_at, stride = _rows(logits)
    weights = _empty((tokens, k), (k, 1), dtype=torch.float32, device=device)
    ids = _empty((tokens, k), (k, 1), dtype=torch.int32, device=device)
    if tokens:
        with _native.on_device(device):
            _native.call(
                "dsa_route_experts", logits_at, stride, code, tokens, experts, k,
                _native.ptr(bias), scoring == "softmax", groups, top_groups, bool(renormalize),
                scale, weights.data_ptr(), ids.data_ptr(), _native.raw_stream(device))
    return weights, ids


def _exponents(scale, shape, what):
    """Powers of two as e8m0 of ``shape`` (from fp32: every one has to be one)."""
    if scale.shape != shape:
        raise ValueError(f"{what} must be {list(shape)}: a scale for every 128 by 128")
    if scale.dtype == SCALES:
        return scale.clone(memory_format=torch.contiguous_format)
    if scale.dtype != torch.float32:
        raise ValueError(f"{what} must be e8m0 or FP32")
    bits = scale.contiguous().view(torch.int32)
    power = bits >> 23
    if not bool(((bits & 0x7FFFFF == 0) & (power > 0) & (power < 255)).all()):
        raise ValueError(f"{what} must hold powers of two")
    return power.to(torch.uint8).view(SCALES)


def _tiles(weight, parts):
    """``[E, N, K]`` codes as tiles of 16 rows by 128 in the order in which a wave reads
    them: ``[E, N / 16, K / 128, 2, 4, 16, 16 bytes]``, lane (g, r) of plane p holding bytes
    64 p + 16 g .. of row r. A wave takes four tiles: 64 / ``parts`` neighbouring rows of
    each of the ``parts`` equal parts of N, so dealt out that four lanes' results are
    neighbours: with n = 4 / ``parts`` tiles of a part, row 4 a + i of its tile t is row
    4 n a + 4 t + i of the 16 n; the parts' tiles in turn."""
    experts, rows, columns = weight.shape
    if weight.data_ptr() % 16 or weight.storage_offset() % 16:
        weight = weight.clone()
    units = weight.view(torch.uint8).view(torch.complex128)  # 16 bytes each
    each = 4 // parts
    units = units.view(experts, parts, rows // 64, 4, each, 4, columns // SCALE_BLOCK, 2, 4)
    return units.permute(0, 2, 4, 1, 6, 7, 8, 3, 5).contiguous().view(torch.uint8)


class ExpertWeights:
    """The gated MLPs of a rank's experts, laid out once for ``expert_mlp``.

    ``gate_up`` e4m3 ``[E, 2 I, D]`` (the gate's rows, then up's) and ``down`` e4m3
    ``[E, D, I]``, contiguous, D and I in whole blocks of 128, each with a power-of-two
    scale for every 128 by 128: ``gate_up_scale`` ``[E, 2 I / 128, D / 128]``,
    ``down_scale`` ``[E, D / 128, I / 128]`` (e8m0, or fp32 powers of two, which are
    checked). The experts are those numbered ``first .. first + E - 1`` of the model's
    ``total`` (default ``first + E``, at most 2^30): other choices are other ranks'.
    ``total`` only tells how many rows an expert may expect.

    Codes (in another order) and scales are copied; the given tensors are not kept.
    """

    def __init__(self, gate_up, gate_up_scale, down, down_scale, *, first=0, total=None):
        if gate_up.ndim != 3 or down.ndim != 3 or gate_up.shape[0] != down.shape[0]:
            raise ValueError("Expected gate_up [E, 2 I, D] and down [E, D, I]")
        experts, dim, inner = down.shape
        if gate_up.shape != (experts, 2 * inner, dim):
            raise ValueError("Expected gate_up [E, 2 I, D] and down [E, D, I]")
        if not 1 <= experts <= MAX_EXPERTS:
            raise ValueError(f"experts must number 1 to {MAX_EXPERTS}")
        if not dim or not inner or dim % SCALE_BLOCK or inner % SCALE_BLOCK or max(dim, inner) > 32768:
            raise ValueError("D and I must be whole blocks of 128, 32768 at most")
        if gate_up.dtype != CODES or down.dtype != CODES:
            raise ValueError("weights must be e4m3 (torch.float8_e4m3fn)")
        if not gate_up.is_contiguous() or not down.is_contiguous():
            raise ValueError("weights must be contiguous")
        tensors = (gate_up, gate_up_scale, down, down_scale)
        if any(t.device != down.device for t in tensors):
            raise ValueError("weights and scales must be on the same device")
        if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
            raise ValueError("the experts' MLP has no backward pass")
        if type(first) is not int or first < 0:
            raise ValueError("first must be a nonnegative integer")
        if total is None:
            total = first + experts
        if type(total) is not int or not first + experts <= total <= 1 << 30:
            raise ValueError("total must be at least first + E, at most 2^30")
        blocks, inner_blocks = dim // SCALE_BLOCK, inner // SCALE_BLOCK
        self.gate_up_scale = _exponents(gate_up_scale, (experts, 2 * inner_blocks, blocks),
                                        "gate_up_scale")
        self.down_scale = _exponents(down_scale, (experts, blocks, inner_blocks), "down_scale")
        self.gate_up = _tiles(gate_up, 2)
        self.down = _tiles(down, 1)
        self.experts, self.dim, self.inner = experts, dim, inner
        self.first, self.total = first, total
        self.device = down.device


def expert_mlp(x, x_scale, experts, ids, weights, *, dtype=torch.bfloat16, out=None):
    """Each token's experts applied to it and summed:
    ``sum_j weights[t, j] * down(silu(gate(x)) * up(x))`` over the choices ``ids[t, j]``.

    ``x`` e4m3 ``[T, D]`` with ``x_scale`` e8m0 ``[T, D / 128]`` (as
    ``residual_rms_norm`` gives them), ``experts`` an ``ExpertWeights``, ``ids`` int32
    and ``weights`` fp32 ``[T, k]``, k up to 64 (as ``route_experts`` gives them).
    Choices outside ``experts.first .. first + E - 1`` add nothing (an expert of another
    rank, or -1 for none); a token may choose an expert twice. T up to 2^22, but refused
    where the products' row tiles (of 32 to 128 choices) by their columns (I / 128 or
    D / 256) would number 2^24. The workspace of a long call holds some 2 D + I bytes for
    each of the T k choices, whichever rank's.

    Returns ``[T, D]`` in ``dtype`` (bf16, fp16 or fp32), or writes it to ``out``
    (contiguous, of ``dtype``); a token without a choice here gives zeros. Sums are in
    32 bits, but for what the matrix unit cuts off each of eight neighbouring products
    (below 2^-13 of the largest; nothing from gate's and up's up to 16 choices an expert or
    2^20 hidden values: in longer calls one row in 100 is 5e-3 of its size off the formula,
    the worst of thousands 4e-2, as a hidden code of the largest moves by a step; the others
    are off by bf16's own 1.7e-3, as shorter calls' are). ``silu(gate) * up`` is rounded to
    e4m3 codes with a power-of-two scale for every 128 (the rule of
    ``indexer.quantize_index``: 2^-22 at least, so that what is below 2^-32 is lost), and an
    expert's result, before it is weighted, to no fewer than 11 bits (down to 2^-29 of the
    largest of its 64 neighbours).
    ``out`` must not overlap the inputs. Forward only.
    """
    if not isinstance(experts, ExpertWeights):
        raise ValueError("experts must be an ExpertWeights")
    device, dim = experts.device, experts.dim
    if x.ndim != 2 or x.shape[1] != dim or x.dtype != CODES or x.device != device:
        raise ValueError("x must be e4m3 [T, D] on the experts' device")
    tokens = x.shape[0]
    if tokens > 1 << 22:
        raise ValueError("tokens must number 0 to 2^22")
    if (x_scale.shape != (tokens, dim // SCALE_BLOCK) or x_scale.dtype != SCALES
            or x_scale.device != device):
        raise ValueError("x_scale must be e8m0 [T, D / 128] on the experts' device")
    if (ids.ndim != 2 or ids.shape[0] != tokens or not 1 <= ids.shape[1] <= MAX_CHOICES
            or ids.dtype != torch.int32 or ids.device != device):
        raise ValueError(f"ids must be int32 [T, k] with k of 1 to {MAX_CHOICES} on the experts' "
                         "device")
    if weights.shape != ids.shape or weights.dtype != torch.float32 or weights.device != device:
        raise ValueError("weights must be FP32 [T, k] on the experts' device")
    if out is not None:
        if (out.shape != (tokens, dim) or out.dtype != dtype or out.device != device
                or not out.is_contiguous() or out.data_ptr() % 16):
            raise ValueError("out must be a contiguous, 16-byte aligned [T, D] tensor of dtype on "
                             "the experts' device")
        if tokens and (_over(out, x) or _over(out, x_scale) or _over(out, ids) or _over(out, weights)):
            raise ValueError("out must not overlap the inputs")
    code = _native.DTYPE_CODES.get(dtype)
    if code is None:
        raise ValueError("dtype must be bf16, fp16 or fp32")
    if torch.is_grad_enabled() and (x.requires_grad or x_scale.requires_grad
                                    or weights.requires_grad):
        raise ValueError("the experts' MLP has no backward pass")
    _native.require_gfx950(device, "the experts' MLP")
    if out is None:
        out = _empty((tokens, dim), (dim, 1), dtype=dtype, device=device)
    if not tokens:
        return out
    x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()
    x_scale, ids, weights = x_scale.contiguous(), ids.contiguous(), weights.contiguous()
    choices = ids.shape[1]
    with _native.on_device(device):
        needed = _native.size_of("dsa_expert_mlp_workspace_bytes", device.index, tokens, choices,
                                 dim, experts.inner, experts.experts, experts.total)
        workspace = _empty((needed,), (1,), dtype=torch.uint8, device=device)
        _native.call(
            "dsa_expert_mlp_fp8", x.data_ptr(), x_scale.data_ptr(), tokens, dim, experts.inner,
            experts.gate_up.data_ptr(), experts.gate_up_scale.data_ptr(),
            experts.down.data_ptr(), experts.down_scale.data_ptr(), experts.experts,
            experts.first, experts.total, ids.data_ptr(), weights.data_ptr(), choices,
            out.data_ptr(), code, workspace.data_ptr(), needed, _native.raw_stream(device))
    return out
