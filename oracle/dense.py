"""Dense attention, rotary pairs and cache writes in 64 bits (TEST INFRASTRUCTURE ONLY).

The formulas themselves, one sequence and head at a time, for the operators
``attention.prompt_attention``, ``attention.shared_prefix_mla``,
``attention.write_kv_fp8`` and ``projections.apply_rope_pair``. Each attention
function also returns what bounds a 16-bit kernel's error element by element:
the mean of |v| under the row's probabilities.

Pinned by ``tests/test_oracle_dense.py`` on closed forms.
"""

import torch


def attend(q, k, v, scale, sees):
    """``q [n, d]``, ``k [m, d]``, ``v [m, e]`` in float64, ``sees`` bool ``[n, m]``:
    ``(out, mean of |v|, largest sum of |q k| scale)``, zeros for a row that sees nothing."""
    out = torch.zeros(len(q), v.shape[1], dtype=torch.float64)
    size = torch.zeros_like(out)
    reach = torch.zeros(len(q), dtype=torch.float64)
    for i in range(len(q)):
        keys = sees[i].nonzero().flatten()
        if not len(keys):
            continue
        s = k[keys] @ q[i] * scale
        p = (s - s.max()).exp()
        out[i] = p @ v[keys] / p.sum()
        size[i] = p @ v[keys].abs() / p.sum()
        reach[i] = (k[keys].abs() @ q[i].abs()).max() * scale
    return out, size, reach


def prompt_attention(q, k, v, scale, cu_q, cu_k, causal=True):
    """Packed sequences; returns ``out``, ``size`` ``[Tq, H, Dv]`` and ``reach`` ``[Tq, H]``
    (zeros outside the sequences)."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    heads, group = q.shape[1], q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape[0], heads, v.shape[2], dtype=torch.float64)
    size, reach = torch.zeros_like(out), torch.zeros(q.shape[0], heads, dtype=torch.float64)
    for b in range(len(cu_q) - 1):
        a, e = int(cu_q[b]), int(cu_q[b + 1])
        c, f = int(cu_k[b]), int(cu_k[b + 1])
        n, m = e - a, f - c
        sees = torch.ones(n, m, dtype=torch.bool)
        if causal:
            sees = torch.arange(m)[None, :] <= torch.arange(n)[:, None] + m - n
        for h in range(heads):
            got = attend(q[a:e, h], k[c:f, h // group], v[c:f, h // group], scale, sees)
            out[a:e, h], size[a:e, h], reach[a:e, h] = got
    return out, size, reach


def shared_prefix_mla(q, prefix, suffixes, cu_q, scale):
    """``prefix [P, 576]`` and one ``[n, 576]`` of ``suffixes`` per branch, as the values
    their records stand for."""
    q = q.detach().cpu().double()
    out = torch.zeros(q.shape[0], q.shape[1], 512, dtype=torch.float64)
    size, reach = torch.zeros_like(out), torch.zeros(q.shape[:2], dtype=torch.float64)
    for b, suffix in enumerate(suffixes):
        a, e = int(cu_q[b]), int(cu_q[b + 1])
        keys = torch.cat([prefix, suffix]).double()
        for i in range(e - a):
            seen = len(prefix) + max(len(suffix) - (e - a) + 1 + i, 0)
            sees = torch.ones(q.shape[1], seen, dtype=torch.bool)
            got = attend(q[a + i], keys[:seen], keys[:seen, :512], scale, sees)
            out[a + i], size[a + i], reach[a + i] = got
    return out, size, reach


def attention_bound(out, size, reach, keys, eps, dim, tiny=0.0):
    """How far a kernel may be off, element by element, that forms scores in fp32, rounds
    probabilities and its result to a type of ``eps`` (each by at most half a step,
    ``eps / 2``) and sums in fp32.

    With p_j (1 + e_j), |e_j| <= d, in both sums, the result moves by at most
    2 d / (1 - d) size. d: the rounding of p (eps / 2), what the score's fp32 sum of
    ``dim`` products is off (at most (dim + 2) 2^-24 reach, taken twice as the unit's
    order and internal rounding are its own), exp2 and its argument (reach 2^-22 and
    2^-21). The fp32 sums over the keys add (keys + 2) 2^-23 size, the final rounding
    eps / 2 of the result (2^-24 where it is tiny). ``tiny``: the largest |v| for a
    type whose probabilities may be subnormal (fp16: off by up to 2^-25 each, among
    probabilities that sum to at least 1), which moves the result by up to
    2 keys 2^-25 tiny. (Held against 2^7 at the maximum they sum to at least that: a
    test that has to see small ones passes 2^-7 of it.)
    """
    score = (2 * (dim + 2) * 2.0 ** -24 + 2.0 ** -22) * reach + 2.0 ** -21
    d = (eps / 2 + score)[..., None]
    inner = 2 * d / (1 - d) * size + (keys + 2) * 2.0 ** -23 * size + keys * 2.0 ** -24 * tiny
    return inner + eps / 2 * (out.abs() + inner) + 2.0 ** -24


def rope(x, positions, frequencies, offset, interleaved, magnitude, inverse=False):
    """``x [T, H, D]`` with its rotated part turned, in float64."""
    x = x.detach().cpu().double().clone()
    half = len(frequencies)
    angle = positions.cpu().double()[:, None] * frequencies.cpu().double()[None, :]
    cos, sin = magnitude * angle.cos()[:, None], magnitude * angle.sin()[:, None]
    if inverse:
        sin = -sin
    i = torch.arange(half)
    a = offset + (2 * i if interleaved else i)
    b = a + 1 if interleaved else a + half
    u, v = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = u * cos - v * sin, v * cos + u * sin
    return x


def rms_norm(latent, weight, eps):
    latent = latent.detach().cpu().double()
    return latent / (latent.square().mean(1, keepdim=True) + eps).sqrt() * weight.cpu().double()
