"""Float64 restatement of the operators of the language model that encodes the prompts (not in the reference).

Independent checks (``tests/test_oracle_prompt.py``): closed forms (a constant row's norm, one key's attention, a quarter
turn) and torch's own ``softmax`` / ``rms_norm`` in float64 on whole inputs.
"""

from __future__ import annotations

import torch


def residual_rmsnorm(x, residual, weight, eps):
    """``(t, y)``: the sum and its RMSNorm, float64."""
    t = x.double() if residual is None else x.double() + residual.double()
    return t, t / (t.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()


def rotate_axes(x, weight, eps, positions, sections, theta, ladder):
    """``(y, pair, angle)``: the (normalised, where a weight is given) and turned vectors of x ``[S, H, D]``; the sizes
    ``|y_i| + |y_{i+h}|`` of each channel's pair (of the channel itself past the rotated ones) and the angles [S, pairs]."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    angles = []
    half = sum(sections)
    for axis, count in enumerate(sections):
        before = sum(sections[:axis])
        for i in range(count):
            power = i / count if ladder == "per_axis" else (before + i) / half
            angles.append(positions[axis].double() * float(theta) ** -power)
    angle = torch.stack(angles, -1)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b, rest = y[..., :half], y[..., half:2 * half], y[..., 2 * half:]
    size = a.abs() + b.abs()
    return torch.cat([a * c - b * s, b * c + a * s, rest], -1), torch.cat([size, size, rest.abs()], -1), angle


def attend(q, k, v, last, scale):
    """Rows q ``[N, H, D]`` over keys k, v ``[M, H_kv, D]``, row i seeing keys 0 .. last[i]: ``(out, size, score)`` with
    ``size = sum p |v|`` and ``score`` the largest ``scale sum |q_d k_d|`` of a row and head over the keys it sees. A row
    without keys gives zeros. Keys that a row does not see take no part, whatever they hold."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(n, heads, dim, dtype=torch.float64)
    size, score = torch.zeros_like(out), torch.zeros(n, heads, dtype=torch.float64)
    for i in range(n):
        m = int(last[i]) + 1
        if m <= 0:
            continue
        qi = q[i].double().view(k.shape[1], group, dim)
        ki, vi = k[:m].double().transpose(0, 1), v[:m].double().transpose(0, 1)
        p = torch.softmax((qi @ ki.transpose(1, 2)) * scale, -1)
        out[i] = (p @ vi).reshape(heads, dim)
        size[i] = (p @ vi.abs()).reshape(heads, dim)
        score[i] = ((qi.abs() @ ki.abs().transpose(1, 2)) * scale).amax(-1).reshape(heads)
    return out, size, score


def packed(q, k, v, bounds, scale):
    """Causal attention of the packed sequences between ``bounds``; rows of no sequence are NaN."""
    out = torch.full(q.shape, torch.nan, dtype=torch.float64)
    size, score = out.clone(), out[..., 0].clone()
    for a, b in zip(bounds, bounds[1:]):
        if b > a:
            out[a:b], size[a:b], score[a:b] = attend(q[a:b], k[a:b], v[a:b], range(b - a), scale)
    return out, size, score


def cached(q, k_cache, v_cache, lengths, scale):
    """New tokens q ``[B, N, H, D]`` over their caches."""
    n = q.shape[1]
    parts = [attend(q[b], k_cache[b], v_cache[b], [m - n + i for i in range(n)], scale) for b, m in enumerate(lengths)]
    return tuple(torch.stack(t) for t in zip(*parts))
