"""Float64 restatement of the operators that serve many requests' recurrent states and adapters (not in the reference).

Independent checks (``tests/test_oracle_recurrent.py``): the sum over all earlier tokens without a state, the Gated DeltaNet's
oracle, a closed form for one channel, adapters by ``F.linear``.
"""

from __future__ import annotations

import torch


def linear_recurrence(q, k, v, log_decay, scale, initial=None):
    """One sequence: q, k ``[T, H_qk, D]``, v ``[T, H, D]``, log_decay ``[H]``. ``(out, out_size, state, state_size)`` with the
    sizes ``sum a^d (1 + d |log2 a|) |terms|``: what an error of the decays, relative to ``1 + d |log2 a|``, can reach."""
    steps, heads, dim = v.shape
    group = heads // q.shape[1]
    a = torch.exp(log_decay.double()).view(heads, 1, 1)
    depth = torch.where(a > 0, -log_decay.double().view(heads, 1, 1) / 0.6931471805599453, 0.0).abs()
    depth = torch.where(a > 0, depth, 0.0)
    s = torch.zeros(heads, dim, dim, dtype=torch.float64, device=v.device) if initial is None else initial.double().clone()
    plain = s.abs()
    size = plain.clone()
    out = torch.empty(steps, heads, dim, dtype=torch.float64, device=v.device)
    out_size = torch.empty_like(out)
    for t in range(steps):
        kt, qt = (x[t].double().repeat_interleave(group, 0) for x in (k, q))
        vt = v[t].double()
        s = torch.where(a > 0, a * s, 0.0) + vt[:, :, None] * kt[:, None]
        add = vt.abs()[:, :, None] * kt.abs()[:, None]
        size = a * (size + depth * plain) + add
        plain = a * plain + add
        out[t] = scale * (s @ qt[..., None])[..., 0]
        out_size[t] = abs(scale) * (size @ qt.abs()[..., None])[..., 0]
    return out, out_size, s, size


def delta_recurrence(q, k, v, beta, g, initial):
    """The gated delta rule over tokens of one request (q, k ``[N, H_qk, D]``, v ``[N, H, D]``): ``(out, out_size, state,
    state_size)``, the sizes with every term's absolute value."""
    steps, heads, dim = v.shape
    group = heads // q.shape[1]
    s, size = initial.double().clone(), initial.double().abs()
    outs, sizes = [], []
    for t in range(steps):
        kt, qt = (x[t].double().repeat_interleave(group, 0) for x in (k, q))
        a, b = torch.exp(g[t].double()).view(heads, 1, 1), beta[t].double().view(heads, 1, 1)
        vk = v[t].double()[:, :, None] * kt[:, None]
        s = a * (s - b * (s @ kt[..., None]) * kt[:, None]) + b * vk
        size = a * (size + b.abs() * (size @ kt.abs()[..., None]) * kt.abs()[:, None]) + b.abs() * vk.abs()
        outs.append((s @ qt[..., None])[..., 0])
        sizes.append((size @ qt.abs()[..., None])[..., 0])
    return torch.stack(outs), torch.stack(sizes), s, size


def adapters(y, x, down, up, scales, index):
    """``y + s_i B_i A_i x`` by row (no adapter where the index is none): ``(out, size)``, the size with absolute values."""
    out, size = y.double().clone(), y.double().abs()
    for i in range(down.shape[0]):
        mine = index == i
        a, b, s = down[i].double(), up[i].double(), float(scales[i])
        out[mine] += s * (x[mine].double() @ a.t()) @ b.t()
        size[mine] += abs(s) * (x[mine].double().abs() @ a.abs().t()) @ b.abs().t()
    return out, size
