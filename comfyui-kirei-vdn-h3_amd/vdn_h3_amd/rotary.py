"""Rotary positions on several axes (time, height, width) for grouped-head q / k on MI355X.

``RotaryAxes`` says which axis turns which channel pairs and how fast; ``normalise_qk_axes`` applies it to the raw q and k
of a projection, with their RMSNorm fused in, from the rows' positions: the angles are computed on the device, in 64 bits
up to the fraction of a turn, so no table of rotations is kept per row. ``hybrid.normalise_qk`` is the same pass for
tables of 2x2 matrices. Forward-only; there is no CPU path.
"""

from __future__ import annotations

import math

import torch

from . import _lib

LADDERS = ("shared", "per_axis")
_POSITION_CODES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


class RotaryAxes:
    """The channel pairs of each axis and their frequencies.

    ``sections[a]`` pairs belong to axis ``a``, in order; ``rot_dim = 2 * sum(sections)`` channels turn, pair ``i`` being
    channels ``i`` and ``i + rot_dim / 2`` (split-half, as in the block). Pair ``i`` turns by ``theta ** (-i / n)`` per
    position: with ``ladder="shared"`` over all ``n = rot_dim / 2`` pairs (one ladder of frequencies, cut into axes), with
    ``"per_axis"`` over the ``n = sections[a]`` pairs of its own axis, counted from the axis's first pair. The object holds the
    frequencies on the device: it has to outlive graphs that were captured with it.
    """

    def __init__(self, sections, theta: float = 10000.0, ladder: str = "shared"):
        self.sections = tuple(int(n) for n in sections)
        if not self.sections or any(n < 0 for n in self.sections) or sum(self.sections) == 0:
            raise ValueError(f"sections must be pair counts of the axes, got {tuple(sections)}")
        if ladder not in LADDERS:
            raise ValueError(f"ladder={ladder!r}; expected one of {LADDERS}")
        if not (math.isfinite(theta) and theta > 0):
            raise ValueError(f"theta must be positive and finite, got {theta}")
        self.theta, self.ladder = float(theta), ladder
        self.rot_dim = 2 * sum(self.sections)
        if self.rot_dim % 16:
            raise ValueError(f"rot_dim {self.rot_dim} (twice the sum of the sections) must be a multiple of 16")
        self._tables: dict[torch.device, tuple[torch.Tensor, torch.Tensor]] = {}

    @property
    def axes(self) -> int:
        return len(self.sections)

    def frequencies(self) -> tuple[torch.Tensor, torch.Tensor]:
        """``(radians per position float64, axis int32)`` of each pair, on the CPU."""
        axis = torch.repeat_interleave(torch.arange(self.axes, dtype=torch.int32), torch.tensor(self.sections))
        pair = torch.arange(self.rot_dim // 2, dtype=torch.float64)
        count = torch.full_like(pair, self.rot_dim // 2)
        if self.ladder == "per_axis":
            widths = torch.tensor(self.sections, dtype=torch.float64)
            pair = pair - (widths.cumsum(0) - widths)[axis.long()]
            count = widths[axis.long()]
        return torch.pow(torch.tensor(self.theta, dtype=torch.float64), -pair / count), axis

    def table(self, device) -> tuple[torch.Tensor, torch.Tensor]:
        """``(turns per position float64, axis int32)`` on ``device``, made once per device (a copy from the host, so a
        graph capture needs one call, or this method, before it)."""
        hit = self._tables.get(device)
        if hit is None:
            radians, axis = self.frequencies()
            hit = self._tables[device] = ((radians / (2 * math.pi)).to(device), axis.to(device))
        return hit


def _norm_weight(weight, dim: int, name: str):
    if weight is None:
        return None
    if weight.numel() != dim:
        raise ValueError(f"{name} must have {dim} entries")
    return _lib.operand(weight.reshape(-1).to(torch.bfloat16))


def normalise_qk_axes(q_raw: torch.Tensor, k_raw: torch.Tensor, positions: torch.Tensor, axes: RotaryAxes,
                      q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                      k_eps: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """q ``[S, H, D]`` and k ``[S, H_kv, D]``, normalised over D where a weight is given, turned by their rows' positions.

    ``positions``: ``[axes, S]`` int32, int64 or float32 on the GPU, any strides, or ``[S]`` for the same position on every
    axis; positions past 2**53 turns lose their fraction. ``eps`` is q's epsilon, ``k_eps`` k's (``eps`` when ``None``).
    D is a multiple of 8 up to 128. Returns new contiguous bf16 tensors (fp32 inside, 64 bits for the norm of vectors whose squares
    leave it, one rounding).
    """
    if q_raw.ndim != 3 or k_raw.ndim != 3 or q_raw.shape[0] != k_raw.shape[0] or q_raw.shape[2] != k_raw.shape[2]:
        raise ValueError("q must be [sequence, heads, dim] and k [sequence, kv_heads, dim]; "
                         f"got {tuple(q_raw.shape)} and {tuple(k_raw.shape)}")
    if q_raw.dtype != torch.bfloat16 or k_raw.dtype != torch.bfloat16:
        raise TypeError(f"normalise_qk_axes computes in bf16; got {q_raw.dtype}/{k_raw.dtype}")
    _lib.forward_only("normalise_qk_axes", q_raw, k_raw, q_weight, k_weight, positions)
    seq, heads, dim = q_raw.shape
    kv_heads = k_raw.shape[1]
    _lib.int32_sizes("normalise_qk_axes", seq, heads, kv_heads)
    device = _lib.require_device(q_raw, k_raw, q_weight, k_weight, positions)
    code = _POSITION_CODES.get(positions.dtype)
    if code is None:
        raise TypeError(f"positions must be int32, int64 or float32, got {positions.dtype}")
    if positions.ndim == 1:
        positions = positions.expand(axes.axes, positions.shape[0])
    if tuple(positions.shape) != (axes.axes, seq):
        raise ValueError(f"positions must be [{axes.axes}, {seq}], got {tuple(positions.shape)}")
    if axes.rot_dim > dim or dim % 8 or not 0 < dim <= 128:
        raise ValueError(f"head dim {dim} must be a multiple of 8 up to 128 and hold the {axes.rot_dim} rotated channels")
    wq, wk = _norm_weight(q_weight, dim, "q_weight"), _norm_weight(k_weight, dim, "k_weight")
    q, k = _lib.operand(q_raw), _lib.operand(k_raw)
    qn = torch.empty(seq, heads, dim, dtype=torch.bfloat16, device=device)
    kn = torch.empty(seq, kv_heads, dim, dtype=torch.bfloat16, device=device)
    if seq == 0:
        return qn, kn
    turns, axis = axes.table(device)
    _lib.launch("vdnh3_qk_rotary_axes", _lib.lib().vdnh3_qk_rotary_axes, device,
                q.data_ptr(), q.stride(0), q.stride(1), _lib.ptr(wq), float(eps), qn.data_ptr(), heads * dim, dim, heads,
                k.data_ptr(), k.stride(0), k.stride(1), _lib.ptr(wk), float(eps if k_eps is None else k_eps), kn.data_ptr(),
                kv_heads * dim, dim, kv_heads, positions.data_ptr(), code, *positions.stride(), turns.data_ptr(),
                axis.data_ptr(), axes.rot_dim, seq, dim)
    return qn, kn


__all__ = ["LADDERS", "RotaryAxes", "normalise_qk_axes"]
