"""Low-rank adapters of many requests beside a shared projection on MI355X.

A projection runs once for the rows of all requests; each row's own adapter is added to its output::

    out_t = y_t + s_i B_i (A_i x_t),   i = index[t]

``LowRankAdapters`` holds the adapters of one projection, ``add`` applies them; ``linear.HipLinear`` takes both
(``adapters=``, ``adapter_index=``). The index is read on the device: a captured call can be replayed with another.
Forward-only; there is no CPU path.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib
from .causal import _INTEGERS

_NAME = "LowRankAdapters.add"


@lru_cache(maxsize=4096)
def _add_plan(xs, xt, xd, ys, yt, yd, ins, it, ind, width: int, out_width: int, count: int, rank: int) -> tuple[int, int, bool]:
    """What the layouts of a call say, checked once for each set of them: ``(rows, workspace bytes, whether no operand has to be
    copied but for an address off 16 bytes)``."""
    rows = xs[0] if len(xs) == 2 else -1
    if len(xs) != 2 or tuple(xs) != (rows, width) or tuple(ys) != (rows, out_width):
        raise ValueError(f"y must be [rows, {out_width}] and x [rows, {width}]; got {tuple(ys)} and {tuple(xs)}")
    if xd != torch.bfloat16 or yd != torch.bfloat16:
        raise TypeError(f"LowRankAdapters.add computes in bf16; got {yd}/{xd}")
    if tuple(ins) != (rows,) or ind not in _INTEGERS:
        raise ValueError(f"index must be a tensor of {rows} integers, one per row")
    _lib.int32_sizes(_NAME, rows)

    def whole(t):
        return t[1] == 1 and (rows < 2 or t[0] % 8 == 0)

    as_they_lie = whole(xt) and whole(yt) and ind == torch.int32 and (rows < 2 or it[0] == 1)
    return rows, _lib.lib().vdnh3_adapter_workspace_wanted(rows, width, count, rank), as_they_lie


def _layouts(down: torch.Tensor, up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """A and B in the kernels' order (``include/vdnh3.h``), the rank filled up with zeros to 16 or a multiple of 32, the widths
    to multiples of 64 and 32."""
    n, rank, width = down.shape
    out = up.shape[1]
    ranks = 16 if rank <= 16 else -(-rank // 32) * 32
    pad = torch.nn.functional.pad
    a = pad(down, (0, -width % 64, 0, ranks - rank)).view(n, ranks // 16, 16, -1, 2, 4, 8)
    b = pad(up, (0, ranks - rank, 0, -out % 32))
    if ranks == 16:
        b = b.view(n, -1, 4, 2, 4, 4, 4).permute(0, 1, 5, 2, 4, 3, 6)
    else:
        b = b.view(n, -1, 4, 2, 4, ranks // 32, 4, 8).permute(0, 1, 5, 3, 6, 2, 4, 7)
    return a.permute(0, 3, 1, 4, 5, 2, 6).contiguous(), b.contiguous()


class LowRankAdapters:
    """The adapters of one projection ``[out, width]``: ``down`` ``[n, rank, width]`` (A) and ``up`` ``[n, out, rank]`` (B), bf16 on
    the GPU, and ``scales``, ``n`` numbers (a tensor or a sequence; ``None``: ones), kept in fp32.

    Widths are multiples of 8 (at most 2**30), ranks at most 1024. The object keeps copies, A and B in the kernels' order (a later
    change of the tensors is not seen), and has to outlive graphs that were captured with it. ``from_pairs`` takes adapters of
    different ranks.
    """

    def __init__(self, down: torch.Tensor, up: torch.Tensor, scales=None):
        if not isinstance(down, torch.Tensor) or not isinstance(up, torch.Tensor) or down.ndim != 3 or up.ndim != 3 or \
                down.shape[0] != up.shape[0] or down.shape[1] != up.shape[2] or 0 in down.shape or 0 in up.shape:
            raise ValueError("down must be [adapters, rank, width] and up [adapters, out, rank]")
        if down.dtype != torch.bfloat16 or up.dtype != torch.bfloat16:
            raise TypeError(f"LowRankAdapters computes in bf16; got {down.dtype}/{up.dtype}")
        self.count, self.rank, self.width = (int(n) for n in down.shape)
        self.out_width = int(up.shape[1])
        if self.width % 8 or self.out_width % 8 or max(self.width, self.out_width) > 2 ** 30:
            raise ValueError(f"the projection's widths must be multiples of 8, at most 2**30, got {self.width} -> "
                             f"{self.out_width}")
        if self.rank > 1024:
            raise ValueError(f"ranks up to 1024 are supported, got {self.rank}")
        _lib.forward_only("LowRankAdapters", down, up, scales)
        if scales is not None:
            scales = torch.as_tensor(scales, dtype=torch.float32, device=down.device).detach().reshape(-1).clone()
            if scales.numel() != self.count:
                raise ValueError(f"scales must be {self.count} numbers, got {scales.numel()}")
        _lib.require_device(down, up, scales)
        self.down, self.up = _layouts(down.detach(), up.detach())
        self.scales = scales

    @classmethod
    def from_pairs(cls, pairs, scales=None) -> "LowRankAdapters":
        """From ``(down [rank_i, width], up [out, rank_i])`` of each adapter; smaller ranks are filled up with zeros
        (which are a NaN times an infinite x)."""
        pairs = list(pairs)
        if not pairs or any(a.ndim != 2 or b.ndim != 2 or a.shape[0] != b.shape[1] or a.shape[1] != pairs[0][0].shape[1] or
                            b.shape[0] != pairs[0][1].shape[0] for a, b in pairs):
            raise ValueError("pairs must be (down [rank, width], up [out, rank]) of one projection")
        rank = max(a.shape[0] for a, _ in pairs)
        pad = torch.nn.functional.pad
        return cls(torch.stack([pad(a, (0, 0, 0, rank - a.shape[0])) for a, _ in pairs]),
                   torch.stack([pad(b, (0, rank - b.shape[1])) for _, b in pairs]), scales)

    def add(self, y: torch.Tensor, x: torch.Tensor, index: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
        """``y`` ``[T, out]`` with each row's adapter applied to ``x`` ``[T, width]`` added, both bf16: a new tensor, or ``out``,
        which may be ``y`` itself (but not overlap it, or x, otherwise).

        ``index`` (``[T]`` integers on the GPU) names a row's adapter; a number outside ``[0, n)`` (-1 by custom) names none, and
        the row keeps ``y``. The sum is rounded once; ``A x`` is fp32. Rows of one adapter are fastest next to each other.
        A number that is not finite stays in its row: infinities of A and x come out as by the formula, those of B as no finite
        numbers.
        """
        return self.apply(self.checked(y, x, index, out), y, x, index, out)

    def checked(self, y: torch.Tensor, x: torch.Tensor, index: torch.Tensor, out: torch.Tensor | None) -> tuple:
        """What ``apply`` needs to know of a call, after every check of its arguments, before anything is written."""
        if not isinstance(index, torch.Tensor):
            raise ValueError(f"index must be a tensor of integers, one per row, got {type(index).__name__}")
        rows, size, as_they_lie = _add_plan(x.shape, x.stride(), x.dtype, y.shape, y.stride(), y.dtype, index.shape, index.stride(),
                                            index.dtype, self.width, self.out_width, self.count, self.rank)
        _lib.forward_only(_NAME, y, x, out)
        device = _lib.require_device(self.down, y, x, index, out)
        if out is not None and (
                out is not y and (tuple(out.shape) != (rows, self.out_width) or out.dtype != torch.bfloat16) or
                not _lib.in_place(out) or (rows > 1 and out.stride(0) < self.out_width)):
            raise ValueError(f"out must be a bf16 [{rows}, {self.out_width}] tensor with 16-byte aligned rows that do not overlap")
        return rows, size, as_they_lie, device

    def apply(self, plan: tuple, y: torch.Tensor, x: torch.Tensor, index: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
        """``add`` of arguments that ``checked`` gave a plan for."""
        rows, size, as_they_lie, device = plan
        if out is None:
            out = torch.empty(rows, self.out_width, dtype=torch.bfloat16, device=device)
        if rows == 0:
            return out
        if not as_they_lie or x.data_ptr() % 16 or y.data_ptr() % 16:
            x, y = _lib.operand(x), _lib.operand(y)
            if index.dtype == torch.int64:
                index = index.clamp(-1, self.count)  # outside stays outside in 32 bits
            index = index.to(torch.int32).contiguous()
        workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        _lib.launch(_NAME, _lib.lib().vdnh3_adapter_add, device,
                    y.data_ptr(), y.stride(0), x.data_ptr(), x.stride(0), self.down.data_ptr(), self.up.data_ptr(),
                    _lib.ptr(self.scales), index.data_ptr(), out.data_ptr(), out.stride(0), rows, self.width, self.out_width,
                    self.count, self.rank, _lib.ptr(workspace), size)
        return out


__all__ = ["LowRankAdapters"]
