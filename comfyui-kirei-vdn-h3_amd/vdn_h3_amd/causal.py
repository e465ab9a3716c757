"""Causal softmax attention with grouped key / value heads on MI355X, for the language model that encodes the prompts.

* ``causal_softmax_packed``: whole prompts of different lengths, packed one behind another;
* ``causal_softmax_cached``: one or several new tokens of each request over the requests' key / value caches.

Both take bf16 and hold scores, sums and softmax statistics in fp32 (q . k, before the scale too, has to stay inside its range).
The products with the values take the probabilities as bf16 (2.0e-3 of the result, with the result's own rounding of 1.6e-3), in
ranges of long caches as two bf16 numbers (1.7e-3). Query head ``h`` reads key / value head ``h // (heads // kv_heads)``. Sequence
bounds are read on the device: a call needs no copy to the host, and a captured one can be replayed with other lengths. Rows that
see an infinity are computed one by one, in a time that grows with the square of the tokens. Forward-only; there is no CPU path.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib
from .window import KERNEL_HEAD_DIMS, padded_head_dim, zero_pad_channels

_INTEGERS = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)


def _check_heads(query, key, value, name):
    if query.dtype != torch.bfloat16 or key.dtype != torch.bfloat16 or value.dtype != torch.bfloat16:
        raise TypeError(f"{name} computes in bf16; got {query.dtype}/{key.dtype}/{value.dtype}")
    heads, kv_heads = query.shape[-2], key.shape[-2]
    if kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} query heads are no multiple of {kv_heads} key / value heads")


def _sequence_bounds(cu_seqlens, rows: int, device) -> torch.Tensor:
    """``cu_seqlens`` as a contiguous int32 device tensor; bounds that the host holds are checked."""
    if not isinstance(cu_seqlens, torch.Tensor):
        cu_seqlens = torch.tensor(list(cu_seqlens))
    if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 1 or cu_seqlens.dtype not in _INTEGERS:
        raise ValueError("cu_seqlens must hold the sequences + 1 integer bounds")
    if cu_seqlens.is_cpu:
        bounds = cu_seqlens.tolist()
        if bounds[0] < 0 or bounds[-1] > rows or any(a > b for a, b in zip(bounds, bounds[1:])):
            raise ValueError(f"cu_seqlens must rise from 0 to at most {rows}, got {bounds[:8]}"
                             f"{' ...' if len(bounds) > 8 else ''}")
        return cu_seqlens.to(torch.int32).to(device)
    if cu_seqlens.get_device() != device.index:
        raise RuntimeError(f"tensors on different devices: {device} and {cu_seqlens.device}")
    return _int32(cu_seqlens, rows)


def _int32(counts: torch.Tensor, most: int) -> torch.Tensor:
    """Counts on the GPU as contiguous int32; wider ones are cut to ``[0, most]`` first, as the kernels cut."""
    if counts.dtype == torch.int32 and counts.is_contiguous():
        return counts
    if counts.dtype == torch.int64:
        counts = counts.clamp(0, most)
    return counts.to(torch.int32).contiguous()


def _output(out, shape, device):
    if out is None:
        return torch.empty(*shape, dtype=torch.bfloat16, device=device)  # 0.8 us less than from a torch.Size
    if tuple(out.shape) != tuple(shape) or out.dtype != torch.bfloat16 or out.stride(-1) != 1:
        raise ValueError(f"out must be a bf16 {list(shape)} tensor with a contiguous last dim")
    if not _lib.in_place(out) or any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise ValueError("out must be 16-byte aligned with strides that are multiples of 8 elements and not 0")
    return out


def causal_softmax_packed(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, cu_seqlens, scale: float, *,
                          out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed sequences: q ``[T, H, D]``, k and v ``[T, H_kv, D]``, all bf16; returns ``[T, H, D]``.

    Sequence ``b`` is the rows ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` (int32 on the GPU; a list or a CPU tensor is
    checked and copied, another integer type on the GPU is converted); row ``i`` of a sequence attends to its rows 0 to
    ``i``. Sequences may be empty. Rows outside every sequence are not written: in a new output they hold anything, in
    ``out`` what it held. Bounds on the GPU are not checked, but cut to ``[0, T]``. ``out`` must not overlap the inputs.
    Head dims 64 and 128 run natively, others up to 128 with zero channels added. Rows of k and v are at most 2**23 elements
    apart.
    """
    if query.ndim != 3 or key.ndim != 3 or key.shape != value.shape or query.shape[0] != key.shape[0] or \
            query.shape[2] != key.shape[2]:
        raise ValueError("query must be [rows, heads, dim], key and value [rows, kv_heads, dim]; got "
                         f"{tuple(query.shape)}, {tuple(key.shape)} and {tuple(value.shape)}")
    _check_heads(query, key, value, "causal_softmax_packed")
    if not 0 < query.shape[2] <= KERNEL_HEAD_DIMS[-1]:
        raise ValueError(f"causal_softmax_packed supports head dims 1 to {KERNEL_HEAD_DIMS[-1]}, got {query.shape[2]}")
    _lib.forward_only("causal_softmax_packed", query, key, value, out)
    rows, heads, dim = query.shape
    _lib.int32_sizes("causal_softmax_packed", rows, heads)
    device = _lib.require_device(query, key, value, out)
    if dim not in KERNEL_HEAD_DIMS:
        width = padded_head_dim(dim)
        if out is not None and (out.shape != query.shape or out.dtype != torch.bfloat16):
            raise ValueError("out must be a bf16 [rows, heads, dim] tensor")
        padded = None if out is None else zero_pad_channels(out, width)  # keeps rows outside every sequence
        res = causal_softmax_packed(*(zero_pad_channels(t, width) for t in (query, key, value)), cu_seqlens,
                                    scale, out=padded)[..., :dim]
        return res.contiguous() if out is None else out.copy_(res)
    cu = _sequence_bounds(cu_seqlens, rows, device)
    out = _output(out, query.shape, device)
    if rows == 0 or heads == 0 or cu.numel() == 1:
        return out
    q, k, v = _lib.operand(query), _lib.operand(key), _lib.operand(value)
    _lib.launch("causal_softmax_packed", _lib.lib().vdnh3_causal_attn_packed, device,
                q.data_ptr(), *q.stride()[:-1], k.data_ptr(), *k.stride()[:-1], v.data_ptr(), *v.stride()[:-1],
                out.data_ptr(), *out.stride()[:-1], cu.data_ptr(), cu.numel() - 1, rows, heads, key.shape[1], dim,
                float(scale))
    return out


@lru_cache(maxsize=1024)
def _cut(batch: int, new: int, room: int, heads: int, kv_heads: int, dim: int) -> tuple[int, int]:
    """The ranges of keys that a call of these sizes takes and the bytes of their partial results."""
    lib = _lib.lib()
    ranges = lib.vdnh3_causal_cached_ranges(batch, new, room, heads, kv_heads, dim)
    return ranges, lib.vdnh3_causal_partial_bytes(new, heads, dim, ranges)


def causal_softmax_cached(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, lengths: torch.Tensor,
                          scale: float, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens over their requests' caches: q ``[B, N, H, D]``, the caches ``[B, room, H_kv, D]`` bf16;
    returns ``[B, N, H, D]``.

    ``lengths`` (``[B]`` int32 on the GPU, another integer type is converted) counts a request's valid cache rows, the
    new tokens' own keys and values (its last N rows) among them: token ``i`` attends to rows 0 to ``lengths[b] - N + i``.
    A token in front of the first row (``lengths[b] < N``) attends to nothing and gives zeros. Rows behind a length are
    not used, whatever they hold. Lengths are cut to ``[0, room]``. Kernel and ranges go by the whole batch, so that a request's last
    bits can differ with the requests beside it. Head dims 64 and 128; the caches are read in place, so
    their layout has to suit the kernel (16-byte rows, at most 2**23 elements apart). ``out`` must not overlap the inputs.
    """
    if query.ndim != 4 or key_cache.ndim != 4 or key_cache.shape != value_cache.shape or \
            query.shape[0] != key_cache.shape[0] or query.shape[3] != key_cache.shape[3]:
        raise ValueError("query must be [batch, new, heads, dim], the caches [batch, room, kv_heads, dim]; got "
                         f"{tuple(query.shape)}, {tuple(key_cache.shape)} and {tuple(value_cache.shape)}")
    _check_heads(query, key_cache, value_cache, "causal_softmax_cached")
    batch, new, heads, dim = query.shape
    room, kv_heads = key_cache.shape[1], key_cache.shape[2]
    _lib.int32_sizes("causal_softmax_cached", batch, new, room, heads)
    if not isinstance(lengths, torch.Tensor):
        raise TypeError(f"lengths must be a tensor of {batch} integers, got {type(lengths).__name__}")
    if lengths.ndim != 1 or lengths.numel() != batch or lengths.dtype not in _INTEGERS:
        raise ValueError(f"lengths must hold {batch} integers, got {tuple(lengths.shape)} {lengths.dtype}")
    if dim not in KERNEL_HEAD_DIMS:
        raise ValueError(f"causal_softmax_cached supports head dims {KERNEL_HEAD_DIMS}, got {dim}")
    _lib.forward_only("causal_softmax_cached", query, key_cache, value_cache, out)
    device = _lib.require_device(query, key_cache, value_cache, lengths, out)
    if not (_lib.in_place(key_cache) and _lib.in_place(value_cache)):
        raise ValueError("the caches must be 16-byte aligned with contiguous channels and strides that are multiples of 8 "
                         "elements (a cache is not copied per call)")
    q = _lib.operand(query)
    out = _output(out, query.shape, device)
    if query.numel() == 0:
        return out
    if room == 0:
        return out.zero_()
    lengths = _int32(lengths, room)
    ranges, size = _cut(batch, new, room, heads, kv_heads, dim)
    partial = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _lib.launch("causal_softmax_cached", _lib.lib().vdnh3_causal_attn_cached, device,
                q.data_ptr(), *q.stride()[:-1], key_cache.data_ptr(), *key_cache.stride()[:-1], value_cache.data_ptr(),
                *value_cache.stride()[:-1], out.data_ptr(), *out.stride()[:-1], lengths.data_ptr(), batch, new, room, heads,
                kv_heads, dim, float(scale), ranges, _lib.ptr(partial), size)
    return out


__all__ = ["causal_softmax_cached", "causal_softmax_packed"]
