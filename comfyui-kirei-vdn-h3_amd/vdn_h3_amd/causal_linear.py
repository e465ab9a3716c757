"""Causal linear attention with a decay for each head on MI355X, for language models with recurrent layers: per value head ``h``
with an fp32 state ``S`` (dv x dk, as in ``gdn``) and ``a = exp(log_decay[h])``::

    S_t = a S_{t-1} + v_t k_t^T,   o_t = scale S_t q_t

* ``causal_linear_packed``: whole prompts of different lengths, packed one behind another, in chunks of 64 tokens;
* ``causal_linear_step``: one or several new tokens of each request, over a pool of the requests' states.

Both take bf16 and hold states and sums in fp32; outputs are rounded once. Value head ``h`` reads query / key head
``h // (heads // qk_heads)``; expanded views (stride 0) are read in place. Sequence bounds and slots are read on the device: a call
needs no copy to the host, and a captured one can be replayed with others. Forward-only; there is no CPU path.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache

import torch

from . import _lib
from .causal import _INTEGERS, _output, _sequence_bounds
from .window import KERNEL_HEAD_DIMS, padded_head_dim, zero_pad_channels


def _head_checks(name: str, dtypes, heads: int, qk_heads: int, dim: int) -> None:
    if any(d != torch.bfloat16 for d in dtypes):
        raise TypeError(f"{name} computes in bf16; got {dtypes[0]}/{dtypes[1]}/{dtypes[2]}")
    if (heads > 0 and qk_heads == 0) or (qk_heads and heads % qk_heads):
        raise ValueError(f"{heads} value heads are no multiple of {qk_heads} query / key heads")
    if not 0 < dim <= KERNEL_HEAD_DIMS[-1]:
        raise ValueError(f"{name} supports head dims 1 to {KERNEL_HEAD_DIMS[-1]}, got {dim}")


def _decays(log_decay, heads: int, name: str) -> torch.Tensor:
    if not isinstance(log_decay, torch.Tensor) or tuple(log_decay.shape) != (heads,) or not log_decay.is_floating_point():
        raise ValueError(f"{name}: log_decay must be a tensor of {heads} numbers, one per value head")
    return log_decay.float().contiguous()


def _states(state, shape, name: str) -> torch.Tensor:
    if not isinstance(state, torch.Tensor) or tuple(state.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {list(shape)}")
    if state.dtype != torch.float32:
        raise TypeError(f"{name} must be fp32, got {state.dtype}")
    return state


@lru_cache(maxsize=1024)
def _cut(rows: int, sequences: int, heads: int, dim: int) -> tuple[int, int]:
    """The ranges of chunks that a call of these sizes takes and the bytes of the states between them."""
    lib = _lib.lib()
    ranges = lib.vdnh3_causal_linear_ranges(rows, sequences, heads, dim)
    return ranges, lib.vdnh3_causal_linear_workspace_bytes(ranges, heads, dim)


def causal_linear_packed(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, log_decay: torch.Tensor, cu_seqlens,
                         scale: float, *, initial_state: torch.Tensor | None = None, output_final_state: bool = False,
                         out: torch.Tensor | None = None):
    """``(o [T, H, D] bf16, final states [B, H, D, D] fp32 or None)`` of packed sequences: q and k ``[T, H_qk, D]``, v
    ``[T, H, D]``, all bf16, ``log_decay`` ``[H]`` (0 keeps everything, -inf nothing).

    Sequence ``b`` is the rows ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` as in ``causal_softmax_packed``; its state starts from
    ``initial_state[b]`` (``[B, H, D, D]`` fp32, dv rows, dk columns) or zeros. An empty sequence's final state is its initial
    one. Rows outside every sequence are not written. A value (or a number of an initial state's row) that is no finite number
    ends its channel: from its token on that channel's outputs and states are none either, rows in front of it are as without it.
    A token behind a row takes no part in it, whatever it holds. ``out`` must not overlap the inputs. Head dims 64 and 128 run
    natively, others up to 128 with zero channels added. Rows are at most 2**23 elements apart.
    """
    name = "causal_linear_packed"
    if query.ndim != 3 or query.shape != key.shape or value.ndim != 3 or query.shape[0] != value.shape[0] or \
            query.shape[2] != value.shape[2]:
        raise ValueError("query and key must be [rows, qk_heads, dim], value [rows, heads, dim]; got "
                         f"{tuple(query.shape)}, {tuple(key.shape)} and {tuple(value.shape)}")
    _head_checks(name, (query.dtype, key.dtype, value.dtype), value.shape[1], query.shape[1], query.shape[2])
    _lib.forward_only(name, query, key, value, log_decay, initial_state, out)
    rows, heads, dim = value.shape
    _lib.int32_sizes(name, rows, heads)
    decays = _decays(log_decay, heads, name)
    device = _lib.require_device(query, key, value, decays, initial_state, out)
    cu = _sequence_bounds(cu_seqlens, rows, device)
    sequences = cu.numel() - 1
    if initial_state is not None:
        _states(initial_state, (sequences, heads, dim, dim), "initial_state")
    if dim not in KERNEL_HEAD_DIMS:
        width = padded_head_dim(dim)
        if out is not None and (out.shape != value.shape or out.dtype != torch.bfloat16):
            raise ValueError("out must be a bf16 [rows, heads, dim] tensor")
        padded = None if out is None else zero_pad_channels(out, width)  # keeps rows outside every sequence
        begin = None
        if initial_state is not None:
            begin = torch.zeros(sequences, heads, width, width, dtype=torch.float32, device=device)
            begin[..., :dim, :dim] = initial_state
        res, final = causal_linear_packed(*(zero_pad_channels(t, width) for t in (query, key, value)), decays, cu, scale,
                                          initial_state=begin, output_final_state=output_final_state, out=padded)
        res = res[..., :dim].contiguous() if out is None else out.copy_(res[..., :dim])
        return res, None if final is None else final[..., :dim, :dim].contiguous()
    out = _output(out, value.shape, device)
    final = torch.empty(sequences, heads, dim, dim, dtype=torch.float32, device=device) if output_final_state else None
    if heads == 0 or sequences == 0:
        return out, final
    if rows == 0:
        if final is not None:
            final.zero_() if initial_state is None else final.copy_(initial_state)
        return out, final
    begin = initial_state
    if begin is not None and (not begin.is_contiguous() or begin.data_ptr() % 16):
        begin = begin.clone(memory_format=torch.contiguous_format)
    q, k, v = _lib.operand(query), _lib.operand(key), _lib.operand(value)
    ranges, size = _cut(rows, sequences, heads, dim)
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _lib.launch(name, _lib.lib().vdnh3_causal_linear_packed, device,
                q.data_ptr(), *q.stride()[:-1], k.data_ptr(), *k.stride()[:-1], v.data_ptr(), *v.stride()[:-1],
                out.data_ptr(), *out.stride()[:-1], decays.data_ptr(), cu.data_ptr(), _lib.ptr(begin), _lib.ptr(final),
                sequences, rows, heads, query.shape[1], dim, float(scale), ranges, _lib.ptr(workspace), size)
    return out, final


@lru_cache(maxsize=4096)
def _step_plan(name: str, *layouts) -> tuple:
    """What the layouts of a step call say, checked and put down for the library once for each set of them, not per call (that
    took more than half of a call's 15 us): shape, strides and dtype of q, k, v, the pool, slots, out (``None`` three times
    without them) and the gates. Returns ``(vdnh3_step_layout, out's shape, whether operands have to be copied first)``."""
    (qs, qt, qd), (ks, kt, kd), (vs, vt, vd), (ps, pt, pd), (ss, st, sd), (os, ot, od), *gates = zip(*[iter(layouts)] * 3)
    if len(qs) != 4 or qs != ks or len(vs) != 4 or qs[:2] != vs[:2] or qs[3] != vs[3]:
        raise ValueError("query and key must be [batch, new, qk_heads, dim], value [batch, new, heads, dim]; got "
                         f"{tuple(qs)}, {tuple(ks)} and {tuple(vs)}")
    _head_checks(name, (qd, kd, vd), vs[2], qs[2], qs[3])
    batch, new, heads, dim = vs
    _lib.int32_sizes(name, *vs)
    if len(ps) != 4 or tuple(ps[1:]) != (heads, dim, dim):
        raise ValueError(f"{name}: state must be [slots, {heads}, {dim}, {dim}], got {tuple(ps)}")
    if pd != torch.float32:
        raise TypeError(f"{name}: state must be fp32, got {pd}")
    if dim > 1 and (pt[3] != 1 or pt[2] != dim):
        raise ValueError(f"{name}: each head's state must be contiguous (it is updated in place)")
    _lib.int32_sizes(name, ps[0])
    if ss is None:
        if batch > ps[0]:
            raise ValueError(f"{name}: {batch} requests need a state each, the pool has {ps[0]}")
    elif tuple(ss) != (batch,) or sd not in _INTEGERS:
        raise ValueError(f"{name}: slots must be a tensor of {batch} integers")
    if os is None:
        ot = (new * heads * dim, heads * dim, dim, 1)
    elif os != vs or od != torch.bfloat16 or (dim > 1 and ot[3] != 1) or any(n > 1 and s == 0 for n, s in zip(os, ot)):
        raise ValueError(f"out must be a bf16 {list(vs)} tensor with a contiguous last dim and no stride of 0")
    shape = (heads,) if len(gates) == 1 else (batch, new, heads)
    for gs, _, gd in gates:
        if tuple(gs) != shape or not gd.is_floating_point:
            what = "log_decay must be a tensor" if len(gates) == 1 else "beta and g must be tensors"
            raise ValueError(f"{name}: {what} of shape {list(shape)}, floating-point")
    # the channels next to each other; slots in 32 bits; gates in fp32, one per head next to each other
    copies = any(t[3] != 1 and dim != 1 for t in (qt, kt, vt)) or (
        ss is not None and (sd != torch.int32 or (batch > 1 and st[0] != 1))) or any(
        gd != torch.float32 or (len(gates) == 1 and heads > 1 and gt[0] != 1) for _, gt, gd in gates)
    gate_strides = (0,) * 6 if len(gates) == 1 else (*gates[0][1], *gates[1][1])
    layout = (ctypes.c_int64 * 26)(*qt[:3], *kt[:3], *vt[:3], *ot[:3], pt[0], pt[1], *gate_strides, ps[0], batch, new, heads,
                                   qs[2], dim)
    return layout, tuple(vs), copies


def _step_copies(query, key, value, slots, gates, count: int):
    """The operands as the kernels take them, where a call's layouts need copies."""
    if slots is not None:
        if slots.dtype == torch.int64:
            slots = slots.clamp(-1, count)  # outside the pool stays outside in 32 bits
        slots = slots.to(torch.int32).contiguous()
    gates = tuple(g.float().contiguous() for g in gates)
    return *(t if t.stride(-1) == 1 else t.contiguous() for t in (query, key, value)), slots, gates


def _step(name: str, fn, query, key, value, state, slots, gates, out, *scale):
    """A step call of either rule: ``gates`` are its decays (one number a head), or beta and g (one a token and head)."""
    try:
        layouts = (query.shape, query.stride(), query.dtype, key.shape, key.stride(), key.dtype, value.shape, value.stride(),
                   value.dtype, state.shape, state.stride(), state.dtype,
                   *((None, None, None) if slots is None else (slots.shape, slots.stride(), slots.dtype)),
                   *((None, None, None) if out is None else (out.shape, out.stride(), out.dtype)),
                   *(x for g in gates for x in (g.shape, g.stride(), g.dtype)))
    except AttributeError:
        raise TypeError(f"{name} takes tensors (query, key, value, the gates, state, slots, out)") from None
    layout, shape, copies = _step_plan(name, *layouts)
    _lib.forward_only(name, query, key, value, state, out, *gates)
    device = _lib.require_device(query, key, value, state, slots, out, *gates)
    if out is None:
        out = torch.empty(*shape, dtype=torch.bfloat16, device=device)
    if 0 in shape:
        return out
    if state.shape[0] == 0:
        return out.zero_()
    if copies:
        query, key, value, slots, gates = _step_copies(query, key, value, slots, gates, state.shape[0])
        return _step(name, fn, query, key, value, state, slots, gates, out, *scale)
    _lib.launch(name, fn, device, query.data_ptr(), key.data_ptr(), value.data_ptr(), out.data_ptr(),
                *[g.data_ptr() for g in gates], state.data_ptr(), None if slots is None else slots.data_ptr(), layout, *scale)
    return out


def causal_linear_step(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, log_decay: torch.Tensor,
                       state: torch.Tensor, scale: float, *, slots: torch.Tensor | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """New tokens over the requests' states: q and k ``[B, N, H_qk, D]``, v ``[B, N, H, D]`` bf16; returns ``[B, N, H, D]``.

    ``state`` is the pool ``[slots, H, D, D]`` fp32 (a head's state contiguous, any strides of slots and heads), updated in place:
    request ``b`` has ``state[slots[b]]`` (``slots`` ``[B]`` integers on the GPU; ``None``: ``state[b]``) and takes its tokens
    in order. A slot outside the pool (-1 by custom) is an idle request: its rows are zeros and nothing is updated. A slot that an
    earlier request of the batch names belongs to that one: the later request's rows are NaN. Head dims up to 128.
    ``out`` must not overlap the inputs.
    """
    return _step("causal_linear_step", _lib.lib().vdnh3_causal_linear_step, query, key, value, state, slots, (log_decay,), out,
                 float(scale))


__all__ = ["causal_linear_packed", "causal_linear_step"]
