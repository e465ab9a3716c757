"""Refusals of the operators that serve many requests' states and adapters, which need no GPU: arguments are checked before any
device work."""

from __future__ import annotations

import ctypes

import pytest
import torch

BF = torch.bfloat16


def _z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def _f(*shape):
    return torch.zeros(shape)


def test_packed_refusals(built_lib):
    from vdn_h3_amd.causal_linear import causal_linear_packed as op

    q, v, d = _z(6, 2, 64), _z(6, 4, 64), _f(4)
    for bad in [lambda: op(q, _z(5, 2, 64), v, d, [0, 6], 0.1), lambda: op(q, _z(6, 4, 64), v, d, [0, 6], 0.1),
                lambda: op(q, q, _z(5, 4, 64), d, [0, 6], 0.1), lambda: op(q, q, _z(6, 4, 32), d, [0, 6], 0.1),
                lambda: op(q[0], q[0], v, d, [0, 6], 0.1), lambda: op(q, q, _z(6, 3, 64), _f(3), [0, 6], 0.1),
                lambda: op(_z(6, 0, 64), _z(6, 0, 64), v, d, [0, 6], 0.1), lambda: op(q, q, v, _f(3), [0, 6], 0.1),
                lambda: op(q, q, v, torch.zeros(4, dtype=torch.int64), [0, 6], 0.1), lambda: op(q, q, v, -0.1, [0, 6], 0.1),
                lambda: op(_z(6, 2, 136), _z(6, 2, 136), _z(6, 4, 136), d, [0, 6], 0.1),
                lambda: op(_z(6, 2, 0), _z(6, 2, 0), _z(6, 4, 0), d, [0, 6], 0.1)]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        op(q.float(), q, v, d, [0, 6], 0.1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        op(q, q, v, d, [0, 6], 0.1)
    for grad in (q.clone().requires_grad_(), d.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="causal_linear_packed is forward-only"):
            op(grad if grad.ndim == 3 else q, q, v, d if grad.ndim == 3 else grad, [0, 6], 0.1)
    with pytest.raises(RuntimeError, match="causal_linear_packed is forward-only"):
        op(q, q, v, d, [0, 6], 0.1, out=_z(6, 4, 64).requires_grad_())
    far = q[:1].expand(2 ** 32 + 6, 2, 64)
    with pytest.raises(ValueError, match="too large"):
        op(far, far, v[:1].expand(2 ** 32 + 6, 4, 64), d, [0, 6], 0.1)


def test_step_refusals(built_lib):
    from vdn_h3_amd.causal_linear import causal_linear_step as linear
    from vdn_h3_amd.gdn import gated_delta_step as delta

    q, v, pool = _z(3, 1, 2, 64), _z(3, 1, 4, 64), _f(5, 4, 64, 64)
    slots = torch.zeros(3, dtype=torch.int32)

    def both(q=q, k=None, v=v, d=None, pool=pool, slots=slots, out=None):
        k = q if k is None else k
        return [lambda: linear(q, k, v, _f(4) if d is None else d, pool, 0.1, slots=slots, out=out),
                lambda: delta(q, k, v, _f(3, 1, 4) if d is None else d, _f(3, 1, 4) if d is None else d, pool, slots=slots,
                              out=out)]

    for case in [both(q=_z(3, 2, 64)), both(k=_z(3, 1, 4, 64)), both(k=_z(2, 1, 2, 64)), both(v=_z(3, 2, 4, 64)),
                 both(v=_z(3, 1, 4, 32)), both(q=_z(3, 1, 3, 64), k=_z(3, 1, 3, 64)), both(d=_f(5)), both(d=_f(3, 1, 2)),
                 both(d=torch.zeros(4, dtype=torch.int32)), both(pool=_f(5, 4, 64, 32)), both(pool=_f(5, 2, 64, 64)),
                 both(pool=_f(4, 64, 64)), both(pool=_f(5, 4, 64, 64).transpose(2, 3)), both(pool=_f(5, 4, 64, 128)[..., :64]),
                 both(pool=_f(2, 4, 64, 64), slots=None), both(slots=slots[:2]), both(slots=slots.float()),
                 both(slots=slots[:, None]), both(out=_z(3, 1, 4, 32)), both(out=_f(3, 1, 4, 64)),
                 both(out=_z(3, 1, 4, 128)[..., ::2]), both(out=_z(3, 1, 1, 64).expand(3, 1, 4, 64)),
                 both(q=_z(3, 1, 2, 136), v=_z(3, 1, 4, 136), pool=_f(5, 4, 136, 136))]:
        for bad in case:
            with pytest.raises(ValueError):
                bad()
    for bad in both(pool=pool.half()) + both(q=q.float(), k=q) + both(slots=[0, 1, 2]):
        with pytest.raises(TypeError):
            bad()
    for good in both():
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            good()
    for bad in both(pool=pool.clone().requires_grad_()) + both(out=_z(3, 1, 4, 64).requires_grad_()):
        with pytest.raises(RuntimeError, match="forward-only"):
            bad()
    with pytest.raises(TypeError):
        linear(q, q, v, 0.5, pool, 0.1)


def test_adapter_refusals(built_lib):
    from vdn_h3_amd.adapters import LowRankAdapters

    for bad in [lambda: LowRankAdapters(_z(2, 8, 64), _z(3, 32, 8)), lambda: LowRankAdapters(_z(2, 8, 64), _z(2, 32, 4)),
                lambda: LowRankAdapters(_z(8, 64), _z(32, 8)), lambda: LowRankAdapters(_z(0, 8, 64), _z(0, 32, 8)),
                lambda: LowRankAdapters(_z(2, 8, 60), _z(2, 32, 8)), lambda: LowRankAdapters(_z(2, 8, 64), _z(2, 30, 8)),
                lambda: LowRankAdapters(_z(2, 8, 64), _z(2, 32, 8), [1.0]), lambda: LowRankAdapters(_z(1, 1032, 8), _z(1, 8, 1032)),
                lambda: LowRankAdapters.from_pairs([]), lambda: LowRankAdapters.from_pairs([(_z(8, 64), _z(32, 4))]),
                lambda: LowRankAdapters.from_pairs([(_z(8, 64), _z(32, 8)), (_z(8, 32), _z(32, 8))])]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        LowRankAdapters(_f(2, 8, 64), _z(2, 32, 8))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        LowRankAdapters(_z(2, 8, 64), _z(2, 32, 8))
    with pytest.raises(RuntimeError, match="forward-only"):
        LowRankAdapters(_z(2, 8, 64).requires_grad_(), _z(2, 32, 8))

    # a handle as __init__ leaves it, on the CPU: add refuses before it looks at the device
    handle = object.__new__(LowRankAdapters)
    handle.count, handle.rank, handle.width, handle.out_width = 2, 8, 64, 32
    handle.down = handle.up = _z(1)
    handle.scales = None
    y, x, index = _z(5, 32), _z(5, 64), torch.zeros(5, dtype=torch.int32)
    for bad in [lambda: handle.add(_z(4, 32), x, index), lambda: handle.add(y, _z(5, 32), index), lambda: handle.add(y, _z(64), index),
                lambda: handle.add(y, x, index[:4]), lambda: handle.add(y, x, index.float()), lambda: handle.add(y, x, [0] * 5),
                lambda: handle.add(y, x[:, None], index)]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        handle.add(y, x.float(), index)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        handle.add(y, x, index)
    with pytest.raises(RuntimeError, match="forward-only"):
        handle.add(y.clone().requires_grad_(), x, index)


def test_layouts_of_the_adapters():
    """Every number of A and B at the place that include/vdnh3.h gives it, zeros elsewhere."""
    from vdn_h3_amd.adapters import _layouts

    for n, rank, width, out in ((2, 8, 72, 40), (1, 16, 64, 32), (2, 24, 64, 8), (1, 40, 200, 72), (1, 100, 8, 64)):
        down = torch.arange(1, n * rank * width + 1).view(n, rank, width).double()
        up = torch.arange(1, n * out * rank + 1).view(n, out, rank).double()
        a, b = _layouts(down, up)
        ranks = 16 if rank <= 16 else -(-rank // 32) * 32
        assert a.shape == (n, -(-width // 64), ranks // 16, 2, 4, 16, 8) and a.count_nonzero() == down.numel()
        for i in range(n):
            for r in range(rank):
                for c in (0, 7, width // 2, width - 1):
                    assert a[i, c // 64, r // 16, c % 64 // 32, c % 32 // 8, r % 16, c % 8] == down[i, r, c]
            for c in range(out):
                m, t = (c % 32 // 8, c % 4), c % 8 // 4
                for r in (0, rank // 2, rank - 1):
                    at = b[(i, c // 32, r // 4, *m, t, r % 4) if ranks == 16 else (i, c // 32, r // 32, t, r % 32 // 8, *m, r % 8)]
                    assert at == up[i, c, r]
        assert b.count_nonzero() == up.numel()


def test_c_entry_points_refuse_before_any_launch(built_lib):
    """Null and misaligned operands, sizes that the kernels do not take: a status, never a launch."""
    from vdn_h3_amd import _lib

    lib, p = _lib.lib(), 1 << 20  # an address that is never read

    def packed(q=p, q_row=128, k=p, v=p, v_head=64, out=p, o_row=256, decay=p, cu=p, initial=p, final=p, n=1, rows=4, h=4, kh=2,
               dim=64, scale=0.1, ranges=1, work=None, size=0):
        return lib.vdnh3_causal_linear_packed(q, q_row, 64, k, 128, 64, v, 256, v_head, out, o_row, 64, decay, cu, initial, final,
                                              n, rows, h, kh, dim, scale, ranges, work, size, None)

    need = lib.vdnh3_causal_linear_workspace_bytes(3, 4, 64)
    assert need >= 3 * 4 * 64 * 64 * 4 and lib.vdnh3_causal_linear_workspace_bytes(1, 4, 64) == 0
    for bad in [dict(q=None), dict(q=p + 8), dict(q_row=100), dict(q_row=(1 << 23) + 8), dict(k=None), dict(v=p + 2),
                dict(v_head=-64), dict(out=None), dict(o_row=12), dict(decay=None), dict(cu=None), dict(initial=p + 4),
                dict(final=p + 8), dict(n=0), dict(rows=0), dict(h=5), dict(kh=0), dict(h=0), dict(dim=80),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(ranges=0), dict(ranges=3), dict(ranges=3, work=p, size=need - 1),
                dict(ranges=3, work=p + 8, size=need), dict(rows=(1 << 31) - 1, n=(1 << 31) - 1)]:
        assert packed(**bad) == _lib.VDNH3_ERR_INVALID, bad
        assert "causal_linear" in _lib.last_error()
    assert packed(ranges=1 << 20, h=64, kh=64, work=p, size=1 << 62) == _lib.VDNH3_ERR_INVALID and "too many" in _lib.last_error()

    names = [a + b for a in "qkvo" for b in ("_batch", "_row", "_head")] + ["slot", "state_head"] + \
        [a + b for a in ("beta", "g") for b in ("_batch", "_row", "_head")] + ["slots", "batch", "new", "heads", "qk_heads", "dim"]
    base = dict.fromkeys(names, 256) | dict(slot=4 * 4096, state_head=4096, slots=3, batch=2, new=1, heads=4, qk_heads=2, dim=64)

    def step(delta, q=p, k=p, v=p, out=p, beta=p, decay=p, pool=p, slots=p, scale=0.1, layout=True, **sizes):
        values = (ctypes.c_int64 * 26)(*(base | sizes).values()) if layout else None
        if delta:
            return lib.vdnh3_gated_delta_step(q, k, v, out, beta, decay, pool, slots, values, None)
        return lib.vdnh3_causal_linear_step(q, k, v, out, decay, pool, slots, values, scale, None)

    for bad in [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(decay=None), dict(pool=None), dict(layout=False),
                dict(slots=0), dict(batch=0), dict(new=0), dict(heads=0), dict(qk_heads=0), dict(dim=0), dict(dim=129), dict(heads=5),
                dict(batch=1 << 31), dict(new=1 << 40), dict(slot=4096), dict(state_head=4095), dict(slot=0), dict(state_head=0),
                dict(slot=4 * 4096 - 1), dict(batch=1 << 30, heads=1 << 10),
                dict(heads=1 << 30, qk_heads=1, state_head=4096, slot=1 << 60)]:
        for delta in (False, True):
            sizes = dict(bad)
            if sizes.get("slots") == 0:
                sizes = dict(sizes, slots=p)
                values = base | dict(slots=0)
                layout = (ctypes.c_int64 * 26)(*values.values())
                rc = (lib.vdnh3_gated_delta_step(p, p, p, p, p, p, p, p, layout, None) if delta else
                      lib.vdnh3_causal_linear_step(p, p, p, p, p, p, p, layout, 0.1, None))
            else:
                rc = step(delta, **sizes)
            assert rc == _lib.VDNH3_ERR_INVALID, bad
            assert ("gated_delta_step" if delta else "causal_linear_step") in _lib.last_error()
    assert step(True, beta=None) == _lib.VDNH3_ERR_INVALID
    assert step(False, scale=float("inf")) == _lib.VDNH3_ERR_INVALID
    assert step(False, slots=None, batch=4) == _lib.VDNH3_ERR_INVALID and "need a state each" in _lib.last_error()

    def add(y=p, y_row=64, x=p, x_row=128, down=p, up=p, index=p, out=p, out_row=64, rows=200, width=128, out_width=64, n=2, rank=8,
            work=p, size=1 << 30):
        return lib.vdnh3_adapter_add(y, y_row, x, x_row, down, up, None, index, out, out_row, rows, width, out_width, n, rank, work,
                                     size, None)

    need = lib.vdnh3_adapter_workspace_bytes(200, 40)
    assert need == 200 * 64 * 4 and lib.vdnh3_adapter_workspace_bytes(64, 64) == 0 and lib.vdnh3_adapter_workspace_bytes(0, 8) == 0
    for bad in [dict(y=None), dict(y=p + 8), dict(y_row=60), dict(y_row=-64), dict(x=p + 2), dict(x_row=-8), dict(down=None),
                dict(down=p + 8), dict(up=p + 8), dict(index=None), dict(out=None), dict(out=p + 16, out_row=0), dict(out_row=128),
                dict(rows=0), dict(width=0), dict(width=124), dict(out_width=60), dict(n=0), dict(rank=0), dict(rank=1025),
                dict(work=None), dict(work=p + 8), dict(rank=40, size=need - 1)]:
        assert add(**bad) == _lib.VDNH3_ERR_INVALID, bad
        assert "adapter_add" in _lib.last_error()
    assert add(rows=(1 << 31) - 64, size=1 << 62) == _lib.VDNH3_ERR_INVALID and "too many" in _lib.last_error()


def test_ranges_of_a_call(built_lib):
    """The host's rule: one round of workgroups, two chunks of each or more, and nothing for sizes that are none."""
    from vdn_h3_amd import _lib

    lib = _lib.lib()
    assert lib.vdnh3_causal_linear_ranges(77, 1, 40, 128) == 1
    assert lib.vdnh3_causal_linear_ranges(512, 1, 40, 128) == 4
    assert lib.vdnh3_causal_linear_ranges(40688, 1, 40, 128) == 6
    assert lib.vdnh3_causal_linear_ranges(500, 500, 40, 128) == 6
    assert lib.vdnh3_causal_linear_ranges(8000, 1, 56, 64) == 9
    assert lib.vdnh3_causal_linear_ranges(8000, 1, 1000, 128) == 1
    for bad in [(0, 1, 1, 64), (1, 0, 1, 64), (1, 1, 0, 64), (1, 1, 1, 80)]:
        assert lib.vdnh3_causal_linear_ranges(*bad) == 0


def test_sizes_at_the_end_of_32_bits_are_refused(built_lib):
    """Block counts of the largest rows and widths that a call can name: a status, not a launch of a count that wrapped around."""
    from vdn_h3_amd import _lib
    from vdn_h3_amd.adapters import LowRankAdapters

    lib, p = _lib.lib(), 1 << 20  # an address that is never read

    def add(rows=200, width=128, out_width=64, n=2, rank=8):
        return lib.vdnh3_adapter_add(p, out_width, p, width, p, p, None, p, p, out_width, rows, width, out_width, n, rank, p,
                                     1 << 62, None)

    top = (1 << 31) - 1
    for bad in [dict(rows=top), dict(rows=top - 62), dict(rows=top, rank=1024), dict(out_width=top - 7), dict(width=top - 7),
                dict(rows=1, out_width=top - 7), dict(rows=top, out_width=top - 7, n=top)]:
        assert add(**bad) == _lib.VDNH3_ERR_INVALID, bad
        assert "adapter_add" in _lib.last_error()
    assert lib.vdnh3_causal_linear_ranges(top, top, 1, 64) == 512  # chunks counted past 32 bits
    one = _z(1)
    for width, out in ((2 ** 30 + 8, 8), (8, 2 ** 30 + 8)):
        with pytest.raises(ValueError, match="widths"):
            LowRankAdapters(one.expand(1, 1, width), one.expand(1, out, 1))


def test_launches_of_the_adapters(built_lib):
    """The workspace that a call wants says which form it takes: one launch (none) for few rows, two where many rows of wide x fall
    to few adapters."""
    from vdn_h3_amd import _lib

    lib = _lib.lib()
    want = lib.vdnh3_adapter_workspace_wanted
    for rows, width, adapters in ((1, 5120, 1), (16, 2 ** 20, 1), (32, 5120, 1), (64, 2560, 1), (64, 5120, 2), (64, 5120, 16),
                                  (64, 13824, 16), (17, 9600, 1), (33, 5120, 2 ** 31 - 1)):
        assert want(rows, width, adapters, 64) == 0, (rows, width, adapters)
    for rows, width, adapters in ((33, 5120, 1), (64, 5120, 1), (64, 2568, 1), (24, 13824, 1), (48, 13824, 4), (64, 5128, 2),
                                  (64, 2 ** 30, 64)):
        assert want(rows, width, adapters, 8) == rows * 16 * 4 and want(rows, width, adapters, 40) == rows * 64 * 4
    for rows, rank in ((65, 8), (200, 40), (1, 65), (64, 1024)):  # what a call needs, it wants
        assert want(rows, 64, 3, rank) == lib.vdnh3_adapter_workspace_bytes(rows, rank) > 0
    for bad in ((0, 64, 1, 8), (8, 0, 1, 8), (8, 64, 0, 8), (8, 64, 1, 0), (8, 64, 1, 1025)):
        assert want(*bad) == 0
