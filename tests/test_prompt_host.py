"""Refusals of the prompt encoder's operators, which need no GPU: arguments are checked before any device work."""

from __future__ import annotations

import pytest
import torch

BF = torch.bfloat16


def _z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def test_norm_refusals(built_lib):
    from vdn_h3_amd import linear
    from vdn_h3_amd.block_kernels import residual_rmsnorm_quantize as op

    x, w = _z(4, 64), _z(64)
    for bad in [lambda: op(_z(4, 64, dtype=torch.float32), x, w, 1e-6, 1), lambda: op(_z(64), None, w, 1e-6, 1),
                lambda: op(x, _z(3, 64), w, 1e-6, 1), lambda: op(x, x.float(), w, 1e-6, 1),
                lambda: op(x, x, _z(32), 1e-6, 1), lambda: op(_z(4, 60), None, _z(60), 1e-6, 1),
                lambda: op(_z(4, 0), None, _z(0), 1e-6, 1), lambda: op(x, x, w, 1e-6, 3),
                lambda: op(x, None, w, 1e-6, 1, sum_out=_z(4, 64)), lambda: op(x, x, w, 1e-6, 1, sum_out=_z(4, 128)[:, ::2]),
                lambda: op(x, x, w, 1e-6, 1, sum_out=x[:1].expand(4, 64))]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        op(x, x, w, 1e-6, linear.KIND_I8)
    with pytest.raises(RuntimeError, match="residual_rmsnorm_quantize is forward-only"):
        op(x, x.clone().requires_grad_(), w, 1e-6, linear.KIND_I8)
    with pytest.raises(RuntimeError, match="residual_rmsnorm_quantize is forward-only"):
        op(x, x, w, 1e-6, linear.KIND_I8, sum_out=_z(4, 64).requires_grad_())
    with pytest.raises(ValueError, match="too large"):
        op(x[:1].expand(2 ** 31, 64), None, w, 1e-6, 1)


def test_rotary_refusals(built_lib):
    from vdn_h3_amd.rotary import RotaryAxes, normalise_qk_axes as op

    for bad in [lambda: RotaryAxes(()), lambda: RotaryAxes((0, 0)), lambda: RotaryAxes((9, -1)), lambda: RotaryAxes((3, 2)),
                lambda: RotaryAxes((8,), theta=0.0), lambda: RotaryAxes((8,), theta=float("inf")),
                lambda: RotaryAxes((8,), ladder="other")]:
        with pytest.raises(ValueError):
            bad()
    axes = RotaryAxes((8, 12, 12))
    assert axes.rot_dim == 64 and axes.axes == 3
    q, k, pos = _z(5, 4, 64), _z(5, 2, 64), torch.zeros(3, 5, dtype=torch.int64)
    for bad in [lambda: op(q, _z(4, 2, 64), pos, axes), lambda: op(q, _z(5, 2, 128), pos, axes),
                lambda: op(q[0], k, pos, axes)]:
        with pytest.raises(ValueError):
            bad()
    for bad in [lambda: op(q.float(), k, pos, axes)]:
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        op(q, k, pos, axes)
    with pytest.raises(ValueError, match="too large"):
        op(q[:1].expand(2 ** 32 + 5, 4, 64), k[:1].expand(2 ** 32 + 5, 2, 64), pos[:, :1].expand(3, 2 ** 32 + 5), axes)
    with pytest.raises(RuntimeError, match="normalise_qk_axes is forward-only"):
        op(q.requires_grad_(), k, pos, axes)


def test_attention_refusals(built_lib):
    from vdn_h3_amd.causal import causal_softmax_cached as cached, causal_softmax_packed as packed

    q, k = _z(6, 4, 64), _z(6, 2, 64)
    for bad in [lambda: packed(q, _z(5, 2, 64), _z(5, 2, 64), [0, 6], 0.1), lambda: packed(q, k, _z(6, 4, 64), [0, 6], 0.1),
                lambda: packed(q, _z(6, 3, 64), _z(6, 3, 64), [0, 6], 0.1), lambda: packed(q, k[..., :32], k[..., :32], [0, 6], 1),
                lambda: packed(q, _z(6, 0, 64), _z(6, 0, 64), [0, 6], 0.1), lambda: packed(q[0], k, k, [0, 6], 0.1)]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        packed(q, k.float(), k.float(), [0, 6], 0.1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        packed(q, k, k, [0, 6], 0.1)
    with pytest.raises(RuntimeError, match="causal_softmax_packed is forward-only"):
        packed(q.clone().requires_grad_(), k, k, [0, 6], 0.1)
    with pytest.raises(RuntimeError, match="causal_softmax_packed is forward-only"):
        packed(q, k, k, [0, 6], 0.1, out=_z(6, 4, 64).requires_grad_())
    far, near = q[:1].expand(2 ** 32 + 6, 4, 64), k[:1].expand(2 ** 32 + 6, 2, 64)
    with pytest.raises(ValueError, match="too large"):
        packed(far, near, near, [0, 6], 0.1)
    q, k, n = _z(2, 1, 4, 64), _z(2, 9, 2, 64), torch.zeros(2, dtype=torch.int32)
    for bad in [lambda: cached(q, k[:1], k[:1], n, 0.1), lambda: cached(q, k, _z(2, 8, 2, 64), n, 0.1),
                lambda: cached(q, k, k, n[:1], 0.1), lambda: cached(q, k, k, n.float(), 0.1),
                lambda: cached(_z(2, 1, 3, 64), k, k, n, 0.1), lambda: cached(_z(2, 1, 4, 80), _z(2, 9, 2, 80), _z(2, 9, 2, 80), n, 0.1)]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cached(q, k, k, n, 0.1)
    with pytest.raises(RuntimeError, match="causal_softmax_cached is forward-only"):
        cached(q, k.clone().requires_grad_(), k, n, 0.1)
    far = k[:, :1].expand(2, 2 ** 32 + 9, 2, 64)
    with pytest.raises(ValueError, match="too large"):
        cached(q, far, far, n, 0.1)


def test_bounds_that_the_host_holds_are_checked():
    from vdn_h3_amd.causal import _sequence_bounds

    device = torch.device("cuda:0")
    for bad in ([0, 7], [-1, 3], [0, 4, 3], [], torch.tensor([0.0, 3.0]), [0, 2.5], [False, True],
                torch.tensor([[0, 3]]), torch.tensor([0, 9])):
        with pytest.raises(ValueError):
            _sequence_bounds(bad, 6, device)


def test_c_entry_points_refuse_before_any_launch(built_lib):
    """Null and misaligned operands, sizes that the kernels do not take: a status, never a launch."""
    from vdn_h3_amd import _lib

    lib, p = _lib.lib(), 1 << 20  # an address that is never read

    def norm(kind=1, x=p, x_row=64, res=p, res_row=64, w=p, eps=1e-6, rows=4, hidden=64, out=p, out_row=64, scale=p, s=p,
             s_row=64):
        return lib.vdnh3_residual_rmsnorm_quant_rows(kind, x, x_row, res, res_row, w, eps, rows, hidden, out, out_row, scale, s,
                                                     s_row, None)

    for bad in [dict(kind=3), dict(kind=-1), dict(x=None), dict(x=p + 8), dict(x_row=60), dict(x_row=8), dict(res=p + 2),
                dict(w=None), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(rows=0), dict(hidden=0),
                dict(hidden=60), dict(out=None), dict(out=p + 4), dict(out_row=32), dict(scale=None), dict(s=p + 8),
                dict(s_row=0), dict(kind=0, out=p + 8)]:
        assert norm(**bad) == _lib.VDNH3_ERR_INVALID, bad
        assert "residual_rmsnorm" in _lib.last_error()

    def rotary(q=p, q_row=256, qh=4, out=p, kh=2, pos=p, kind=1, turns=p, axis=p, rot=64, rows=3, dim=64, w=None):
        return lib.vdnh3_qk_rotary_axes(q, q_row, 64, w, 1e-6, out, 256, 64, qh, p, 128, 64, None, 1e-6, p, 128, 64, kh, pos,
                                        kind, 3, 1, turns, axis, rot, rows, dim, None)

    for bad in [dict(q=None), dict(q=p + 8), dict(q_row=100), dict(qh=0), dict(out=None), dict(kh=0), dict(pos=None),
                dict(kind=3), dict(turns=None), dict(axis=None), dict(rot=0), dict(rot=24), dict(rot=80), dict(rows=0),
                dict(dim=60), dict(dim=136), dict(w=p + 2)]:
        assert rotary(**bad) == _lib.VDNH3_ERR_INVALID, bad

    def far_rotary():
        return lib.vdnh3_qk_rotary_axes(p, 256, 64, None, float("nan"), p, 256, 64, 4, p, 128, 64, None, 1e-6, p, 128, 64, 2, p,
                                        1, 3, 1, p, p, 64, 3, 64, None)

    assert far_rotary() == _lib.VDNH3_ERR_INVALID and "eps" in _lib.last_error()
    # more threads than a launch holds
    assert norm(rows=1 << 24) == _lib.VDNH3_ERR_INVALID and "too many" in _lib.last_error()
    assert rotary(rows=1 << 26) == _lib.VDNH3_ERR_INVALID and "too many" in _lib.last_error()

    def packed(q=p, q_row=256, k=p, out=p, cu=p, n=1, rows=4, h=4, kh=2, dim=64, scale=0.1):
        return lib.vdnh3_causal_attn_packed(q, q_row, 64, k, 128, 64, p, 128, 64, out, 256, 64, cu, n, rows, h, kh, dim, scale,
                                            None)

    for bad in [dict(q=None), dict(q=p + 8), dict(q_row=100), dict(k=None), dict(out=p + 8), dict(cu=None), dict(n=0),
                dict(rows=0), dict(h=5), dict(kh=0), dict(h=0), dict(dim=80), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("nan")), dict(scale=float("inf"))]:
        assert packed(**bad) == _lib.VDNH3_ERR_INVALID, bad
    assert packed(rows=1 << 30, h=64, kh=2) == _lib.VDNH3_ERR_INVALID and "too many" in _lib.last_error()
    assert packed(rows=1 << 26, h=64, kh=64, n=1 << 23) == _lib.VDNH3_ERR_INVALID and "too many" in _lib.last_error()

    def cached(q=p, k=p, k_row=128, lengths=p, batch=2, new=1, room=64, h=4, kh=2, dim=64, scale=0.1, ranges=0, part=None,
               size=0):
        return lib.vdnh3_causal_attn_cached(q, 256, 256, 64, k, 8192, k_row, 64, p, 8192, 128, 64, p, 256, 256, 64, lengths,
                                            batch, new, room, h, kh, dim, scale, ranges, part, size, None)

    for bad in [dict(q=None), dict(k=p + 2), dict(k_row=(1 << 23) + 8), dict(k_row=-8), dict(lengths=None), dict(batch=0),
                dict(new=0), dict(room=0), dict(h=3), dict(dim=96), dict(scale=float("inf")), dict(ranges=-1),
                dict(ranges=2), dict(ranges=2, part=p, size=8), dict(ranges=2, part=p + 8, size=1 << 20),
                dict(room=(1 << 31) - 1), dict(ranges=2, room=(1 << 31) - 100),
                dict(batch=1 << 30, new=1 << 20, h=1 << 10, kh=1 << 10),
                dict(ranges=1, batch=1 << 30, new=1 << 30, h=1 << 10, kh=1 << 10), dict(ranges=1, batch=1 << 20, new=1 << 12),
                dict(ranges=1, batch=1 << 16, room=1 << 25)]:
        assert cached(**bad) == _lib.VDNH3_ERR_INVALID, bad


def test_ranges_of_a_call(built_lib):
    """The host's rule: never more parts than the buffer's size counts, one range where one takes the caches, the prompt
    kernel (0) for many tokens over short caches, and nothing for sizes that are none."""
    from vdn_h3_amd import _lib

    lib = _lib.lib()
    assert lib.vdnh3_causal_cached_ranges(1, 1, 64, 40, 8, 128) <= 1
    assert lib.vdnh3_causal_cached_ranges(64, 1, 8192, 40, 8, 128) == 32
    assert lib.vdnh3_causal_cached_ranges(16, 64, 2048, 40, 8, 128) == 0
    assert lib.vdnh3_causal_cached_ranges(1, 32, 40960, 40, 8, 128) > 1
    for bad in [(0, 1, 1, 1, 1, 64), (1, 0, 1, 1, 1, 64), (1, 1, 0, 1, 1, 64), (1, 1, 1, 3, 2, 64), (1, 1, 1, 0, 1, 64),
                (1, 1, 1, 1, 0, 64), (1, 1, 1, 1, 1, 0), (1, 1, 2 ** 31 - 1, 4, 4, 64),
                (2 ** 31 - 1, 2 ** 31 - 1, 64, 2 ** 31 - 1, 1, 128)]:
        assert lib.vdnh3_causal_cached_ranges(*bad) == 0
    assert lib.vdnh3_causal_partial_bytes(3, 10, 64, 1) == 0
    assert lib.vdnh3_causal_partial_bytes(3, 10, 64, 4) == 4 * 2 * 30 * 66 * 4


def test_launch_makes_the_tensors_device_current(monkeypatch):
    from vdn_h3_amd import _lib

    entered = []

    class Guard:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            entered.append(self.device)

        def __exit__(self, *_):
            entered.append(None)

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(_lib, "stream_handle", lambda device: 77)
    seen = []

    def call(*args):
        seen.append((args, list(entered)))
        return 0

    _lib.launch("x", call, torch.device("cuda:0"), 1, 2)
    _lib.launch("x", call, torch.device("cuda:1"), 3)
    assert seen[0] == ((1, 2, 77), []) and seen[1] == ((3, 77), [torch.device("cuda:1")]) and entered[-1] is None


def test_scales_past_fp32_are_refused(built_lib):
    """The kernels take scale * log2(e): a finite scale whose product is none gave NaNs. Nothing is launched either way: the null
    bounds and lengths are refused behind the scale."""
    from vdn_h3_amd import _lib

    lib, p = _lib.lib(), 1 << 20
    for scale, word in ((3e38, "scale"), (2.4e38, "scale"), (2.3e38, "null")):
        assert lib.vdnh3_causal_attn_packed(p, 256, 64, p, 128, 64, p, 128, 64, p, 256, 64, None, 1, 4, 4, 2, 64, scale,
                                            None) == _lib.VDNH3_ERR_INVALID
        assert word in _lib.last_error(), (scale, _lib.last_error())
        assert lib.vdnh3_causal_attn_cached(p, 256, 256, 64, p, 8192, 128, 64, p, 8192, 128, 64, p, 256, 256, 64, None, 2, 1, 64, 4,
                                            2, 64, scale, 0, None, 0, None) == _lib.VDNH3_ERR_INVALID
        assert word in _lib.last_error(), (scale, _lib.last_error())


def test_attention_names_itself_where_it_refuses(built_lib):
    """Head dims that no kernel takes, and lengths that are no tensor."""
    from vdn_h3_amd.causal import causal_softmax_cached as cached, causal_softmax_packed as packed

    for dim in (0, 136):
        q, k = _z(6, 4, dim), _z(6, 2, dim)
        with pytest.raises(ValueError, match="causal_softmax_packed supports head dims"):
            packed(q, k, k, [0, 6], 0.1)
    q, k = _z(2, 1, 4, 64), _z(2, 9, 2, 64)
    for lengths in ([3, 4], 3, None):
        with pytest.raises(TypeError, match="lengths must be a tensor"):
            cached(q, k, k, lengths, 0.1)
