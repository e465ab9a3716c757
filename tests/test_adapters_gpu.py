"""Low-rank adapters of many requests against float64 (GPU).

Bar, from the arithmetic, relative to the absolute values of the terms (`size`, y among them): the products with A are fp32 sums
of `width` terms, width 2^-24; s A x is one product more and meets B as two bf16 numbers, 2^-16; the products with B are sums of
`rank` terms, 2 rank 2^-24, and the sum with y one more. The result is rounded once, 2^-8 of itself.
"""

from __future__ import annotations

import pytest
import torch

from oracle import recurrent_oracle as ro

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _case(rows, width, out, n, rank, device, seed=0):
    g = torch.Generator().manual_seed(rows + width + seed)
    x, y = torch.randn(rows, width, generator=g).to(BF), torch.randn(rows, out, generator=g).to(BF)
    down = (torch.randn(n, rank, width, generator=g) * width ** -0.5).to(BF)
    up = torch.randn(n, out, rank, generator=g).to(BF)
    return [t.to(device) for t in (x, y, down, up, torch.rand(n, generator=g) - 0.3)], g


def _check(got, x, y, down, up, scales, index):
    want, size = ro.adapters(y, x, down, up, scales if scales is not None else [1.0] * down.shape[0], index)
    bar = ((x.shape[1] + 2 * down.shape[1] + 8) * 2.0 ** -24 + 2.0 ** -16) * size + 2.0 ** -8 * want.abs()
    d = (got.double() - want).abs()
    assert (d <= bar).all(), (d / bar.clamp_min(1e-30)).max()
    none = (index < 0) | (index >= down.shape[0])
    assert torch.equal(got[none], y[none])


def _runs(rows, lengths, choices):
    index = torch.full((rows,), -1, dtype=torch.int32)
    at = 0
    for n, c in zip(lengths, choices):
        index[at:at + n] = c
        at += n
    return index


CASES = [  # rows, width, out, adapters, rank
    (1, 64, 64, 1, 8), (1, 5120, 640, 8, 16), (3, 8, 8, 2, 8), (17, 136, 264, 3, 16), (64, 512, 512, 16, 16), (65, 1000, 72, 70, 8),
    (130, 256, 1032, 4, 24), (200, 2048, 256, 3, 64), (333, 640, 320, 5, 40), (64, 384, 128, 2, 128), (100, 256, 64, 3, 136),
    (70, 128, 64, 2, 264), (20000, 64, 64, 3, 32), (48, 5120, 64, 2, 48)]


@pytest.mark.parametrize("rows,width,out,n,rank", CASES)
def test_against_float64(device, rows, width, out, n, rank):
    from vdn_h3_amd.adapters import LowRankAdapters

    print(f"case adapters {rows} x {width} -> {out}, {n} of rank {rank}", flush=True)
    (x, y, down, up, scales), g = _case(rows, width, out, n, rank, device)
    handle = LowRankAdapters(down, up, scales)
    any_order = torch.randint(-1, n + 1, (rows,), generator=g, dtype=torch.int32)
    runs = torch.randint(-1, n, (rows,), generator=g, dtype=torch.int32).sort()[0]
    same = torch.full((rows,), n - 1, dtype=torch.int32)
    none = torch.full((rows,), -1, dtype=torch.int32)
    for index in (any_order, runs, same, none):
        index = index.to(device)
        got = handle.add(y, x, index)
        _check(got, x, y, down, up, scales, index)
        again = y.clone()
        assert handle.add(again, x, index.long(), out=again) is again and torch.equal(again, got)
    # views: columns of wider matrices, off 16 bytes, one row for all
    wide_x = torch.cat([x, x], 1)[:, width:]
    wide_y = torch.cat([y, y], 1)[:, :out]
    off = torch.empty(x.numel() + 1, dtype=BF, device=device)[1:].view_as(x).copy_(x)
    index = any_order.to(device)
    got = handle.add(y, x, index)
    for args in ((wide_y, wide_x), (y, off)):
        assert torch.equal(handle.add(*args, index), got)
    to = torch.full((rows, out + 8), 7.0, dtype=BF, device=device)
    assert torch.equal(handle.add(y, x, index, out=to[:, :out]), got) and (to[:, out:] == 7).all()
    one = handle.add(y[:1].expand(rows, out), x[:1].expand(rows, width), index)
    assert torch.equal(one, handle.add(y[:1].expand(rows, out).contiguous(), x[:1].expand(rows, width).contiguous(), index))


def test_ranks_scales_and_pairs(device):
    from vdn_h3_amd.adapters import LowRankAdapters

    (x, y, down, up, scales), g = _case(50, 128, 96, 3, 12, device)
    index = torch.randint(0, 3, (50,), generator=g).to(device)
    _check(LowRankAdapters(down, up).add(y, x, index), x, y, down, up, None, index)
    _check(LowRankAdapters(down, up, scales.tolist()).add(y, x, index), x, y, down, up, scales, index)
    _check(LowRankAdapters(down, up, scales.double().cpu()).add(y, x, index), x, y, down, up, scales, index)
    lone = LowRankAdapters.from_pairs([(down[0], up[0]), (down[1, :5], up[1, :, :5]), (down[2, :1], up[2, :, :1])], scales)
    down, up = down.clone(), up.clone()
    down[1, 5:], down[2, 1:], up[1, :, 5:], up[2, :, 1:] = 0, 0, 0, 0
    _check(lone.add(y, x, index), x, y, down, up, scales, index)
    turned = LowRankAdapters(down.transpose(1, 2).contiguous().transpose(1, 2), up, scales)
    assert torch.equal(turned.add(y, x, index), lone.add(y, x, index))


def test_a_row_keeps_to_itself(device):
    """Infinities and NaN of a row, or of an adapter that others use, stay there."""
    from vdn_h3_amd.adapters import LowRankAdapters

    (x, y, down, up, scales), g = _case(90, 256, 128, 4, 16, device)
    index = torch.randint(0, 3, (90,), generator=g, dtype=torch.int32).to(device)
    index[7] = 3
    want = LowRankAdapters(down, up, scales).add(y, x, index)
    for value in (torch.inf, torch.nan):
        bad = x.clone()
        bad[11, 5] = value
        got = LowRankAdapters(down, up, scales).add(y, bad, index)
        assert not got[11].isfinite().any() and torch.equal(got[:11], want[:11]) and torch.equal(got[12:], want[12:])
        poisoned = down.clone()
        poisoned[3] = value
        got = LowRankAdapters(poisoned, up, scales).add(y, x, index)
        assert not got[7].isfinite().any()
        got[7] = want[7]
        assert torch.equal(got, want)


def test_beside_a_projection(device):
    from vdn_h3_amd.adapters import LowRankAdapters
    from vdn_h3_amd.linear import HipLinear

    (x, _, down, up, scales), g = _case(77, 256, 384, 3, 16, device)
    weight = (torch.randn(384, 256, generator=g) / 16).to(BF).to(device)
    index = torch.randint(-1, 3, (77,), generator=g, dtype=torch.int32).to(device)
    handle = LowRankAdapters(down, up, scales)
    for precision in ("bf16", "int8", "fp8"):
        layer = HipLinear(weight, precision)
        base = layer(x)
        got = layer(x, adapters=handle, adapter_index=index)
        assert torch.equal(got, handle.add(base, x, index))
        out = torch.zeros(77, 384, dtype=BF, device=device)
        assert layer(x.float(), out=out, adapters=handle, adapter_index=index) is out and torch.equal(out, got)
        with pytest.raises(ValueError):
            layer(x, out=out, accumulate=True, adapters=handle, adapter_index=index)
        with pytest.raises(ValueError):
            layer(x, adapter_index=index)


def test_replays_take_another_index(device):
    from vdn_h3_amd.adapters import LowRankAdapters

    (x, y, down, up, scales), g = _case(40, 512, 256, 5, 16, device)
    index = torch.zeros(40, dtype=torch.int32, device=device)
    handle, out = LowRankAdapters(down, up, scales), torch.zeros_like(y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        handle.add(y, x, index, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        handle.add(y, x, index, out=out)
    for seed in range(4):
        index.copy_(torch.randint(-1, 6, (40,), generator=g, dtype=torch.int32))
        x.add_(0.25)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, handle.add(y, x, index))


def test_layouts_of_rows_and_kept_scales(device):
    """Rows that overlap or lie far apart (past 32 bits), one row with any stride; the object keeps the scales that it was given."""
    from vdn_h3_amd.adapters import LowRankAdapters

    (x, y, down, up, scales), g = _case(70, 256, 128, 3, 40, device)
    index = torch.randint(-1, 3, (70,), generator=g, dtype=torch.int32).to(device)
    handle = LowRankAdapters(down, up, scales)
    want = handle.add(y, x, index)
    scales.zero_()
    assert torch.equal(handle.add(y, x, index), want)
    sliding = x.flatten().as_strided((70, 256), (8, 1))
    assert torch.equal(handle.add(y, sliding, index), handle.add(y, sliding.contiguous(), index))
    room = torch.empty(70 * 2 ** 25 + 256, dtype=BF, device=device)
    far_x, far_y = room.as_strided((70, 256), (2 ** 25, 1)), room.as_strided((70, 128), (2 ** 25, 1), 512)
    far_x.copy_(x)
    far_y.copy_(y)
    assert torch.equal(handle.add(far_y, far_x, index), want) and handle.add(far_y, far_x, index, out=far_y) is far_y
    assert torch.equal(far_y, want) and torch.equal(far_x, x)
    one = x.flatten()[:300].as_strided((1, 256), (3, 1))
    assert torch.equal(handle.add(y[:1].as_strided((1, 128), (1, 1)), one, index[:1]), handle.add(y[:1], one.clone(), index[:1]))


def test_a_projection_refuses_adapters_of_another(device):
    """Before anything is written."""
    from vdn_h3_amd.adapters import LowRankAdapters
    from vdn_h3_amd.linear import HipLinear

    (x, _, down, up, scales), _ = _case(9, 256, 128, 3, 16, device)
    layer, out = HipLinear(torch.zeros(128, 256, dtype=BF, device=device)), torch.full((9, 128), 7.0, dtype=BF, device=device)
    index = torch.zeros(9, dtype=torch.int32, device=device)
    for handle, at in ((LowRankAdapters(down[..., :128], up), index), (LowRankAdapters(down, up[:, :64]), index),
                       (LowRankAdapters(down, up), None)):
        with pytest.raises(ValueError):
            layer(x, out=out, adapters=handle, adapter_index=at)
    assert (out == 7.0).all()


@pytest.mark.parametrize("precision", ["bf16", "int8", "fp8"])
def test_a_projection_refuses_operands_of_its_adapters(device, precision):
    """An index or an output that the adapters do not take: before anything is written."""
    from vdn_h3_amd.adapters import LowRankAdapters
    from vdn_h3_amd.linear import HipLinear

    (x, _, down, up, scales), _ = _case(9, 256, 128, 3, 16, device)
    layer, handle = HipLinear(torch.zeros(128, 256, dtype=BF, device=device), precision), LowRankAdapters(down, up, scales)
    room = torch.full((9 * 200,), 7.0, device=device)
    good, wide = room.to(BF)[:9 * 128].view(9, 128), room.to(BF)
    index = torch.zeros(9, dtype=torch.int32, device=device)
    at = dict(x=x, out=good, adapter_index=index)
    for error, change in [(ValueError, dict(adapter_index=index[:8])), (ValueError, dict(adapter_index=index[:, None])),
                          (ValueError, dict(adapter_index=index.float())), (ValueError, dict(adapter_index=[0] * 9)),
                          (RuntimeError, dict(adapter_index=index.cpu())), (TypeError, dict(out=room[:9 * 128].view(9, 128))),
                          (ValueError, dict(out=wide[1:1 + 9 * 128].view(9, 128))),
                          (ValueError, dict(out=wide.as_strided((9, 128), (132, 1)))),
                          (ValueError, dict(out=wide.as_strided((9, 128), (64, 1)))), (ValueError, dict(out=good[:8])),
                          (ValueError, dict(x=x[:8])), (ValueError, dict(x=x[:, :128]))]:
        with pytest.raises(error):
            layer(adapters=handle, **(at | change))
        assert (change.get("out", good) == 7.0).all() and (good == 7.0).all(), change
    with pytest.raises(RuntimeError, match="forward-only"):
        layer(adapters=handle, **(at | dict(out=good.clone().requires_grad_())))
    assert layer(adapters=handle, **at) is good
    assert torch.equal(good, layer(x, adapters=handle, adapter_index=index))


@pytest.mark.parametrize("rows", [24, 200])
@pytest.mark.parametrize("width,rank", [(64, 1), (72, 1), (64, 8), (136, 16), (256, 24), (264, 40), (72, 64), (520, 136)])
def test_infinities_of_x(device, rows, width, rank):
    """An infinite channel of x gives the infinities of the formula: neither the second number of s A x nor the channels and ranks
    that the kernels add make a NaN of them. With one rank the signs are any, with more all are positive (else it is inf - inf)."""
    from vdn_h3_amd.adapters import LowRankAdapters

    (x, y, down, up, scales), _ = _case(rows, width, 72, 3, rank, device)
    if rank > 1:
        down, up = down.abs() + 2.0 ** -10, up.abs() + 2.0 ** -10
    down, up, scales = torch.where(down == 0, 1.0, down).to(BF), torch.where(up == 0, 1.0, up).to(BF), scales.abs() + 0.1
    index = (torch.arange(rows, device=device, dtype=torch.int32) % 4) - 1
    plain = LowRankAdapters(down, up, scales).add(y, x, index)
    bad = x.clone()
    places = [(0, torch.inf), (width - 1, torch.inf), (width // 2, -torch.inf), (width - 8, -torch.inf), (width - 3, torch.nan),
              (5, torch.inf)]
    for row, (channel, value) in enumerate(places):
        bad[3 * row + 1, channel] = value
    got = LowRankAdapters(down, up, scales).add(y, bad, index)
    want, _ = ro.adapters(y, bad, down, up, scales, index)
    touched = ~bad.isfinite().all(1) & (index >= 0)
    assert touched.sum() >= 4 and torch.equal(got[~touched], plain[~touched])
    assert torch.equal(got[touched].isnan(), want[touched].isnan()) and not got[touched].isfinite().any()
    assert torch.equal(torch.nan_to_num(got[touched].double(), 0.0, 1.0, -1.0), torch.nan_to_num(want[touched], 0.0, 1.0, -1.0))


@pytest.mark.parametrize("rows,width,n,rank", [(33, 5120, 1, 16), (64, 5120, 1, 32), (64, 13824, 4, 64), (24, 13824, 1, 8)])
def test_one_launch_and_two_are_equal(device, rows, width, n, rank):
    """Calls of few rows with the workspace that they want, without one and with one off 16 bytes: the same bits."""
    from vdn_h3_amd import _lib
    from vdn_h3_amd.adapters import LowRankAdapters

    (x, y, down, up, scales), g = _case(rows, width, 264, n, rank, device)
    handle, lib = LowRankAdapters(down, up, scales), _lib.lib()
    index = torch.randint(-1, n, (rows,), generator=g, dtype=torch.int32).to(device)
    size = lib.vdnh3_adapter_workspace_wanted(rows, width, n, rank)
    assert size > 0 and lib.vdnh3_adapter_workspace_bytes(rows, rank) == 0
    got = handle.add(y, x, index)
    _check(got, x, y, down, up, scales, index)
    work = torch.zeros(size + 16, dtype=torch.uint8, device=device)
    for at, room, used in ((None, 0, False), (work.data_ptr(), size - 1, False), (work.data_ptr() + 8, size, False),
                           (work.data_ptr(), size, True)):
        out = torch.full_like(y, 7.0)
        _lib.check(lib.vdnh3_adapter_add(y.data_ptr(), 264, x.data_ptr(), width, handle.down.data_ptr(), handle.up.data_ptr(),
                                         handle.scales.data_ptr(), index.data_ptr(), out.data_ptr(), 264, rows, width, 264, n, rank,
                                         at, room, _lib.stream_handle(device)), "add")
        assert torch.equal(out, got) and work.any().item() == used


TALL = [  # rows, width, out, adapters, rank: blocks of 32 and 64 rows with every number of rank tiles, several steps of columns
    (9000, 64, 72, 3, 8), (9000, 72, 40, 3, 24), (9000, 64, 64, 4, 64), (9000, 136, 72, 2, 136), (17000, 64, 72, 3, 8),
    (17000, 72, 64, 3, 64), (17000, 64, 40, 2, 136), (64, 72, 8712, 16, 16), (63, 64, 8712, 17, 40), (64, 64, 8712, 16, 24),
    (16001, 64, 4104, 3, 8), (16001, 64, 4104, 2, 32), (16001, 64, 4104, 2, 40), (16001, 64, 4104, 2, 136)]


@pytest.mark.parametrize("rows,width,out,n,rank", TALL)
def test_blocks_and_steps_against_float64(device, rows, width, out, n, rank):
    from vdn_h3_amd.adapters import LowRankAdapters

    print(f"case adapters {rows} x {width} -> {out}, {n} of rank {rank}", flush=True)
    (x, y, down, up, scales), g = _case(rows, width, out, n, rank, device)
    handle = LowRankAdapters(down, up, scales)
    any_order = torch.randint(-1, n + 1, (rows,), generator=g, dtype=torch.int32)
    few = torch.where(torch.rand(rows, generator=g) < 0.3, any_order, -1)  # fewer than 16 rows of each in a block
    half = torch.where(torch.arange(rows) % 64 < 20, any_order, n - 1)  # up to 64 of the last, few of the others
    runs = torch.randint(-1, n, (rows,), generator=g, dtype=torch.int32).sort()[0]
    for index in (any_order, few, half, runs):
        index = index.to(torch.int32).to(device)
        got = handle.add(y, x, index)
        _check(got, x, y, down, up, scales, index)
        again = y.clone()
        assert handle.add(again, x, index, out=again) is again and torch.equal(again, got)
