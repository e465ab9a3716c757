"""q / k RMSNorm and rotary positions on several axes against float64 (GPU).

Bar (u = 2^-24): the normalised channels y_i, y_{i+h} of a pair are off by at most 24 u of themselves (the sum over at most
128 squares in chains of 8 and a tree of 4, root, quotient, two products). The fraction of a turn is rounded to fp32 (2 pi
2^-26 < 2 u), its cosine and sine are off by a few units (8 u), the two products and their sum by 2 u; with the product
position * frequency in 64 bits, off by 2^-51 of the angle. Together (40 u + 2^-51 angle) (|y_i| + |y_{i+h}|), and 2^-8 of the
result for its rounding to bf16.
"""

from __future__ import annotations

import pytest
import torch

from oracle import prompt_oracle as po

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _case(rows, heads, kv, dim, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = (2 * torch.randn(rows, heads + 2 * kv, dim, generator=g)).to(BF)
    wq, wk = ((1 + 0.2 * torch.randn(dim, generator=g)).to(BF) for _ in range(2))
    return qkv, wq, wk, g


def _check(got, x, w, eps, positions, axes):
    y, size, angle = po.rotate_axes(x, w, eps, positions, axes.sections, axes.theta, axes.ladder)
    far = torch.zeros(size.shape[0], 1, size.shape[2], dtype=torch.float64)
    half = angle.shape[1]
    far[:, 0, :half] = far[:, 0, half:2 * half] = angle.abs()
    bar = (40 * 2.0 ** -24 + far * 2.0 ** -51) * size + (2.0 ** -8) * y.abs()
    d = (got.double().cpu() - y).abs()
    assert (d <= bar).all(), (d / bar.clamp_min(1e-30)).max()


CASES = [  # rows, heads, kv heads, dim, sections, ladder, with norm
    (1, 1, 1, 8 * 2, (8,), "shared", True), (1, 40, 8, 128, (8, 28, 28), "shared", False),
    (1001, 40, 8, 128, (8, 28, 28), "per_axis", True), (130, 5, 5, 128, (16, 16), "shared", True),
    (257, 28, 4, 128, (64,), "shared", True), (333, 14, 2, 64, (4, 14, 14), "per_axis", True),
    (65, 16, 2, 64, (0, 8, 0, 8), "shared", False), (77, 6, 3, 80, (10, 14, 16), "shared", True),
    (50, 3, 1, 96, (24,), "shared", True), (31, 7, 1, 40, (3, 5), "per_axis", True), (4500, 8, 1, 128, (64,), "shared", True),
    (1025, 2, 1, 128, (8, 28, 28), "per_axis", True), (2047, 3, 1, 64, (12, 12), "shared", True),
    (2049, 2, 2, 64, (32,), "shared", False), (4099, 1, 1, 64, (16, 16), "per_axis", True), (2050, 1, 1, 24, (8,), "shared", True)]


@pytest.mark.parametrize("rows,heads,kv,dim,sections,ladder,norm", CASES)
def test_against_float64(device, rows, heads, kv, dim, sections, ladder, norm):
    from vdn_h3_amd.rotary import RotaryAxes, normalise_qk_axes

    print(f"case rotary {rows}x{heads}/{kv}x{dim} {sections} {ladder} norm={norm}", flush=True)
    axes = RotaryAxes(sections, theta=10000.0, ladder=ladder)
    qkv, wq, wk, g = _case(rows, heads, kv, dim, rows + dim)
    pos = torch.randint(0, 40688, (len(sections), rows), generator=g)
    dev = qkv.to(device)
    q, k = dev[:, :heads], dev[:, heads:heads + kv]
    qw, kw = (wq, wk) if norm else (None, None)
    got = normalise_qk_axes(q, k, pos.to(device), axes, *(None if t is None else t.to(device) for t in (qw, kw)), 1e-5, 1e-3)
    assert got[0].shape == (rows, heads, dim) and got[1].shape == (rows, kv, dim)
    _check(got[0], qkv[:, :heads], qw, 1e-5, pos, axes)
    _check(got[1], qkv[:, heads:heads + kv], kw, 1e-3, pos, axes)
    assert torch.equal(dev.cpu(), qkv)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32])
def test_positions_of_every_type_far_and_strided(device, dtype):
    from vdn_h3_amd.rotary import RotaryAxes, normalise_qk_axes

    print(f"case rotary positions {dtype}", flush=True)
    axes = RotaryAxes((16, 24, 24), theta=500000.0)
    qkv, wq, wk, g = _case(64, 4, 2, 128, 3)
    if dtype == torch.float32:  # frames at a rate that is no whole number, and rows in front of the first
        pos = torch.randn(3, 64, generator=g) * 1000
    else:
        pos = torch.randint(-5, 2 ** 31 - 1 if dtype == torch.int32 else 2 ** 40, (3, 64), generator=g).to(dtype)
    dev = qkv.to(device)
    want = normalise_qk_axes(dev[:, :4], dev[:, 4:6], pos.to(device), axes, wq.to(device), wk.to(device))
    _check(want[0], qkv[:, :4], wq, 1e-6, pos, axes)
    _check(want[1], qkv[:, 4:6], wk, 1e-6, pos, axes)
    across = pos.t().contiguous().to(device).t()  # [rows, axes] storage
    heads_first = dev.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(64 * 8 * 128 + 1, dtype=BF, device=device)[1:].view(64, 8, 128).copy_(dev)  # off 16 bytes: copied
    for x in (heads_first, odd):
        got = normalise_qk_axes(x[:, :4], x[:, 4:6], across, axes, wq.to(device), wk.to(device))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = normalise_qk_axes(dev[:, :4], dev[:, 4:6], pos[0].to(device), axes)
    _check(one[0], qkv[:, :4], None, 0.0, pos[:1].expand(3, 64), axes)


def test_same_rotation_as_a_table(device):
    """Against the table form of the pass: the table's fp32 matrices and the angles computed here differ by a unit of fp32."""
    from vdn_h3_amd.hybrid import normalise_qk
    from vdn_h3_amd.rotary import RotaryAxes, normalise_qk_axes

    axes = RotaryAxes((8, 28, 28))
    qkv, wq, wk, g = _case(300, 4, 4, 128, 8)
    pos = torch.randint(0, 5000, (3, 300), generator=g)
    radians, axis = axes.frequencies()
    angle = pos.double()[axis.long()].t() * radians
    c, s = angle.cos().float(), angle.sin().float()
    table = torch.stack([torch.stack([c, -s], -1), torch.stack([s, c], -1)], -2).to(device)
    dev = qkv.to(device)
    want = normalise_qk(dev[:, :4], dev[:, 4:8], wq.to(device), wk.to(device), 1e-6, rope_freqs=table)
    got = normalise_qk_axes(dev[:, :4], dev[:, 4:8], pos.to(device), axes, wq.to(device), wk.to(device))
    for a, b in zip(got, want):
        assert (a.float() - b.float()).abs().max() <= 2 ** -6 * b.float().abs().max() and (a == b).float().mean() > 0.99


def test_refusals_streams_and_graph(device):
    from vdn_h3_amd.rotary import RotaryAxes, normalise_qk_axes

    axes = RotaryAxes((4, 4, 8))
    qkv, wq, wk, g = _case(20, 4, 2, 64, 4)
    dev, pos = qkv.to(device), torch.randint(0, 99, (3, 20), generator=g).to(device)
    q, k = dev[:, :4], dev[:, 4:6]
    for bad in [lambda: normalise_qk_axes(q, k, pos[:2], axes), lambda: normalise_qk_axes(q, k, pos[:, :19], axes),
                lambda: normalise_qk_axes(q, k, pos, RotaryAxes((40,))), lambda: normalise_qk_axes(q, k, pos, axes, wq[:8].to(device)),
                lambda: normalise_qk_axes(q[..., :60], k[..., :60], pos, axes)]:
        with pytest.raises(ValueError):
            bad()
    for dtype in (torch.float64, torch.int16, torch.bfloat16):
        with pytest.raises(TypeError):
            normalise_qk_axes(q, k, pos.to(dtype), axes)
    assert normalise_qk_axes(q[:0], k[:0], pos[:, :0], axes)[0].shape == (0, 4, 64)
    want = normalise_qk_axes(q, k, pos, axes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = normalise_qk_axes(q, k, pos, axes)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = normalise_qk_axes(q, k, pos, axes)
    for _ in range(3):
        pos.add_(17)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, normalise_qk_axes(q, k, pos, axes)))


@pytest.mark.parametrize("rows,heads,kv,dim,sections", [(9, 5, 1, 128, (64,)), (2100, 2, 1, 64, (8, 8)), (5000, 3, 3, 80, (10, 14, 16))])
def test_vectors_near_the_largest_and_the_smallest_numbers(device, rows, heads, kv, dim, sections):
    """The norm of a vector does not depend on its size, where its squares pass fp32 and where they fall under it; an infinity
    or a NaN stays in its vector."""
    from vdn_h3_amd.rotary import RotaryAxes, normalise_qk_axes

    print(f"case rotary ends of the range {rows}x{heads}/{kv}x{dim}", flush=True)
    axes = RotaryAxes(sections)
    qkv, wq, wk, g = _case(rows, heads, kv, dim, 70)
    for row, by in ((0, 2.0 ** 70), (1, 2.0 ** 120), (2, 2.0 ** -80), (3, 2.0 ** -120), (rows - 1, 2.0 ** 100)):
        qkv[row] = (qkv[row].float() * by).to(BF)
    qkv[4, 0], qkv[4, 1] = qkv[4, 0].sign() * 3e38, qkv[4, 1].sign() * 2.0 ** -133
    pos = torch.randint(0, 4000, (len(sections), rows), generator=g)
    dev = qkv.to(device)
    call = lambda x: normalise_qk_axes(x[:, :heads], x[:, heads:heads + kv], pos.to(device), axes, wq.to(device), wk.to(device), 0.0)
    want = call(dev)
    _check(want[0], qkv[:, :heads], wq, 0.0, pos, axes)
    _check(want[1], qkv[:, heads:heads + kv], wk, 0.0, pos, axes)
    dev[6, 1, 3], dev[7, 0, 5] = torch.nan, torch.inf
    got = call(dev)
    for (row, head) in ((6, 1), (7, 0)):
        assert got[0][row, head].isnan().any()
        got[0][row, head] = want[0][row, head] = 0
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
