"""The residual addition, RMSNorm and 8-bit codes in one pass against float64 (GPU).

Bars, from the arithmetic (u = 2^-24, one fp32 operation): t = fl(x + residual) is off by u |t|. The sum of squares adds at
most L = hidden / 64 + 14 terms one behind another, so y = t r w is off by at most R |y|, R = (L + 16) u (half of the sum's
error enters the root; the rest covers the squares, the mean, the root, the quotient and two products). A stored bf16 adds
2^-8 of the value. The scale is off by (R + 4 u) of itself, a quotient y / s by 2^-23 more; an int8 code is half a step of the
scale off, an e4m3 code 2^-4 of the value or, below the smallest normal number, 2^-10 of the scale.
"""

from __future__ import annotations

import pytest
import torch

from oracle import prompt_oracle as po

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF = torch.bfloat16
KINDS = {"bf16": 0, "int8": 1, "fp8": 2}


def _case(rows, hidden, seed):
    g = torch.Generator().manual_seed(seed)
    loud = 1 + 30 * (torch.rand(hidden, generator=g) < 0.02)
    x = torch.randn(rows, hidden, generator=g).to(BF)
    res = (3 * torch.randn(rows, hidden, generator=g) * loud).to(BF)
    return x, res, (1 + 0.3 * torch.randn(hidden, generator=g)).to(BF)


def _check(got, kind, x, res, w, eps):
    codes, scale, total = got
    t, y = po.residual_rmsnorm(x, res, w, eps)
    r = (x.shape[1] / 64 + 30) * U
    if res is not None:
        assert ((total.double().cpu() - t).abs() <= (2.0 ** -8 + 2 * U) * t.abs()).all()
    c = codes.double().cpu()
    if kind == "bf16":
        assert scale is None and codes.dtype == BF
        assert ((c - y).abs() <= (2.0 ** -8 + 2 * r) * y.abs()).all()
        return
    most = {"int8": 127.0, "fp8": 448.0}[kind]
    s = (y.abs().amax(-1, keepdim=True) / most).clamp_min(1e-12)
    assert scale.shape == (x.shape[0], 1) and ((scale.double().cpu() - s).abs() <= (r + 4 * U) * s).all()
    assert c.abs().max() <= most
    step = 0.5 * s if kind == "int8" else torch.maximum(y.abs() * 2.0 ** -4, 2.0 ** -10 * s)
    assert ((c * scale.double().cpu() - y).abs() <= step * (1 + 2 * r) + y.abs() * (2 * r + 2.0 ** -22)).all()


# widths of one chunk, ragged ones, one at each edge of a lane's chunks, and one past what registers hold
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows,hidden", [(1, 8), (3, 72), (1, 5120), (2, 2048), (2, 2056), (5, 5128), (513, 5120), (7, 8192),
                                         (3, 8200), (2, 16384), (2, 20008), (1030, 256), (2051, 1024), (4099, 2048),
                                         (4098, 24)])
def test_against_float64(device, kind, rows, hidden):
    from vdn_h3_amd.block_kernels import residual_rmsnorm_quantize

    print(f"case residual norm {kind} {rows}x{hidden}", flush=True)
    x, res, w = _case(rows, hidden, rows + hidden)
    dx, dr, dw = x.to(device), res.to(device), w.to(device)
    for r, dres in ((res, dr), (None, None)):
        got = residual_rmsnorm_quantize(dx, dres, dw, 1e-6, KINDS[kind])
        _check(got, kind, x, r, w, 1e-6)
        if r is None:
            assert got[2] is dx
    assert torch.equal(dx.cpu(), x) and torch.equal(dr.cpu(), res)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows,hidden", [(9, 1024), (9, 5120), (9, 8200), (2100, 1024)])
def test_strided_repeated_and_in_place(device, kind, rows, hidden):
    from vdn_h3_amd.block_kernels import residual_rmsnorm_quantize

    print(f"case residual norm strides {kind} {rows} {hidden}", flush=True)
    x, res, w = _case(rows, hidden, 5)
    wide = torch.full((rows, hidden + 64), 7.0, dtype=BF, device=device)
    wide[:, 8:8 + hidden] = x.to(device)
    want = residual_rmsnorm_quantize(x.to(device), res.to(device), w.to(device), 1e-5, KINDS[kind])

    def same(got):
        assert all(a is b or torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got[:2], want[:2]))
        assert torch.equal(got[2], want[2])

    same(residual_rmsnorm_quantize(wide[:, 8:8 + hidden], res.to(device), w.to(device), 1e-5, KINDS[kind]))
    odd = torch.empty(rows * hidden + 1, dtype=BF, device=device)[1:].view(rows, hidden).copy_(x)  # rows off 16 bytes: copied
    same(residual_rmsnorm_quantize(odd, res.to(device), w.to(device), 1e-5, KINDS[kind]))
    for which in range(2):  # the sum over x or over the residual
        a, b = x.to(device), res.to(device)
        got = residual_rmsnorm_quantize(a, b, w.to(device), 1e-5, KINDS[kind], sum_out=(a, b)[which])
        assert got[2] is (a, b)[which]
        same(got)
    out = torch.full((rows, hidden + 16), 5.0, dtype=BF, device=device)
    same(residual_rmsnorm_quantize(x.to(device), res.to(device), w.to(device), 1e-5, KINDS[kind], sum_out=out[:, :hidden]))
    assert (out[:, hidden:] == 5).all() and (wide[:, :8] == 7).all()
    one = residual_rmsnorm_quantize(x.to(device), res[:1].to(device).expand(rows, hidden), w.to(device), 1e-5, KINDS[kind])
    _check(one, kind, x, res[:1].expand(rows, hidden), w, 1e-5)


def test_squares_under_the_smallest_numbers(device):
    """With no epsilon the norm of a row does not depend on its size."""
    from vdn_h3_amd.block_kernels import residual_rmsnorm_quantize

    for hidden in (256, 5120, 9216):
        x, res, w = _case(5, hidden, 30)
        for kind in KINDS:
            for by in (2.0 ** -70, 2.0 ** 60):
                a, b = (x.float() * by).to(BF), (res.float() * by).to(BF)
                _check(residual_rmsnorm_quantize(a.to(device), b.to(device), w.to(device), 0.0, KINDS[kind]), kind, a, b, w, 0.0)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hidden,times", [(512, 1), (5120, 1), (9216, 1), (512, 300), (2048, 300)])
def test_borders(device, kind, hidden, times):
    """Zero rows, rows far up and far down in bf16's range, and rows that are not finite."""
    from vdn_h3_amd.block_kernels import residual_rmsnorm_quantize

    print(f"case residual norm borders {kind} {hidden} x {times}", flush=True)
    x, res, w = _case(8, hidden, 6)
    x[0], res[0] = 0, 0
    x[1], res[1] = x[1] * 2.0 ** 100, res[1] * 2.0 ** 100  # the squares pass fp32
    x[2], res[2] = x[2] * 2.0 ** -60, res[2] * 2.0 ** -60
    res[3] = -x[3]
    x[4, hidden // 2] = torch.inf
    res[5, hidden - 1] = torch.nan
    x[6, 0], res[6, 0] = -3e38, -3e38  # the sum passes fp32
    got = residual_rmsnorm_quantize(x.to(device).repeat(times, 1), res.to(device).repeat(times, 1), w.to(device), 1e-6, KINDS[kind])
    for t in got:  # the same rows give the same results
        if t is not None:
            bits = t.view(torch.uint8).view(times, 8, -1)
            assert torch.equal(bits, bits[:1].expand_as(bits))
    got = [None if t is None else t[:8] for t in got]
    fine = [0, 1, 2, 3, 7]
    _check([None if t is None else t[fine] for t in got], kind, x[fine], res[fine], w, 1e-6)
    for row in (4, 5, 6):
        if kind == "bf16":
            assert got[0][row].isnan().any()
        else:
            assert got[1][row].isnan().all() and (got[0][row].float() == 0).all()


def test_codes_feed_the_w8a8_product(device):
    """The codes and scales are those that quantize_rows makes of the norm where bf16 holds the norm exactly, and the
    product of HipLinear's int8 weights takes them as they are."""
    from vdn_h3_amd import linear
    from vdn_h3_amd.block_kernels import residual_rmsnorm_quantize

    g = torch.Generator().manual_seed(3)
    # rows of +-2^e: the norm of each is a power of two times +-1, exactly
    x = (torch.randint(0, 2, (64, 1024), generator=g) * 2.0 - 1).to(BF)
    w = torch.full((1024,), 4.0, dtype=BF)
    for kind, precision in ((linear.KIND_I8, "int8"), (linear.KIND_F8, "fp8")):
        q, s, t = residual_rmsnorm_quantize(x.to(device), x.to(device), w.to(device), 0.0, kind)
        y = (4 * x).to(device)
        q2, s2 = linear.quantize_rows(y, kind)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
        assert torch.equal(t.cpu(), 2 * x)
        layer = linear.HipLinear(torch.randn(96, 1024, generator=g).to(BF).to(device), precision)
        assert torch.equal(linear.gemm_w8a8(q, s, layer.weight, layer.weight_scale), layer(y))


def test_streams_and_graph(device):
    from vdn_h3_amd.block_kernels import residual_rmsnorm_quantize

    x, res, w = (t.to(device) for t in _case(40, 2048, 9))
    want = residual_rmsnorm_quantize(x, res, w, 1e-6, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = residual_rmsnorm_quantize(x, res, w, 1e-6, 1)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = residual_rmsnorm_quantize(x, res, w, 1e-6, 1)
    for seed in range(3):
        a, b, _ = (t.to(device) for t in _case(40, 2048, 20 + seed))
        x.copy_(a), res.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, residual_rmsnorm_quantize(x, res, w, 1e-6, 1)))


def test_no_rows(device):
    from vdn_h3_amd.block_kernels import residual_rmsnorm_quantize

    x = torch.empty(0, 64, dtype=BF, device=device)
    q, s, t = residual_rmsnorm_quantize(x, x, torch.ones(64, dtype=BF, device=device), 1e-6, 2)
    assert q.shape == (0, 64) and s.shape == (0, 1) and t.shape == (0, 64)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hidden,times", [(512, 1), (5120, 1), (9216, 1), (512, 300), (2048, 300)])
def test_weights_whose_products_pass_fp32(device, kind, hidden, times):
    """t w is past fp32's largest number, or under its smallest, while the norm, t r w, is one that bf16 holds."""
    from vdn_h3_amd.block_kernels import residual_rmsnorm_quantize

    print(f"case residual norm products {kind} {hidden} x {times}", flush=True)
    for t_up, w_up, eps in ((45, 90, 1e-6), (-42, -105, 0.0)):
        x, res, w = _case(8, hidden, 31)
        x, res, w = ((t.float() * 2.0 ** up).to(BF) for t, up in ((x, t_up), (res, t_up), (w, w_up)))
        z = (x.float() + res.float()).abs() * w.float().abs()
        assert (z.amax(1).isinf() if t_up > 0 else z.median(1).values < 2.0 ** -140).all()
        got = residual_rmsnorm_quantize(x.to(device).repeat(times, 1), res.to(device).repeat(times, 1), w.to(device), eps,
                                        KINDS[kind])
        _check([None if t is None else t[-8:] for t in got], kind, x, res, w, eps)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hidden,times", [(512, 1), (5120, 1), (9216, 1), (512, 300), (2048, 300)])
def test_rows_near_the_largest_and_the_smallest_numbers(device, kind, hidden, times):
    """Whole rows up to bf16's largest numbers and down to its smallest: their norm is an ordinary one."""
    from vdn_h3_amd.block_kernels import residual_rmsnorm_quantize

    print(f"case residual norm ends of the range {kind} {hidden} x {times}", flush=True)
    x, res, w = _case(8, hidden, 32)
    sign = x.float().sign()
    x[0], res[0] = sign[0] * 1e37, 0
    x[1], res[1] = sign[1] * 3e38, 0
    x[2], res[2] = sign[2] * 1.6e38, sign[2] * 1.6e38
    x[3], res[3] = x[3] * 1e36, res[3] * 1e34
    x[4, 1:], res[4], x[4, 0] = 0, 0, 3e38  # one channel alone
    x[5], res[5] = x[5] * 2.0 ** -120, res[5] * 2.0 ** -120
    x[6], res[6] = sign[6] * 2.0 ** -133, 0  # the smallest number
    got = residual_rmsnorm_quantize(x.to(device).repeat(times, 1), res.to(device).repeat(times, 1), w.to(device), 0.0, KINDS[kind])
    over = x.to(device).repeat(times, 1)  # the sum over x
    got2 = residual_rmsnorm_quantize(over, res.to(device).repeat(times, 1), w.to(device), 0.0, KINDS[kind], sum_out=over)
    assert all(a is b or torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, got2))
    for t in got:  # the same rows give the same results
        if t is not None:
            bits = t.view(torch.uint8).view(times, 8, -1)
            assert torch.equal(bits, bits[:1].expand_as(bits))
    _check([None if t is None else t[:8] for t in got], kind, x, res, w, 0.0)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hidden,times", [(512, 1), (5120, 1), (9216, 1), (512, 300), (2048, 300)])
def test_norms_past_fp32(device, kind, hidden, times):
    """A row whose norm, not only a product on its way, is past fp32: the 8-bit kinds have the scale NaN, bf16 the infinity."""
    from vdn_h3_amd.block_kernels import residual_rmsnorm_quantize

    print(f"case residual norm past fp32 {kind} {hidden} x {times}", flush=True)
    x, res, w = _case(8, hidden, 33)
    x[:] = res[:] = 0
    x[:6, 3], x[:6, 5], w[3], w[5] = 1.5, -0.75, 3e38, 1.0  # t w overflows, and t r w the more
    x[6:, 5] = 1.0  # y = sqrt(hidden) in a channel, none in the others
    x[5, 3], res[5, 3] = 0.01, 0.01  # t w does not overflow, t r w does
    x[5, 5] = 0
    got = residual_rmsnorm_quantize(x.to(device).repeat(times, 1), res.to(device).repeat(times, 1), w.to(device), 0.0, KINDS[kind])
    assert (po.residual_rmsnorm(x, res, w, 0.0)[1][:6, 3].abs() > 2.0 ** 128).all()
    codes, scale, _ = (None if t is None else t[-8:] for t in got)
    if kind == "bf16":
        assert (codes[:6, 3] == torch.inf).all() and codes[:, [i for i in range(hidden) if i != 3]].isfinite().all()
    else:
        assert scale[:6].isnan().all() and (codes[:6].float() == 0).all()
    _check([None if t is None else t[-2:] for t in got], kind, x[6:], res[6:], w, 0.0)
