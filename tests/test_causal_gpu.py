"""Causal attention of packed prompts and of new tokens over caches against float64 (GPU).

Bar, from the arithmetic: a score is a sum of D products in fp32, off by at most (D + 8) 2^-24 of scale sum |q_d k_d| (`score`
below), and an exponential by 2^-20 of itself with its argument's rounding, so each probability by e = (D + 8) 2^-24 score
+ 2^-20 (1 + score). Probabilities are rounded to bf16 for the products with the values (2^-8 each), in the sum of the
values and in the row's sum alike: with A = sum p |v| the result is off by at most 2 (2^-8 + e) A, and 2^-8 of itself for
its own rounding.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import prompt_oracle as po

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _qkv(rows, heads, kv, dim, seed, loud=1.0):
    g = torch.Generator().manual_seed(seed)
    return ((loud * torch.randn(rows, heads, dim, generator=g)).to(BF), torch.randn(rows, kv, dim, generator=g).to(BF),
            torch.randn(rows, kv, dim, generator=g).to(BF))


def _check(got, want, dim):
    out, size, score = want
    e = ((dim + 8) * 2.0 ** -24 * score + 2.0 ** -20 * (1 + score))[..., None]
    bar = 2 * (2.0 ** -8 + e) * size + 2.0 ** -8 * out.abs()
    g = got.double().cpu()
    live = ~out.isnan()
    d = (g - out).abs()[live]
    assert (d <= bar[live]).all(), (d / bar[live].clamp_min(1e-30)).max()


def _cached_in(ranges, q, k, v, lengths, scale):
    """``vdnh3_causal_attn_cached`` in that many ranges, into an output of sevens and a buffer of NaNs."""
    from vdn_h3_amd import _lib

    lib = _lib.lib()
    (batch, new, heads, dim), (room, kv) = q.shape, k.shape[1:3]
    size = lib.vdnh3_causal_partial_bytes(new, heads, dim, ranges)
    partial = torch.full((max(size, 16),), 0xFF, dtype=torch.uint8, device=q.device)
    out = torch.full(q.shape, 7.0, dtype=BF, device=q.device)
    _lib.check(lib.vdnh3_causal_attn_cached(
        q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], out.data_ptr(),
        *out.stride()[:3], lengths.data_ptr(), batch, new, room, heads, kv, dim, scale, ranges, partial.data_ptr(), size,
        _lib.stream_handle(q.device)), "cached")
    return out


PACKED = [  # lengths, heads, kv heads, dim
    ([1], 1, 1, 64), ([2], 5, 1, 128), ([5, 1, 33], 4, 4, 64), ([0, 3, 0, 1, 64, 0], 8, 2, 128), ([95, 96, 97], 5, 1, 128),
    ([255, 256, 257], 2, 2, 128), ([51, 52, 103], 10, 2, 128), ([640], 40, 8, 128), ([1, 500, 63], 14, 2, 64),
    ([700], 3, 3, 64), ([130, 31], 7, 1, 128), ([600], 32, 1, 64), ([200], 6, 2, 80), ([90, 7], 4, 4, 24),
    ([1] * 40, 8, 1, 128), ([1300, 900], 40, 8, 128), ([2100], 20, 20, 64), ([17, 1, 1, 300] * 3, 20, 20, 64)]


@pytest.mark.parametrize("lengths,heads,kv,dim", PACKED)
def test_packed_against_float64(device, lengths, heads, kv, dim):
    from vdn_h3_amd.causal import causal_softmax_packed

    print(f"case packed {lengths} {heads}/{kv}x{dim}", flush=True)
    bounds = [0]
    for n in lengths:
        bounds.append(bounds[-1] + n)
    rows = bounds[-1]
    q, k, v = _qkv(rows, heads, kv, dim, rows + dim, loud=2.0)
    scale = dim ** -0.5
    cu = torch.tensor(bounds, dtype=torch.int32, device=device)
    got = causal_softmax_packed(q.to(device), k.to(device), v.to(device), cu, scale)
    want = po.packed(q, k, v, bounds, scale)
    _check(got, want, dim)
    if dim % 8 == 0:  # views of one projection, and heads in front of rows
        fused = torch.cat([q, k, v], 1).to(device).split((heads, kv, kv), 1)
        first = [t.to(device).transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
        assert torch.equal(causal_softmax_packed(*fused, bounds, scale), got)
        assert torch.equal(causal_softmax_packed(*first, cu.long(), scale), got)


def test_rows_outside_every_sequence_stay(device):
    from vdn_h3_amd.causal import causal_softmax_packed

    for dim in (128, 80):
        q, k, v = _qkv(300, 4, 2, dim, 1)
        for bounds in ([20, 130, 130, 260], [0, 0], [300, 300], [299, 300], [7, 8]):
            out = torch.full((300, 4, dim), 3.0, dtype=BF, device=device)
            # what lies outside a sequence takes no part, whatever it holds
            a, b = bounds[0], bounds[-1]
            dk, dv = k.clone(), v.clone()
            dk[:a], dk[b:], dv[:a], dv[b:] = torch.nan, torch.inf, torch.inf, torch.nan
            got = causal_softmax_packed(q.to(device), dk.to(device), dv.to(device),
                                        torch.tensor(bounds, dtype=torch.int32, device=device), 0.1, out=out)
            assert got is out and (out[:a] == 3).all() and (out[b:] == 3).all()
            _check(got, po.packed(q, k, v, bounds, 0.1), dim)


def test_bounds_on_the_device_are_cut(device):
    from vdn_h3_amd.causal import causal_softmax_packed

    q, k, v = _qkv(100, 2, 1, 64, 2)
    cu = torch.tensor([-7, 40, 2000000000], dtype=torch.int32, device=device)
    got = causal_softmax_packed(q.to(device), k.to(device), v.to(device), cu, 0.125)
    _check(got, po.packed(q, k, v, [0, 40, 100], 0.125), 64)


@pytest.mark.parametrize("dim,kv", [(128, 1), (64, 4)])
def test_infinities_and_nans_where_a_row_does_not_look(device, dim, kv):
    """Keys and values behind a row, or of another sequence, are not a number: the row does not change. Rows that see one
    hold what the softmax gives."""
    from vdn_h3_amd.causal import causal_softmax_packed

    print(f"case non-finite {dim} {kv}", flush=True)
    bounds, heads = [0, 150, 340], 4
    q, k, v = _qkv(340, heads, kv, dim, 11)
    k[100], v[120] = torch.nan, torch.inf
    v[120, :, 1::2] = torch.nan
    k[150 + 96], v[150 + 97] = -torch.inf, torch.nan
    k[339], v[339] = torch.inf, torch.nan
    got = causal_softmax_packed(q.to(device), k.to(device), v.to(device), bounds, dim ** -0.5).cpu()
    seen = [i for i in range(340) if i < 100 or 150 <= i < 150 + 96]
    want = [t[seen] for t in po.packed(q, k, v, bounds, dim ** -0.5)]
    assert not want[0].isnan().any()
    _check(got[seen], want, dim)
    assert got[100:150].isnan().all()  # a key that is no number
    assert got[150 + 97:].isnan().all()  # a value that is none, or a key of infinities


def test_scores_at_the_ends_of_the_range(device):
    """One key far above the rest, all keys equal, scores in the thousands either way."""
    from vdn_h3_amd.causal import causal_softmax_packed

    q, k, v = _qkv(400, 2, 1, 64, 12, loud=40.0)
    got = causal_softmax_packed(q.to(device), k.to(device), v.to(device), [0, 400], 4.0)
    _check(got, po.packed(q, k, v, [0, 400], 4.0), 64)
    same = k[:1].expand(400, 1, 64).contiguous()
    got = causal_softmax_packed(q.to(device), same.to(device), v.to(device), [0, 400], 4.0)
    _check(got, po.packed(q, same, v, [0, 400], 4.0), 64)
    down = (-q.float().abs().mean((0, 1)))[None, None].expand(400, 1, 64).to(BF).contiguous()
    up = q.abs()
    got = causal_softmax_packed(up.to(device), down.to(device), v.to(device), [0, 400], 1.0)
    _check(got, po.packed(up, down, v, [0, 400], 1.0), 64)


CACHED = [  # new, room, lengths, heads, kv heads, dim
    (1, 1, [1], 1, 1, 64), (1, 70, [0, 1, 2, 63, 64, 65, 70], 5, 1, 128), (1, 1000, [1000, 31, 999], 40, 8, 128),
    (1, 257, [256, 257, 5], 16, 16, 64), (2, 300, [0, 1, 2, 3, 299], 8, 2, 128), (5, 400, [3, 5, 128, 400], 28, 4, 128),
    (1, 500, [500, 77], 32, 1, 128), (9, 130, [130, 9, 100], 14, 2, 64), (70, 200, [200, 70, 10, 0], 6, 2, 128),
    (300, 640, [640, 400, 257], 5, 1, 64), (1, 4100, [4100], 4, 1, 128), (4, 2500, [2500, 0, 1300], 6, 1, 64),
    (40, 96, [96] * 3, 1, 1, 128), (1, 90, [45] * 70, 2, 1, 64)]


@pytest.mark.parametrize("new,room,lengths,heads,kv,dim", CACHED)
def test_cached_against_float64(device, new, room, lengths, heads, kv, dim):
    from vdn_h3_amd.causal import causal_softmax_cached

    print(f"case cached {new}/{room} {lengths} {heads}/{kv}x{dim}", flush=True)
    batch = len(lengths)
    q, k, v = _qkv(batch * max(new, room), heads, kv, dim, room + new, loud=2.0)
    q = q[:batch * new].view(batch, new, heads, dim)
    k, v = (t[:batch * room].view(batch, room, kv, dim) for t in (k, v))
    scale = dim ** -0.5
    want = po.cached(q, k, v, lengths, scale)
    n = torch.tensor(lengths, dtype=torch.int32, device=device)
    got = causal_softmax_cached(q.to(device), k.to(device), v.to(device), n, scale)
    _check(got, want, dim)
    # heads in front of rows in the caches, stale rows that are no numbers, a view of q, an output with a wider row
    dk, dv = (t.transpose(1, 2).contiguous().to(device).transpose(1, 2) for t in (k, v))
    for b, m in enumerate(lengths):
        dk[b, m:], dv[b, m:] = torch.nan, torch.inf
    wide = torch.full((batch, new, heads + 3, dim), 9.0, dtype=BF, device=device)
    view = torch.cat([q, q], 2).to(device)[:, :, :heads]
    got2 = causal_softmax_cached(view, dk, dv, n.long(), scale, out=wide[:, :, :heads])
    assert torch.equal(got2, got) and (wide[:, :, heads:] == 9).all()


@pytest.mark.parametrize("new,heads,kv,dim", [(1, 5, 1, 128), (1, 4, 4, 64), (3, 12, 2, 64), (7, 10, 2, 128), (9, 10, 2, 128),
                                                (7, 20, 4, 64), (20, 10, 2, 128), (33, 3, 1, 64)])
def test_cached_however_it_is_cut(device, new, heads, kv, dim):
    """Whole rows and every number of ranges, more than there are tiles for among them; lengths of every kind at once."""
    from vdn_h3_amd import _lib

    lengths = [0, 1, 31, 32, 33, 700, 64, 0, 257, 128, 96, 1, 0]
    batch, room = len(lengths), 704
    q, k, v = _qkv(batch * room, heads, kv, dim, 40 + new, loud=2.0)
    q, k, v = q[:batch * new].view(batch, new, heads, dim), k.view(batch, room, kv, dim), v.view(batch, room, kv, dim)
    want = po.cached(q, k, v, lengths, 0.1)
    n = torch.tensor(lengths, dtype=torch.int32, device=device)
    dq, dk, dv = q.to(device), k.to(device), v.to(device)
    for ranges in (0, 1, 2, 3, 5, 8, 13, 17, 40, 256):
        print(f"case {ranges} ranges, {new} new tokens {heads}/{kv}x{dim}", flush=True)
        out = _cached_in(ranges, dq, dk, dv, n, 0.1)
        _check(out, want, dim)
    lib, partial = _lib.lib(), torch.empty(64, dtype=torch.uint8, device=device)
    assert lib.vdnh3_causal_attn_cached(
        dq.data_ptr(), *dq.stride()[:3], dk.data_ptr(), *dk.stride()[:3], dv.data_ptr(), *dv.stride()[:3], out.data_ptr(),
        *out.stride()[:3], n.data_ptr(), batch, new, room, heads, kv, dim, 0.1, 4, partial.data_ptr(), 64,
        _lib.stream_handle(device)) == _lib.VDNH3_ERR_INVALID  # too small a buffer


def test_many_requests(device):
    """More requests than a workgroup has threads, some without keys."""
    from vdn_h3_amd.causal import causal_softmax_cached

    batch, room = 700, 40
    g = torch.Generator().manual_seed(50)
    lengths = torch.randint(0, room + 1, (batch,), generator=g)
    q, k, v = _qkv(batch * room, 4, 2, 64, 51)
    q, k, v = q[:batch * 2].view(batch, 2, 4, 64), k.view(batch, room, 2, 64), v.view(batch, room, 2, 64)
    want = po.cached(q, k, v, lengths.tolist(), 0.125)
    dq, dk, dv = q.to(device), k.to(device), v.to(device)
    _check(causal_softmax_cached(dq, dk, dv, lengths.to(device), 0.125), want, 64)
    for ranges in (1, 7, 64, 300):
        print(f"case {ranges} ranges of {batch} requests", flush=True)
        _check(_cached_in(ranges, dq, dk, dv, lengths.to(device, torch.int32), 0.125), want, 64)


def test_many_sequences(device):
    """More packed sequences than a wavefront has lanes, empty ones among them."""
    from vdn_h3_amd.causal import causal_softmax_packed

    g = torch.Generator().manual_seed(52)
    lengths = torch.randint(0, 40, (150,), generator=g)
    lengths[:3], lengths[63:66], lengths[128], lengths[-2:] = 0, 0, 300, 0
    bounds = [0] + lengths.cumsum(0).tolist()
    for heads, kv, dim in ((5, 1, 64), (4, 4, 128)):
        q, k, v = _qkv(bounds[-1], heads, kv, dim, 53)
        cu = torch.tensor(bounds, dtype=torch.int32, device=device)
        got = causal_softmax_packed(q.to(device), k.to(device), v.to(device), cu, 0.125)
        _check(got, po.packed(q, k, v, bounds, 0.125), dim)
    # thousands, nearly all of them empty or of one row
    lengths = (torch.rand(9000, generator=g) < 0.1).long()
    lengths[[0, 4095, 4097, 8999]] = torch.tensor([3, 70, 130, 2])
    bounds = [0] + lengths.cumsum(0).tolist()
    q, k, v = _qkv(bounds[-1], 4, 2, 64, 54)
    got = causal_softmax_packed(q.to(device), k.to(device), v.to(device), bounds, 0.125)
    _check(got, po.packed(q, k, v, bounds, 0.125), 64)


def test_cached_infinities_behind_a_new_token(device):
    from vdn_h3_amd.causal import causal_softmax_cached

    for new in (4, 40):
        q, k, v = _qkv(200, 4, 2, 64, 14)
        q, k, v = q[None, :new], k[None], v[None]
        v[0, 199], k[0, 198] = torch.nan, torch.nan  # what only the last two tokens see
        n = torch.tensor([200], dtype=torch.int32, device=device)
        want = po.cached(q, k, v, [200], 0.125)
        dq, dk, dv = q.to(device), k.to(device), v.to(device)
        for got in [causal_softmax_cached(dq, dk, dv, n, 0.125)] + [_cached_in(r, dq, dk, dv, n, 0.125) for r in (0, 1, 3)]:
            got = got.cpu()
            _check(got[:, :-2], [t[:, :-2] for t in want], 64)
            assert got[:, -2:].isnan().all()


@pytest.mark.parametrize("new", [1, 4, 40, 200])
def test_infinities_and_largest_numbers_that_a_row_sees(device, new):
    """An infinity among the values gives an infinity, values near the largest number sum to numbers; the other channels and
    the tokens in front do not change. New tokens over caches of one part and of several, and whole prompts."""
    from vdn_h3_amd.causal import causal_softmax_cached, causal_softmax_packed

    for room, dim in ((60, 128), (900, 64), (900, 128)):
        new = min(new, room)
        print(f"case infinities seen {new} of {room} x {dim}", flush=True)
        q, k, v = _qkv(room, 4, 2, dim, 16)
        big = (torch.rand(room, generator=torch.Generator().manual_seed(17)) * 0.1 + 0.9) * 3e38
        v[room // 2, :, 3], v[-1, :, 5] = torch.inf, -torch.inf
        v[:, :, 7], v[:, :, 8] = big[:, None].to(BF), -big[:, None].to(BF)
        whole = po.packed(q, k, v, [0, room], dim ** -0.5)
        n = torch.tensor([room], dtype=torch.int32, device=device)
        caches = (q[None, -new:].to(device), k[None].to(device), v[None].to(device), n, dim ** -0.5)
        some = [causal_softmax_cached(*caches)] + [_cached_in(r, *caches) for r in (0, 1, 3)]
        full = causal_softmax_packed(q.to(device), k.to(device), v.to(device), [0, room], dim ** -0.5)
        for got, want in [(t[0], [w[-new:] for w in whole]) for t in some] + [(full, whole)]:
            odd = want[0].isinf()
            assert odd.any() and torch.equal(got.cpu()[odd], want[0][odd].to(BF))
            rest = [want[0].masked_fill(odd, 0), want[1].masked_fill(odd, 0), want[2]]
            assert got.cpu()[~odd].isfinite().all()
            _check(got.cpu().masked_fill(odd, 0), rest, dim)


def test_counts_past_32_bits_are_cut(device):
    from vdn_h3_amd.causal import causal_softmax_cached, causal_softmax_packed

    q, k, v = _qkv(90, 4, 2, 64, 18)
    far = torch.tensor([2 ** 32 + 5, -2 ** 32 + 5], dtype=torch.int64, device=device)
    got = causal_softmax_cached(q[:2, None].to(device), *(t.expand(2, -1, -1, -1).to(device) for t in (k, v)), far, 0.125)
    _check(got, po.cached(q[:2, None], *(t.expand(2, -1, -1, -1) for t in (k, v)), [90, 0], 0.125), 64)
    got = causal_softmax_packed(q.to(device), k.to(device), v.to(device), far.flip(0), 0.125)
    _check(got, po.packed(q, k, v, [0, 90], 0.125), 64)


# row 1,199 starts at element 2.5e9; rows as far apart as they may be
@pytest.mark.parametrize("new,room,row", [(1, 1200, 1 << 21), (40, 1200, 1 << 21), (1, 300, 1 << 23), (70, 300, 1 << 23)])
def test_offsets_past_32_bits(device, new, room, row):
    """Caches whose rows lie more than 2^32 bytes, and 2^31 elements, behind their first."""
    from vdn_h3_amd.causal import causal_softmax_cached

    print(f"case cached far {new} {room} x {row}", flush=True)
    store = torch.empty(room * row, dtype=BF, device=device)
    k, v = (torch.as_strided(store, (1, room, 2, 64), (8, row, 64, 1), off) for off in (0, 1 << 20))
    q, hk, hv = _qkv(room, 4, 2, 64, 15)
    k.copy_(hk[None]), v.copy_(hv[None])
    q = q[None, :new]
    n = torch.tensor([room - 1], dtype=torch.int32, device=device)
    want = po.cached(q, hk[None], hv[None], [room - 1], 0.125)
    _check(causal_softmax_cached(q.to(device), k, v, n, 0.125), want, 64)
    for ranges in (0, 1, 5):
        _check(_cached_in(ranges, q.to(device), k, v, n, 0.125), want, 64)


def test_strides_of_single_elements_do_not_count(device):
    from vdn_h3_amd.block_kernels import residual_rmsnorm_quantize
    from vdn_h3_amd.causal import causal_softmax_cached, causal_softmax_packed
    from vdn_h3_amd.rotary import RotaryAxes, normalise_qk_axes

    def odd(t):  # a stride of 3 wherever a dimension has one element
        return torch.as_strided(t, t.shape, tuple(3 if n == 1 else s for n, s in zip(t.shape, t.stride())))

    for rows, heads, kv in ((1, 4, 1), (1, 1, 1), (40, 1, 1)):
        q, k, v = (t.to(device) for t in _qkv(rows, heads, kv, 64, 60))
        want = causal_softmax_packed(q, k, v, [0, rows], 0.125)
        assert torch.equal(causal_softmax_packed(odd(q), odd(k), odd(v), [0, rows], 0.125), want)
        n = torch.tensor([rows], dtype=torch.int32, device=device)
        got = causal_softmax_cached(odd(q[None, -1:]), odd(k[None]), odd(v[None]), n, 0.125)
        _check(got[0], [t[-1:] for t in po.packed(q.cpu(), k.cpu(), v.cpu(), [0, rows], 0.125)], 64)
        pos = torch.arange(rows, device=device)
        axes = RotaryAxes((32,))
        assert all(torch.equal(a, b) for a, b in zip(normalise_qk_axes(odd(q), odd(k), pos, axes),
                                                     normalise_qk_axes(q, k, pos, axes)))
    x, w = torch.randn(1, 64, device=device).to(BF), torch.ones(64, dtype=BF, device=device)
    out = torch.empty_like(x)
    got = residual_rmsnorm_quantize(odd(x), odd(x), w, 1e-6, 1, sum_out=odd(out))
    assert torch.equal(got[0], residual_rmsnorm_quantize(x, x, w, 1e-6, 1)[0]) and torch.equal(out, 2 * x)


def test_cache_layout_and_lengths_are_checked(device):
    from vdn_h3_amd.causal import causal_softmax_cached, causal_softmax_packed

    q, k = torch.zeros(2, 1, 4, 64, dtype=BF, device=device), torch.zeros(2, 9, 2, 72, dtype=BF, device=device)
    n = torch.ones(2, dtype=torch.int32, device=device)
    for bad in (k[..., 1:65], torch.zeros(2, 9, 64, 2, dtype=BF, device=device).transpose(2, 3)):
        with pytest.raises(ValueError, match="in place|copied"):
            causal_softmax_cached(q, bad, bad, n, 0.1)
    good = k[..., :64]
    with pytest.raises(ValueError, match="out"):
        causal_softmax_cached(q, good, good, n, 0.1, out=torch.zeros(2, 1, 4, 64, device=device))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            causal_softmax_cached(q, good, good, n, scale)
        with pytest.raises(ValueError, match="scale"):
            causal_softmax_packed(q[:, 0], good[:, 0], good[:, 0], [0, 2], scale)
    with pytest.raises(RuntimeError, match="CPU"):
        causal_softmax_cached(q, good, good, n.cpu(), 0.1)
    with pytest.raises(ValueError, match="out"):
        causal_softmax_cached(q, good, good, n, 0.1, out=torch.zeros(1, 1, 4, 64, dtype=BF, device=device).expand(2, 1, 4, 64))
    empty = causal_softmax_cached(q, good[:, :0], good[:, :0], n, 0.1)
    assert (empty == 0).all()
    assert causal_softmax_packed(q[:0, 0], good[:0, 0], good[:0, 0], [0], 0.1).shape == (0, 4, 64)
    assert causal_softmax_cached(q[:0], good[:0], good[:0], n[:0], 0.1).shape == (0, 1, 4, 64)


def test_repeatable_on_streams_and_in_graphs(device):
    """The same bits again; on another stream; and from a graph replayed with other lengths and other bounds."""
    from vdn_h3_amd.causal import causal_softmax_cached, causal_softmax_packed

    q, k, v = (t.to(device) for t in _qkv(1500, 10, 2, 128, 16))
    cu = torch.tensor([0, 700, 1500], dtype=torch.int32, device=device)
    qc, kc, vc = q[:6].view(2, 3, 10, 128), k.view(2, 750, 2, 128), v.view(2, 750, 2, 128)
    n = torch.tensor([750, 20], dtype=torch.int32, device=device)
    q1 = q[:2].view(2, 1, 10, 128)

    def calls():
        return (causal_softmax_packed(q, k, v, cu, 0.1), causal_softmax_cached(qc, kc, vc, n, 0.1),
                causal_softmax_cached(q1, kc, vc, n, 0.1))

    want = calls()
    assert all(torch.equal(a, b) for a, b in zip(calls(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = calls()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for first, lengths in ((700, (750, 20)), (1, (1, 0)), (1499, (333, 749)), (0, (640, 2))):
        cu.copy_(torch.tensor([0, first, 1500], dtype=torch.int32))
        n.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, calls())), (first, lengths)
    assert math.isfinite(got[0].float().abs().max().item())


@pytest.mark.parametrize("dim", [64, 128])
def test_infinities_far_below_a_rows_maximum(device, dim):
    """An infinite value counts however small its key's probability is (an exponential under fp32's smallest number), in
    front of larger scores and behind them; opposite infinities give a NaN; a score of minus infinity leaves none of it."""
    from vdn_h3_amd.causal import causal_softmax_cached, causal_softmax_packed

    room, heads, kv = 700, 4, 2
    g = torch.Generator().manual_seed(61)
    q = torch.zeros(room, heads, dim)
    q[..., 0] = 8.0
    k = 0.1 * torch.randn(room, kv, dim, generator=g)
    v = torch.randn(room, kv, dim, generator=g).to(BF)
    k[..., 0] = 0.0
    for j, score in ((5, -110.0), (40, -400.0), (300, -600.0), (301, -130.0), (302, -88.0), (640, -650.0)):
        k[j, :, 0] = score / 8
    k[400:, :, 0] += 12.0  # scores 96 above those in front
    k[640, :, 0] = -600.0 / 8
    q, k = q.to(BF), k.to(BF)
    v[5, :, 1], v[40, :, 2], v[300, :, 3], v[640, :, 4] = torch.inf, -torch.inf, torch.inf, -torch.inf
    v[301, :, 5], v[302, :, 5] = torch.inf, -torch.inf
    for new in (1, 60, 350):
        print(f"case infinities far below {new} of {room} x {dim}", flush=True)
        out, size, score = po.packed(q, k, v, [0, room], 1.0)
        assert (out[-1, :, [1, 3]] == torch.inf).all() and (out[-1, :, [2, 4]] == -torch.inf).all() and out[-1, :, 5].isnan().all()
        n = torch.tensor([room], dtype=torch.int32, device=device)
        caches = (q[None, -new:].to(device), k[None].to(device), v[None].to(device), n, 1.0)
        some = [causal_softmax_cached(*caches)] + [_cached_in(r, *caches) for r in (0, 1, 3, 9)]
        full = causal_softmax_packed(q.to(device), k.to(device), v.to(device), [0, room], 1.0)
        for got, want in [(t[0], [w[-new:] for w in (out, size, score)]) for t in some] + [(full, (out, size, score))]:
            got = got.cpu()
            odd = ~want[0].isfinite()
            assert torch.equal(got[odd].nan_to_num(7.0), want[0][odd].to(BF).nan_to_num(7.0))
            assert got[~odd].isfinite().all()
            _check(got.masked_fill(odd, 0), [want[0].masked_fill(odd, 0), want[1].masked_fill(odd, 0), want[2]], dim)
