"""Every block height of the causal kernels, asserted through the host's rule (GPU): workgroups of 128 and of 256 rows on whole
prompts and over caches, and of 16, 32 and 48 rows over ranges of caches.

The first test needs no tolerance but for one rounding. With queries of zeros every probability is exactly 1 and the row's sum
the number of its keys, n; values of 1 in a channel of its own for each of D keys at a time make each output channel one key's
probability, 1 / n (the fp32 quotient and one rounding to bf16), or 0 for a key that the row does not see. A key that is lost,
counted twice or seen by a wrong row shows, whichever it is.
"""

from __future__ import annotations

import pytest
import torch

from oracle import prompt_oracle as po
from test_causal_gpu import _cached_in, _check, _qkv

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _one_key_each(first, like):
    """Values that are 1 where channel d meets key first + d of a cache or a sequence's row first + d."""
    v = torch.zeros_like(like)
    room, dim = v.shape[-3], v.shape[-1]
    j = torch.arange(first, min(first + dim, room), device=v.device)
    v[..., j, :, j - first] = 1
    return v


def _quotients(seen, keys):
    """1 / keys where seen, as fp32 divides; [rows, dim]."""
    return torch.where(seen, 1.0 / keys[:, None].float().clamp_min(1), 0.0)


def _same_quotients(got, want):
    """``got`` ``[..., heads, dim]`` against ``want`` ``[..., dim]``: zeros are zeros, the others off by a rounding to bf16 and two
    units of fp32 (the reciprocal and its product)."""
    want = want.unsqueeze(-2)
    return ((got.float() - want).abs() <= (2.0 ** -8 + 2.0 ** -23) * want).all()


PACKED = [  # lengths, heads, kv heads, dim, rows of a workgroup
    ([1300, 1, 0, 333, 307], 40, 8, 128, 256), ([4600, 8], 16, 16, 128, 256), ([51, 0, 2349, 1, 300], 28, 4, 128, 256),
    ([900, 1200, 204], 32, 1, 128, 256), ([2900, 1, 1300], 32, 8, 64, 256), ([6560], 20, 20, 64, 256),
    ([97, 4500, 0, 5000], 14, 2, 64, 256), ([1, 500, 63, 0, 900], 40, 8, 128, 128), ([2100, 77], 20, 20, 64, 128)]


@pytest.mark.parametrize("lengths,heads,kv,dim,height", PACKED)
def test_every_key_of_a_prompt_counts_once(device, built_lib, lengths, heads, kv, dim, height):
    from vdn_h3_amd.causal import causal_softmax_packed

    print(f"case every key {lengths} {heads}/{kv}x{dim}", flush=True)
    bounds = torch.tensor([0] + lengths).cumsum(0).tolist()
    rows = bounds[-1]
    assert built_lib.vdnh3_causal_block_rows(1, rows, heads, kv, dim, 0) == height
    q = torch.zeros(rows, heads, dim, dtype=BF, device=device)
    k = torch.randn(rows, kv, dim, device=device).to(BF)
    row = torch.arange(rows, device=device)
    start = torch.cat([torch.full((n,), a) for a, n in zip(bounds, lengths)]).to(device)
    for first in range(0, rows, dim):
        got = causal_softmax_packed(q, k, _one_key_each(first, k), bounds, 0.125)
        key = first + torch.arange(dim, device=device)
        seen = (key[None] >= start[:, None]) & (key[None] <= row[:, None])
        assert _same_quotients(got, _quotients(seen, row - start + 1)), first


CACHED = [  # new tokens, lengths, room, heads, kv heads, dim, rows of a workgroup of ranges
    (1, [0, 1, 31, 32, 33, 700, 64, 0, 257, 128, 96, 1, 0], 704, 5, 1, 128, 16),
    (3, [0, 1, 31, 32, 33, 700, 64, 0, 257, 128, 96, 2, 3], 704, 12, 2, 64, 32),
    (20, [0, 1, 31, 32, 33, 700, 64, 0, 257, 128, 96, 19, 20], 704, 10, 2, 128, 48),
    (33, [700, 20, 33, 0, 650], 700, 4, 4, 64, 48), (1, [4100], 4100, 8, 1, 64, 16), (8, [2500, 0, 1300], 2500, 8, 2, 128, 32)]


@pytest.mark.parametrize("new,lengths,room,heads,kv,dim,height", CACHED)
def test_every_key_of_a_cache_counts_once(device, built_lib, new, lengths, room, heads, kv, dim, height):
    batch = len(lengths)
    q = torch.zeros(batch, new, heads, dim, dtype=BF, device=device)
    k = torch.randn(batch, room, kv, dim, device=device).to(BF)
    n = torch.tensor(lengths, dtype=torch.int32, device=device)
    last = (n[:, None] - new + torch.arange(new, device=device)).view(-1)
    for ranges in (0, 1, 2, 3, 5, 8, 13, 32, 40, 256):
        print(f"case every key {ranges} ranges, {new} new tokens {lengths} {heads}/{kv}x{dim}", flush=True)
        assert built_lib.vdnh3_causal_block_rows(batch, new, heads, kv, dim, ranges) == (height if ranges else 128)
        for first in range(0, room, dim):
            got = _cached_in(ranges, q, k, _one_key_each(first, k), n, 0.125)
            key = first + torch.arange(dim, device=device)
            want = _quotients(key[None] <= last[:, None], last + 1)
            assert _same_quotients(got.view(-1, heads, dim), want), (ranges, first)


HIGH_CACHED = [  # new tokens, lengths, room, heads, kv heads, dim: the prompt kernel over caches, 256 rows a workgroup
    (1000, [1500, 600, 0], 1500, 40, 8, 128), (700, [700, 1100, 33, 2], 1100, 28, 4, 128),
    (1100, [1100, 0, 40, 2000], 2000, 32, 8, 64), (2300, [2300, 2301, 5], 2304, 20, 20, 64)]


@pytest.mark.parametrize("new,lengths,room,heads,kv,dim", HIGH_CACHED)
def test_many_new_tokens_over_caches(device, built_lib, new, lengths, room, heads, kv, dim):
    print(f"case high blocks over caches {new} {lengths} {heads}/{kv}x{dim}", flush=True)
    batch = len(lengths)
    assert built_lib.vdnh3_causal_block_rows(batch, new, heads, kv, dim, 0) == 256
    n = torch.tensor(lengths, dtype=torch.int32, device=device)
    q, k, v = (t.view(batch, -1, t.shape[1], dim) for t in _qkv(batch * max(new, room), heads, kv, dim, 70, loud=2.0))
    q, k, v = q[:, :new], k[:, :room], v[:, :room]
    got = _cached_in(0, q.to(device), k.to(device), v.to(device), n, dim ** -0.5).cpu()
    for b, m in enumerate(lengths):
        some = _edges(new, heads // kv, 256)
        want = po.attend(q[b, some], k[b], v[b], [m - new + i for i in some], dim ** -0.5)
        _check(got[b, some], want, dim)
        assert (got[b, :max(0, new - m)] == 0).all()
    # each key once here too
    zero, dk = torch.zeros_like(q).to(device), k.to(device)
    last = (n[:, None] - new + torch.arange(new, device=device)).view(-1)
    for first in range(0, room, 4 * dim + dim // 2):
        key = first + torch.arange(dim, device=device)
        out = _cached_in(0, zero, dk, _one_key_each(first, dk), n, 0.125)
        assert _same_quotients(out.view(-1, heads, dim), _quotients(key[None] <= last[:, None], last + 1)), first


def _edges(tokens, group, height):
    """The tokens at the first blocks' edges, at the last ones' and in between."""
    at = {0, 1, tokens - 2, tokens - 1} | set(range(0, tokens, max(1, tokens // 12)))
    for b in list(range(1, 6)) + list(range(tokens * group // height - 2, tokens * group // height + 1)):
        at |= {b * height // group + i for i in (-1, 0, 1)}
    return sorted(i for i in at if 0 <= i < tokens)


@pytest.mark.parametrize("lengths,heads,kv,dim,height", [c for c in PACKED if c[-1] == 256])
def test_high_blocks_against_float64(device, built_lib, lengths, heads, kv, dim, height):
    """Rows of random prompts; then values and keys that are not finite near the sequences' ends: rows in front of them are right
    as before, and rows that see them hold what the softmax gives."""
    from vdn_h3_amd.causal import causal_softmax_packed

    print(f"case high blocks {lengths} {heads}/{kv}x{dim}", flush=True)
    bounds = torch.tensor([0] + lengths).cumsum(0).tolist()
    assert built_lib.vdnh3_causal_block_rows(1, bounds[-1], heads, kv, dim, 0) == height
    q, k, v = _qkv(bounds[-1], heads, kv, dim, 71, loud=2.0)
    scale = dim ** -0.5
    fine = causal_softmax_packed(q.to(device), k.to(device), v.to(device), bounds, scale).cpu()
    for a, n in zip(bounds, lengths):
        some = _edges(n, heads // kv, height)
        if some:
            _check(fine[a:a + n][some], po.attend(q[a:a + n][some], k[a:a + n], v[a:a + n], some, scale), dim)
    k, v = k.clone(), v.clone()
    clean = torch.ones(bounds[-1], dtype=torch.bool)
    ends = []
    for a, n in zip(bounds, lengths):
        if n < 60:
            continue
        e = a + n
        v[e - 40, :, 3], v[e - 39, :, 4], v[e - 30], k[e - 20, :, 1] = torch.inf, -torch.inf, torch.nan, torch.nan
        clean[e - 40:e] = False
        ends.append((a, e))
    got = causal_softmax_packed(q.to(device), k.to(device), v.to(device), bounds, scale).cpu()
    # rows whose tiles hold one are made key by key, the others as before
    assert got[clean].isfinite().all()
    for a, e in ends:
        at = [e - a - i for i in (60, 45, 41)]
        _check(got[a:e][at], po.attend(q[a:e][at], k[a:e], v[a:e], at, scale), dim)
        assert (got[e - 40:e - 30, :, 3] == torch.inf).all() and (got[e - 39:e - 30, :, 4] == -torch.inf).all()
        at = [e - a - i for i in (40, 35, 31)]
        out, size, score = po.attend(q[a:e][at], k[a:e], v[a:e], at, scale)
        odd = ~out.isfinite()
        _check(got[a:e][at].masked_fill(odd, 0), (out.masked_fill(odd, 0), size.masked_fill(odd, 0), score), dim)
        assert got[e - 30:e].isnan().all()


@pytest.mark.parametrize("new,heads,kv,dim", [(1, 10, 2, 128), (5, 8, 1, 64), (40, 6, 2, 128)])
def test_a_request_beside_others_of_other_lengths(device, new, heads, kv, dim):
    """By the prompt kernel and in one range a request's result does not depend on the lengths beside it."""
    print(f"case beside others {new} {heads}/{kv}x{dim}", flush=True)
    q, k, v = (t.view(4, -1, t.shape[1], dim).to(device) for t in _qkv(4 * 600, heads, kv, dim, 72, loud=2.0))
    q = q[:, :new]
    for ranges in (0, 1):
        seen = []
        for lengths in ([600, 431, 0, 77], [3, 431, 600, 599], [431, 431, 431, 1]):
            n = torch.tensor(lengths, dtype=torch.int32, device=device)
            seen.append(_cached_in(ranges, q, k, v, n, 0.1)[1])
        assert torch.equal(seen[0], seen[1]) and torch.equal(seen[0], seen[2]), ranges
