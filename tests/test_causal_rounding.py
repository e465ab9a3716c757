"""Over ranges of caches a probability is two bf16 numbers: a bar that tells them from one.

From the arithmetic: p as a bf16 number and the rest as another is off by 2^-8 * 2^-8 = 2^-16 of p. A score is off by
(D + 8) 2^-24 of scale sum |q_d k_d| (`score`), an exponential by 2^-20 of itself with its argument's rounding: e = (D + 8)
2^-24 score + 2^-20 (1 + score), for p itself, where a later maximum scales it, and where the wavefronts' and the ranges'
sums are merged. Sums of n keys in fp32, each number's two parts on a quarter of the tiles, add at most n + 64 roundings one
behind another, in the values' sum and in the row's alike. With A = sum p |v| the result is off by 2 (2^-16 + 3 e + (n + 64)
2^-24) A and 2^-8 of itself. One bf16 number is off by up to 2^-8 of p: near-equal probabilities of values with either sign
make results that are small next to A, where that shows.
"""

from __future__ import annotations

import pytest
import torch

from oracle import prompt_oracle as po

BF = torch.bfloat16


def _case(batch, new, room, heads, kv, dim, seed):
    g = torch.Generator().manual_seed(seed)
    q = (0.25 * torch.randn(batch, new, heads, dim, generator=g)).to(BF)
    return q, *(torch.randn(batch, room, kv, dim, generator=g).to(BF) for _ in range(2))


def _over(got, want, keys, dim):
    """The largest error in parts of the bar."""
    out, size, score = want
    e = ((dim + 8) * 2.0 ** -24 * score + 2.0 ** -20 * (1 + score))[..., None]
    bar = 2 * (2.0 ** -16 + 3 * e + (keys + 64) * 2.0 ** -24) * size + 2.0 ** -8 * out.abs()
    return ((got.double().cpu() - out).abs() / bar.clamp_min(1e-30)).max().item()


CASES = [  # new tokens, lengths, heads, kv heads, dim
    (1, [64, 100, 300, 5], 40, 8, 128), (4, [200, 33, 300], 12, 2, 64), (20, [300, 140], 10, 2, 128)]


@pytest.mark.parametrize("new,lengths,heads,kv,dim", CASES)
def test_the_bar_tells_one_number_from_two(new, lengths, heads, kv, dim):
    q, k, v = _case(len(lengths), new, max(lengths), heads, kv, dim, 80)
    scale = dim ** -0.5
    want = po.cached(q, k, v, lengths, scale)
    group = heads // kv
    for parts in (1, 2):
        worst = 0.0
        for b, m in enumerate(lengths):
            got = torch.zeros(new, heads, dim, dtype=torch.float64)
            for i in range(max(0, new - m), new):
                n = m - new + i + 1
                s = torch.einsum("hgd,jhd->hgj", q[b, i].double().view(kv, group, dim), k[b, :n].double()) * scale
                p = torch.exp(s - s.amax(-1, keepdim=True)).float()
                rounded = p.to(BF).double()
                if parts == 2:
                    rounded += (p - p.to(BF).float()).to(BF).double()
                out = torch.einsum("hgj,jhd->hgd", rounded, v[b, :n].double()) / rounded.sum(-1, keepdim=True)
                got[i] = out.reshape(heads, dim)
            worst = max(worst, _over(got.to(BF), [w[b] for w in want], m, dim))
        assert worst > 2 if parts == 1 else worst <= 1, (parts, worst)


@pytest.mark.gpu
@pytest.mark.parametrize("new,lengths,heads,kv,dim", CASES)
def test_ranges_keep_two_numbers(device, new, lengths, heads, kv, dim):
    from test_causal_gpu import _cached_in

    q, k, v = _case(len(lengths), new, max(lengths), heads, kv, dim, 81)
    scale = dim ** -0.5
    want = po.cached(q, k, v, lengths, scale)
    n = torch.tensor(lengths, dtype=torch.int32, device=device)
    for ranges in (1, 2, 3, 8):
        print(f"case rounding {ranges} ranges, {new} new tokens {heads}/{kv}x{dim}", flush=True)
        got = _cached_in(ranges, q.to(device), k.to(device), v.to(device), n, scale)
        for b, m in enumerate(lengths):
            over = _over(got[b], [w[b] for w in want], m, dim)
            assert over <= 1, (ranges, b, over)
