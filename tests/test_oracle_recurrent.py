"""The float64 oracle of recurrent states and adapters against forms that share no step with it."""

from __future__ import annotations

import torch
import torch.nn.functional as F

from oracle import gdn_oracle, recurrent_oracle as ro


def test_linear_recurrence_is_the_sum_over_all_earlier_tokens():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(11, h, 6, generator=g).double() for h in (2, 2, 4))
    rate = -torch.rand(4, generator=g).double()
    s0 = torch.randn(4, 6, 6, generator=g).double()
    out, size, s, ssize = ro.linear_recurrence(q, k, v, rate, 0.5, s0)
    i = torch.arange(11).double()
    for h in range(4):
        w = torch.exp(rate[h] * (i[:, None] - i)).tril() * (q[:, h // 2] @ k[:, h // 2].t())
        want = 0.5 * (w @ v[:, h] + torch.exp(rate[h] * (i + 1))[:, None] * (q[:, h // 2] @ s0[h].t()))
        assert torch.allclose(out[:, h], want, rtol=1e-12)
        end = torch.exp(rate[h] * 11) * s0[h] + (v[:, h] * torch.exp(rate[h] * (10 - i))[:, None]).t() @ k[:, h // 2]
        assert torch.allclose(s[h], end, rtol=1e-12)
    assert (size >= out.abs() - 1e-12).all() and (ssize >= s.abs() - 1e-12).all()


def test_one_channel_by_hand():
    one = torch.ones(4, 1, 1)
    half = torch.tensor([0.5]).log()
    out, size, s, _ = ro.linear_recurrence(one, one, one, half, 1.0)
    assert torch.allclose(out.flatten(), torch.tensor([1.0, 1.5, 1.75, 1.875], dtype=torch.float64), atol=1e-7)
    # sum of 2^-d (1 + d): 1, 2, 2.75, 3.25
    assert torch.allclose(size.flatten(), torch.tensor([1.0, 2.0, 2.75, 3.25], dtype=torch.float64), atol=1e-6)
    gone, _, s, _ = ro.linear_recurrence(one, one, 3 * one, torch.tensor([-torch.inf]), 1.0, torch.full((1, 1, 1), 7.0))
    assert (gone == 3).all() and (s == 3).all()


def test_delta_recurrence_is_the_gated_deltanets():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(5, 3, 7, generator=g) for _ in range(3))
    beta, rate, s0 = torch.rand(5, 3, generator=g), -torch.rand(5, 3, generator=g), torch.randn(3, 7, 7, generator=g)
    out, size, s, ssize = ro.delta_recurrence(q, k, v, beta, rate, s0)
    want, end = gdn_oracle.recurrence(q, k, v, beta, rate, s0)
    assert torch.allclose(out, want, rtol=1e-11) and torch.allclose(s, end, rtol=1e-11)
    assert (size >= out.abs() - 1e-12).all() and (ssize >= s.abs() - 1e-12).all()


def test_adapters_by_linear_layers():
    g = torch.Generator().manual_seed(3)
    x, y = torch.randn(5, 8, generator=g).double(), torch.randn(5, 6, generator=g).double()
    down, up = torch.randn(2, 3, 8, generator=g).double(), torch.randn(2, 6, 3, generator=g).double()
    out, size = ro.adapters(y, x, down, up, torch.tensor([2.0, -1.0]), torch.tensor([0, 1, -1, 1, 9]))
    assert torch.equal(out[2], y[2]) and torch.equal(out[4], y[4])
    assert torch.allclose(out[0], y[0] + 2 * F.linear(F.linear(x[0], down[0]), up[0]))
    assert torch.allclose(out[[1, 3]], y[[1, 3]] - F.linear(F.linear(x[[1, 3]], down[1]), up[1]))
    assert (size >= out.abs() - 1e-12).all()
