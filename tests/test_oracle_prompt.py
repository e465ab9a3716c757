"""The float64 oracle of the prompt encoder's operators against closed forms and torch in float64."""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from oracle import prompt_oracle as po


def test_norm_of_a_constant_row_and_against_torch():
    x = torch.full((1, 16), 3.0)
    t, y = po.residual_rmsnorm(x, -x / 3, torch.full((16,), 2.0), 0.0)
    assert torch.equal(t, torch.full((1, 16), 2.0, dtype=torch.float64)) and torch.allclose(y, torch.full_like(y, 2.0))
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(5, 40, generator=g).double(), torch.randn(40, generator=g).double()
    assert torch.allclose(po.residual_rmsnorm(x, None, w, 1e-3)[1], F.rms_norm(x, (40,), w, 1e-3), rtol=1e-13)


def test_quarter_turns_per_axis():
    # theta 1: every pair turns by its axis's position in radians
    x = torch.zeros(3, 1, 18, dtype=torch.float64)
    x[..., :8] = 1.0
    x[..., 16:] = 5.0
    pos = torch.tensor([[0.0, math.pi / 2, math.pi], [math.pi, 0.0, math.pi / 2]], dtype=torch.float64)
    y, size, angle = po.rotate_axes(x, None, 0.0, pos, (3, 5), 1.0, "shared")
    want = {0: (1, 0), 1: (0, 1), 2: (-1, 0)}
    for row in range(3):
        assert torch.allclose(y[row, 0, 0:3], torch.full((3,), float(want[row][0]), dtype=torch.float64), atol=1e-15)
        assert torch.allclose(y[row, 0, 8:11], torch.full((3,), float(want[row][1]), dtype=torch.float64), atol=1e-15)
    assert torch.allclose(y[0, 0, 3:8], torch.full((5,), -1.0, dtype=torch.float64)) and (y[..., 16:] == 5).all()
    assert torch.equal(size[..., :16], torch.ones_like(size[..., :16])) and angle.shape == (3, 8)


def test_ladders():
    pos = torch.ones(2, 1)
    x = torch.zeros(1, 1, 16)
    shared = po.rotate_axes(x, None, 0.0, pos, (2, 6), 16.0, "shared")[2][0]
    own = po.rotate_axes(x, None, 0.0, pos, (2, 6), 16.0, "per_axis")[2][0]
    assert torch.allclose(shared, 16.0 ** (-torch.arange(8).double() / 8))
    assert torch.allclose(own, torch.cat([16.0 ** (-torch.arange(n).double() / n) for n in (2, 6)]))


def test_attention_against_torch_and_by_hand():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(9, h, 8, generator=g).double() for h in (6, 2, 2))
    out, size, score = po.packed(q, k, v, [0, 4, 4, 9], 0.5)
    for a, b in ((0, 4), (4, 9)):
        want = F.scaled_dot_product_attention(*(t[a:b].transpose(0, 1).repeat_interleave(6 // t.shape[1], 0)
                                                for t in (q, k, v)), is_causal=True, scale=0.5).transpose(0, 1)
        assert torch.allclose(out[a:b], want, rtol=1e-12)
    assert torch.allclose(out[4], v[4].repeat_interleave(3, 0)) and (size >= out.abs() - 1e-12).all()
    # new tokens over a cache are the last rows of the whole; one in front of the first key sees nothing
    o, _, _ = po.cached(q[None, 7:], k[None], v[None], [9], 0.5)
    whole = po.packed(q, k, v, [0, 9], 0.5)[0]
    assert torch.allclose(o[0], whole[7:])
    o, _, _ = po.cached(q[None, 7:], k[None], v[None], [1], 0.5)
    assert (o[0, 0] == 0).all() and torch.allclose(o[0, 1], v[0].repeat_interleave(3, 0))
