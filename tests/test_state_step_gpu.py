"""New tokens over pools of recurrent states against float64 (GPU): linear attention and the gated delta rule.

Bar, from the arithmetic, relative to the absolute values of the terms: each token's update of a state is one rounding of the
decay, one of the product and one fused addition (3 2^-24, the decay's exponential 2^-22), the delta rule's dot product with the
key D more, the readout D more. N tokens add up. Outputs are rounded to bf16, 2^-8 of themselves.
"""

from __future__ import annotations

import pytest
import torch

from oracle import recurrent_oracle as ro

pytestmark = pytest.mark.gpu

BF = torch.bfloat16

CASES = [  # batch, new, slots, value heads, q / k heads, dim
    (1, 1, 1, 1, 1, 128), (3, 1, 5, 4, 2, 128), (2, 4, 2, 3, 3, 64), (5, 2, 9, 6, 2, 80), (4, 3, 6, 2, 1, 24), (2, 7, 4, 2, 2, 17),
    (2, 1, 3, 3, 1, 1), (70, 1, 90, 2, 2, 64), (130, 2, 130, 1, 1, 100), (1, 33, 2, 2, 2, 128), (16, 1, 16, 40, 40, 128),
    (3, 2, 4, 2, 2, 66), (3, 2, 4, 2, 2, 127)]


def _case(batch, new, count, heads, qk, dim, device, delta, seed=0):
    g = torch.Generator().manual_seed(dim + batch + seed)
    q, k = (torch.randn(batch, new, qk, dim, generator=g) for _ in range(2))
    if delta:
        q, k = (t / t.norm(dim=-1, keepdim=True) for t in (q, k))
    q, k = q.to(BF).to(device), k.to(BF).to(device)
    v = torch.randn(batch, new, heads, dim, generator=g).to(BF).to(device)
    pool = torch.randn(count, heads, dim, dim, generator=g).to(device)
    slots = torch.randperm(count, generator=g)[:batch].to(torch.int32).to(device)
    if delta:
        gates = (torch.rand(batch, new, heads, generator=g).to(device), -torch.rand(batch, new, heads, generator=g).to(device))
    else:
        gates = (-torch.exp2(-8.0 * torch.arange(heads) / heads).to(device),)
    return q, k, v, gates, pool, slots


def _step(delta, q, k, v, gates, pool, **kw):
    from vdn_h3_amd.causal_linear import causal_linear_step
    from vdn_h3_amd.gdn import gated_delta_step

    return gated_delta_step(q, k, v, *gates, pool, **kw) if delta else causal_linear_step(q, k, v, *gates, pool, 0.3, **kw)


def _want(delta, q, k, v, gates, pool, slots):
    parts = []
    for b, slot in enumerate(slots.tolist()):
        if delta:
            parts.append(ro.delta_recurrence(q[b], k[b], v[b], gates[0][b], gates[1][b], pool[slot]))
        else:
            parts.append(ro.linear_recurrence(q[b], k[b], v[b], gates[0], 0.3, pool[slot]))
    return [torch.stack(x) for x in zip(*parts)]


def _check(got, pool, want, slots, new, dim, delta):
    out, size, s, ssize = want
    per = 2.0 ** -22 + (8 + (2 * dim if delta else 0)) * 2.0 ** -24
    d = (got.double() - out).abs()
    bar = (new * per + (dim + 8) * 2.0 ** -24) * size + 2.0 ** -8 * out.abs() + 2.0 ** -134  # bf16's smallest step, halved
    assert (d <= bar).all(), (d / bar).max()
    d = (pool[slots.long()].double() - s).abs()
    bar = new * per * ssize
    assert (d <= bar).all(), (d / bar.clamp_min(1e-30)).max()


@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("batch,new,count,heads,qk,dim", CASES)
def test_against_float64(device, batch, new, count, heads, qk, dim, delta):
    print(f"case step {batch}x{new} of {count}, {heads}/{qk}x{dim} delta {delta}", flush=True)
    q, k, v, gates, pool, slots = _case(batch, new, count, heads, qk, dim, device, delta)
    before = pool.clone()
    want = _want(delta, q, k, v, gates, pool, slots)
    got = _step(delta, q, k, v, gates, pool, slots=slots)
    _check(got, pool, want, slots, new, dim, delta)
    rest = torch.ones(count, dtype=torch.bool, device=device)
    rest[slots.long()] = False
    assert torch.equal(pool[rest], before[rest])
    # without slots, views of one projection, odd strides, wide indices
    own = before[slots.long()].clone()
    assert torch.equal(_step(delta, q, k, v, gates, own), got) and torch.equal(own, pool[slots.long()])
    fused = torch.cat([q, k, v], 2).split((qk, qk, heads), 2)
    wide = before.clone()
    assert torch.equal(_step(delta, *fused, gates, wide, slots=slots.long()), got) and torch.equal(wide, pool)
    odd = [torch.empty(*t.shape[:3], dim + 3, dtype=BF, device=device)[..., 1:dim + 1].copy_(t) for t in (q, k, v)]
    again, out = before.clone(), torch.empty(batch, new, heads, dim + 1, dtype=BF, device=device)[..., :dim]
    # number by number instead of in 16 bytes: the same sums
    assert _step(delta, *odd, gates, again, slots=slots, out=out) is out
    assert torch.equal(out, got) and torch.equal(again, pool)


@pytest.mark.parametrize("delta", [False, True])
def test_pools_of_layers_and_of_heads(device, delta):
    q, k, v, gates, pool, slots = _case(3, 2, 5, 4, 2, 64, device, delta)
    layers = torch.zeros(5, 3, 4, 64, 64, device=device)
    layers[:, 1] = pool
    by_head = pool.transpose(0, 1).contiguous().transpose(0, 1)
    off = torch.zeros(pool.numel() + 1, device=device)[1:].view_as(pool).copy_(pool)  # off 16 bytes
    want = _step(delta, q, k, v, gates, pool, slots=slots)
    for view in (layers[:, 1], by_head, off):
        assert torch.equal(_step(delta, q, k, v, gates, view, slots=slots), want) and torch.equal(view, pool)
    assert not layers[:, 0].any() and not layers[:, 2].any()


@pytest.mark.parametrize("delta", [False, True])
def test_idle_requests_and_a_slot_named_twice(device, delta):
    q, k, v, gates, pool, _ = _case(70, 2, 12, 2, 1, 64, device, delta)
    slots = torch.full((70,), -1, dtype=torch.int32, device=device)
    live = {3: 7, 5: 0, 66: 11}
    for b, s in live.items():
        slots[b] = s
    slots[8], slots[9], slots[10] = 12, -2 ** 31, 2 ** 31 - 1  # outside the pool
    slots[6], slots[68] = 7, 0  # taken by requests 3 and 5
    before, want = pool.clone(), {}
    for b, s in live.items():
        alone = before[s:s + 1].clone()
        one = (gates[0][b:b + 1], gates[1][b:b + 1]) if delta else gates
        want[b] = _step(delta, q[b:b + 1], k[b:b + 1], v[b:b + 1], one, alone)[0], alone[0]
    out = _step(delta, q, k, v, gates, pool, slots=slots)
    for b in range(70):
        if b in live:
            assert torch.equal(out[b], want[b][0]) and torch.equal(pool[live[b]], want[b][1])
        elif b in (6, 68):
            assert out[b].isnan().all()
        else:
            assert (out[b] == 0).all()
    others = [s for s in range(12) if s not in live.values()]
    assert torch.equal(pool[others], before[others])


@pytest.mark.parametrize("delta", [False, True])
def test_values_that_are_no_numbers_end_their_channel(device, delta):
    q, k, v, gates, pool, _ = _case(2, 3, 2, 2, 2, 80, device, delta)
    clean = pool.clone()
    want = _step(delta, q, k, v, gates, clean)
    v[0, 1, 0, 5] = torch.inf
    got = _step(delta, q, k, v, gates, pool)
    assert not got[0, 1:, 0, 5].isfinite().any() and not pool[0, 0, 5].isfinite().any()
    got[0, 1:, 0, 5], pool[0, 0, 5] = want[0, 1:, 0, 5], clean[0, 0, 5]
    assert torch.equal(got, want) and torch.equal(pool, clean)


def test_prompts_then_tokens(device):
    """A prompt in chunks and the rest token by token is the prompt in chunks: both forms of both rules."""
    from vdn_h3_amd.causal_linear import causal_linear_packed, causal_linear_step
    from vdn_h3_amd.gdn import chunk_gated_delta_rule, gated_delta_step

    for dim in (128, 48):
        q, k, v, (decay,), _, _ = _case(1, 90, 1, 4, 4, dim, device, False)
        whole, end = causal_linear_packed(q[0], k[0], v[0], decay, [0, 90], 0.3, output_final_state=True)
        _, size, _, ssize = ro.linear_recurrence(q[0], k[0], v[0], decay, 0.3)
        head, state = causal_linear_packed(q[0, :70], k[0, :70], v[0, :70], decay, [0, 70], 0.3, output_final_state=True)
        tail = [causal_linear_step(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], decay, state, 0.3)[0] for t in range(70, 90)]
        d = (torch.cat([head, *tail]).double() - whole.double()).abs()
        assert (d <= 2 * (2.0 ** -14 * size + 2.0 ** -8 * whole.double().abs())).all()
        assert ((state[0].double() - end[0].double()).abs() <= 2.0 ** -14 * ssize).all()

        q, k, v, (beta, g), _, _ = _case(1, 90, 1, 4, 4, dim, device, True)
        _, state = chunk_gated_delta_rule(q[0, :70], k[0, :70], v[0, :70], beta[0, :70], g[0, :70], output_final_state=True)
        tail = gated_delta_step(q[:, 70:], k[:, 70:], v[:, 70:], beta[:, 70:], g[:, 70:], state[None])
        whole, end = chunk_gated_delta_rule(q[0], k[0], v[0], beta[0], g[0], output_final_state=True)
        # the chunk form rounds its operands to bf16 (W, U, K and Q with decays): a few 2^-8 of rows of unit keys
        for a, b in ((tail[0], whole[70:]), (state[:, :, :], end)):
            a, b = a.double(), b.double()
            assert (a - b).norm() <= 4 * 2.0 ** -8 * b.norm()


@pytest.mark.parametrize("delta", [False, True])
def test_replays_take_other_slots_and_states(device, delta):
    q, k, v, gates, pool, slots = _case(4, 1, 9, 2, 2, 128, device, delta)
    out, mirror = torch.zeros_like(v), pool.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(delta, q, k, v, gates, pool.clone(), slots=slots, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(delta, q, k, v, gates, pool, slots=slots, out=out)
    for now in (slots.tolist(), [8, -1, 2, 3], [0, 1, 2, 3], [5, 5, -1, 8]):
        slots.copy_(torch.tensor(now, dtype=torch.int32))
        v.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        want = _step(delta, q, k, v, gates, mirror, slots=slots)
        assert torch.equal(torch.nan_to_num(out, 9.0), torch.nan_to_num(want, 9.0)) and torch.equal(pool, mirror)


@pytest.mark.parametrize("delta", [False, True])
def test_pools_past_32_bits(device, delta):
    """States at 2^31 elements and more, between slots and between heads."""
    count = 66000
    q, k, v, gates, _, _ = _case(2, 1, 2, 2, 2, 128, device, delta)
    whole = torch.empty(2, count, 128, 128, device=device)
    for pool in (whole.view(count, 2, 128, 128), whole.transpose(0, 1)):
        small = torch.randn(2, 2, 128, 128, device=device)
        pool[0], pool[count - 1] = small[0], small[1]
        pool[count - 2] = 5.0
        slots = torch.tensor([0, count - 1], dtype=torch.int64, device=device)
        got = _step(delta, q, k, v, gates, pool, slots=slots)
        assert torch.equal(got, _step(delta, q, k, v, gates, small))
        assert torch.equal(pool[0], small[0]) and torch.equal(pool[count - 1], small[1]) and (pool[count - 2] == 5.0).all()
