"""The operators of a layer that serves many requests, together as they are used (GPU): a projection with each request's adapter,
prompts packed one behind another, new tokens over the pool of states, the projection out. Every stage is held against float64 on
the inputs that it had, so its bar is its own:

projections: the product is rounded to bf16 (2^-8 of itself), and so is its sum with the adapter's (2^-8 of the sum; its other terms
are those of test_adapters_gpu); attention and states: the bars of test_causal_linear_gpu and test_state_step_gpu.
"""

from __future__ import annotations

import pytest
import torch

from oracle import recurrent_oracle as ro

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
WIDTH, HEADS, QK, DIM, SLOTS = 320, 4, 2, 64, 6
SCALE = DIM ** -0.5


class _Layer:
    def __init__(self, device, delta):
        from vdn_h3_amd.adapters import LowRankAdapters
        from vdn_h3_amd.linear import HipLinear

        g = torch.Generator().manual_seed(11)
        rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        inner = (HEADS + 2 * QK) * DIM
        self.weights = [(rand(inner, WIDTH) * WIDTH ** -0.5).to(BF).to(device), (rand(WIDTH, HEADS * DIM) * 0.06).to(BF).to(device)]
        self.pairs = [((rand(3, rank, w.shape[1]) * w.shape[1] ** -0.5).to(BF).to(device),
                       (rand(3, w.shape[0], rank) * 0.3).to(BF).to(device), torch.rand(3, generator=g).to(device))
                      for w, rank in zip(self.weights, (16, 40))]
        self.adapters = [LowRankAdapters(*p) for p in self.pairs]
        self.projections = [HipLinear(w) for w in self.weights]
        self.gate = (rand(HEADS, WIDTH) * WIDTH ** -0.5).to(BF).to(device)
        self.decay = -torch.exp2(-4.0 * torch.arange(HEADS) / HEADS).to(device)
        self.delta = delta

    def project(self, i, x, index, check):
        got = self.projections[i](x, adapters=self.adapters[i], adapter_index=index)
        if check:
            down, up, scales = self.pairs[i]
            base, room = x.double() @ self.weights[i].double().t(), x.double().abs() @ self.weights[i].double().abs().t()
            want, size = ro.adapters(base, x, down, up, scales, index)
            bar = ((x.shape[1] + 2 * down.shape[1] + 8) * 2.0 ** -24 + 2.0 ** -16) * (size + room) + \
                2.0 ** -8 * (base.abs() * (1 + 2.0 ** -8) + want.abs())
            d = (got.double() - want).abs()
            assert (d <= bar).all(), (d / bar).max()
        return got

    def operands(self, x, index, check):
        qkv = self.project(0, x, index, check)
        q, k, v = (t.unflatten(1, (-1, DIM)) for t in qkv.split((QK * DIM, QK * DIM, HEADS * DIM), 1))
        q, k = (torch.nn.functional.normalize(t.float(), dim=-1).to(BF) for t in (q, k))
        return q, k, v

    def gates(self, x):
        from vdn_h3_amd.linear import sigmoid_linear

        beta = sigmoid_linear(x, self.gate).float()
        return beta, -beta.flip(-1)

    def prompts(self, x, bounds, index, pool, slots, check=True):
        """The prompts of requests whose states go to ``pool[slots]``."""
        from vdn_h3_amd.causal_linear import causal_linear_packed
        from vdn_h3_amd.gdn import chunk_gated_delta_rule

        q, k, v = self.operands(x, index, check)
        if self.delta:
            beta, g = self.gates(x)
            o = torch.empty_like(v)
            for i, slot in enumerate(slots):
                a, b = bounds[i], bounds[i + 1]
                wide = [t[a:b].repeat_interleave(HEADS // QK, 1) for t in (q, k)]
                o[a:b], pool[slot] = chunk_gated_delta_rule(*wide, v[a:b], beta[a:b], g[a:b], output_final_state=True)
        else:
            o, states = causal_linear_packed(q, k, v, self.decay, bounds, SCALE, output_final_state=True)
            pool[slots] = states
            for i, (a, b) in enumerate(zip(bounds, bounds[1:]) if check else ()):
                out, size, s, ssize = ro.linear_recurrence(q[a:b], k[a:b], v[a:b], self.decay, SCALE)
                bar = ((DIM + b - a + 64) * 2.0 ** -24 + 2.0 ** -16 + 2.0 ** -22) * size + 2.0 ** -8 * out.abs()
                assert ((o[a:b].double() - out).abs() <= bar).all()
                assert ((states[i].double() - s).abs() <= ((b - a + 64) * 2.0 ** -24 + 2.0 ** -22) * ssize).all()
        return self.project(1, o.flatten(1), index, check)

    def tokens(self, x, index, pool, slots, check=True):
        """New tokens ``x`` ``[requests, new, width]`` over their states."""
        from vdn_h3_amd.causal_linear import causal_linear_step
        from vdn_h3_amd.gdn import gated_delta_step

        batch, new, _ = x.shape
        rows = x.flatten(0, 1)
        each = index if new == 1 else index.repeat_interleave(new)
        q, k, v = (t.unflatten(0, (batch, new)) for t in self.operands(rows, each, check))
        before = pool.clone() if check else None
        if self.delta:
            beta, g = (t.unflatten(0, (batch, new)) for t in self.gates(rows))
            o = gated_delta_step(q, k, v, beta, g, pool, slots=slots)
        else:
            o = causal_linear_step(q, k, v, self.decay, pool, SCALE, slots=slots)
        if check:
            per = 2.0 ** -22 + (8 + (2 * DIM if self.delta else 0)) * 2.0 ** -24
            for i, slot in enumerate(slots.tolist()):
                if slot < 0:
                    assert not o[i].any()
                    continue
                if self.delta:
                    out, size, s, ssize = ro.delta_recurrence(q[i], k[i], v[i], beta[i], g[i], before[slot])
                else:
                    out, size, s, ssize = ro.linear_recurrence(q[i], k[i], v[i], self.decay, SCALE, before[slot])
                bar = (new * per + (DIM + 8) * 2.0 ** -24) * size + 2.0 ** -8 * out.abs()
                assert ((o[i].double() - out).abs() <= bar).all()
                assert ((pool[slot].double() - s).abs() <= new * per * ssize).all()
                before[slot] = pool[slot]
            assert torch.equal(torch.nan_to_num(pool, 7.0), torch.nan_to_num(before, 7.0))  # nobody else's state
        return self.project(1, o.flatten(2).flatten(0, 1), each, check).unflatten(0, (batch, new))


def _inputs(device, *shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + shape[0])).to(BF).to(device)


def _integers(device, *values):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _started(device, layer, check=False):
    bounds, slots = [0, 130, 131, 196], [4, 0, 2]
    index = _integers(device, -1, 1, 0)
    pool = torch.full((SLOTS, HEADS, DIM, DIM), torch.nan, device=device)
    of_rows = index.repeat_interleave(torch.tensor([130, 1, 65], device=device))
    y = layer.prompts(_inputs(device, 196, WIDTH), bounds, of_rows, pool, slots, check)
    assert y.isfinite().all()
    return pool, index, _integers(device, *slots)


@pytest.mark.parametrize("delta", [False, True])
def test_prompts_then_tokens(device, delta):
    layer = _Layer(device, delta)
    pool, index, slots = _started(device, layer, True)
    for new, now in ((1, slots), (1, _integers(device, 4, -1, 2)), (4, slots), (1, slots)):
        y = layer.tokens(_inputs(device, 3, new, WIDTH, seed=new), index, pool, now)
        assert y.isfinite().all()
    assert pool[[1, 3, 5]].isnan().all() and pool[[0, 2, 4]].isfinite().all()


@pytest.mark.parametrize("delta", [False, True])
def test_two_graphs_over_one_pool(device, delta):
    """Tokens of two and of three requests, captured; replays in turn with prompts and eager tokens between, against an eager copy."""
    layer = _Layer(device, delta)
    pool, _, _ = _started(device, layer)
    mirror = pool.clone()
    graphs = []
    for batch in (2, 3):
        x, index, slots = _inputs(device, batch, 1, WIDTH), _integers(device, *range(batch)), _integers(device, *[0, 2, 4][:batch])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer.tokens(x, index, pool.clone(), slots, False)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer.tokens(x, index, pool, slots, False)
        graphs.append((graph, x, index, slots, y))
    for turn, (names, where) in enumerate([((1, -1), (2, 0)), ((0, 2, 1), (4, -1, 0)), ((2, 2), (4, 2)), ((-1, 0, 0), (0, 2, 4))]):
        graph, x, index, slots, y = graphs[turn % 2]
        index.copy_(_integers(device, *names))
        slots.copy_(_integers(device, *where))
        x.copy_(_inputs(device, *x.shape, seed=20 + turn))
        graph.replay()
        want = layer.tokens(x, index, mirror, slots, False)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(torch.nan_to_num(pool, 7.0), torch.nan_to_num(mirror, 7.0)), turn
        for p in (pool, mirror):
            layer.prompts(_inputs(device, 70, WIDTH, seed=turn), [0, 70], torch.ones(70, dtype=torch.int32, device=device), p, [0], False)


@pytest.mark.parametrize("delta", [False, True])
def test_on_another_stream(device, delta):
    layer = _Layer(device, delta)
    results = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            pool, index, slots = _started(device, layer)
            results.append([layer.tokens(_inputs(device, 3, n, WIDTH, seed=n), index, pool, slots, False) for n in (1, 2)] + [pool])
        stream.synchronize()
    assert all(torch.equal(torch.nan_to_num(a, 7.0), torch.nan_to_num(b, 7.0)) for a, b in zip(*results))


def test_calls_of_two_streams_at_once(device):
    """Prompts, tokens and adapters of two streams in turn, without a wait between them: the results of one after another."""
    layers = [_Layer(device, False), _Layer(device, True)]
    pools = [_started(device, layer) for layer in layers]
    prompts = [_inputs(device, 900 + 64 * i, WIDTH, seed=i) for i in range(2)]
    tokens = [_inputs(device, 3, 1, WIDTH, seed=50 + i) for i in range(2)]
    rows = [torch.arange(x.shape[0], device=device, dtype=torch.int32) % 4 - 1 for x in prompts]

    def turn(i, pool):
        y = layers[i].prompts(prompts[i], [0, prompts[i].shape[0]], rows[i], pool, [1], False)
        return y, layers[i].tokens(tokens[i], pools[i][1], pool, pools[i][2], False)

    want = []
    for i in range(2):
        pool = pools[i][0].clone()
        want.append([turn(i, pool) for _ in range(4)] + [pool])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(turn(i, pools[i][0]))
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(torch.nan_to_num(pools[i][0], 7.0), torch.nan_to_num(want[i][-1], 7.0))
        assert all(torch.equal(a, b) for x, y in zip(got[i], want[i]) for a, b in zip(x, y))


def _leave_in_memory(value):
    """Memory of every size that an allocation is cut from, freed with ``value`` (None: normal numbers) in it."""
    blocks = [torch.empty(1 << n, device="cuda") for n in (26, 24, 22, 20, 18, 16, 12) for _ in range(4)]
    for t in blocks:
        t.normal_() if value is None else t.fill_(value)


def test_calls_repeat_bit_for_bit(device):
    """Every operator on the same inputs, whatever its outputs and workspaces held before and whatever ran in between."""
    from vdn_h3_amd.adapters import LowRankAdapters
    from vdn_h3_amd.causal_linear import causal_linear_packed, causal_linear_step
    from vdn_h3_amd.gdn import gated_delta_step
    from vdn_h3_amd.linear import HipLinear

    g = torch.Generator().manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    calls = []
    for bounds, heads, dim in (([0, 1135], 20, 64), ([0, 77, 78, 78, 1000, 1500], 8, 128), ([0, 6000], 4, 128), ([0, 30], 8, 128)):
        q, k, v = (rand(bounds[-1], n, dim).to(BF).to(device) for n in (heads // 4, heads // 4, heads))
        decay, initial = -torch.rand(heads, generator=g).to(device), rand(len(bounds) - 1, heads, dim, dim).to(device)
        calls.append(lambda a=(q, k, v, decay, bounds, 0.1), s=initial: causal_linear_packed(
            *a, initial_state=s, output_final_state=True))
    for batch, new, dim in ((9, 1, 128), (5, 4, 64), (3, 2, 80)):
        q, k, v = (rand(batch, new, n, dim).to(BF).to(device) for n in (4, 4, 8))
        pool, beta = rand(batch, 8, dim, dim).to(device), torch.rand(batch, new, 8, generator=g).to(device)

        def steps(a=(q, k / 8, v), pool=pool, beta=beta):
            pools = pool.clone(), pool.clone()
            return causal_linear_step(*a, -beta[0, 0], pools[0], 0.1), gated_delta_step(*a, beta, -beta, pools[1]), *pools

        calls.append(steps)
    for rows, width, out, n, rank in ((1, 640, 5120, 2, 16), (64, 5120, 256, 1, 32), (60, 640, 512, 9, 64), (700, 256, 384, 3, 40),
                                      (9000, 64, 128, 3, 8)):
        layer = HipLinear((rand(out, width) * width ** -0.5).to(BF).to(device))
        handle = LowRankAdapters(rand(n, rank, width).to(BF).to(device), rand(n, out, rank).to(BF).to(device))
        x, index = rand(rows, width).to(BF).to(device), torch.randint(-1, n, (rows,), generator=g, dtype=torch.int32).to(device)
        calls.append(lambda layer=layer, x=x, h=handle, i=index: (layer(x, adapters=h, adapter_index=i),))
    want = [call() for call in calls]
    for value in (torch.nan, None, 0.0, None):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        _leave_in_memory(value)
        got = [call() for call in calls]
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
