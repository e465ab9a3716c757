"""Causal linear attention of packed prompts against float64 (GPU).

Bar, from the arithmetic, relative to the absolute values of the terms (`size`, weighted by 1 + d |log2 a| for a term d tokens
back): a dot product of D bf16 products in fp32 is off by at most D 2^-24, the scores and the state that meet q are two bf16
numbers, off by 2^-17 (2^-8 of 2^-9), the decays are off by 2^-22 (1 + d |log2 a|) (log2 a and its multiple rounded, v_exp_f32),
and of T terms added one after another in fp32 each sum rounds once, T 2^-24. The states take no part of it in fewer than 24 bits.
Outputs are rounded once more: 2^-8 of themselves.
"""

from __future__ import annotations

import pytest
import torch

from oracle import recurrent_oracle as ro

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _case(rows, heads, qk, dim, seed, device, sequences=0):
    g = torch.Generator().manual_seed(seed)
    q, k = ((torch.randn(rows, qk, dim, generator=g)).to(BF).to(device) for _ in range(2))
    v = torch.randn(rows, heads, dim, generator=g).to(BF).to(device)
    decay = -torch.exp2(-8.0 * torch.arange(heads) / heads).to(device)
    initial = torch.randn(sequences, heads, dim, dim, generator=g).to(device) if sequences else None
    return q, k, v, decay, initial


def _want(q, k, v, decay, bounds, scale, initial):
    parts = [ro.linear_recurrence(q[a:b], k[a:b], v[a:b], decay, scale, None if initial is None else initial[i])
             for i, (a, b) in enumerate(zip(bounds, bounds[1:]))]
    return [torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]), torch.stack([p[2] for p in parts]),
            torch.stack([p[3] for p in parts])]


def _check(got, want, dim, longest):
    o, final = got
    out, size, s, ssize = want
    bar = ((dim + longest + 64) * 2.0 ** -24 + 2.0 ** -16 + 2.0 ** -22) * size + 2.0 ** -8 * out.abs()
    d = (o.double() - out).abs()
    assert (d <= bar).all(), (d / bar.clamp_min(1e-30)).max()
    d = (final.double() - s).abs()
    bar = ((longest + 64) * 2.0 ** -24 + 2.0 ** -22) * ssize
    assert (d <= bar).all(), (d / bar.clamp_min(1e-30)).max()


def _bounds(lengths):
    bounds = [0]
    for n in lengths:
        bounds.append(bounds[-1] + n)
    return bounds


def _in_ranges(ranges, q, k, v, decay, bounds, scale, initial):
    """``vdnh3_causal_linear_packed`` in that many ranges, a workspace of NaNs and outputs of sevens."""
    from vdn_h3_amd import _lib

    lib = _lib.lib()
    rows, heads, dim = v.shape
    size = lib.vdnh3_causal_linear_workspace_bytes(ranges, heads, dim)
    work = torch.full((max(size, 16),), 0xFF, dtype=torch.uint8, device=q.device)
    out = torch.full(v.shape, 7.0, dtype=BF, device=q.device)
    final = torch.full((len(bounds) - 1, heads, dim, dim), 7.0, device=q.device)
    cu = torch.tensor(bounds, dtype=torch.int32, device=q.device)
    _lib.check(lib.vdnh3_causal_linear_packed(
        q.data_ptr(), *q.stride()[:2], k.data_ptr(), *k.stride()[:2], v.data_ptr(), *v.stride()[:2], out.data_ptr(),
        *out.stride()[:2], decay.data_ptr(), cu.data_ptr(), _lib.ptr(initial), final.data_ptr(), len(bounds) - 1, rows, heads,
        q.shape[1], dim, scale, ranges, work.data_ptr(), size, _lib.stream_handle(q.device)), "packed")
    return out, final


CASES = [  # lengths, value heads, q / k heads, dim
    ([1], 1, 1, 64), ([1], 3, 1, 128), ([2, 63], 4, 4, 64), ([64], 2, 2, 128), ([65, 0, 1], 6, 2, 128), ([0, 0, 130, 0], 4, 2, 64),
    ([127, 128, 129], 2, 1, 128), ([77, 1, 300, 0, 64], 8, 8, 64), ([1000], 5, 5, 128), ([640, 3], 16, 4, 64),
    ([200, 1, 90], 6, 2, 80), ([100], 4, 4, 24), ([33, 70], 3, 3, 17), ([5] * 70, 2, 2, 128), ([1] * 600, 1, 1, 64)]


@pytest.mark.parametrize("lengths,heads,qk,dim", CASES)
@pytest.mark.parametrize("begun", [False, True])
def test_against_float64(device, lengths, heads, qk, dim, begun):
    from vdn_h3_amd.causal_linear import causal_linear_packed

    print(f"case linear {lengths[:8]} {heads}/{qk}x{dim} {begun}", flush=True)
    bounds = _bounds(lengths)
    q, k, v, decay, initial = _case(bounds[-1], heads, qk, dim, len(lengths) + dim, device, len(lengths) if begun else 0)
    scale = dim ** -0.5
    cu = torch.tensor(bounds, dtype=torch.int32, device=device)
    got = causal_linear_packed(q, k, v, decay, cu, scale, initial_state=initial, output_final_state=True)
    _check(got, _want(q, k, v, decay, bounds, scale, initial), dim, max(lengths))
    out, none = causal_linear_packed(q, k, v, decay, bounds, scale, initial_state=initial)
    assert none is None and torch.equal(out, got[0])
    if dim % 8 == 0:  # views of one projection, heads in front of rows, one head's keys for all
        fused = torch.cat([q, k, v], 1).split((qk, qk, heads), 1)
        first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
        for args in (fused, first):
            again = causal_linear_packed(*args, decay, cu.long(), scale, initial_state=initial, output_final_state=True)
            assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
        wide = causal_linear_packed(q[:, :1].expand(-1, heads, -1), k[:, :1].expand(-1, heads, -1), v, decay, cu, scale,
                                    initial_state=initial)[0]
        assert torch.equal(wide, causal_linear_packed(q[:, :1], k[:, :1], v, decay, cu, scale, initial_state=initial)[0])


@pytest.mark.parametrize("lengths,heads,dim", [([700], 2, 128), ([130, 0, 1, 333, 64, 65], 3, 64), ([0, 64, 64, 0], 2, 128),
                                               ([1], 2, 64), ([2000], 1, 128)])
@pytest.mark.parametrize("begun", [False, True])
def test_every_number_of_ranges(device, lengths, heads, dim, begun):
    bounds = _bounds(lengths)
    q, k, v, decay, initial = _case(bounds[-1], heads, heads, dim, 5, device, len(lengths) if begun else 0)
    want = _want(q, k, v, decay, bounds, 0.3, initial)
    for ranges in (1, 2, 3, 4, 7, 12, 40):
        print(f"ranges {ranges}", flush=True)
        _check(_in_ranges(ranges, q, k, v, decay, bounds, 0.3, initial), want, dim, max(lengths))


def test_long_sequence_and_slow_decays(device):
    """6,000 tokens in the ranges of the host's rule, decays of 0 (nothing fades), tiny, -inf (nothing stays) and huge."""
    from vdn_h3_amd.causal_linear import causal_linear_packed

    q, k, v, _, initial = _case(6000, 8, 2, 128, 9, device, 1)
    decay = torch.tensor([0.0, -1e-6, -1e-3, -0.1, -3.0, -40.0, -1e30, -torch.inf], device=device)
    got = causal_linear_packed(q, k, v, decay, [0, 6000], 0.1, initial_state=initial, output_final_state=True)
    _check(got, _want(q, k, v, decay, [0, 6000], 0.1, initial), 128, 6000)


def test_rows_outside_every_sequence_stay(device):
    from vdn_h3_amd.causal_linear import causal_linear_packed

    for dim in (128, 80):
        q, k, v, decay, _ = _case(300, 4, 2, dim, 1, device)
        for bounds in ([20, 130, 130, 260], [0, 0], [300, 300], [299, 300], [7, 8]):
            out = torch.full((300, 4, dim), 7.0, dtype=BF, device=device)
            cu = torch.tensor(bounds, dtype=torch.int32, device=device)
            res, final = causal_linear_packed(q, k, v, decay, cu, 0.2, out=out, output_final_state=True)
            assert res is out and (out[:bounds[0]] == 7).all() and (out[bounds[-1]:] == 7).all()
            a, b = bounds[0], bounds[-1]
            alone, end = causal_linear_packed(q[a:b], k[a:b], v[a:b], decay, [n - a for n in bounds], 0.2, output_final_state=True)
            assert torch.equal(out[a:b], alone) and torch.equal(final, end)


def test_bounds_outside_the_rows_are_cut(device):
    from vdn_h3_amd.causal_linear import causal_linear_packed

    q, k, v, decay, _ = _case(150, 2, 2, 64, 2, device)
    for bad, good in (([-5, 70, 2000], [0, 70, 150]), ([100, 40, 150], [100, 100, 100]), ([2 ** 31 - 1] * 2, [150, 150])):
        cu = torch.tensor(bad, dtype=torch.int32, device=device)
        out, final = causal_linear_packed(q, k, v, decay, cu, 0.2, output_final_state=True)
        if bad[1] >= bad[0]:
            want, end = causal_linear_packed(q, k, v, decay, good, 0.2, output_final_state=True)
            a, b = good[0], good[-1]
            assert torch.equal(out[a:b], want[a:b]) and torch.equal(final, end)


@pytest.mark.parametrize("dim", [128, 64])
def test_later_tokens_take_no_part_whatever_they_hold(device, dim):
    from vdn_h3_amd.causal_linear import causal_linear_packed

    q, k, v, decay, initial = _case(200, 2, 2, dim, 3, device, 1)
    for at in (0, 1, 37, 63, 64, 100, 199):
        want = causal_linear_packed(q[:at], k[:at], v[:at], decay, [0, at], 0.2, initial_state=initial)[0] if at else v[:0]
        for value in (torch.nan, torch.inf, -torch.inf):
            for which in ("k", "v", "q"):
                t = {"q": q, "k": k, "v": v}
                t[which] = t[which].clone()
                t[which][at, 0, 5] = value
                o, s = causal_linear_packed(t["q"], t["k"], t["v"], decay, [0, 200], 0.2, initial_state=initial,
                                            output_final_state=True)
                plain, end = causal_linear_packed(q, k, v, decay, [0, 200], 0.2, initial_state=initial, output_final_state=True)
                # rows in front: as if the sequence ended there, but for the order of the sums of a chunk's end
                assert torch.equal(o[:at], plain[:at]) and (o[:at].float() - want.float()).abs().max() <= 2.0 ** -7 * 8 \
                    if at else True
                assert torch.equal(o[:, 1], plain[:, 1]) and torch.equal(s[0, 1], end[0, 1])  # the other head
                if which == "v":  # the channel ends there, the others go on
                    others = [c for c in range(dim) if c != 5]
                    assert not o[at:, 0, 5].isfinite().any() and torch.equal(o[:, 0, others], plain[:, 0, others])
                    assert not s[0, 0, 5].isfinite().any() and torch.equal(s[0, 0, others], end[0, 0, others])
                elif which == "k":
                    assert not o[at:, 0].isfinite().any() and not s[0, 0, :, 5].isfinite().any()
                else:
                    assert not o[at, 0].isfinite().any() and torch.equal(o[at + 1:], plain[at + 1:]) and torch.equal(s, end)


def test_prompts_in_pieces(device):
    """A prompt in two calls, the second from the first's state: the same outputs and state within the bar, twice."""
    from vdn_h3_amd.causal_linear import causal_linear_packed

    q, k, v, decay, _ = _case(500, 4, 2, 128, 4, device)
    whole, end = causal_linear_packed(q, k, v, decay, [0, 500], 0.1, output_final_state=True)
    _, size, _, ssize = _want(q, k, v, decay, [0, 500], 0.1, None)
    for cut in (1, 64, 250, 499):
        a, s = causal_linear_packed(q[:cut], k[:cut], v[:cut], decay, [0, cut], 0.1, output_final_state=True)
        b, s = causal_linear_packed(q[cut:], k[cut:], v[cut:], decay, [0, 500 - cut], 0.1, initial_state=s, output_final_state=True)
        d = (torch.cat([a, b]).double() - whole.double()).abs()
        assert (d <= 2 * (2.0 ** -14 * size + 2.0 ** -8 * whole.double().abs())).all()
        assert ((s[0].double() - end[0].double()).abs() <= 2.0 ** -14 * ssize[0]).all()


def test_replays_take_other_lengths(device):
    from vdn_h3_amd.causal_linear import causal_linear_packed

    q, k, v, decay, initial = _case(400, 2, 2, 128, 6, device, 3)
    cu = torch.tensor([0, 100, 250, 400], dtype=torch.int32, device=device)
    out, final = torch.zeros_like(v), None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        causal_linear_packed(q, k, v, decay, cu, 0.2, initial_state=initial, output_final_state=True, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, final = causal_linear_packed(q, k, v, decay, cu, 0.2, initial_state=initial, output_final_state=True, out=out)
    for bounds in ([0, 100, 250, 400], [0, 0, 400, 400], [0, 1, 2, 3], [0, 399, 399, 400]):
        cu.copy_(torch.tensor(bounds, dtype=torch.int32))
        v.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        want, end = causal_linear_packed(q, k, v, decay, cu, 0.2, initial_state=initial, output_final_state=True)
        assert torch.equal(out[:bounds[-1]], want[:bounds[-1]]) and torch.equal(final, end)


def test_strides_of_single_rows_and_heads_and_past_32_bits(device):
    """A single row or head has no stride, whatever its tensor says; offsets and states past 2^31 elements."""
    from vdn_h3_amd.causal_linear import causal_linear_packed

    for heads in (1, 3):
        q, k, v, decay, initial = _case(1, heads, 1, 64, 3, device, 1)
        want = causal_linear_packed(q, k, v, decay, [0, 1], 0.1, initial_state=initial, output_final_state=True)
        odd = [t.flatten().as_strided(t.shape, (5, 64 if t.shape[1] > 1 else 3, 1)) for t in (q, k, v)]
        out = torch.zeros(heads * 64, dtype=BF, device=device).as_strided((1, heads, 64), (7, 64 if heads > 1 else 1, 1))
        got = causal_linear_packed(*odd, decay, [0, 1], 0.1, initial_state=initial, output_final_state=True, out=out)
        assert got[0] is out and torch.equal(out, want[0]) and torch.equal(got[1], want[1])
    q, k, v, decay, _ = _case(300, 2, 2, 64, 4, device)
    want = causal_linear_packed(q, k, v, decay, [0, 130, 300], 0.1, output_final_state=True)
    room = torch.empty(300 * 2 ** 23, dtype=BF, device=device)
    far = [room.as_strided((300, 2, 64), (2 ** 23, 64 * (i + 1), 1), 1024 * i) for i in range(4)]
    for t, x in zip(far, (q, k, v)):
        t.copy_(x)
    got = causal_linear_packed(*far[:3], decay, [0, 130, 300], 0.1, output_final_state=True, out=far[3])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # 70,000 sequences of a token each over 2 heads x 128: 2.3e9 numbers of states
    q, k, v, decay, _ = _case(1, 2, 2, 128, 5, device)
    cu = torch.zeros(70001, dtype=torch.int32, device=device)
    cu[-1] = 1
    del room, far, got
    final = causal_linear_packed(q, k, v, decay, cu, 0.1, output_final_state=True)[1]
    one = causal_linear_packed(q, k, v, decay, [0, 1], 0.1, output_final_state=True)[1]
    assert torch.equal(final[-1], one[0]) and not final[69998].any() and not final[:5].any()


@pytest.mark.parametrize("lengths,heads,dim", [([700], 2, 128), ([130, 0, 1, 333, 64, 65], 3, 64), ([0, 64, 64, 0], 2, 128),
                                               ([1], 2, 64), ([1300, 700], 1, 64)])
def test_what_a_workspace_held_takes_no_part(device, lengths, heads, dim):
    """Every number of ranges, with token counts of another call where the ranges' own go: a count that the first pass left out
    would add a state that is none, or one of NaNs."""
    from vdn_h3_amd import _lib

    lib, bounds = _lib.lib(), _bounds(lengths)
    q, k, v, decay, initial = _case(bounds[-1], heads, heads, dim, 5, device, len(lengths))
    cu, want = torch.tensor(bounds, dtype=torch.int32, device=device), _want(q, k, v, decay, bounds, 0.3, initial)
    for ranges in (2, 3, 4, 7, 12, 17, 18, 40):
        results = []
        for tokens, state in ((-1, torch.nan), (64, torch.nan), (0, 1.0), (640, 1e30)):
            print(f"ranges {ranges} over {tokens} {state}", flush=True)
            size = lib.vdnh3_causal_linear_workspace_bytes(ranges, heads, dim)
            work = torch.full((size // 4,), state, device=device)
            work.view(torch.int32)[-ranges:] = tokens
            out, final = torch.zeros_like(v), torch.zeros(len(lengths), heads, dim, dim, device=device)
            _lib.check(lib.vdnh3_causal_linear_packed(
                q.data_ptr(), *q.stride()[:2], k.data_ptr(), *k.stride()[:2], v.data_ptr(), *v.stride()[:2], out.data_ptr(),
                *out.stride()[:2], decay.data_ptr(), cu.data_ptr(), initial.data_ptr(), final.data_ptr(), len(lengths), bounds[-1],
                heads, heads, dim, 0.3, ranges, work.data_ptr(), size, _lib.stream_handle(device)), "packed")
            results.append((out, final))
        _check(results[0], want, dim, max(lengths))
        assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(r, results[0]))


@pytest.mark.parametrize("dim", [128, 64, 40])
def test_a_state_that_is_no_number_ends_its_channel(device, dim):
    from vdn_h3_amd.causal_linear import causal_linear_packed

    q, k, v, decay, initial = _case(700, 2, 2, dim, 8, device, 3)
    bounds = [0, 300, 300, 700]
    want, end = causal_linear_packed(q, k, v, decay, bounds, 0.2, initial_state=initial, output_final_state=True)
    for value in (torch.nan, torch.inf):
        bad = initial.clone()
        bad[2, 1, 5, 7] = bad[1, 0, 3, 0] = value
        o, s = causal_linear_packed(q, k, v, decay, bounds, 0.2, initial_state=bad, output_final_state=True)
        assert not o[300:, 1, 5].isfinite().any() and not s[2, 1, 5, 7].isfinite() and not s[1, 0, 3, 0].isfinite()
        o[300:, 1, 5], s[2, 1, 5], s[1, 0, 3, 0] = want[300:, 1, 5], end[2, 1, 5], end[1, 0, 3, 0]
        assert torch.equal(o, want) and torch.equal(s, end)
