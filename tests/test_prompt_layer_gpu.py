"""One layer of a prompt encoder built from the operators, prompts first and then token by token (GPU).

norm + int8 codes -> W8A8 q/k/v projection -> q/k norm and rotary positions -> causal attention -> W8A8 output projection ->
residual addition + norm. A prompt taken whole and the same prompt taken token by token over caches are the same layer, so
their outputs differ only by rounding: each row's codes and projections are the same bits in both, the attention's outputs
are within its bar, twice.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize("precision", ["int8", "fp8"])
def test_prompts_whole_and_token_by_token(device, precision):
    from vdn_h3_amd import linear
    from vdn_h3_amd.block_kernels import residual_rmsnorm_quantize
    from vdn_h3_amd.causal import causal_softmax_cached, causal_softmax_packed
    from vdn_h3_amd.rotary import RotaryAxes, normalise_qk_axes

    kind = linear.KIND_I8 if precision == "int8" else linear.KIND_F8
    heads, kv, dim, hidden, lengths = 10, 2, 128, 1280, [33, 1, 70]
    g = torch.Generator().manual_seed(21)

    def rand(*shape):
        return torch.randn(*shape, generator=g)

    qkv_proj = linear.HipLinear((rand((heads + 2 * kv) * dim, hidden) * hidden ** -0.5).to(BF).to(device), precision)
    out_proj = linear.HipLinear((rand(hidden, heads * dim) * hidden ** -0.5).to(BF).to(device), precision)
    w1, w2 = ((1 + 0.1 * rand(hidden)).to(BF).to(device) for _ in range(2))
    wq, wk = ((1 + 0.1 * rand(dim)).to(BF).to(device) for _ in range(2))
    axes = RotaryAxes((16, 24, 24))
    rows, room = sum(lengths), 96
    x, res = rand(rows, hidden).to(BF).to(device), (2 * rand(rows, hidden)).to(BF).to(device)
    starts = [0, 33, 34]
    pos = torch.cat([torch.arange(n) for n in lengths]).expand(3, rows).contiguous().to(device)
    cu = torch.tensor([0, 33, 34, 104], dtype=torch.int32, device=device)

    def project(x, res, pos):
        codes, scale, total = residual_rmsnorm_quantize(x, res, w1, 1e-6, kind)
        qkv = linear.gemm_w8a8(codes, scale, qkv_proj.weight, qkv_proj.weight_scale).view(-1, heads + 2 * kv, dim)
        q, k = normalise_qk_axes(qkv[:, :heads], qkv[:, heads:heads + kv], pos, axes, wq, wk)
        return total, q, k, qkv[:, heads + kv:]

    def close(attended, total):
        return residual_rmsnorm_quantize(out_proj(attended.flatten(1)), total, w2, 1e-6, kind)

    total, q, k, v = project(x, res, pos)
    attended = causal_softmax_packed(q, k, v, cu, dim ** -0.5)
    codes, scale, _ = close(attended, total)

    caches = [torch.full((3, room, kv, dim), torch.nan, dtype=BF, device=device) for _ in range(2)]
    rows_of = {}
    for step in range(max(lengths)):
        live = [b for b, n in enumerate(lengths) if step < n]
        at = torch.tensor([starts[b] + step for b in live], device=device)
        t1, q1, k1, v1 = project(x[at], res[at], pos[:, at].contiguous())
        assert torch.equal(t1, total[at]) and torch.equal(q1, q[at]) and torch.equal(k1, k[at]) and torch.equal(v1, v[at])
        who = torch.tensor(live, device=device)
        caches[0][who, step], caches[1][who, step] = k1, v1
        n = torch.full((len(live),), step + 1, dtype=torch.int32, device=device)
        o = causal_softmax_cached(q1[:, None], caches[0][who], caches[1][who], n, dim ** -0.5)[:, 0]
        for i, row in enumerate(at.tolist()):
            rows_of[row] = o[i]
    stepped = torch.stack([rows_of[i] for i in range(rows)])
    # 2 (2 2^-8 A + 2^-8 |o|) with A = sum p |v| at most the largest |v| of the keys: 6 2^-8 max |v|
    assert (stepped.float() - attended.float()).abs().max() <= 6 * 2.0 ** -8 * v.float().abs().max()
    codes2, scale2, _ = close(stepped, total)
    a, b = (c.float() * s for c, s in ((codes, scale), (codes2, scale2)))
    assert torch.nn.functional.cosine_similarity(a, b).min() > 0.999
