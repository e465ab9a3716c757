"""Operators of a language model with linear-attention layers that serves many requests at once, next to the prompt
encoder's operators and the Gated DeltaNet.

Kinds of call (``case["kind"]``):

* ``prompt``  - causal linear attention with a decay for each head over packed prompts, states in and out
* ``token``   - its recurrent form: new tokens of requests whose states lie in a pool
* ``delta``   - the recurrent form of the Gated DeltaNet, over such a pool too
* ``adapter`` - each row's low-rank adapter added to the output of a projection that all requests share

``run`` computes them in plain torch (fp32, one rounding at the end) or, with ``own`` set, through the calls of
``vdn_h3_amd``. ``exact`` restates each in float64: the prompts as one sum over all earlier tokens, without chunks.
"""

import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
BF16 = torch.bfloat16


def _framework():
    path = os.path.join(os.getcwd(), "comfyui-kirei-vdn-h3_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import vdn_h3_amd.adapters as adapters
    import vdn_h3_amd.causal_linear as causal_linear
    import vdn_h3_amd.gdn as gdn
    return causal_linear, gdn, adapters


# ---- the cases ---------------------------------------------------------------------------------------------

def listed():
    return [
        # one prompt of the text rows' length; its final state is what the tokens behind it start from
        dict(name="prompt_512", kind="prompt", lengths="512", heads=40, qk_heads=40, dim=128, begun=False),
        # the prompts of a batch that continue conversations (states in), one of a single token, queries and keys shared
        # by the heads of a group
        dict(name="prompt_ragged", kind="prompt", lengths="77 1 1000 209 512 1807 333", heads=40, qk_heads=8, dim=128,
             begun=True),
        # every row of a full-length sequence of the block
        dict(name="prompt_40688", kind="prompt", lengths="40688", heads=40, qk_heads=40, dim=128, begun=False),
        # the next token of one request: latency
        dict(name="token_b1", kind="token", batch=1, new=1, slots=8, heads=40, qk_heads=40, dim=128),
        # four tokens that a draft proposed, for each of 16 requests, narrow heads
        dict(name="token_b16_n4", kind="token", batch=16, new=4, slots=24, heads=32, qk_heads=8, dim=64),
        # the next token of a full batch
        dict(name="token_b64", kind="token", batch=64, new=1, slots=96, heads=40, qk_heads=40, dim=128),
        # the same two ends for the gated delta rule
        dict(name="delta_b1", kind="delta", batch=1, new=1, slots=8, heads=40, qk_heads=40, dim=128),
        dict(name="delta_b64", kind="delta", batch=64, new=1, slots=96, heads=32, qk_heads=16, dim=128),
        # one token through the block's fused projection
        dict(name="adapter_r1", kind="adapter", requests=1, rows=1, adapters=8, rank=16, width=5120, out=15360),
        # the next token of 64 requests, each with its own choice of 16 adapters or none
        dict(name="adapter_r64", kind="adapter", requests=64, rows=64, adapters=16, rank=16, width=5120, out=15360),
        # the prompts of a batch, ragged
        dict(name="adapter_r3939", kind="adapter", requests=7, rows=3939, adapters=8, rank=32, width=5120, out=5120),
        # all rows of the block at full length through its output projection, one style each for a few requests
        dict(name="adapter_r40688", kind="adapter", requests=3, rows=40688, adapters=4, rank=64, width=5120, out=5120),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


#: value heads, query / key heads, channels of a head
_HEADS = ((40, 40, 128), (40, 8, 128), (32, 16, 128), (16, 16, 128), (8, 4, 128), (20, 20, 64), (32, 8, 64), (56, 56, 64))


def draw(rng):
    kind = rng.choice(("prompt", "token", "delta", "adapter"))
    heads, qk_heads, dim = rng.choice(_HEADS)
    if kind == "prompt":
        # sequences until about the drawn number of tokens is full
        total, lengths = _log_int(rng, 16, 24000), []
        while sum(lengths) < total and len(lengths) < 24:
            lengths.append(min(_log_int(rng, 1, 24000), total - sum(lengths)))
        return dict(kind=kind, lengths=" ".join(map(str, lengths)), heads=heads, qk_heads=qk_heads, dim=dim,
                    begun=rng.random() < 0.5)
    if kind in ("token", "delta"):
        batch = _log_int(rng, 1, 64)
        return dict(kind=kind, batch=batch, new=rng.choice((1, 1, 1, 2, rng.randint(3, 8))), slots=rng.randint(batch, 96),
                    heads=heads, qk_heads=qk_heads, dim=dim)
    rows = _log_int(rng, 1, 24000)
    return dict(kind=kind, requests=rng.randint(1, min(rows, 64)), rows=rows, adapters=rng.randint(1, 16 if rows < 4096 else 6),
                rank=rng.choice((8, 16, 16, 32, 64)), width=rng.choice((1024, 2048, 4096, 5120, 8 * rng.randint(64, 640))),
                out=rng.choice((1024, 4096, 5120, 8 * rng.randint(64, 640))))


# ---- inputs ------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(0xADA + 7919 * int(seed))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE)


def _unit(x):
    return x / x.norm(dim=-1, keepdim=True).clamp_min(1e-6)


def _lengths(case):
    return [int(n) for n in case["lengths"].split()]


_CHUNK = 64


def _chunks(lengths):
    """Chunks of 64 tokens that end with their sequence: first row, tokens, sequence, tokens of the sequence before it."""
    table, start = [], 0
    for b, n in enumerate(lengths):
        table += [(start + a, min(_CHUNK, n - a), b, a) for a in range(0, n, _CHUNK)]
        start += n
    return torch.tensor(table).t().contiguous().to(DEVICE)


def prepare(case, seed):
    g = _generator(seed)
    state = dict(case)
    if case["kind"] == "adapter":
        rows, n, rank = case["rows"], case["adapters"], case["rank"]
        state["x"] = _randn(g, rows, case["width"]).to(BF16)
        state["y"] = _randn(g, rows, case["out"]).to(BF16)
        down = (_randn(g, n, rank, case["width"]) * case["width"] ** -0.5).to(BF16)
        up = (0.5 * _randn(g, n, case["out"], rank) * rank ** -0.5).to(BF16)
        scale = 0.5 + torch.rand(n, generator=g, device=DEVICE)
        # requests are runs of rows, of ragged lengths, each with its adapter or none
        cuts = torch.rand(case["requests"] - 1, generator=g, device=DEVICE).mul(rows).long().sort()[0]
        if rows == case["requests"]:
            request = torch.arange(rows, device=DEVICE)
        else:
            request = torch.searchsorted(cuts, torch.arange(rows, device=DEVICE), right=True)
        least = 0 if case["requests"] == 1 else -1
        choice = torch.randint(least, n, (case["requests"],), generator=g, device=DEVICE)
        state["index"] = choice[request].to(torch.int32)
        state["down"], state["up"], state["scales"] = down, up, scale
        if own:
            _, _, adapters = _framework()
            state["handle"] = adapters.LowRankAdapters(down, up, scale)
        return state
    heads, qk_heads, dim = case["heads"], case["qk_heads"], case["dim"]
    state["scale"] = dim ** -0.5
    # a geometric row of decays, from 0.4 to 0.996 a token
    state["log_decay"] = -torch.exp2(-8.0 * torch.arange(heads, device=DEVICE) / heads)
    if case["kind"] == "prompt":
        lengths = _lengths(case)
        rows = sum(lengths)
        # normalised queries and keys and the values, views of one buffer of rows
        qkv = _randn(g, rows, 2 * qk_heads + heads, dim).to(BF16)
        state["q"], state["k"], state["v"] = qkv.split((qk_heads, qk_heads, heads), 1)
        state["cu_seqlens"] = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(DEVICE)
        state["chunks"] = _chunks(lengths)
        state["initial"] = 2 * _randn(g, len(lengths), heads, dim, dim) if case["begun"] else None
        return state
    batch, new = case["batch"], case["new"]
    q, k = _randn(g, batch, new, qk_heads, dim), _randn(g, batch, new, qk_heads, dim)
    if case["kind"] == "delta":  # the delta rule's keys are unit vectors
        q, k = _unit(q), _unit(k)
        state["beta"] = torch.sigmoid(_randn(g, batch, new, heads))
        state["g"] = -0.1 * torch.nn.functional.softplus(_randn(g, batch, new, heads))
    state["q"], state["k"], state["v"] = q.to(BF16), k.to(BF16), _randn(g, batch, new, heads, dim).to(BF16)
    state["pool"] = _randn(g, case["slots"], heads, dim, dim)
    state["at"] = torch.randperm(case["slots"], generator=g, device=DEVICE)[:batch].to(torch.int32)
    return state


# ---- the plain forms and the framework's calls -------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_plain(state):
    return {"prompt": _plain_prompt, "token": _plain_token, "delta": _plain_delta, "adapter": _plain_adapter}[state["kind"]](state)


def _run_own(state):
    causal_linear, gdn, _ = _framework()
    kind = state["kind"]
    if kind == "prompt":
        return list(causal_linear.causal_linear_packed(state["q"], state["k"], state["v"], state["log_decay"],
                                                       state["cu_seqlens"], state["scale"], initial_state=state["initial"],
                                                       output_final_state=True))
    if kind == "token":
        out = causal_linear.causal_linear_step(state["q"], state["k"], state["v"], state["log_decay"], state["pool"],
                                               state["scale"], slots=state["at"])
        return [out, state["pool"]]
    if kind == "delta":
        out = gdn.gated_delta_step(state["q"], state["k"], state["v"], state["beta"], state["g"], state["pool"],
                                   slots=state["at"])
        return [out, state["pool"]]
    return state["handle"].add(state["y"], state["x"], state["index"])


def _per_head(x, heads):
    """Heads of queries or keys, in the last but one place, repeated for the value heads of their group."""
    return x.float().repeat_interleave(heads // x.shape[-2], -2)


def _plain_prompt(state):
    heads, dim, scale, log_decay = state["heads"], state["dim"], state["scale"], state["log_decay"]
    first, count, owner, before = state["chunks"]
    rows, sequences = state["v"].shape[0], len(_lengths(state))
    i = torch.arange(_CHUNK, device=DEVICE)
    live = i < count[:, None]
    at = (first[:, None] + i).clamp_max(rows - 1)
    q, k, v = (_per_head(state[name], heads)[at].permute(2, 0, 1, 3).contiguous() for name in "qkv")  # [H, chunks, 64, D]

    def decay(tokens):  # a^tokens by head, 0 where there is a negative number of tokens between
        tokens = tokens.float()
        return torch.exp(log_decay.view(-1, *[1] * tokens.ndim) * tokens).masked_fill(tokens < 0, 0.0)

    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * decay(i[:, None] - i)[:, None]
    inside = torch.matmul(scores, v)
    # what each chunk adds to the state [Dv, Dk] at its end, and the states at the chunks' beginnings
    weight = decay(torch.where(live, count[:, None] - 1 - i, -1))
    added = torch.matmul((v * weight[..., None]).transpose(2, 3).contiguous(), k)
    between = torch.where(owner[:, None] == owner, before[:, None] - (before + count), -1)
    begin = torch.matmul(decay(between), added.flatten(2)).view_as(added)
    initial = state["initial"]
    if initial is not None:
        begin = begin + decay(before)[..., None, None] * initial.transpose(0, 1)[:, owner]
    carried = torch.matmul(q, begin.transpose(2, 3).contiguous()) * decay(i + 1)[:, None, :, None]
    out = torch.empty(rows, heads, dim, dtype=BF16, device=DEVICE)
    out[at[live]] = ((inside + carried) * scale).to(BF16).permute(1, 2, 0, 3)[live]
    end = decay(count)[..., None, None] * begin + added
    last = torch.searchsorted(owner, torch.arange(sequences, device=DEVICE), right=True) - 1
    return [out, end[:, last].transpose(0, 1).contiguous()]


def _plain_token(state):
    heads, new, at = state["heads"], state["new"], state["at"].long()
    q, k = (_per_head(state[name], heads).transpose(1, 2) for name in "qk")  # [B, H, N, D]
    v = state["v"].float().transpose(1, 2)
    i = torch.arange(new, device=DEVICE)
    log_decay = state["log_decay"][:, None]
    old = state["pool"][at]
    weight = torch.exp(log_decay[..., None] * (i[:, None] - i).clamp_min(0)).tril()
    out = torch.matmul(torch.matmul(q, k.transpose(2, 3).contiguous()) * weight, v)
    out = out + torch.exp(log_decay * (i + 1))[..., None] * torch.matmul(q, old.transpose(2, 3).contiguous())
    late = torch.exp(log_decay * (new - 1 - i))[..., None]
    state["pool"][at] = torch.exp(log_decay * new)[..., None] * old + torch.matmul((v * late).transpose(2, 3).contiguous(), k)
    return [(out * state["scale"]).transpose(1, 2).to(BF16).contiguous(), state["pool"]]


def _plain_delta(state):
    heads, at = state["heads"], state["at"].long()
    q, k, v = (_per_head(state[name], heads) for name in "qkv")
    decay, beta = torch.exp(state["g"])[..., None, None], state["beta"][..., None]
    s, out = state["pool"][at], torch.empty_like(v)
    for t in range(state["new"]):  # each token's update needs the state that the one before it left
        kt = k[:, t, :, None]
        s = s * decay[:, t]
        write = (v[:, t] - (s * kt).sum(-1)) * beta[:, t]
        s = s + write[..., None] * kt
        out[:, t] = (s * q[:, t, :, None]).sum(-1)
    state["pool"][at] = s
    return [out.to(BF16), state["pool"]]


def _plain_adapter(state):
    # all rows through all adapters, and each row keeps its own: no loop over adapters, no row counts on the host
    n, rank, index = state["down"].shape[0], state["rank"], state["index"]
    keep = (index[:, None] == torch.arange(n, device=DEVICE)) * state["scales"]
    h = torch.matmul(state["x"].float(), state["down"].float().flatten(0, 1).t().contiguous()).view(-1, n, rank)
    h = (h * keep[..., None]).flatten(1)
    up = state["up"].float().transpose(1, 2).reshape(n * rank, -1)
    return (state["y"].float() + torch.matmul(h, up)).to(BF16)


# ---- work and exact results --------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "adapter":
        rows, width, out = case["rows"], case["width"], case["out"]
        used = min(case["adapters"], case["requests"])
        return {"bytes": 2 * rows * (width + 2 * out) + 2 * used * case["rank"] * (width + out) + 4 * rows,
                "flops": 2 * rows * case["rank"] * (width + out)}
    heads, qk_heads, dim = case["heads"], case["qk_heads"], case["dim"]
    if case["kind"] == "prompt":
        lengths = _lengths(case)
        rows = sum(lengths)
        states = 4 * len(lengths) * heads * dim * dim * (2 if case["begun"] else 1)
        return {"bytes": 4 * rows * (qk_heads + heads) * dim + states, "flops": 4 * rows * heads * dim * dim}
    tokens = case["batch"] * case["new"]
    each = 7 if case["kind"] == "delta" else 5
    gates = 8 * tokens * heads if case["kind"] == "delta" else 0
    return {"bytes": 8 * case["batch"] * heads * dim * dim + 4 * tokens * (qk_heads + heads) * dim + gates,
            "flops": each * tokens * heads * dim * dim}


def exact(case, seed):
    state = prepare(case, seed)
    return {"prompt": _exact_prompt, "token": _exact_token, "delta": _exact_delta, "adapter": _exact_adapter}[case["kind"]](state)


def _exact_prompt(state):
    q, k, v, initial = state["q"], state["k"], state["v"], state["initial"]
    rows, heads, dim = v.shape
    lengths = _lengths(state)
    out = torch.empty(v.shape, dtype=torch.float64, device=DEVICE)
    final = torch.zeros(len(lengths), heads, dim, dim, dtype=torch.float64, device=DEVICE)
    a = 0
    for b, n in enumerate(lengths):
        j = torch.arange(n, device=DEVICE, dtype=torch.float64)
        for h in range(heads):
            rate = float(state["log_decay"][h])
            one = h * q.shape[1] // heads
            qh, kh, vh = q[a:a + n, one].double() * state["scale"], k[a:a + n, one].double(), v[a:a + n, h].double()
            if initial is not None:
                s0 = initial[b, h].double()
                final[b, h] += s0 * math.exp(rate * n)
            for c in range(0, n, 2048):  # blocks of rows against every token up to their last
                e = min(c + 2048, n)
                ago = j[c:e, None] - j[None, :e]
                w = torch.where(ago >= 0, torch.exp(rate * ago.clamp_min_(0)), 0.0)
                o = (w * (qh[c:e] @ kh[:e].t())) @ vh[:e]
                if initial is not None:
                    o += torch.exp(rate * (j[c:e, None] + 1)) * (qh[c:e] @ s0.t())
                out[a + c:a + e, h] = o
            final[b, h] += (vh * torch.exp(rate * (n - 1 - j))[:, None]).t() @ kh
        a += n
    return [out, final]


def _exact_token(state):
    pool, heads = state["pool"].double(), state["heads"]
    rates = torch.exp(state["log_decay"].double())[None, :, None, None]
    at, group = state["at"].long(), heads // state["qk_heads"]
    s, rows = pool[at], []
    for t in range(state["new"]):
        kt, qt = (state[name][:, t].double().repeat_interleave(group, 1) for name in "kq")
        s = s * rates + torch.einsum("bhv,bhk->bhvk", state["v"][:, t].double(), kt)
        rows.append(torch.einsum("bhvk,bhk->bhv", s, qt) * state["scale"])
    pool[at] = s
    return [torch.stack(rows, 1), pool]


def _exact_delta(state):
    pool, group = state["pool"].double(), state["heads"] // state["qk_heads"]
    at = state["at"].long()
    s, rows, eye = pool[at], [], torch.eye(state["dim"], device=DEVICE, dtype=torch.float64)
    for t in range(state["new"]):
        kt, qt = (state[name][:, t].double().repeat_interleave(group, 1) for name in "kq")
        b = state["beta"][:, t].double()[..., None, None]
        turn = eye - b * kt[..., :, None] * kt[..., None, :]
        s = torch.exp(state["g"][:, t].double())[..., None, None] * (s @ turn.contiguous())
        s = s + b * state["v"][:, t].double()[..., :, None] * kt[..., None, :]
        rows.append((s @ qt[..., None])[..., 0])
    pool[at] = s
    return [torch.stack(rows, 1), pool]


def _exact_adapter(state):
    out = state["y"].double()
    for i in range(state["down"].shape[0]):
        mine = state["index"] == i
        h = state["x"][mine].double() @ state["down"][i].double().t()
        out[mine] += (h * state["scales"][i].double()) @ state["up"][i].double().t()
    return out
