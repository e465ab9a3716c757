"""The operators of the language model that encodes the prompts, next to the block that reads its text rows.

Kinds of call (``case["kind"]``):

* ``norm``   - residual addition, RMSNorm and 8-bit (or bf16) activations of one layer's input
* ``rotary`` - q / k RMSNorm and the rotary embedding of positions on several axes (time, height, width)
* ``packed`` - causal attention of several prompts packed into one sequence, grouped key / value heads
* ``cached`` - causal attention of new tokens (one or a few per request) over the requests' key / value caches

``run`` computes them in plain torch (fp32, one rounding at the end) or, with ``own`` set, through the calls of
``vdn_h3_amd``. ``exact`` restates each in float64. Codes are returned as the values they stand for: int8 codes times
their row's scale, e4m3 codes as the e4m3 numbers they are, beside the scales.
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
    import vdn_h3_amd.block_kernels as block_kernels
    import vdn_h3_amd.causal as causal
    import vdn_h3_amd.linear as linear
    import vdn_h3_amd.rotary as rotary
    return block_kernels, rotary, causal, linear


# ---- the cases ---------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of one request through a layer's input norm: launch and latency
        dict(name="norm_int8_r1", kind="norm", codes="int8", rows=1, hidden=5120, residual=True),
        # the text rows of one prompt
        dict(name="norm_int8_r512", kind="norm", codes="int8", rows=512, hidden=5120, residual=True),
        # a ragged batch in front of a projection that stays in bf16 (the first and last layers of a quantised model)
        dict(name="norm_bf16_r8296", kind="norm", codes="bf16", rows=8296, hidden=4096, residual=True),
        # every row of a full-length sequence, fp8 projections behind it
        dict(name="norm_fp8_r40688", kind="norm", codes="fp8", rows=40688, hidden=5120, residual=True),
        # one new token for each of 16 requests, no q/k norm
        dict(name="rotary_b16", kind="rotary", text=16, frames=0, gh=0, gw=0, heads=40, kv_heads=8, dim=128, rot=128,
             norm=False, ladder="shared"),
        # a prompt with a short ragged clip in it, grouped heads, half of the channels rotated
        dict(name="rotary_f37_11x19", kind="rotary", text=563, frames=37, gh=11, gw=19, heads=32, kv_heads=4, dim=128,
             rot=64, norm=True, ladder="shared"),
        # text and video rows of the block at full length, each axis with its own ladder of frequencies
        dict(name="rotary_f31_48x27", kind="rotary", text=512, frames=31, gh=48, gw=27, heads=40, kv_heads=40, dim=128,
             rot=128, norm=True, ladder="per_axis"),
        # one prompt of the text rows' length
        dict(name="packed_512", kind="packed", lengths="512", heads=40, kv_heads=8, dim=128),
        # the prompts of a batch, one of a single token and one with a clip among them
        dict(name="packed_ragged", kind="packed", lengths="77 1 1000 209 512 1807 333", heads=40, kv_heads=8, dim=128),
        # one long prompt (a document, or a clip's rows)
        dict(name="packed_8296", kind="packed", lengths="8296", heads=40, kv_heads=8, dim=128),
        # the next token of one request behind a long context
        dict(name="cached_b1_40688", kind="cached", batch=1, new=1, room=40960, least=40688, most=40688, heads=40,
             kv_heads=8, dim=128),
        # the next token of a batch of requests of mixed lengths
        dict(name="cached_b64", kind="cached", batch=64, new=1, room=8192, least=16, most=8192, heads=40, kv_heads=8,
             dim=128),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


#: query heads, key / value heads, channels of a head
_HEADS = ((40, 8, 128), (40, 40, 128), (32, 8, 128), (32, 4, 128), (28, 4, 128), (16, 2, 128), (8, 1, 128), (20, 20, 64),
          (32, 8, 64), (14, 2, 64))


def draw(rng):
    kind = rng.choice(("norm", "rotary", "packed", "cached"))
    heads, kv_heads, dim = rng.choice(_HEADS)
    if kind == "norm":
        hidden = rng.choice((1024, 2048, 4096, 5120, 8192, 8 * rng.randint(64, 1024)))
        most = 40688 * 5120 // hidden
        return dict(kind=kind, codes=rng.choice(("int8", "fp8", "bf16")), rows=_log_int(rng, 1, min(most, 40688)),
                    hidden=hidden, residual=rng.random() < 0.85)
    if kind == "rotary":
        while True:
            c = dict(text=_log_int(rng, 1, 2048), frames=rng.choice((0, 1, rng.randint(2, 72))), gh=rng.randint(4, 48),
                     gw=rng.randint(4, 48))
            if c["text"] + c["frames"] * c["gh"] * c["gw"] <= 40688:
                break
        return dict(kind=kind, **c, heads=heads, kv_heads=kv_heads, dim=dim, rot=rng.choice((dim, dim, dim // 2)),
                    norm=rng.random() < 0.7, ladder=rng.choice(("shared", "per_axis")))
    if kind == "packed":
        # sequences until about the drawn number of tokens is full
        total, lengths = _log_int(rng, 16, 8000), []
        while sum(lengths) < total and len(lengths) < 24:
            lengths.append(min(_log_int(rng, 1, 8000), total - sum(lengths)))
        return dict(kind=kind, lengths=" ".join(map(str, lengths)), heads=heads, kv_heads=kv_heads, dim=dim)
    batch = _log_int(rng, 1, 64)
    room = _log_int(rng, 64, min(40960, 64 * 8192 // batch))
    new = rng.choice((1, 1, 1, 2, rng.randint(3, 9)))
    most = rng.randint(room // 2, room)
    return dict(kind=kind, batch=batch, new=min(new, room // 2), room=room, least=rng.randint(0, most), most=most,
                heads=heads, kv_heads=kv_heads, dim=dim)


# ---- inputs ------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(0x5EED + 7919 * int(seed))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE)


def _sections(rot):
    """Pairs of channels per axis (time, height, width): a quarter, and the rest in halves."""
    time = rot // 8
    height = (rot // 2 - time + 1) // 2
    return time, height, rot // 2 - time - height


def _positions(case, g):
    """``[3, rows]`` int64: text rows count on all axes together, video rows carry (frame, row, column) behind them.
    Without video the rows are new tokens of requests that are anywhere in their context."""
    text, frames, gh, gw = case["text"], case["frames"], case["gh"], case["gw"]
    if not frames:
        return torch.randint(0, 40688, (1, text), generator=g, device=DEVICE).expand(3, text).contiguous()
    head = torch.arange(text, device=DEVICE).expand(3, text)
    t, h, w = torch.meshgrid(*(torch.arange(n, device=DEVICE) for n in (frames, gh, gw)), indexing="ij")
    return torch.cat([head, text + torch.stack([t, h, w]).reshape(3, -1)], 1).contiguous()


def prepare(case, seed):
    g = _generator(seed)
    state = dict(case)
    if case["kind"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        # a residual stream has a few channels far above the rest
        loud = 1 + 20 * (torch.rand(hidden, generator=g, device=DEVICE) < 0.004).float()
        state["x"] = _randn(g, rows, hidden).to(BF16)
        state["residual"] = (3 * _randn(g, rows, hidden) * loud).to(BF16) if case["residual"] else None
        state["weight"] = (1 + 0.2 * _randn(g, hidden)).to(BF16)
        state["eps"] = 1e-6
        return state
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    state["scale"] = dim ** -0.5
    if case["kind"] == "rotary":
        state["positions"] = _positions(case, g)
        rows = state["positions"].shape[1]
        # views of a fused projection's rows, as in the block
        qkv = (2 * _randn(g, rows, (heads + 2 * kv_heads) * dim)).to(BF16).view(rows, heads + 2 * kv_heads, dim)
        state["q"], state["k"] = qkv[:, :heads], qkv[:, heads:heads + kv_heads]
        norm = case["norm"]
        state["q_weight"] = (1 + 0.1 * _randn(g, dim)).to(BF16) if norm else None
        state["k_weight"] = (1 + 0.1 * _randn(g, dim)).to(BF16) if norm else None
        state["eps"], state["theta"] = 1e-6, 10000.0
        if own:
            _, rotary, _, _ = _framework()
            state["axes"] = rotary.RotaryAxes(_sections(case["rot"]), theta=state["theta"], ladder=case["ladder"])
        return state
    if case["kind"] == "packed":
        lengths = [int(n) for n in case["lengths"].split()]
        rows = sum(lengths)
        # normalised queries and keys and the values, views of one buffer of rows
        qkv = _randn(g, rows, heads + 2 * kv_heads, dim).to(BF16)
        state["q"], state["k"], state["v"] = qkv.split((heads, kv_heads, kv_heads), 1)
        ends = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
        state["cu_seqlens"] = ends.to(DEVICE)
        return state
    batch, new, room = case["batch"], case["new"], case["room"]
    lengths = torch.randint(case["least"], case["most"] + 1, (batch,), generator=g, device=DEVICE)
    state["lengths"] = lengths.to(torch.int32)
    state["q"] = _randn(g, batch, new, heads, dim).to(BF16)
    # behind a request's length the cache holds rows of requests that came before
    state["k_cache"] = _randn(g, batch, room, kv_heads, dim).to(BF16)
    state["v_cache"] = _randn(g, batch, room, kv_heads, dim).to(BF16)
    return state


# ---- the plain forms and the framework's calls -------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_plain(state):
    return {"norm": _plain_norm, "rotary": _plain_rotary, "packed": _plain_packed, "cached": _plain_cached}[state["kind"]](state)


def _run_own(state):
    block_kernels, rotary, causal, linear = _framework()
    kind = state["kind"]
    if kind == "norm":
        code = {"bf16": linear.KIND_BF16, "int8": linear.KIND_I8, "fp8": linear.KIND_F8}[state["codes"]]
        y, scale, total = block_kernels.residual_rmsnorm_quantize(state["x"], state["residual"], state["weight"],
                                                                  state["eps"], code)
        if state["codes"] == "int8":
            y = torch.mul(y, scale, out=torch.empty(y.shape, dtype=BF16, device=y.device))
        return [y, scale, total if state["residual"] is not None else None]
    if kind == "rotary":
        return list(rotary.normalise_qk_axes(state["q"], state["k"], state["positions"], state["axes"],
                                             state["q_weight"], state["k_weight"], state["eps"]))
    if kind == "packed":
        return causal.causal_softmax_packed(state["q"], state["k"], state["v"], state["cu_seqlens"], state["scale"])
    return causal.causal_softmax_cached(state["q"], state["k_cache"], state["v_cache"], state["lengths"],
                                        state["scale"])


def _plain_norm(state):
    total = state["x"].float()
    if state["residual"] is not None:
        total = total + state["residual"].float()
    y = total * torch.rsqrt(total.square().mean(-1, keepdim=True) + state["eps"]) * state["weight"].float()
    out = total.to(BF16) if state["residual"] is not None else None
    if state["codes"] == "bf16":
        return [y.to(BF16), None, out]
    most = 127.0 if state["codes"] == "int8" else 448.0
    scale = (y.abs().amax(-1, keepdim=True) / most).clamp_min(1e-12)
    if state["codes"] == "int8":
        return [((y / scale).round().clamp(-most, most) * scale).to(BF16), scale, out]
    return [(y / scale).clamp(-most, most).to(torch.float8_e4m3fn), scale, out]


def _turns(case, dtype, device):
    """``(frequency, axis)`` of each pair of channels: theta^(-i / n) over all n pairs, or over the pairs of its axis."""
    sections = _sections(case["rot"])
    axis = torch.repeat_interleave(torch.arange(3, device=device), torch.tensor(sections, device=device))
    i = torch.arange(case["rot"] // 2, device=device, dtype=dtype)
    n = torch.full_like(i, case["rot"] // 2)
    if case["ladder"] == "per_axis":
        starts = torch.tensor([0, sections[0], sections[0] + sections[1]], device=device, dtype=dtype)
        i, n = i - starts[axis], torch.tensor(sections, device=device, dtype=dtype)[axis]
    return torch.pow(torch.tensor(10000.0, dtype=dtype, device=device), -i / n), axis


def _plain_rotary(state):
    # angles in 64 bits: at position 40,688 a 32-bit angle is off by up to 2e-3
    frequency, axis = _turns(state, torch.float64, state["q"].device)
    angle = state["positions"].double()[axis].t() * frequency
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half = state["rot"] // 2
    both = []
    for x, weight in ((state["q"], state["q_weight"]), (state["k"], state["k_weight"])):
        y = x.float()
        if weight is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + state["eps"]) * weight.float()
        a, b = y[..., :half], y[..., half:2 * half]
        both.append(torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half:]], -1).to(BF16))
    return both


def _softmax_value(scores, seen, value):
    """``softmax(scores where seen) value`` over the last axis; a row that sees nothing gives zeros."""
    scores = scores.masked_fill(~seen, -torch.inf)
    most = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(scores.dtype).min)
    p = torch.exp(scores.sub_(most))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, value) / torch.where(total > 0, total, 1.0)


def _plain_packed(state):
    q, k, v, ends = state["q"], state["k"], state["v"], state["cu_seqlens"]
    rows, heads, dim = q.shape
    kv_heads = k.shape[1]
    at = torch.arange(rows, device=q.device)
    sequence = torch.searchsorted(ends, at.to(ends.dtype), right=True)
    seen = (sequence[:, None] == sequence[None]) & (at[:, None] >= at[None])
    qf = q.float().view(rows, kv_heads, heads // kv_heads, dim).permute(1, 2, 0, 3)
    kf = (k.float() * state["scale"]).permute(1, 2, 0).contiguous()[:, None]
    vf = v.float().transpose(0, 1).contiguous()[:, None]
    out = _softmax_value(torch.matmul(qf, kf), seen, vf)
    return out.permute(2, 0, 1, 3).reshape(rows, heads, dim).to(BF16)


def _plain_cached(state):
    q, k, v, lengths = state["q"], state["k_cache"], state["v_cache"], state["lengths"]
    batch, new, heads, dim = q.shape
    room, kv_heads = k.shape[1], k.shape[2]
    group = heads // kv_heads
    last = lengths[:, None] - new + torch.arange(new, device=q.device)  # the last key a new token sees
    seen = torch.arange(room, device=q.device) <= last[..., None]
    qf = q.float().view(batch, new, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, new * group, dim)
    kf = (k.float() * state["scale"]).permute(0, 2, 3, 1).contiguous()
    vf = v.float().transpose(1, 2).contiguous()
    seen = seen[:, None, :, None].expand(batch, 1, new, group, room).reshape(batch, 1, new * group, room)
    out = _softmax_value(torch.matmul(qf, kf), seen, vf)
    return out.view(batch, kv_heads, new, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, new, heads, dim).to(BF16)


# ---- work and exact results --------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "norm":
        n = case["rows"] * case["hidden"]
        each = 2 + (4 if case["residual"] else 0) + (2 if case["codes"] == "bf16" else 1)
        return {"bytes": n * each + 2 * case["hidden"] + (0 if case["codes"] == "bf16" else 4 * case["rows"]),
                "flops": 6 * n}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if kind == "rotary":
        rows = case["text"] + case["frames"] * case["gh"] * case["gw"]
        n = rows * (heads + kv_heads) * dim
        return {"bytes": 4 * n + 24 * rows, "flops": (7 if case["norm"] else 3) * n}
    if kind == "packed":
        lengths = [int(n) for n in case["lengths"].split()]
        return {"bytes": 2 * sum(lengths) * 2 * (heads + kv_heads) * dim,
                "flops": 4 * dim * heads * sum(n * (n + 1) // 2 for n in lengths)}
    # the lengths lie evenly between the two ends
    keys = case["batch"] * (case["least"] + case["most"]) / 2
    return {"bytes": 4 * keys * kv_heads * dim + 4 * case["batch"] * case["new"] * heads * dim,
            "flops": 4 * dim * heads * keys * case["new"]}


def _round_e4m3(y):
    """The nearest e4m3 number (ties to even): three bits behind the leading one, the smallest step 2^-9."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "packed": _exact_packed, "cached": _exact_cached}[case["kind"]](state)


def _exact_norm(state):
    parts = []
    for rows in torch.arange(state["rows"], device=DEVICE).split(4096):
        r = state["x"][rows].double()
        if state["residual"] is not None:
            r += state["residual"][rows].double()
        length = torch.sqrt((r * r).sum(1) / r.shape[1] + state["eps"])
        y = r / length[:, None] * state["weight"].double()
        scale = None
        if state["codes"] != "bf16":
            most = {"int8": 127, "fp8": 448}[state["codes"]]
            scale = torch.clamp(y.abs().max(1, keepdim=True).values / most, min=1e-12)
            y = torch.round(y / scale) * scale if state["codes"] == "int8" else _round_e4m3(y / scale)
        parts.append((y, scale, r if state["residual"] is not None else None))
    return [None if p[0] is None else torch.cat(p) for p in zip(*parts)]


def _exact_rotary(state):
    frequency, axis = _turns(state, torch.float64, state["q"].device)
    turn = torch.polar(torch.ones_like(frequency), state["positions"].double().t()[:, axis] * frequency)[:, None]
    half, both = frequency.numel(), []
    for name in ("q", "k"):
        y, weight = state[name].double(), state[name + "_weight"]
        if weight is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + state["eps"]) * weight.double()
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
        both.append(torch.cat((z.real, z.imag, y[..., 2 * half:]), -1))
    return both


def _exact_rows(q, k, v, first, scale):
    """One head: row i of ``q`` sees the keys 0 .. first + i."""
    s = (q.double() @ k.double().t().contiguous()) * scale
    s = torch.where(torch.ones_like(s).tril(first) > 0, s, -torch.inf)
    return torch.softmax(s, 1) @ v.double()


def _exact_packed(state):
    q, k, v = state["q"], state["k"], state["v"]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    ends = state["cu_seqlens"].tolist()
    for a, b in zip(ends, ends[1:]):
        for h in range(q.shape[1]):
            g = h * k.shape[1] // q.shape[1]
            out[a:b, h] = _exact_rows(q[a:b, h], k[a:b, g], v[a:b, g], 0, state["scale"])
    return out


def _exact_cached(state):
    q, k, v = state["q"], state["k_cache"], state["v_cache"]
    new, heads, kv_heads = q.shape[1], q.shape[2], k.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, n in enumerate(state["lengths"].tolist()):
        idle = max(0, new - n)  # new tokens in front of the first key see nothing
        if idle >= new:
            continue
        for g in range(kv_heads):
            one = slice(g * (heads // kv_heads), (g + 1) * (heads // kv_heads))
            kd, vd = k[b, :n, g].double(), v[b, :n, g].double()
            s = torch.einsum("ihd,jd->ihj", q[b, idle:, one].double(), kd) * state["scale"]
            j = torch.arange(n, device=q.device)
            i = torch.arange(idle, new, device=q.device)
            s = torch.where(j <= (n - new + i)[:, None, None], s, -torch.inf)
            out[b, idle:, one] = torch.einsum("ihj,jd->ihd", torch.softmax(s, -1), vd)
    return out
