"""Cases of the dense and state-space operators beside the routed experts of a
hybrid (Mamba-2 / MoE) model, for timing and for checking their values.

  linear  a dense projection with bias, activation and residual in its epilogue
  conv    the causal depthwise convolution over packed prompts
  scan    the selective state-space scan over packed prompts
  token   convolution, scan and gated norm for one new token of each sequence
  norm    the gated RMS norm of the scan's output, per group of channels

``run`` computes each in plain torch operations, or through
``ervf_b200.GPUKernels`` where ``own`` is true.  ``exact`` computes them in 64
bits, token by token, from the recurrences.
"""

import functools
import math

import torch

own = False

HIDDEN = 2688     # hidden size of the hybrid
INNER = 4096      # heads * head_dim of its state-space layers
SHARED = 3712     # width of its shared expert
VOCAB = 131072    # rows of its output head
EPS = 1e-5
QUANTUM = 64      # chunk length of the plain scan


def listed():
    return [
        # one decoded token through a state-space layer's output projection, onto the f32 residual stream
        {"name": "linear_token", "op": "linear", "rows": HIDDEN, "cols": INNER, "tokens": 1,
         "act": "none", "bias": False, "resid": True, "out": "f32"},
        # the output head for a decode batch, f32 logits
        {"name": "linear_head", "op": "linear", "rows": VOCAB, "cols": HIDDEN, "tokens": 19,
         "act": "none", "bias": False, "resid": False, "out": "f32"},
        # the shared expert's up projection of one short prompt
        {"name": "linear_up", "op": "linear", "rows": SHARED, "cols": HIDDEN, "tokens": 509,
         "act": "relu2", "bias": True, "resid": False, "out": "bf16"},
        # the shared expert's down projection of a long prompt, with bias and residual
        {"name": "linear_down", "op": "linear", "rows": HIDDEN, "cols": SHARED, "tokens": 8192,
         "act": "none", "bias": True, "resid": True, "out": "bf16"},
        # the convolution of one long prompt
        {"name": "conv_long", "op": "conv", "tokens": 8192, "seqs": 1, "channels": INNER + 2048,
         "width": 4, "type": "bf16"},
        # the convolution of a few ragged prompts, some of them continued, in f32
        {"name": "conv_ragged", "op": "conv", "tokens": 1021, "seqs": 7, "channels": INNER + 2048,
         "width": 4, "type": "f32"},
        # the scan of one long prompt
        {"name": "scan_long", "op": "scan", "tokens": 8192, "seqs": 1, "heads": 64, "head_dim": 64,
         "groups": 8, "d_state": 128, "type": "bf16"},
        # the scan of a batch of ragged prompts, some of them continued
        {"name": "scan_ragged", "op": "scan", "tokens": 4099, "seqs": 13, "heads": 64, "head_dim": 64,
         "groups": 8, "d_state": 128, "type": "bf16"},
        # one token of one sequence: latency
        {"name": "token_one", "op": "token", "seqs": 1, "heads": 64, "head_dim": 64, "groups": 8,
         "d_state": 128, "width": 4, "type": "f32"},
        # one token of each sequence of a decode batch
        {"name": "token_batch", "op": "token", "seqs": 96, "heads": 64, "head_dim": 64, "groups": 8,
         "d_state": 128, "width": 4, "type": "bf16"},
        # the norm behind the scan of a long prompt
        {"name": "norm_long", "op": "norm", "tokens": 8192, "groups": 8, "group_size": 512, "type": "bf16"},
        # the same for a short one in f32
        {"name": "norm_short", "op": "norm", "tokens": 67, "groups": 8, "group_size": 512, "type": "f32"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("linear", "linear", "conv", "scan", "scan", "token", "norm"))
    if op == "linear":
        cols = 8 * _spread(rng, 16, 512)
        if rng.random() < 0.2:
            rows, tokens = _spread(rng, 16384, VOCAB), _spread(rng, 1, 64)
        else:
            rows = _spread(rng, 128, 8192)
            tokens = min(_spread(rng, 1, 8192), 8192 * HIDDEN * SHARED // (rows * cols))
        return {"op": op, "rows": rows, "cols": cols, "tokens": tokens,
                "act": rng.choice(("none", "relu2", "silu", "gelu")), "bias": rng.random() < 0.5,
                "resid": rng.random() < 0.5, "out": rng.choice(("f32", "bf16"))}
    if op == "conv":
        tokens = _spread(rng, 1, 8192)
        return {"op": op, "tokens": tokens, "seqs": min(tokens, _spread(rng, 1, 32)),
                "channels": _spread(rng, 256, INNER + 2048), "width": rng.choice((2, 3, 4)),
                "type": rng.choice(("f32", "bf16"))}
    if op == "scan":
        tokens, groups = _spread(rng, 1, 8192), rng.choice((1, 2, 4, 8))
        return {"op": op, "tokens": tokens, "seqs": min(tokens, _spread(rng, 1, 32)),
                "heads": groups * rng.randint(1, 8), "head_dim": 64, "groups": groups,
                "d_state": rng.choice((64, 128)), "type": "bf16"}
    if op == "token":
        groups = rng.choice((1, 2, 4, 8))
        return {"op": op, "seqs": _spread(rng, 1, 96), "heads": groups * rng.randint(1, 8),
                "head_dim": rng.choice((32, 64)), "groups": groups, "d_state": rng.choice((64, 96, 128)),
                "width": rng.choice((2, 3, 4)), "type": rng.choice(("f32", "bf16"))}
    return {"op": op, "tokens": _spread(rng, 1, 8192), "groups": rng.choice((1, 2, 4, 8)),
            "group_size": 8 * _spread(rng, 8, 64), "type": rng.choice(("f32", "bf16"))}


def _type(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _lengths(case, g):
    """Token counts of the packed prompts, made from the seed."""
    t, s = case["tokens"], case["seqs"]
    cuts = torch.randint(0, t + 1, (s - 1,), generator=g).sort().values
    ends = torch.cat([cuts, torch.tensor([t])])
    return torch.diff(ends, prepend=torch.tensor([0]))


def _packing(case, seed, dev):
    """What a serving loop knows of its packed prompts: offsets, longest
    length, the state slot of each and whether it continues an earlier one."""
    g = torch.Generator().manual_seed(seed)
    lens, s = _lengths(case, g), case["seqs"]
    cu = torch.zeros(s + 1, dtype=torch.int32)
    cu[1:] = lens.cumsum(0)
    slots = torch.randperm(s + 2, generator=g)[:s].int()
    has = (torch.rand(s, generator=g) < 0.5) if s > 1 else torch.zeros(1, dtype=torch.bool)
    return {"cu": cu.to(dev), "longest": int(lens.max()), "slots": slots.to(dev),
            "has": has.to(torch.uint8).to(dev)}


def _heads(case, rnd, dev):
    """The scan's parameters as a model holds them: steps of 0.001 to 0.1,
    decay rates of 1 to 16."""
    h = case["heads"]
    step = torch.exp(rnd(h, uniform=True) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    return {"A": -(1 + 15 * rnd(h, uniform=True)), "D": 1 + 0.1 * rnd(h),
            "dt_bias": step + torch.log(-torch.expm1(-step))}


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def rnd(*shape, uniform=False):
        make = torch.rand if uniform else torch.randn
        return make(*shape, generator=gen, device=dev)

    op, s = case["op"], dict(case)
    if op == "linear":
        rows, cols, tokens = case["rows"], case["cols"], case["tokens"]
        s["W"] = (rnd(rows, cols) * 0.02).bfloat16()
        s["x"] = rnd(tokens, cols).bfloat16()
        s["b"] = 0.1 * rnd(rows) if case["bias"] else None
        s["r"] = rnd(tokens, rows).to(_type(case["out"])) if case["resid"] else None
        s["y"] = torch.empty(tokens, rows, dtype=_type(case["out"]), device=dev)
        return s
    ty = _type(case["type"])
    if op == "norm":
        n = case["groups"] * case["group_size"]
        s["x"], s["z"] = rnd(case["tokens"], n).to(ty), rnd(case["tokens"], n).to(ty)
        s["w"] = 1 + 0.1 * rnd(n)
        s["y"] = torch.empty_like(s["x"])
        return s
    if op == "conv":
        ch, w = case["channels"], case["width"]
        s.update(_packing(case, seed, dev))
        s["x"] = rnd(case["tokens"], ch).to(ty)
        s["w"], s["b"] = rnd(ch, w) / math.sqrt(w), 0.1 * rnd(ch)
        s["state"] = rnd(case["seqs"] + 2, w - 1, ch).to(ty)
        s["y"] = torch.empty_like(s["x"])
        return s
    h, p, gr, n = case["heads"], case["head_dim"], case["groups"], case["d_state"]
    width = h * p + 2 * gr * n
    s.update(_heads(case, rnd, dev))
    if op == "scan":
        # x, B and C lie side by side in the convolution's output
        s.update(_packing(case, seed, dev))
        s["xbc"] = torch.nn.functional.silu(rnd(case["tokens"], width)).to(ty)
        s["dt"] = rnd(case["tokens"], h).to(ty)
        s["state"] = 0.3 * rnd(case["seqs"] + 2, h, p, n)
        s["y"] = torch.empty(case["tokens"], h * p, dtype=ty, device=dev)
        return s
    # one row of the input projection: gate, convolved channels, steps
    b, w = case["seqs"], case["width"]
    s["row"] = rnd(b, (h * p + width + h + 7) // 8 * 8).to(ty)
    s["cw"], s["cb"] = rnd(width, w) / math.sqrt(w), 0.1 * rnd(width)
    s["nw"] = 1 + 0.1 * rnd(h * p)
    s["slots"] = torch.randperm(b + 2, generator=torch.Generator().manual_seed(seed))[:b].int().to(dev)
    s["conv"] = rnd(b + 2, w - 1, width).to(ty)
    s["state"] = 0.3 * rnd(b + 2, h, p, n)
    s["y"] = torch.empty(b, h * p, dtype=ty, device=dev)
    return s


# ------------------------------------------------------------ plain forms


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(torch.clamp(v, max=20))))


def _silu(v):
    return v / (1 + torch.exp(-v))


def _act(v, act):
    if act == "relu2":
        return torch.clamp(v, min=0) ** 2
    if act == "silu":
        return _silu(v)
    return v * 0.5 * (1 + torch.erf(v * math.sqrt(0.5))) if act == "gelu" else v


def _linear(s):
    v = s["x"].float() @ s["W"].float().t()
    if s["b"] is not None:
        v = v + s["b"]
    v = _act(v, s["act"])
    if s["r"] is not None:
        v = v + s["r"].float()
    return v.to(s["y"].dtype)


def _norm(y, z, w, groups):
    v = (y * _silu(z)).unflatten(-1, (groups, -1))
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    return v.flatten(-2) * w


def _padded(s, quantum):
    """[seqs, longest] token indices of the packed rows, and which are real."""
    cu = s["cu"].long()
    at = torch.arange(-(-max(1, s["longest"]) // quantum) * quantum, device=cu.device)
    real = at < (cu[1:] - cu[:-1])[:, None]
    return torch.where(real, cu[:-1, None] + at, 0), real


def _conv(s):
    x, w = s["x"].float(), s["w"]
    k, slots, cu = w.shape[1], s["slots"].long(), s["cu"].long()
    old = torch.where(s["has"].bool()[:, None, None], s["state"][slots].float(), 0)
    at = torch.arange(x.shape[0], device=x.device)
    seq = torch.searchsorted(cu[1:].contiguous(), at, right=True)
    back = at[:, None] - (k - 1) + torch.arange(k, device=x.device)
    before = back < cu[seq][:, None]                     # taps that lie in the carried state
    carried = (back - cu[seq][:, None]) + (k - 1)
    taps = torch.where(before[..., None], old[seq[:, None], carried.clamp(0, k - 2)], x[back.clamp(min=0)])
    y = _silu((taps * w.t()).sum(1) + s["b"])
    # the last k - 1 inputs of each sequence, older ones from its carried state
    last = cu[1:, None] - (k - 1) + torch.arange(k - 1, device=x.device)
    early = last < cu[:-1, None]
    kept = (last - cu[:-1, None] + (k - 1)).clamp(0, k - 2)
    new = torch.where(early[..., None], torch.gather(old, 1, kept[..., None].expand(-1, -1, x.shape[1])),
                      x[last.clamp(min=0)])
    s["state"][slots] = new.to(s["state"].dtype)
    return y.to(s["x"].dtype), s["state"]


def _scan(s):
    """The scan in chunks: inside a chunk as a masked product, between chunks
    through the chunks' states."""
    h, p, gr, n, q = s["heads"], s["head_dim"], s["groups"], s["d_state"], QUANTUM
    at, real = _padded(s, q)
    b, c = at.shape[0], at.shape[1] // q
    xbc = s["xbc"].float()[at].unflatten(1, (c, q))
    x = xbc[..., :h * p].unflatten(-1, (h, p))
    bb = xbc[..., h * p:h * p + gr * n].unflatten(-1, (gr, n))
    cc = xbc[..., h * p + gr * n:].unflatten(-1, (gr, n))
    dt = _softplus(s["dt"].float()[at] + s["dt_bias"])
    dt = torch.where(real[..., None], dt, 0).unflatten(1, (c, q))
    cum = (dt * s["A"]).cumsum(2)                                    # [b, c, q, h]
    cum_t = cum.permute(0, 1, 3, 2)
    low = torch.ones(q, q, dtype=torch.bool, device=x.device).tril()
    decay = torch.exp(torch.where(low, cum_t[..., :, None] - cum_t[..., None, :], -math.inf))
    scores = torch.einsum("bcqgn,bckgn->bcgqk", cc, bb).repeat_interleave(h // gr, 2) * decay
    dtx = dt[..., None] * x
    y = torch.einsum("bchqk,bckhp->bcqhp", scores, dtx)
    to_end = torch.exp(cum[:, :, -1:] - cum)
    made = torch.einsum("bckgip,bckgn->bcgipn", (to_end[..., None] * dtx).unflatten(3, (gr, -1)), bb)
    made = made.flatten(2, 3)                                        # each chunk's own state
    total = torch.nn.functional.pad(cum[:, :, -1].double().cumsum(1), (0, 0, 1, 0))  # [b, c + 1, h]
    total = total.permute(0, 2, 1)
    past = torch.ones(c + 1, c, dtype=torch.bool, device=x.device).tril(-1)
    carry = torch.exp(torch.where(past, total[..., :, None] - total[..., None, 1:], -math.inf)).float()
    slots = s["slots"].long()
    first = torch.where(s["has"].bool()[:, None, None, None], s["state"][slots], 0)
    starts = torch.einsum("bhzc,bchpn->bzhpn", carry, made)
    starts = starts + torch.exp(total).float().permute(0, 2, 1)[..., None, None] * first[:, None]
    inter = torch.einsum("bcqgn,bcgipn->bcqgip", cc, starts[:, :-1].unflatten(2, (gr, -1))).flatten(3, 4)
    y = y + torch.exp(cum)[..., None] * inter + s["D"][:, None] * x
    out = torch.empty_like(s["y"])
    out[at[real]] = y.flatten(1, 2)[real].flatten(1).to(out.dtype)
    s["state"][slots] = starts[:, -1]
    return out, s["state"]


def _token(s):
    h, p, gr, n = s["heads"], s["head_dim"], s["groups"], s["d_state"]
    row, slots = s["row"].float(), s["slots"].long()
    width = h * p + 2 * gr * n
    z, dt = row[:, :h * p], row[:, h * p + width:h * p + width + h]
    taps = torch.cat([s["conv"][slots].float(), row[:, None, h * p:h * p + width]], 1)
    v = _silu((taps * s["cw"].t()).sum(1) + s["cb"])
    s["conv"][slots] = taps[:, 1:].to(s["conv"].dtype)
    x = v[:, :h * p].unflatten(1, (h, p))
    bb = v[:, h * p:h * p + gr * n].unflatten(1, (gr, n)).repeat_interleave(h // gr, 1)
    cc = v[:, h * p + gr * n:].unflatten(1, (gr, n)).repeat_interleave(h // gr, 1)
    dt = _softplus(dt + s["dt_bias"])
    new = torch.exp(dt * s["A"])[..., None, None] * s["state"][slots]
    new = new + (dt[..., None] * x)[..., None] * bb[:, :, None]
    s["state"][slots] = new
    y = (new * cc[:, :, None]).sum(-1) + s["D"][:, None] * x
    return _norm(y.flatten(1), z, s["nw"], gr).to(s["y"].dtype), s["conv"], s["state"]


@functools.lru_cache(None)
def _kernels():
    from ervf_b200 import GPUKernels

    return GPUKernels()


def _call(s):
    """The calls a user's program makes."""
    k, op = _kernels(), s["op"]
    if op == "linear":
        k.linear_bf16(s["y"], s["W"], s["x"], s["rows"], s["cols"], s["tokens"], bias=s["b"], act=s["act"],
                      resid=s["r"])
        return s["y"]
    if op == "norm":
        k.gated_norm(s["y"], s["x"], s["z"], s["w"], s["tokens"], s["groups"], s["group_size"], eps=EPS)
        return s["y"]
    if op == "conv":
        k.conv1d_prompt(s["y"], s["x"], s["w"], s["b"], s["state"], s["cu"], s["seqs"], s["tokens"],
                        s["channels"], s["width"], slots=s["slots"], has_state=s["has"])
        return s["y"], s["state"]
    h, p, gr, n = s["heads"], s["head_dim"], s["groups"], s["d_state"]
    width = h * p + 2 * gr * n
    if op == "scan":
        x, b, c = s["xbc"][:, :h * p], s["xbc"][:, h * p:h * p + gr * n], s["xbc"][:, h * p + gr * n:]
        k.ssm_prompt(s["y"], x, s["dt"], s["A"], b, c, s["D"], s["dt_bias"], s["state"], s["cu"], s["seqs"],
                     s["tokens"], h, p, gr, n, slots=s["slots"], has_state=s["has"])
        return s["y"], s["state"]
    z, xbc, dt = s["row"][:, :h * p], s["row"][:, h * p:h * p + width], s["row"][:, h * p + width:]
    k.ssm_token(s["y"], xbc, dt, s["cw"], s["cb"], s["conv"], s["A"], s["D"], s["dt_bias"], s["state"],
                s["seqs"], h, p, gr, n, s["width"], z=z, norm_w=s["nw"], eps=EPS, slots=s["slots"])
    return s["y"], s["conv"], s["state"]


def run(state):
    if own:
        return _call(state)
    return {"linear": _linear, "conv": _conv, "scan": _scan, "token": _token,
            "norm": lambda s: _norm(s["x"].float(), s["z"].float(), s["w"], s["groups"]).to(s["y"].dtype)
            }[state["op"]](state)


def work(case):
    op = case["op"]
    if op == "linear":
        r, c, t, o = case["rows"], case["cols"], case["tokens"], 4 if case["out"] == "f32" else 2
        return {"bytes": 2 * r * c + 2 * t * c + t * r * o * (1 + case["resid"]) + 4 * r * case["bias"],
                "flops": 2 * r * c * t}
    e = 4 if case["type"] == "f32" else 2
    if op == "norm":
        n = case["tokens"] * case["groups"] * case["group_size"]
        return {"bytes": 3 * n * e + 4 * case["groups"] * case["group_size"], "flops": 8 * n}
    if op == "conv":
        t, ch, w, b = case["tokens"], case["channels"], case["width"], case["seqs"]
        return {"bytes": 2 * t * ch * e + 4 * ch * (w + 1) + 2 * b * ch * (w - 1) * e,
                "flops": t * ch * (2 * w + 4)}
    h, p, gr, n, b = case["heads"], case["head_dim"], case["groups"], case["d_state"], case["seqs"]
    if op == "scan":
        t = case["tokens"]
        return {"bytes": t * e * (2 * h * p + 2 * gr * n + h) + 4 * b * h * p * n * (2 if b > 1 else 1),
                "flops": 5 * t * h * p * n}
    width, w = h * p + 2 * gr * n, case["width"]
    return {"bytes": b * e * (2 * h * p + width + h + 2 * (w - 1) * width) + 8 * b * h * p * n
            + 4 * width * (w + 1), "flops": 5 * b * h * p * n}


# ------------------------------------------------------------ in 64 bits


def _gate(v):
    return v * torch.sigmoid(v)


def _exact_norm(y, z, w, groups):
    v = (y * _gate(z)).reshape(y.shape[0], groups, -1)
    scale = torch.linalg.vector_norm(v, dim=-1, keepdim=True) / math.sqrt(v.shape[-1])
    return (v / torch.sqrt(scale ** 2 + EPS)).reshape(y.shape) * w.double()


def _steps(dt, bias):
    return torch.logaddexp(dt.double() + bias.double(), torch.zeros((), dtype=torch.float64, device=dt.device))


def _exact_conv(s):
    x, w, cu = s["x"].double(), s["w"].double(), s["cu"].tolist()
    k, y, state = w.shape[1], torch.empty_like(s["x"], dtype=torch.float64), s["state"].double()
    for i, slot in enumerate(s["slots"].tolist()):
        head = state[slot] if s["has"][i] else torch.zeros_like(state[slot])
        line = torch.cat([head, x[cu[i]:cu[i + 1]]])
        m = cu[i + 1] - cu[i]
        total = s["b"].double().expand(m, -1)
        for j in range(k):
            total = total + line[j:j + m] * w[:, j]
        y[cu[i]:cu[i + 1]] = _gate(total)
        state[slot] = line[line.shape[0] - (k - 1):]
    return y, state


def _exact_scan(s):
    h, p, gr, n = s["heads"], s["head_dim"], s["groups"], s["d_state"]
    cu, slots = s["cu"].long(), s["slots"].long()
    state, all_y = s["state"].double(), torch.empty(s["y"].shape, dtype=torch.float64, device=cu.device)
    xbc, dt = s["xbc"].double(), _steps(s["dt"], s["dt_bias"])
    decay = torch.exp(dt * s["A"].double())
    now = torch.where(s["has"].bool()[:, None, None, None], state[slots], 0)
    order = torch.argsort(cu[1:] - cu[:-1], descending=True)
    lens = (cu[1:] - cu[:-1])[order].tolist()
    now, begin = now[order], cu[:-1][order]
    live = len(lens)
    for t in range(s["longest"]):
        while lens[live - 1] <= t:
            live -= 1
        at = begin[:live] + t
        x = xbc[at, :h * p].reshape(live, h, p)
        b = xbc[at, h * p:h * p + gr * n].reshape(live, gr, 1, n)
        c = xbc[at, h * p + gr * n:].reshape(live, gr, n, 1)
        m = now[:live]
        m.mul_(decay[at][..., None, None])
        m.view(live, gr, -1, n).add_((dt[at][..., None] * x).reshape(live, gr, -1, 1) * b)
        y = torch.matmul(m.view(live, gr, -1, n), c).reshape(live, h, p)
        all_y[at] = (y + s["D"].double()[:, None] * x).reshape(live, h * p)
    state[slots[order]] = now
    return all_y, state


def _exact_token(s):
    h, p, gr, n = s["heads"], s["head_dim"], s["groups"], s["d_state"]
    width, slots = h * p + 2 * gr * n, s["slots"].long()
    row, conv, state = s["row"].double(), s["conv"].double(), s["state"].double()
    line = torch.cat([conv[slots], row[:, None, h * p:h * p + width]], 1)
    v = s["cb"].double().expand(line.shape[0], -1)
    for j in range(line.shape[1]):
        v = v + line[:, j] * s["cw"].double()[:, j]
    v = _gate(v)
    conv[slots] = line[:, 1:]
    dt = _steps(row[:, h * p + width:h * p + width + h], s["dt_bias"])
    y = torch.empty(row.shape[0], h, p, dtype=torch.float64, device=row.device)
    now = state[slots]
    for i in range(h):
        g = i // (h // gr)
        x = v[:, i * p:(i + 1) * p]
        b = v[:, h * p + g * n:h * p + (g + 1) * n]
        c = v[:, h * p + gr * n + g * n:h * p + gr * n + (g + 1) * n]
        now[:, i] = now[:, i] * torch.exp(dt[:, i] * s["A"][i].double())[:, None, None] \
            + (dt[:, i, None] * x)[:, :, None] * b[:, None]
        y[:, i] = torch.matmul(now[:, i], c[:, :, None])[..., 0] + s["D"][i].double() * x
    state[slots] = now
    return _exact_norm(y.reshape(row.shape[0], -1), row[:, :h * p], s["nw"], gr), conv, state


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        v = torch.nn.functional.linear(s["x"].double(), s["W"].double(),
                                       None if s["b"] is None else s["b"].double())
        if case["act"] == "relu2":
            v = torch.relu(v).square()
        elif case["act"] == "silu":
            v = _gate(v)
        elif case["act"] == "gelu":
            v = v * torch.special.ndtr(v)
        return v if s["r"] is None else v + s["r"].double()
    if op == "norm":
        return _exact_norm(s["x"].double(), s["z"].double(), s["w"], case["groups"])
    return {"conv": _exact_conv, "scan": _exact_scan, "token": _exact_token}[op](s)
