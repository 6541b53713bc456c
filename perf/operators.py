"""Cases, plain forms and exact values of the group-limited router and the
block-scaled 8-bit matrix products (dense, shared expert, routed experts).

``listed()`` and ``draw()`` give the cases, ``prepare()`` what a program has
in hand before the call, ``run()`` one call: of the library's entry points
where ``own`` is true, else of the same operator written out in elementary
torch operations in 32 bits. ``exact()`` computes the definition in 64 bits.

Operators (E4M3 values; a 32-bit scale per 128 of a row of activations, one per
128 x 128 block of a weight; a row's block with largest magnitude a >= 1e-12 is
held as e4m3(x * f32(448 / a)) with the scale f32(a / 448)):

    route    scores s of the logits, the best groups by their two best s + bias
             (or their best), the top-k of s + bias in these groups, gates s / sum
    linear   y = x W^T, x quantized in the call, W [N, K] held in 8 bits
    mlp      y = (silu(x G^T) * (x U^T)) D^T, both sets of activations quantized
    experts  the same per routed row with its expert's weights, then the sum of
             a token's rows by gate * scaling
"""

import importlib
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
F8 = torch.float8_e4m3fn
BF16 = torch.bfloat16


# -- cases -----------------------------------------------------------------

def listed():
    return [
        # one token being decoded: nothing but latency
        dict(name="route_1", op="route", t=1, e=256, k=8, groups=8, top=4, act="sigmoid", bias=True),
        # a prompt of odd length, softmax scores, groups judged by their best expert
        dict(name="route_4099_softmax", op="route", t=4099, e=96, k=6, groups=6, top=3, act="softmax", bias=False),
        # a full batch of the size of the largest layer benchmark
        dict(name="route_16384", op="route", t=16384, e=256, k=8, groups=8, top=4, act="sigmoid", bias=True),
        # a projection for one token: the weight is read once, nothing else counts
        dict(name="linear_1", op="linear", m=1, n=4096, k=4096),
        # ragged in every direction: a last block of 16 columns, an odd number of outputs
        dict(name="linear_77_ragged", op="linear", m=77, n=1001, k=1040),
        # a projection over an ordinary batch
        dict(name="linear_4096", op="linear", m=4096, n=4096, k=2048),
        # the largest projection
        dict(name="linear_16384", op="linear", m=16384, n=8192, k=4096),
        # the shared expert beside the small-batch layer
        dict(name="mlp_512", op="mlp", m=512, c=1024, f=2048),
        # the shared expert over half of the largest batch
        dict(name="mlp_8192", op="mlp", m=8192, c=2048, f=1536),
        # one token being decoded: eight experts' weights are read once
        dict(name="experts_1", op="experts", t=1, c=2048, f=1536, e=64, k=8),
        # the small-batch latency layer
        dict(name="experts_512", op="experts", t=512, c=1024, f=2048, e=32, k=2),
        # the largest layer
        dict(name="experts_16384", op="experts", t=16384, c=2048, f=1536, e=64, k=4),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["route", "linear", "linear", "mlp", "experts", "experts"])
    if op == "route":
        groups = rng.choice([2, 4, 6, 8, 16])
        e = groups * rng.randint(2, 256 // groups)
        top = rng.randint(1, groups)
        k = rng.randint(1, min(8, top * (e // groups)))
        return dict(op=op, t=_log(rng, 1, 16384), e=e, k=k, groups=groups, top=top,
                    act=rng.choice(["sigmoid", "softmax"]), bias=rng.random() < 0.7)
    if op == "linear":
        return dict(op=op, m=_log(rng, 1, 16384), n=_log(rng, 64, 8192), k=16 * _log(rng, 8, 256))
    if op == "mlp":
        return dict(op=op, m=_log(rng, 1, 8192), c=128 * rng.randint(2, 16), f=128 * rng.randint(2, 16))
    e = rng.choice([8, 16, 32, 48, 64])
    return dict(op=op, t=_log(rng, 1, 16384), c=128 * rng.randint(2, 16), f=128 * rng.randint(2, 12), e=e,
                k=rng.randint(1, 4))


def work(case):
    op = case["op"]
    if op == "route":
        t, e, k = case["t"], case["e"], case["k"]
        return {"bytes": t * e * 4 + (e * 4 if case["bias"] else 0) + t * k * 10, "flops": 10 * t * e}
    blocks = lambda n, k: 4 * -(-n // BLOCK) * -(-k // BLOCK)  # noqa: E731
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k + blocks(n, k) + 2 * m * n, "flops": 2 * m * n * k}
    c, f = case["c"], case["f"]
    expert = 3 * c * f + 3 * blocks(c, f)
    if op == "mlp":
        return {"bytes": 4 * case["m"] * c + expert, "flops": 6 * case["m"] * c * f}
    t, k = case["t"], case["k"]
    return {"bytes": 4 * t * c + 10 * t * k + min(case["e"], t * k) * expert, "flops": 6 * t * k * c * f}


# -- inputs ----------------------------------------------------------------

def _weight(gen, *shape):
    """A weight ~ N(0, 0.02) as E4M3 values and a scale per 128 x 128 block."""
    n, k = shape[-2:]
    w = torch.randn(*shape, generator=gen, device="cuda").mul_(0.02)
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n))
    w = w.view(*shape[:-2], nb, BLOCK, kb, BLOCK)
    scale = w.abs().amax(dim=(-3, -1)).clamp_(min=1e-12) / E4M3_MAX
    w = (w / scale[..., :, None, :, None]).view(*shape[:-2], nb * BLOCK, kb * BLOCK)
    return w[..., :n, :k].to(F8).contiguous(), scale.contiguous()


def _activations(gen, rows, cols):
    """~ N(0, 1), a few columns eight times as large, as activations have them."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x[:, torch.randint(0, cols, (max(1, cols // 256),), generator=gen, device="cuda")] *= 8.0
    return x.to(BF16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "route":
        logits = torch.randn(case["t"], case["e"], generator=gen, device="cuda")
        bias = torch.randn(case["e"], generator=gen, device="cuda").mul_(0.1) if case["bias"] else None
        return dict(case, logits=logits, expert_bias=bias)
    if op == "linear":
        q, scale = _weight(gen, case["n"], case["k"])
        return dict(case, x=_activations(gen, case["m"], case["k"]), q=q, scale=scale)
    c, f = case["c"], case["f"]
    lead = (case["e"],) if op == "experts" else ()
    gate_up_q, gate_up_scale = _weight(gen, *lead, 2 * f, c)
    down_q, down_scale = _weight(gen, *lead, c, f)
    state = dict(case, gate_up_q=gate_up_q, gate_up_scale=gate_up_scale, down_q=down_q, down_scale=down_scale)
    if op == "mlp":
        return dict(state, x=_activations(gen, case["m"], c))
    t, e, k = case["t"], case["e"], case["k"]
    logits = torch.randn(t, e, generator=gen, device="cuda")
    logits += 0.25 * torch.randn(e, generator=gen, device="cuda")  # some experts are liked more than others
    score, top_idx = torch.topk(torch.sigmoid(logits), k)
    gate = (score / score.sum(-1, keepdim=True)).to(BF16)
    return dict(state, x=_activations(gen, t, c), top_idx=top_idx, gate=gate, scaling=2.5)


# -- one call --------------------------------------------------------------

def run(state):
    op = state["op"]
    if own:
        ops = importlib.import_module("praxis-1-oss_b200").ops
        if op == "route":
            return ops.route(state["logits"], state["expert_bias"], state["k"], state["act"], groups=state["groups"],
                             top_groups=state["top"], group_score="top2" if state["act"] == "sigmoid" else "max")
        if op == "linear":
            return ops.fp8_linear(state["x"], state["q"], state["scale"])
        if op == "mlp":
            return ops.fp8_mlp(state["x"], state["gate_up_q"], state["gate_up_scale"], state["down_q"],
                               state["down_scale"])
        return ops.fp8_moe_forward(state["x"], state["top_idx"], state["gate"], state["gate_up_q"],
                                   state["gate_up_scale"], state["down_q"], state["down_scale"], state["scaling"])
    if op == "route":
        return plain_route(state)
    if op == "linear":
        return (plain_quantized(state["x"].float()) @ plain_weight(state["q"], state["scale"]).T).to(BF16)
    if op == "mlp":
        return plain_swiglu(state["x"].float(), plain_weight(state["gate_up_q"], state["gate_up_scale"]),
                            plain_weight(state["down_q"], state["down_scale"])).to(BF16)
    return plain_experts(state)


def plain_weight(q, scale):
    """The 32-bit values that E4M3 values and block scales stand for."""
    n, k = q.shape[-2:]
    full = scale.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]
    return q.float() * full


def plain_quantized(x):
    """x rounded to E4M3 with a scale per 128 of a row, as the values it then stands for."""
    k = x.shape[-1]
    kb = -(-k // BLOCK)
    b = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).unflatten(-1, (kb, BLOCK))
    amax = b.abs().amax(-1, keepdim=True).clamp(min=1e-12)
    most = torch.full_like(amax, E4M3_MAX)
    return ((b * (most / amax)).to(F8).float() * (amax / most)).flatten(-2)[..., :k]


def plain_swiglu(x, gate_up, down):
    """Rows x [.., R, C] through gate_up [.., 2F, C] and down [.., C, F]."""
    gate, up = (plain_quantized(x) @ gate_up.mT).chunk(2, dim=-1)
    return plain_quantized(gate * torch.sigmoid(gate) * up) @ down.mT


def plain_route(state):
    logits, bias, groups = state["logits"], state["expert_bias"], state["groups"]
    t, e = logits.shape
    if state["act"] == "sigmoid":
        score = torch.reciprocal(1.0 + torch.exp(-logits))
    else:
        p = torch.exp(logits - logits.amax(-1, keepdim=True))
        score = p / p.double().sum(-1, keepdim=True).float()  # in 64 bits: the sum's order moves no border
    choice = score if bias is None else score + bias
    best = torch.sort(choice.view(t, groups, e // groups), dim=-1, descending=True).values
    of_group = best[..., :2].sum(-1) if state["act"] == "sigmoid" else best[..., 0]
    kept = torch.sort(of_group, dim=-1, descending=True, stable=True).indices[:, : state["top"]]
    open_ = torch.zeros(t, groups, dtype=torch.bool, device=logits.device).scatter_(1, kept, True)
    choice = choice.masked_fill(~open_.repeat_interleave(e // groups, 1), -math.inf)
    top_idx = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, : state["k"]].contiguous()
    picked = score.gather(1, top_idx)
    return top_idx, (picked / picked.sum(-1, keepdim=True)).to(BF16)


def plain_experts(state):
    x, top_idx, gate = state["x"], state["top_idx"], state["gate"]
    t, k = top_idx.shape
    e = state["e"]
    weight = gate.float() * state["scaling"]
    if t * k <= e:  # few rows: each with its expert's weights
        pick = top_idx.flatten()
        gate_up = plain_weight(state["gate_up_q"][pick], state["gate_up_scale"][pick])
        down = plain_weight(state["down_q"][pick], state["down_scale"][pick])
        rows = plain_swiglu(x.float().repeat_interleave(k, 0)[:, None], gate_up, down)[:, 0]
        return (rows.view(t, k, -1) * weight[..., None]).sum(1).to(BF16)
    flat = top_idx.flatten()
    order = torch.sort(flat, stable=True).indices
    counts = torch.bincount(flat, minlength=e)
    room = int(counts.max())
    place = torch.arange(t * k, device=x.device) - (counts.cumsum(0) - counts)[flat[order]]
    slot = flat[order] * room + place
    packed = torch.zeros(e * room, x.shape[1], device=x.device)
    packed[slot] = x.float()[order // k]
    rows = plain_swiglu(packed.view(e, room, -1), plain_weight(state["gate_up_q"], state["gate_up_scale"]),
                        plain_weight(state["down_q"], state["down_scale"])).view(e * room, -1)
    back = torch.empty_like(slot)
    back[order] = slot
    return (rows[back].view(t, k, -1) * weight[..., None]).sum(1).to(BF16)


# -- the definition in 64 bits ---------------------------------------------

def _exact_weight(q, scale):
    w = q.double()
    for i in range(scale.shape[-2]):
        for j in range(scale.shape[-1]):
            w[..., i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scale[..., i, j, None, None].double()
    return w


def _exact_rows(x):
    # the two factors of a block, 448 / a and a / 448, are 32-bit numbers by definition
    y = torch.empty_like(x)
    for j in range(0, x.shape[-1], BLOCK):
        b = x[..., j:j + BLOCK]
        a = torch.clamp(torch.amax(torch.abs(b), -1, True), min=1e-12)
        y[..., j:j + BLOCK] = (b * (E4M3_MAX * a.reciprocal()).float()).to(F8).double() * (a / E4M3_MAX).float()
    return y


def _exact_mlp(x, gate_up, down):
    h = torch.matmul(_exact_rows(x), gate_up.transpose(-1, -2))
    f = h.shape[-1] // 2
    g, u = h[..., :f], h[..., f:]
    return torch.matmul(_exact_rows(g / (1 + torch.exp(-g)) * u), down.transpose(-1, -2))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "route":
        z = s["logits"].double()
        z = 1 / (1 + torch.exp(-z)) if case["act"] == "sigmoid" else torch.softmax(z, -1)
        c = z if s["expert_bias"] is None else z + s["expert_bias"].double()
        t, e, groups = case["t"], case["e"], case["groups"]
        g = c.reshape(t, groups, e // groups)
        g = g.topk(min(2, e // groups), -1).values.sum(-1) if case["act"] == "sigmoid" else g.amax(-1)
        shut = torch.ones(t, groups, dtype=torch.bool, device=c.device)
        shut.scatter_(1, g.topk(case["top"], -1).indices, False)
        c = c.reshape(t, groups, -1).masked_fill(shut[..., None], -math.inf).reshape(t, e)
        v = z.gather(1, c.topk(case["k"], -1).indices)
        return None, v / v.sum(-1, keepdim=True)  # indices are whole numbers: no value in 64 bits
    x = s["x"].double()
    if op == "linear":
        return _exact_rows(x) @ _exact_weight(s["q"], s["scale"]).T
    if op == "mlp":
        return _exact_mlp(x, _exact_weight(s["gate_up_q"], s["gate_up_scale"]),
                          _exact_weight(s["down_q"], s["down_scale"]))
    y = torch.zeros_like(x)
    for i in torch.unique(s["top_idx"]).tolist():
        token, place = torch.nonzero(s["top_idx"] == i, as_tuple=True)
        rows = _exact_mlp(x[token], _exact_weight(s["gate_up_q"][i], s["gate_up_scale"][i]),
                          _exact_weight(s["down_q"][i], s["down_scale"][i]))
        y.index_add_(0, token, rows * (s["gate"][token, place].double() * s["scaling"])[:, None])
    return y
