"""The operators of a quantised MoE block, as they are measured: the residual add
and RMSNorm that also leaves its row in 8 bits, the routing of expert groups,
and the expert FFN on 4-bit weights.

Formats (both with one power-of-two scale per 32 consecutive values of a row,
stored as its exponent + 127 in a byte):
  8 bits  e4m3 codes; the scale 2^e is the smallest with max|v| <= 448 * 2^e
  4 bits  e2m1 codes, two per byte, the even column in the low half

A case is a dict of plain values:
  op      norm     r = x + residual; n = rmsnorm(r); n in 8 bits
          route    logits -> the K experts of each token and their weights
          experts  tokens in 8 bits through gate|up, the gated activation in 8
                   bits through down, summed with the routing weights
  T H E K I        tokens, hidden size, experts, top-k, expert width
  dtype            of x, residual and the results
  scoring, bias, groups, topk_groups, group_score, scale   of a route
  act, skew        of the experts; skew: Zipf exponent of their popularity
"""

from __future__ import annotations

import math

import torch

own = False  # True: the framework's own operators instead of the plain forms

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-5
SIGMA_W = 0.02
BLOCK = 32
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _norm_case(T, H, dtype="bf16", bias=False, **name):
    return dict(op="norm", T=T, H=H, dtype=dtype, bias=bias, **name)


def _route_case(T, E, K, scoring, bias, groups=1, topk_groups=1, group_score="max", scale=1.0,
                **name):
    return dict(op="route", T=T, E=E, K=K, scoring=scoring, bias=bias, groups=groups,
                topk_groups=topk_groups, group_score=group_score, scale=scale, **name)


def _experts_case(T, H, E, K, I, dtype="bf16", act="silu", skew=0.0, **name):
    return dict(op="experts", T=T, H=H, E=E, K=K, I=I, dtype=dtype, act=act, skew=skew, **name)


def listed():
    return [
        # One sequence generating: the launch and its latency.
        _norm_case(1, 4096, name="norm_decode_1"),
        # A generating batch of odd size, a norm with a bias.
        _norm_case(37, 2048, dtype="f16", bias=True, name="norm_batch_37"),
        # A long prompt.
        _norm_case(4096, 4096, name="norm_prompt_4096"),
        # A generating batch; softmax scores, the best groups by their best expert.
        _route_case(8, 160, 6, "softmax", False, 8, 3, "max", 16.0, name="route_decode_8"),
        # A prompt of odd length, balanced by a bias, without groups.
        _route_case(999, 64, 6, "sigmoid", True, name="route_prompt_999"),
        # Long prompts of many sequences, groups by the sum of their best two.
        _route_case(16384, 256, 8, "sigmoid", True, 8, 4, "top2", 2.5, name="route_prompt_16384"),
        # One sequence generating: the routed experts' weights stream for one row.
        _experts_case(1, 4096, 8, 2, 14336, name="experts_decode_1"),
        # A generating batch over many small experts.
        _experts_case(16, 2048, 64, 6, 1408, name="experts_fine_decode_16"),
        # A large generating batch, or a short prompt, of odd length.
        _experts_case(197, 4096, 8, 2, 14336, dtype="f16", name="experts_mixed_197"),
        # Sizes that are no multiple of a tile, skewed routing, another activation.
        _experts_case(333, 1248, 12, 3, 3296, act="gelu_tanh", skew=0.8,
                      name="experts_ragged_333"),
        # A long prompt through many small experts.
        _experts_case(4096, 2048, 64, 6, 1408, skew=0.3, name="experts_fine_prompt_4096"),
        # A long prompt through large experts.
        _experts_case(4096, 4096, 8, 2, 14336, skew=0.3, name="experts_prompt_4096"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "route", "route", "experts", "experts", "experts"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "norm":
        return _norm_case(_log_int(rng, 1, 8192), BLOCK * _log_int(rng, 16, 256),
                          dtype=rng.choice(["bf16", "f16", "f32"]), bias=rng.random() < 0.3)
    if op == "route":
        E = rng.choice([8, 16, 24, 60, 64, 96, 128, 160, 192, 256])
        G = rng.choice([g for g in (1, 1, 2, 4, 8, 12, 16) if E % g == 0 and E // g >= 2])
        tg = rng.randint(1, G)
        return _route_case(_log_int(rng, 1, 16384), E, rng.randint(1, min(12, tg * (E // G))),
                           rng.choice(["softmax", "sigmoid"]), rng.random() < 0.6, G, tg,
                           rng.choice(["max", "top2"]), rng.choice([1.0, 2.5]))
    # weights of at most 10^9 elements, most sizes no multiple of a tile
    H, I = BLOCK * _log_int(rng, 16, 160), BLOCK * _log_int(rng, 16, 160)
    most = min(64, int(1e9 / (3 * H * I)))
    E = _log_int(rng, 1, most)
    return _experts_case(_log_int(rng, 1, 2048), H, E, rng.randint(1, min(E, 8)), I, dtype=dtype,
                         act=rng.choice(["silu", "silu", "gelu", "gelu_tanh"]),
                         skew=rng.choice([0.0, 0.3, 1.1]))


# ------------------------------------------------------------------- inputs
def _routing(c, gen):
    """Distinct experts per token with a Zipf popularity, and their weights."""
    T, E, K = c["T"], c["E"], c["K"]
    logits = torch.empty((T, E), device="cuda").normal_(0.0, 1.0, generator=gen)
    rank = torch.randperm(E, generator=gen, device="cuda")
    ids = torch.argsort(logits - c["skew"] * torch.log1p(rank.float()), dim=-1,
                        descending=True)[:, :K].contiguous()
    w = torch.softmax(torch.gather(logits, 1, ids), -1)
    return w.contiguous(), ids


def _weights_4bit(E, N, K, gen):
    """[E, N, K/2] codes and [E, N, K/32] scales of N(0, 0.02) weights, each
    block scaled so that its largest value is at most 6 and above 3."""
    codes = torch.empty((E, N, K // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty((E, N, K // BLOCK), dtype=torch.uint8, device="cuda")
    half = torch.tensor([(a + b) / 2 for a, b in zip(FP4, FP4[1:])], device="cuda")
    for e in range(E):
        w = torch.empty((N, K // BLOCK, BLOCK), device="cuda").normal_(0.0, SIGMA_W, generator=gen)
        m, ex = torch.frexp(w.abs().amax(-1, keepdim=True))  # 6 = 0.75 * 2^3
        ex = torch.where(m <= 0.75, ex - 3, ex - 2)
        w = w * _pow2(127 - ex)
        q = torch.bucketize(w.abs(), half).to(torch.uint8) | (w < 0).to(torch.uint8) * 8
        q = q.reshape(N, K // 2, 2)
        codes[e] = q[..., 0] | q[..., 1] << 4
        scales[e] = (ex[..., 0] + 127).to(torch.uint8)
    return codes, scales


def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    d = {}
    if c["op"] == "route":
        # logits as a router of unit-variance tokens gives them, and a bias of
        # the size that balancing experts leaves
        d["logits"] = torch.empty((c["T"], c["E"]), device="cuda").normal_(0.0, 1.3, generator=gen)
        d["bias"] = torch.empty(c["E"], device="cuda").normal_(0.0, 0.05, generator=gen) \
            if c["bias"] else None
        return d
    dt = DTYPES[c["dtype"]]

    def normal(mean, sigma, *shape):
        return torch.empty(shape, dtype=dt, device="cuda").normal_(mean, sigma, generator=gen)

    d["x"] = normal(0.0, 1.0, c["T"], c["H"])
    if c["op"] == "norm":
        d["residual"] = normal(0.0, 1.0, c["T"], c["H"])
        d["weight"] = normal(1.0, 0.1, c["H"])
        d["bias"] = normal(0.0, 0.1, c["H"]) if c["bias"] else None
        return d
    d["topk_w"], d["topk_ids"] = _routing(c, gen)
    d["w1"] = _weights_4bit(c["E"], 2 * c["I"], c["H"], gen)  # gate rows, then up rows
    d["w2"] = _weights_4bit(c["E"], c["H"], c["I"], gen)
    return d


@torch.no_grad()
def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = case
    if own and case["op"] == "norm":
        from reframework_amd.layers import RMSNorm
        norm = RMSNorm(case["H"], EPS, bias=case["bias"])
        norm.weight.data = d.pop("weight")
        if case["bias"]:
            norm.bias.data = d.pop("bias")
        d["norm"] = norm
    if own and case["op"] == "experts":
        from reframework_amd.moe import Mxfp4Experts
        # the codes of a checkpoint, laid out once for the kernels
        d["experts"] = Mxfp4Experts.from_codes(*d.pop("w1"), *d.pop("w2"))
    return d


# -------------------------------------------------------------- plain forms
def _pow2(b):
    """2^(b - 127) in 32 bits of bytes b in [0, 254], exactly."""
    b = b.int()
    return torch.where(b > 0, b << 23, torch.full_like(b, 1 << 22)).view(torch.float32)


def _to_8bit(v):
    """(codes, scale bytes) of fp32 rows."""
    b = v.reshape(v.shape[0], -1, BLOCK)
    amax = b.abs().amax(-1, keepdim=True)
    m, ex = torch.frexp(amax)  # amax = m * 2^ex, m in [1/2, 1); 448 = 0.875 * 2^9
    ex = torch.where(m <= 0.875, ex - 9, ex - 8).clamp_(min=-127)
    ex = torch.where(amax > 0, ex, torch.full_like(ex, -127))
    codes = (b * _pow2(127 - ex)).to(torch.float8_e4m3fn)
    return codes.reshape(v.shape), (ex + 127).to(torch.uint8).squeeze(-1)


def _from_8bit(codes, scales):
    b = codes.float().reshape(codes.shape[0], -1, BLOCK)
    return (b * _pow2(scales)[..., None]).reshape(codes.shape)


def _from_4bit(codes, scales):
    """fp32 [n, rows, columns] of [n, rows, columns / 2] codes."""
    one = torch.tensor(FP4 + tuple(-v for v in FP4), device=codes.device)
    pairs = torch.stack([one.repeat(16), one.repeat_interleave(16)], -1)  # by byte: low, high
    w = pairs[codes.int()].reshape(*scales.shape, BLOCK)
    w *= _pow2(scales)[..., None]
    return w.reshape(*codes.shape[:-1], -1)


def _act(name, g):
    if name == "silu":
        return g / (1.0 + torch.exp(-g))
    if name == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g / math.sqrt(2.0)))
    return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)))


def _norm_plain(s):
    dt = s["x"].dtype
    res = (s["x"].float() + s["residual"].float()).to(dt)
    r = res.float()
    n = r / torch.sqrt((r * r).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    if s["bias"] is not None:
        n = n + s["bias"].float()
    n = n.to(dt)
    codes, scales = _to_8bit(n.float())
    return n, codes, scales.view(torch.float8_e8m0fnu), res


def _scores(c, logits):
    if c["scoring"] == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits))
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _route_plain(s):
    # in 64 bits: what is chosen lies next to what is not
    c, logits = s["case"], s["logits"].double()
    T, E, K, G = c["T"], c["E"], c["K"], c["groups"]
    scores = _scores(c, logits)
    if s["bias"] is not None:
        choice = scores + s["bias"].double()
    elif c["group_score"] == "top2" and G > 1:
        choice = scores
    else:
        choice = logits  # the scores are in its order
    if G > 1:
        best = torch.sort(choice.reshape(T, G, E // G), dim=-1, descending=True)[0]
        gs = best[..., 0] + best[..., 1] if c["group_score"] == "top2" else best[..., 0]
        kept = torch.sort(gs, dim=-1, descending=True, stable=True)[1][:, :c["topk_groups"]]
        on = torch.zeros((T, G), dtype=torch.bool, device=logits.device)
        on[torch.arange(T, device=logits.device)[:, None], kept] = True
        choice = torch.where(on.repeat_interleave(E // G, 1), choice,
                             torch.full_like(choice, -math.inf))
    ids = torch.sort(choice, dim=-1, descending=True, stable=True)[1][:, :K]
    w = torch.gather(scores, 1, ids)
    w = w / (w.sum(-1, keepdim=True) + 1e-20) * c["scale"]
    return w.float(), ids


def _experts_plain(s):
    c, ids = s["case"], s["topk_ids"]
    T, H, K, I = (c[k] for k in "THKI")
    x = _from_8bit(*_to_8bit(s["x"].float()))
    used, group, count = torch.unique(ids, return_inverse=True, return_counts=True)
    n, most = used.numel(), int(count.max())
    # slot j in the order of its expert, at its place among the expert's slots
    order = torch.argsort(group.reshape(-1), stable=True)
    first = torch.cumsum(count, 0) - count
    g = group.reshape(-1)[order]
    row = torch.empty_like(order)
    row[order] = g * most + torch.arange(T * K, device=ids.device) - first[g]
    xg = torch.zeros((n * most, H), device=x.device)
    xg[row] = x.repeat_interleave(K, 0)
    w1, w2 = ([t[used] for t in s[k]] for k in ("w1", "w2"))
    gu = torch.bmm(xg.reshape(n, most, H), _from_4bit(*w1).transpose(1, 2)).reshape(-1, 2 * I)
    h = _from_8bit(*_to_8bit(_act(c["act"], gu[:, :I]) * gu[:, I:]))
    y = torch.bmm(h.reshape(n, most, I), _from_4bit(*w2).transpose(1, 2)).reshape(-1, H)
    out = (y[row].reshape(T, K, H) * s["topk_w"][..., None]).sum(1)
    return out.to(s["x"].dtype)


@torch.no_grad()
def run(state):
    c = state["case"]
    if not own:
        return {"norm": _norm_plain, "route": _route_plain, "experts": _experts_plain}[c["op"]](state)
    if c["op"] == "norm":
        normed, q, res = state["norm"].forward_add_residual_mxfp8(state["x"], state["residual"])
        return normed, q.codes, q.scales, res
    if c["op"] == "route":
        from reframework_amd.moe import grouped_topk
        return grouped_topk(state["logits"], c["K"], renormalize=True, scoring=c["scoring"],
                            bias=state["bias"], num_groups=c["groups"],
                            topk_groups=c["topk_groups"], group_score=c["group_score"],
                            scale=c["scale"])
    from reframework_amd.moe import fused_experts_mxfp4
    return fused_experts_mxfp4(state["x"], state["experts"], state["topk_w"], state["topk_ids"],
                               activation=c["act"])


def work(case):
    T = case["T"]
    if case["op"] == "route":
        E, K = case["E"], case["K"]
        return {"bytes": T * E * 4 + E * 4 + T * K * 12, "flops": T * E * 8}
    H, esz = case["H"], 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        return {"bytes": T * H * (4 * esz + 1) + T * H // BLOCK + H * esz, "flops": 8 * T * H}
    E, K, I = case["E"], case["K"], case["I"]
    # distinct experts that T tokens of K uniform choices reach
    used = E * (1.0 - (1.0 - K / E) ** T)
    return {"bytes": int(used * 3 * H * I * (0.5 + 1.0 / BLOCK) + 2 * T * H * esz + T * K * 12),
            "flops": 6 * T * K * H * I}


# -------------------------------------------------------------------- exact
def _round_8bit(v):
    """(values of the codes, scales) in 64 bits, from the format's definition."""
    b = v.reshape(v.shape[0], -1, BLOCK)
    amax = b.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(amax / 448.0)).clamp(min=-127.0))
    b = b / scale
    # e4m3: three bits below the leading one, down to 2^-6
    step = torch.exp2(torch.floor(torch.log2(b.abs().clamp(min=2.0 ** -6))) - 3.0)
    return (torch.round(b / step) * step).reshape(v.shape), scale.squeeze(-1)


def _through_8bit(v):
    codes, scale = _round_8bit(v)
    return codes * scale.repeat_interleave(BLOCK, 1)


def _weight64(codes, scales):
    lut = torch.tensor(FP4, dtype=torch.float64, device=codes.device)
    q = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1).long()
    v = lut[q & 7] * (1 - 2 * (q >> 3)).double()
    return v * torch.exp2(scales.double() - 127.0).repeat_interleave(BLOCK, 1)


@torch.no_grad()
def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["op"] == "norm":
        dt = d["x"].dtype
        res = (d["x"].double() + d["residual"].double()).to(dt).double()
        n = res * torch.rsqrt(res.square().mean(-1, keepdim=True) + EPS) * d["weight"].double()
        if d["bias"] is not None:
            n = n + d["bias"].double()
        codes, scale = _round_8bit(n.to(dt).double())  # of the row as it is stored
        return n, codes, scale, res
    if c["op"] == "route":
        E, K, G = c["E"], c["K"], c["groups"]
        x = d["logits"].double()
        p = torch.sigmoid(x) if c["scoring"] == "sigmoid" else torch.softmax(x, -1)
        by = p + (0.0 if d["bias"] is None else d["bias"].double())
        groups = by.reshape(-1, G, E // G)
        gs = groups.topk(2 if c["group_score"] == "top2" else 1, dim=-1)[0].sum(-1)
        last = torch.topk(gs, c["topk_groups"], dim=-1)[0][:, -1:]  # of distinct scores
        groups = groups.masked_fill((gs < last)[..., None], -math.inf)
        ids = torch.topk(groups.reshape(-1, E), K, dim=-1)[1]
        w = torch.gather(p, 1, ids)
        return w / (w.sum(-1, keepdim=True) + 1e-20) * c["scale"], ids
    x = _through_8bit(d["x"].double())
    out = torch.zeros_like(x)
    for e in range(c["E"]):
        tok, slot = torch.nonzero(d["topk_ids"] == e, as_tuple=True)
        if tok.numel():
            w1, w2 = (_weight64(d[k][0][e], d[k][1][e]) for k in ("w1", "w2"))
            g, u = (x[tok] @ w1.t()).chunk(2, -1)
            h = _through_8bit(_act(c["act"], g) * u)
            out.index_add_(0, tok, (h @ w2.t()) * d["topk_w"][tok, slot, None].double())
    return out
