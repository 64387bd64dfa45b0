"""Operators of an MoE block in training and with 8-bit weights, as they are measured:
the residual add and LayerNorm, tokens sorted by expert and back, the product with
weights in 8 bits of one scale per block of 128, and the expert FFN on such weights.

The 8-bit format: e4m3 codes (largest magnitude 448) with fp32 scales. Rows have one
scale per 128 consecutive values, weights one per 128 x 128 block; both blocks start at
multiples of 128, the last of a row or matrix may be smaller. With m the block's largest
magnitude, at least 448 * 2^-126, the scale is m / 448 and a value's code is
value * 448 / m, rounded to nearest even: of that quotient, not of the value over the
rounded scale, which turns 16-bit values' many ties into something near them.

A case is a dict of plain values:
  op      norm     r = x + residual; n = layernorm(r); training: the gradients too
          tokens   rows = x in the order of the experts; out = weighted sums of given
                   rows back in the order of the tokens; training: the gradients too
          product  rows grouped by matrix, quantised, times the matrices; training:
                   the gradient of the rows too
          experts  gate|up, the gated activation in 8 bits, down, summed with the
                   routing weights
  T H E K I        tokens, hidden size, experts, top-k, expert width
  N                result columns of a product; its rows are the T * K slots, its depth H
  dtype            of tokens and results
  train, drop, act, skew   drop: share of slots that go to no expert here; skew: Zipf
                   exponent of the experts' popularity
"""

from __future__ import annotations

import math

import torch

own = False  # True: the framework's own operators instead of the plain forms

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-5
SIGMA_W = 0.02
BLOCK = 128
E4M3_MAX = 448.0
SMALLEST = E4M3_MAX * 2.0 ** -126


def _norm_case(T, H, dtype="bf16", train=False, **name):
    return dict(op="norm", T=T, H=H, dtype=dtype, train=train, **name)


def _tokens_case(T, H, E, K, dtype="bf16", train=False, drop=0.0, skew=0.0, **name):
    return dict(op="tokens", T=T, H=H, E=E, K=K, dtype=dtype, train=train, drop=drop, skew=skew,
                **name)


def _product_case(T, H, E, K, N, dtype="bf16", train=False, skew=0.0, **name):
    return dict(op="product", T=T, H=H, E=E, K=K, N=N, dtype=dtype, train=train, skew=skew, **name)


def _experts_case(T, H, E, K, I, dtype="bf16", act="silu", skew=0.0, **name):
    return dict(op="experts", T=T, H=H, E=E, K=K, I=I, dtype=dtype, act=act, skew=skew, **name)


def listed():
    return [
        # One sequence generating: the launch and its latency.
        _norm_case(1, 4096, name="norm_decode_1"),
        # Training on a short batch of odd length and width.
        _norm_case(777, 1000, dtype="f16", train=True, name="norm_train_777"),
        # Training on a long batch.
        _norm_case(8192, 4096, train=True, name="norm_train_8192"),
        # A generating batch over many small experts.
        _tokens_case(16, 2048, 64, 6, name="tokens_decode_16"),
        # Training on one rank of several that share the experts: half of the slots
        # belong to the others.
        _tokens_case(999, 1248, 12, 3, dtype="f32", train=True, drop=0.5, skew=0.8,
                     name="tokens_train_999"),
        # Training on a long batch.
        _tokens_case(8192, 4096, 8, 2, train=True, skew=0.3, name="tokens_train_8192"),
        # One sequence generating: two experts' weights stream for one row each.
        _product_case(1, 4096, 8, 2, 14336, name="product_decode_1"),
        # Training through sizes that are no multiple of a tile, skewed routing.
        _product_case(333, 1248, 12, 3, 3296, dtype="f16", train=True, skew=0.8,
                      name="product_train_333"),
        # A long prompt through large matrices.
        _product_case(4096, 4096, 8, 2, 14336, skew=0.3, name="product_prompt_4096"),
        # A generating batch over many small experts.
        _experts_case(16, 2048, 64, 6, 1408, name="experts_decode_16"),
        # A large generating batch, or a short prompt, of odd length.
        _experts_case(197, 4096, 16, 2, 6400, act="gelu", name="experts_mixed_197"),
        # A long prompt through large experts.
        _experts_case(4096, 4096, 8, 2, 14336, skew=0.3, name="experts_prompt_4096"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "tokens", "product", "product", "experts", "experts"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    any_dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    skew = rng.choice([0.0, 0.3, 1.1])
    if op == "norm":
        # most widths whole 16 bytes, some not
        H = 8 * _log_int(rng, 16, 1024) + rng.choice([0, 0, 0, 1, 4])
        most = min(8192, int(8192 * 4096 / H / (2 if any_dtype == "f32" else 1)))
        return _norm_case(_log_int(rng, 1, most), H, dtype=any_dtype, train=rng.random() < 0.5)
    E = _log_int(rng, 1, 64)
    K = rng.randint(1, min(E, 8))
    if op == "tokens":
        H = 8 * _log_int(rng, 32, 640) + rng.choice([0, 0, 0, 1, 4])
        most = min(8192, int(16384 * 4096 / (H * K) / (2 if any_dtype == "f32" else 1)))
        return _tokens_case(_log_int(rng, 1, most), H, E, K, dtype=any_dtype,
                            train=rng.random() < 0.5, drop=rng.choice([0.0, 0.0, 0.5]), skew=skew)
    # weights of at most 10^9 elements, most sizes no multiple of a tile
    H, I = 16 * _log_int(rng, 16, 320), 16 * _log_int(rng, 16, 320)
    E = min(E, int(1e9 / (3 * H * I)))
    K = min(K, E)
    if op == "product":
        return _product_case(_log_int(rng, 1, 2048), H, E, K, I, dtype=dtype,
                             train=rng.random() < 0.5, skew=skew)
    return _experts_case(_log_int(rng, 1, 2048), H, E, K, I, dtype=dtype,
                         act=rng.choice(["silu", "silu", "gelu", "gelu_tanh"]), skew=skew)


# ------------------------------------------------------------------- inputs
def _routing(c, gen):
    """Distinct experts per token with a Zipf popularity, and their weights."""
    T, E, K = c["T"], c["E"], c["K"]
    logits = torch.empty((T, E), device="cuda").normal_(0.0, 1.0, generator=gen)
    rank = torch.randperm(E, generator=gen, device="cuda")
    ids = torch.argsort(logits - c["skew"] * torch.log1p(rank.float()), dim=-1,
                        descending=True)[:, :K].contiguous()
    w = torch.softmax(torch.gather(logits, 1, ids), -1)
    if c.get("drop"):
        gone = torch.rand((T, K), device="cuda", generator=gen) < c["drop"]
        ids = torch.where(gone, torch.full_like(ids, -1), ids)
    return w.contiguous(), ids


def _weights_8bit(E, N, K, gen):
    """[E, N, K] codes and [E, N blocks, K blocks] scales of weights whose size differs
    from block to block as trained ones' does."""
    n, k = -(-N // BLOCK), -(-K // BLOCK)
    codes = torch.empty((E, N, K), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((E, n, k), device="cuda")
    for e in range(E):
        size = torch.empty((n, 1, k, 1), device="cuda").normal_(0.0, 0.3, generator=gen)
        w = torch.empty((n, BLOCK, k, BLOCK), device="cuda").normal_(0.0, SIGMA_W, generator=gen)
        w *= torch.exp(size)
        inside = torch.arange(n * BLOCK, device="cuda") < N
        w *= inside.reshape(n, BLOCK, 1, 1)
        w *= (torch.arange(k * BLOCK, device="cuda") < K).reshape(1, 1, k, BLOCK)
        s = w.abs().amax((1, 3), keepdim=True).clamp_(min=SMALLEST) / E4M3_MAX
        codes[e] = (w / s).reshape(n * BLOCK, k * BLOCK)[:N, :K].to(codes.dtype)
        scales[e] = s.reshape(n, k)
    return codes, scales


def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    T, H = c["T"], c["H"]

    def normal(mean, sigma, *shape):
        return torch.empty(shape, dtype=dt, device="cuda").normal_(mean, sigma, generator=gen)

    d = {}
    if c["op"] == "norm":
        # a residual stream whose mean is not zero
        d.update(x=normal(0.0, 1.0, T, H), residual=normal(0.5, 2.0, T, H),
                 weight=normal(1.0, 0.1, H), bias=normal(0.0, 0.1, H))
        if c["train"]:
            d.update(dy=normal(0.0, 1.0, T, H), dres=normal(0.0, 1.0, T, H))
        return d
    d["topk_w"], d["topk_ids"] = _routing(c, gen)
    R, E = T * c["K"], c["E"]
    if c["op"] == "tokens":
        d.update(x=normal(0.0, 1.0, T, H), y=normal(0.0, 1.0, R, H))
        if c["train"]:
            d.update(drows=normal(0.0, 1.0, R, H), dout=normal(0.0, 1.0, T, H))
        return d
    # features of different sizes, as a residual stream has them
    size = torch.exp(torch.empty(H, device="cuda").normal_(0.0, 0.5, generator=gen))
    if c["op"] == "product":
        d["x"] = (normal(0.0, 1.0, R, H) * size).to(dt)
        d["w"] = _weights_8bit(E, c["N"], H, gen)
        if c["train"]:
            d["dout"] = normal(0.0, 1.0, R, c["N"])
        return d
    d["x"] = (normal(0.0, 1.0, T, H) * size).to(dt)
    d["w1"] = _halves(_weights_8bit(2 * E, c["I"], H, gen))  # gate, then up of each expert
    d["w2"] = _weights_8bit(E, H, c["I"], gen)
    return d


def _halves(w):
    """Matrices [2 E, I, H] as [E, 2 I, H], with their scales; the blocks of both halves start
    at their own first row."""
    codes, scales = w
    return (codes.reshape(-1, 2 * codes.shape[1], codes.shape[2]),
            scales.reshape(-1, 2 * scales.shape[1], scales.shape[2]))


def prepare(case, seed):
    c, d = case, _inputs(case, seed)
    d["case"] = c
    if c["op"] == "product":
        # rows arrive grouped by matrix; a program that sorted them knows the counts
        d["counts"] = torch.bincount(d.pop("topk_ids").reshape(-1), minlength=c["E"]).tolist()
    if not own:
        return d
    if c["op"] == "norm":
        from reframework_amd.layers import LayerNorm
        norm = LayerNorm(c["H"], EPS)
        norm.weight.data, norm.bias.data = d.pop("weight"), d.pop("bias")
        d["norm"] = norm.requires_grad_(c["train"])
    if c["op"] == "product":
        from reframework_amd.moe import Fp8Weight
        ends = torch.tensor(d["counts"]).cumsum(0)
        d["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), ends]).int().cuda()
        # the codes of a checkpoint, laid out once; training keeps the transposed matrices too
        d["weight"] = Fp8Weight.from_codes(*d.pop("w"), transposed=c["train"])
    if c["op"] == "experts":
        from reframework_amd.moe import Fp8Experts
        d["experts"] = Fp8Experts.from_codes(*d.pop("w1"), *d.pop("w2"))
    if c.get("train"):
        for k in ("x", "residual", "y", "topk_w"):
            if k in d:
                d[k].requires_grad_()
    return d


# -------------------------------------------------------------- plain forms
def _to_8bit(v):
    """(codes, scales) of fp32 rows, padded to whole blocks."""
    b = torch.nn.functional.pad(v, (0, -v.shape[1] % BLOCK)).reshape(v.shape[0], -1, BLOCK)
    most = b.abs().amax(-1, keepdim=True).clamp(min=SMALLEST)
    return (b * E4M3_MAX / most).to(torch.float8_e4m3fn), most / E4M3_MAX


def _through_8bit(v):
    codes, scale = _to_8bit(v)
    return (codes.float() * scale).reshape(v.shape[0], -1)[:, :v.shape[1]]


def _from_8bit(codes, scales):
    """fp32 [N, K] of one matrix's codes and block scales."""
    s = scales.repeat_interleave(BLOCK, 0)[:codes.shape[0]]
    return codes.float() * s.repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]


def _w1_from_8bit(codes, scales):
    i, n = codes.shape[0] // 2, scales.shape[0] // 2
    return torch.cat([_from_8bit(codes[:i], scales[:n]), _from_8bit(codes[i:], scales[n:])])


def _act(name, g):
    if name == "silu":
        return g / (1.0 + torch.exp(-g))
    if name == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g / math.sqrt(2.0)))
    return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)))


def _norm_plain(s):
    dt = s["x"].dtype
    res = (s["x"].float() + s["residual"].float()).to(dt)
    r, w = res.float(), s["weight"].float()
    xc = r - r.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xhat = xc * rstd
    out = (xhat * w + s["bias"].float()).to(dt)
    if not s["case"]["train"]:
        return out, res
    dy = s["dy"].float()
    g = dy * w
    dr = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    dr = (dr + s["dres"].float()).to(dt)
    return out, res, dr, dr, (dy * xhat).sum(0).to(dt), dy.sum(0).to(dt)


def _tokens_plain(s):
    c, ids, y = s["case"], s["topk_ids"], s["y"]
    T, H, E, K = (c[k] for k in "THEK")
    R, dt, dev = T * K, y.dtype, y.device
    flat = torch.where((ids < 0) | (ids >= E), torch.full_like(ids, E), ids).reshape(-1)
    order = torch.sort(flat, stable=True)[1]
    offsets = (flat[:, None] < torch.arange(E + 1, device=dev)).sum(0).int()
    place = torch.empty_like(order)
    place[order] = torch.arange(R, device=dev)
    used = (flat < E)[:, None]
    rows = torch.where(used[order], s["x"][order // K], torch.zeros((), dtype=dt, device=dev))
    place = place[:, None].expand(R, H)
    mine = torch.where(used, torch.gather(y.float(), 0, place), torch.zeros((), device=dev))
    w = s["topk_w"][..., None]
    out = (mine.reshape(T, K, H) * w).sum(1).to(dt)
    slots = torch.where(used[:, 0], place[:, 0], torch.full_like(order, -1)).reshape(T, K).int()
    if not c["train"]:
        return rows, offsets, slots, out
    dx = torch.where(used, torch.gather(s["drows"].float(), 0, place), torch.zeros((), device=dev))
    dout = s["dout"].float()[:, None]
    dy = torch.zeros((R, H), device=dev)
    dy.scatter_(0, place, torch.where(used, (w * dout).reshape(R, H), torch.zeros((), device=dev)))
    dw = (mine.reshape(T, K, H) * dout).sum(-1)
    return rows, offsets, slots, out, dx.reshape(T, K, H).sum(1).to(dt), dy.to(dt), dw


def _product_plain(s):
    x, (codes, scales), counts = _through_8bit(s["x"].float()), s["w"], s["counts"]
    dt = s["x"].dtype
    w = [_from_8bit(codes[e], scales[e]) if n else None for e, n in enumerate(counts)]
    out = torch.cat([x[a - n:a] @ w[e].t() for e, n, a in _groups(counts)]).to(dt)
    if not s["case"]["train"]:
        return out
    dout = _through_8bit(s["dout"].float())
    return out, torch.cat([dout[a - n:a] @ w[e] for e, n, a in _groups(counts)]).to(dt)


def _groups(counts):
    """(matrix, rows, one past its last row) of the matrices that have any."""
    end = 0
    for e, n in enumerate(counts):
        end += n
        if n:
            yield e, n, end


def _experts_plain(s):
    c, ids = s["case"], s["topk_ids"]
    T, H, K, I = (c[k] for k in "THKI")
    x = _through_8bit(s["x"].float())
    flat = ids.reshape(-1)
    order = torch.sort(flat, stable=True)[1]
    y = torch.empty((T * K, H), device=x.device)
    for e, n, end in _groups(torch.bincount(flat, minlength=c["E"]).tolist()):
        slot = order[end - n:end]
        gu = x[slot // K] @ _w1_from_8bit(s["w1"][0][e], s["w1"][1][e]).t()
        h = _through_8bit(_act(c["act"], gu[:, :I]) * gu[:, I:])
        y[slot] = h @ _from_8bit(s["w2"][0][e], s["w2"][1][e]).t()
    return (y.reshape(T, K, H) * s["topk_w"][..., None]).sum(1).to(s["x"].dtype)


def run(state):
    c = state["case"]
    with torch.set_grad_enabled(own and bool(c.get("train"))):
        if own:
            return _run_own(c, state)
        return {"norm": _norm_plain, "tokens": _tokens_plain, "product": _product_plain,
                "experts": _experts_plain}[c["op"]](state)


def _run_own(c, s):
    if c["op"] == "norm":
        norm = s["norm"]
        out = norm.forward_add_residual(s["x"], s["residual"])
        if c["train"]:
            out += torch.autograd.grad(out, [s["x"], s["residual"], norm.weight, norm.bias],
                                       [s["dy"], s["dres"]])
        return tuple(t.detach() for t in out)
    if c["op"] == "tokens":
        from reframework_amd.moe import combine_tokens, permute_tokens
        rows, order = permute_tokens(s["x"], s["topk_ids"], c["E"])
        out = combine_tokens(s["y"], order, s["topk_w"])
        got = (rows.detach(), order.offsets, order.slot_to_row, out.detach())
        if c["train"]:
            got += torch.autograd.grad([rows, out], [s["x"], s["y"], s["topk_w"]],
                                       [s["drows"], s["dout"]])
        return got
    if c["op"] == "product":
        from reframework_amd.moe import matmul_fp8
        out = matmul_fp8(s["x"], s["weight"], s["offsets"])
        if c["train"]:
            return out.detach(), torch.autograd.grad(out, s["x"], s["dout"])[0]
        return out
    from reframework_amd.moe import fused_experts_fp8
    return fused_experts_fp8(s["x"], s["experts"], s["topk_w"], s["topk_ids"],
                             activation=c["act"])


def work(case):
    c = case
    T, H, train = c["T"], c["H"], bool(c.get("train"))
    esz = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "norm":
        if train:  # x, residual, dy, dres; out, r, their common gradient; the parameters'
            return {"bytes": 7 * T * H * esz + 4 * H * esz, "flops": 24 * T * H}
        return {"bytes": 4 * T * H * esz + 2 * H * esz, "flops": 8 * T * H}
    E, K = c["E"], c["K"]
    R = T * K
    if c["op"] == "tokens":
        kept = R * (1.0 - c["drop"])
        rows = (2 * T * H + R * H + kept * H) * esz + R * 16
        if train:
            rows += (2 * T * H + R * H + kept * H) * esz + R * 4
        return {"bytes": int(rows), "flops": int((6 if train else 2) * kept * H)}
    # distinct experts that T tokens of K uniform choices reach
    used = E * (1.0 - (1.0 - K / E) ** T)
    if c["op"] == "product":
        N = c["N"]
        two = 2 if train else 1
        return {"bytes": int(used * H * N * (1.0 + 4.0 / BLOCK ** 2) + two * R * (H + N) * esz),
                "flops": 2 * two * R * H * N}
    I = c["I"]
    return {"bytes": int(used * 3 * H * I * (1.0 + 4.0 / BLOCK ** 2) + 2 * T * H * esz + R * 12),
            "flops": 6 * R * H * I}


# -------------------------------------------------------------------- exact
def _round_8bit(v):
    """Rows of 64 bits through the 8-bit format, from its definition."""
    out = torch.empty_like(v)
    for a in range(0, v.shape[1], BLOCK):
        b = v[:, a:a + BLOCK]
        most = b.abs().amax(-1, keepdim=True).clamp(min=SMALLEST)
        q = b * E4M3_MAX / most
        # e4m3: three bits below the leading one, down to 2^-6
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3.0)
        out[:, a:a + BLOCK] = torch.round(q / step) * step * (most / E4M3_MAX)
    return out


def _weight64(codes, scales):
    w = codes.double()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            w[BLOCK * i:BLOCK * (i + 1), BLOCK * j:BLOCK * (j + 1)] *= scales[i, j].double()
    return w


def _norm_exact(c, d):
    dt = d["x"].dtype
    r = (d["x"].double() + d["residual"].double()).to(dt).double()
    w, b = d["weight"].double(), d["bias"].double()
    var, mean = torch.var_mean(r, -1, correction=0, keepdim=True)
    rstd = torch.rsqrt(var + EPS)
    xhat = (r - mean) * rstd
    out = xhat * w + b
    if not c["train"]:
        return out, r
    dy = d["dy"].double()
    # the row's Jacobian: without the parts along 1 and along xhat
    v = dy * w
    v = v - v.sum(-1, keepdim=True) / c["H"]
    dr = rstd * (v - xhat * (v * xhat).sum(-1, keepdim=True) / c["H"]) + d["dres"].double()
    return out, r, dr, dr, torch.einsum("th,th->h", dy, xhat), dy.sum(0)


def _tokens_exact(c, d):
    T, H, E, K = (c[k] for k in "THEK")
    ids, w = d["topk_ids"], d["topk_w"].double()
    x, y = d["x"].double(), d["y"].double()
    slots = torch.full((T, K), -1, dtype=torch.int32, device=x.device)
    rows = torch.zeros((T * K, H), dtype=torch.float64, device=x.device)
    out = torch.zeros_like(x)
    if c["train"]:
        drows, dout = d["drows"].double(), d["dout"].double()
        dx, dy, dw = torch.zeros_like(x), torch.zeros_like(rows), torch.zeros_like(w)
    ends = [0]
    for e in range(E):
        tok, k = torch.nonzero(ids == e, as_tuple=True)
        a, b = ends[-1], ends[-1] + tok.numel()
        ends.append(b)
        slots[tok, k] = torch.arange(a, b, dtype=torch.int32, device=x.device)
        rows[a:b] = x[tok]
        out.index_add_(0, tok, w[tok, k, None] * y[a:b])
        if c["train"]:
            dx.index_add_(0, tok, drows[a:b])
            dy[a:b] = w[tok, k, None] * dout[tok]
            dw[tok, k] = (dout[tok] * y[a:b]).sum(-1)
    got = rows, torch.tensor(ends, dtype=torch.int32, device=x.device), slots, out
    return got + (dx, dy, dw) if c["train"] else got


def _product_exact(c, d):
    x, ids = _round_8bit(d["x"].double()), d["topk_ids"].reshape(-1)
    out = torch.empty((x.shape[0], c["N"]), dtype=torch.float64, device=x.device)
    if c["train"]:
        dout, dx = _round_8bit(d["dout"].double()), torch.empty_like(x)
    a = 0
    for e in range(c["E"]):
        b = a + int((ids == e).sum())
        if b > a:
            w = _weight64(d["w"][0][e], d["w"][1][e])
            out[a:b] = x[a:b] @ w.t()
            if c["train"]:
                dx[a:b] = dout[a:b] @ w
        a = b
    return (out, dx) if c["train"] else out


def _experts_exact(c, d):
    x, I = _round_8bit(d["x"].double()), c["I"]
    out = torch.zeros_like(x)
    n = d["w1"][1].shape[1] // 2
    for e in range(c["E"]):
        tok, slot = torch.nonzero(d["topk_ids"] == e, as_tuple=True)
        if tok.numel():
            codes, scales = d["w1"][0][e], d["w1"][1][e]
            g = x[tok] @ _weight64(codes[:I], scales[:n]).t()
            u = x[tok] @ _weight64(codes[I:], scales[n:]).t()
            h = _round_8bit(_act(c["act"], g) * u)
            y = h @ _weight64(d["w2"][0][e], d["w2"][1][e]).t()
            out.index_add_(0, tok, y * d["topk_w"][tok, slot, None].double())
    return out


@torch.no_grad()
def exact(case, seed):
    return {"norm": _norm_exact, "tokens": _tokens_exact, "product": _product_exact,
            "experts": _experts_exact}[case["op"]](case, _inputs(case, seed))
