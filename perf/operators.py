"""Block-scaled 8-bit operators: what they compute, in plain torch operations, and the cases they are
measured on.

A matrix in blocks of 128: every run of 128 values along the contraction of a product (activations and
gradients), or every 128 x 128 tile (weights), has one scale, a power of two, the smallest with which the
block's largest magnitude is at most 448; the values are e4m3. Two operators are built from it:

* ``linear``: ``y = x wᵀ (+ b)``. The products of a training step are ``y`` from x in rows and w in tiles, ``dx``
  from dy in rows and w in the same tiles, ``dw`` from dy and x in blocks of 128 tokens. ``db`` is the plain
  column sum of dy.
* ``mlp``: ``y = (act(x wgᵀ) * (x wuᵀ)) wdᵀ``, the gated feed-forward block, all of whose products are of that
  kind. Gate and up products, ``h``, ``dh`` and the gradients of gate and up are bf16 values, as on the way
  through the layers one by one.

``mode`` "kept" is the forward pass on weights that are in 8 bits already (an encoder that answers
requests), "step" a forward and backward pass on bf16 weights (training), which casts them.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BLOCK, E4M3_MAX = 128, 448.0


def _linear(name, mode, tokens, k, n, bias=False):
    return {"name": name, "op": "linear", "mode": mode, "tokens": tokens, "k": k, "n": n, "bias": bias}


def _mlp(name, mode, tokens, hidden, inner, kind="swiglu"):
    return {"name": name, "op": "mlp", "mode": mode, "tokens": tokens, "hidden": hidden, "inner": inner,
            "kind": kind}


def listed():
    return [
        # the query projection of a 2560-wide embedder for one search request: latency
        _linear("linear_query", "kept", 12, 2560, 4096),
        # a few short texts through the fused, biased projection of a BERT-base layer
        _linear("linear_texts", "kept", 700, 768, 2304, bias=True),
        # a stream of documents through the fused projection of a 4096-wide embedder
        _linear("linear_documents", "kept", 20960, 4096, 6144),
        # the smallest training batches: a few pairs on a narrow model, an odd number of tokens
        _linear("linear_step_small", "step", 257, 1024, 2048, bias=True),
        # a packed training batch of a 2560-wide embedder
        _linear("linear_step", "step", 8191, 2560, 6144),
        # a large batch on a 4096-wide one
        _linear("linear_step_large", "step", 16384, 4096, 4096),
        # one search request through a feed-forward block
        _mlp("mlp_query", "kept", 24, 2560, 9728),
        # several texts on a narrower model
        _mlp("mlp_texts", "kept", 500, 1024, 4096),
        # a stream of documents
        _mlp("mlp_documents", "kept", 20000, 2048, 8192),
        # the narrowest model, tanh-GELU, a short padded batch
        _mlp("mlp_step_small", "step", 1000, 768, 1152, "geglu"),
        # training batches of 2048- and 2560-wide embedders
        _mlp("mlp_step", "step", 4097, 2048, 8192),
        _mlp("mlp_step_large", "step", 16384, 2560, 9728),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    mode = rng.choice(("kept", "step"))
    if rng.random() < 0.5:
        tokens = _log(rng, 1, 16384)
        k, n = 16 * _log(rng, 16, 256), 16 * _log(rng, 16, 384)
        return _linear("", mode, tokens, k, n, rng.random() < 0.4)
    tokens = _log(rng, 1, 12000)
    return _mlp("", mode, tokens, 16 * _log(rng, 16, 160), 128 * _log(rng, 4, 76),
                rng.choice(("swiglu", "swiglu", "geglu")))


# ---------------------------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------------------------
def _scaled(x, rows, cols):
    """e4m3 values, scale exponents (biased by 127) and what they stand for in fp32, of the matrix x in blocks
    of rows x cols."""
    R, C = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -C % cols, 0, -R % rows))
    v = v.view(v.shape[0] // rows, rows, v.shape[1] // cols, cols)
    amax = v.abs().amax(dim=(1, 3), keepdim=True)
    bits = amax.view(torch.int32)
    # 448 = 1.75 * 2^8: one step up where the mantissa of the largest magnitude is above 0.75
    e = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(1, 254)
    e = torch.where(amax == 0, torch.full_like(e, 127), e)
    q = (v * ((254 - e) << 23).view(torch.float32)).to(torch.float8_e4m3fn)
    value = (q.float() * (e << 23).view(torch.float32)).reshape(v.shape[0] * rows, -1)[:R, :C]
    return q, e, value


def _rounded(x, rows, cols):
    return _scaled(x, rows, cols)[2]


def _kept(w):
    """The 8-bit form of a weight that an encoder keeps: bytes [n, k], their rows a multiple of 16 bytes
    apart, and one exponent for each row and 128 columns, four of a row in a word: [ceil(k / 512), n, 4]."""
    n, k = w.shape
    q, e, _ = _scaled(w, BLOCK, BLOCK)
    data = torch.zeros(n, -(-k // 16) * 16, dtype=torch.uint8, device=w.device)
    data[:, :k] = q.view(torch.uint8).reshape(q.shape[0] * BLOCK, -1)[:n, :k]
    rows = e.reshape(q.shape[0], 1, q.shape[2]).expand(-1, BLOCK, -1).reshape(-1, q.shape[2])[:n]
    words = torch.nn.functional.pad(rows, (0, -rows.shape[1] % 4), value=127)
    return data, words.to(torch.uint8).view(n, -1, 4).transpose(0, 1).contiguous()


def _of_kept(data, scales, k):
    e = scales.transpose(0, 1).reshape(data.shape[0], -1).int()
    e = e.repeat_interleave(BLOCK, dim=1)[:, :k]
    return data[:, :k].view(torch.float8_e4m3fn).float() * (e << 23).view(torch.float32)


def _act(g, kind):
    if kind == "swiglu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _bf16(x):
    return x.to(torch.bfloat16).to(x.dtype)


def _plain_linear(s):
    x, b = s["x"], s["b"]
    if s["mode"] == "kept":
        y = _rounded(x, 1, BLOCK) @ _of_kept(*s["w"], x.shape[1]).t()
        return (y if b is None else y + b.float()).to(torch.bfloat16)
    w, dy = s["w"], s["dy"]
    wv = _rounded(w, BLOCK, BLOCK)
    y = _rounded(x, 1, BLOCK) @ wv.t()
    y = y if b is None else y + b.float()
    dx = _rounded(dy, 1, BLOCK) @ wv
    dw = _rounded(dy, BLOCK, 1).t() @ _rounded(x, BLOCK, 1)
    out = [y, dx, dw] + ([] if b is None else [dy.float().sum(0)])
    return [v.to(torch.bfloat16) for v in out]


def _plain_mlp(s):
    x, kind = s["x"], s["kind"]
    if s["mode"] == "kept":
        wv, dv = _of_kept(*s["w"], x.shape[1]), _of_kept(*s["wd"], s["inner"])
    else:
        wv, dv = _rounded(s["w"], BLOCK, BLOCK), _rounded(s["wd"], BLOCK, BLOCK)
    g, u = _bf16(_rounded(x, 1, BLOCK) @ wv.t()).chunk(2, dim=1)
    a, da = _act(g, kind)
    h = _bf16(a * u)
    y = (_rounded(h, 1, BLOCK) @ dv.t()).to(torch.bfloat16)
    if s["mode"] == "kept":
        return y
    dy = s["dy"]
    dh = _bf16(_rounded(dy, 1, BLOCK) @ dv)
    dgu = _bf16(torch.cat([dh * u * da, dh * a], dim=1))
    dx = _rounded(dgu, 1, BLOCK) @ wv
    dw = _rounded(dgu, BLOCK, 1).t() @ _rounded(x, BLOCK, 1)
    dwd = _rounded(dy, BLOCK, 1).t() @ _rounded(h, BLOCK, 1)
    return [y] + [v.to(torch.bfloat16) for v in (dx, dw, dwd)]


# ---------------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------------
def _own_linear(s):
    from lset_b200.ops import fp8_block as fb

    x, b = s["x"], s["b"]
    if s["mode"] == "kept":
        with torch.no_grad():
            return fb.linear_fp8_block(x, fb.Fp8BlockTensor(s["w"][0], x.shape[1], s["w"][1]), b)
    leaves = [x, s["w"]] + ([] if b is None else [b])
    y = fb.linear_fp8_block(*leaves)
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]


def _own_mlp(s):
    from lset_b200.ops import fp8_block as fb

    x = s["x"]
    if s["mode"] == "kept":
        with torch.no_grad():
            return fb.gated_mlp_fp8_block(x, fb.Fp8BlockTensor(s["w"][0], x.shape[1], s["w"][1]), None,
                                          fb.Fp8BlockTensor(s["wd"][0], s["inner"], s["wd"][1]), s["kind"])
    y = fb.gated_mlp_fp8_block(x, s["w"], None, s["wd"], s["kind"])
    return [y.detach(), *torch.autograd.grad(y, [x, s["w"], s["wd"]], s["dy"])]


def run(state):
    if own:
        return _own_linear(state) if state["op"] == "linear" else _own_mlp(state)
    with torch.no_grad():
        return _plain_linear(state) if state["op"] == "linear" else _plain_mlp(state)


# ---------------------------------------------------------------------------------------------
# Inputs, work, exact values
# ---------------------------------------------------------------------------------------------
def _normal(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


def _activations(g, tokens, width):
    """Rows of a residual stream behind its norm: some channels far larger than the others, and zero rows
    where a batch is padded."""
    x = torch.randn(tokens, width, generator=g, device="cuda")
    x *= torch.where(torch.rand(width, generator=g, device="cuda") < 0.01, 16.0, 1.0)
    if tokens >= 64:
        x[tokens - tokens // 32:] = 0
    return x.to(torch.bfloat16)


def _gradients(g, tokens, width):
    """Gradients differ in size from token to token; tokens that no loss looks at have none."""
    dy = torch.randn(tokens, width, generator=g, device="cuda")
    dy *= 1e-3 * torch.exp(torch.randn(tokens, 1, generator=g, device="cuda"))
    if tokens >= 64:
        dy[tokens - tokens // 32:] = 0
    return dy.to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    T, kept = case["tokens"], case["mode"] == "kept"
    s = {"op": case["op"], "mode": case["mode"]}
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        s["x"] = _activations(g, T, k)
        w = _normal(g, n, k, scale=k ** -0.5)
        s["b"] = _normal(g, n, scale=0.5) if case["bias"] else None
        s["w"] = _kept(w) if kept else w
        s["dy"] = None if kept else _gradients(g, T, n)
        leaves = ("x", "w", "b")
    else:
        H, I = case["hidden"], case["inner"]
        s["x"], s["inner"], s["kind"] = _activations(g, T, H), I, case["kind"]
        w, wd = _normal(g, 2 * I, H, scale=H ** -0.5), _normal(g, H, I, scale=I ** -0.5)
        s["w"], s["wd"] = (_kept(w), _kept(wd)) if kept else (w, wd)
        s["dy"] = None if kept else _gradients(g, T, H)
        leaves = ("x", "w", "wd")
    if not kept:
        for name in leaves:
            if s[name] is not None:
                s[name].requires_grad_()
    return s


def work(case):
    T, kept = case["tokens"], case["mode"] == "kept"
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        weight, extra = n * k, 2 * n if case["bias"] else 0
        acts, products = 2 * T * (k + n), T * n * k
    else:
        weight, extra = 3 * case["hidden"] * case["inner"], 0
        acts, products = 2 * T * 2 * case["hidden"], T * weight
    if kept:  # weights in 8 bits
        return {"bytes": acts + weight + extra, "flops": 2 * products}
    return {"bytes": 2 * (acts + 2 * weight + extra), "flops": 6 * products}


def _exact_rounded(x, rows, cols):
    """x (64 bits) in blocks of rows x cols: each value to the nearest multiple of its e4m3 step, ties to even."""
    R, C = x.shape
    v = torch.nn.functional.pad(x, (0, -C % cols, 0, -R % rows))
    v = v.reshape(v.shape[0] // rows, rows, v.shape[1] // cols, cols)
    top = v.abs().amax(dim=(1, 3), keepdim=True)
    m, e = torch.frexp(top / E4M3_MAX)          # top / 448 = m 2^e, 0.5 <= m < 1
    e = torch.where(m == 0.5, e - 1, e)         # the smallest e with top <= 448 2^e
    e = torch.where(top == 0, torch.zeros_like(e), e).clamp(min=-126)
    y = torch.ldexp(v, -e)
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    y = torch.ldexp(torch.round(y / step) * step, e)
    return y.reshape(y.shape[0] * rows, -1)[:R, :C]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        x = s["x"].double()

        def weight(w, k):
            if case["mode"] == "kept":
                e = s[w][1].permute(1, 0, 2).flatten(1).double() - 127
                q = s[w][0][:, :k].view(torch.float8_e4m3fn).double()
                return q * torch.exp2(e)[:, torch.arange(k, device=q.device) // BLOCK]
            return _exact_rounded(s[w].double(), BLOCK, BLOCK)

        if case["op"] == "linear":
            w = weight("w", case["k"])
            y = _exact_rounded(x, 1, BLOCK) @ w.t()
            if s["b"] is not None:
                y = y + s["b"].double()
            if case["mode"] == "kept":
                return y
            dy = s["dy"].double()
            out = [y, _exact_rounded(dy, 1, BLOCK) @ w,
                   _exact_rounded(dy, BLOCK, 1).t() @ _exact_rounded(x, BLOCK, 1)]
            return out + ([] if s["b"] is None else [dy.sum(0)])
        w, wd = weight("w", case["hidden"]), weight("wd", case["inner"])
        gu = _bf16(_exact_rounded(x, 1, BLOCK) @ w.t())
        g, u = gu[:, :case["inner"]], gu[:, case["inner"]:]
        if case["kind"] == "swiglu":
            sg = torch.sigmoid(g)
            a, da = g * sg, sg + g * sg * (1 - sg)
        else:
            z = (2 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3)
            t = torch.tanh(z)
            a = g * (1 + t) / 2
            da = (1 + t) / 2 + g / 2 * (1 - t ** 2) * (2 / math.pi) ** 0.5 * (1 + 0.134145 * g ** 2)
        h = _bf16(a * u)
        y = _exact_rounded(h, 1, BLOCK) @ wd.t()
        if case["mode"] == "kept":
            return y
        dy = s["dy"].double()
        dh = _bf16(_exact_rounded(dy, 1, BLOCK) @ wd)
        dgu = _bf16(torch.cat([dh * u * da, dh * a], dim=1))
        return [y, _exact_rounded(dgu, 1, BLOCK) @ w,
                _exact_rounded(dgu, BLOCK, 1).t() @ _exact_rounded(x, BLOCK, 1),
                _exact_rounded(dy, BLOCK, 1).t() @ _exact_rounded(h, BLOCK, 1)]
