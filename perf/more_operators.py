"""What the 4-bit floating-point linears are timed on: the quantiser and its way back, the product of microscaled codes
(dense, over rows sorted by expert, and the two products of a backward pass), and a mixture-of-experts layer for a few
tokens, through the entry points of ferrisres_amd.Context.

Widths are those of the benchmark and the tests: 2048 x 2048 (the reference's single linear), hidden 2048 / inner 5632,
4096 / 11008 and 5120 / 13824, and 16 experts of which each token takes two.

Conventions. 32 values along the axis that a product sums over share one power of two, held as a byte b that stands for
2^(b - 127): b = max(e, 2) - 2, e the biased exponent of the largest magnitude. A value's code is x * 2^(127 - b) rounded
to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives (ties to the even code, 6 above it). Two codes lie in a
byte, the first in its low half; a row's scales are padded to a multiple of 4 of them. The layer's activations stay as
they are (its weights alone are codes), and so does what lies between its two products.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
MOST_MACS = 2048 * 4096 * 11008  # of a linear's product
MOST_WEIGHTS = 16 * 2048 * 5632  # of one matrix of all experts
_ctx = None


def listed():
    return [
        # activations of a prompt, codes along the rows, and the values that they stand for
        {"name": "quantize_rows_bf16", "kind": "quantize", "m": 2048, "k": 5632, "dtype": "bf16", "mode": "rows"},
        # a layer's f32 weights after an optimiser step, transposed codes for the gradient of the activations
        {"name": "quantize_cols_f32", "kind": "quantize", "m": 11008, "k": 4096, "dtype": "f32", "mode": "cols"},
        # one token through the reference's single linear: latency
        {"name": "linear_1tok_bf16", "kind": "linear", "m": 1, "k": 2048, "n": 2048, "dtype": "bf16"},
        # a full decode batch through the widest linear of a 7B model
        {"name": "linear_16tok_bf16", "kind": "linear", "m": 16, "k": 4096, "n": 11008, "dtype": "bf16"},
        # a chunk of a prompt, an odd number of tokens, f32 in and out, 13B width
        {"name": "linear_333tok_f32", "kind": "linear", "m": 333, "k": 5120, "n": 13824, "dtype": "f32"},
        # prompt processing: the widest linear of a 7B model over 2048 tokens
        {"name": "linear_2048tok_bf16", "kind": "linear", "m": 2048, "k": 4096, "n": 11008, "dtype": "bf16"},
        # the same linear's backward pass in training, an odd number of tokens: dx and dw
        {"name": "grad_1999tok_bf16", "kind": "grad", "m": 1999, "k": 4096, "n": 11008, "dtype": "bf16"},
        # a small f32 batch through one linear of each expert: sort, quantise, dispatch, product, combine
        {"name": "experts_33tok_f32", "kind": "experts", "t": 33, "h": 2048, "n": 5632, "e": 8, "top_k": 4,
         "dtype": "f32"},
        # a prompt chunk through the same
        {"name": "experts_512tok_bf16", "kind": "experts", "t": 512, "h": 2048, "n": 5632, "e": 16, "top_k": 2,
         "dtype": "bf16"},
        # one token through a whole layer, router included: decoding for a single user
        {"name": "moe_1tok_bf16", "kind": "moe", "t": 1, "h": 2048, "i": 5632, "e": 16, "top_k": 2, "dtype": "bf16",
         "routes": "router"},
        # a decode batch through the same
        {"name": "moe_8tok_bf16", "kind": "moe", "t": 8, "h": 2048, "i": 5632, "e": 16, "top_k": 2, "dtype": "bf16",
         "routes": "router"},
        # a larger batch, f32, whose routes come from elsewhere and whose last slots are padding
        {"name": "moe_61tok_f32", "kind": "moe", "t": 61, "h": 2048, "i": 5632, "e": 16, "top_k": 2, "dtype": "f32",
         "routes": "given"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, step):
    return max(step, _log_int(rng, lo, hi) // step * step)


def draw(rng):
    kind = rng.choice(("linear", "linear", "grad", "quantize", "experts", "moe", "moe"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    step = 32 if rng.random() < 0.3 else 128  # widths that leave a step of the kernels unfilled among them
    if kind in ("linear", "grad"):
        m = _log_int(rng, 1, 4096) if kind == "linear" else _log_int(rng, 64, 2048)
        while True:
            k, n = _width(rng, 1024, 14336, step), _width(rng, 1024, 14336, step)
            if m * k * n <= MOST_MACS:
                return {"kind": kind, "m": m, "k": k, "n": n, "dtype": dtype}
    if kind == "quantize":
        while True:
            m, k = _log_int(rng, 16, 16384), _width(rng, 512, 14336, step) - rng.choice((0, 0, 3))
            if m * k <= 11008 * 4096:
                return {"kind": kind, "m": m, "k": k, "dtype": dtype, "mode": rng.choice(("rows", "cols"))}
    top_k = rng.choice((1, 2, 2, 4))
    while True:
        h, n, e = _width(rng, 1024, 4096, step), _width(rng, 1024, 5632, step), rng.choice((8, 16, 32))
        t = _log_int(rng, 1, 1024 if kind == "experts" else 64)
        if h * n * e <= MOST_WEIGHTS and t * top_k * h * n <= 2048 * 2048 * 5632:
            c = {"kind": kind, "t": t, "h": h, "e": e, "top_k": top_k, "dtype": dtype}
            if kind == "experts":
                return {**c, "n": n}
            return {**c, "i": n, "routes": rng.choice(("router", "router", "given"))}


# ---- inputs, all from the seed --------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _acts(g, m, k, dtype):
    """Normalised activations: channels of uneven gain, a few of them far larger than the rest."""
    gain = torch.exp(0.3 * torch.randn((k,), generator=g, device=DEV))
    gain *= torch.where(torch.rand((k,), generator=g, device=DEV) < 1 / 256, 12.0, 1.0)
    return (torch.randn((m, k), generator=g, device=DEV) * gain).to(DT[dtype])


def _grads(g, m, k, dtype):
    """Gradients: tokens of very different weight."""
    gain = 1e-3 * torch.exp(torch.randn((m, 1), generator=g, device=DEV))
    return (torch.randn((m, k), generator=g, device=DEV) * gain).to(DT[dtype])


def _routes(g, t, e, top_k):
    """The experts each token takes, some more popular than others, and their weights. The last tokens of a batch are
    padding: they go nowhere (-1)."""
    logits = torch.randn((t, e), generator=g, device=DEV) + 0.5 * torch.randn((e,), generator=g, device=DEV)
    val, idx = torch.topk(logits, top_k, dim=1)
    idx = idx.to(torch.int32)
    idx[t - t // 16:] = -1
    return idx, torch.softmax(val, dim=1)


def _inputs(c, seed):
    """The tensors a user's program has: activations, gradients, routes or a router, and weights in f32."""
    g = _gen(seed)
    kind = c["kind"]
    weights = lambda *shape: 0.02 * torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    if kind == "quantize":
        m, k = c["m"], c["k"]
        return {"x": _acts(g, m, k, c["dtype"]) if c["mode"] == "rows" else weights(m, k).to(DT[c["dtype"]])}
    if kind in ("linear", "grad"):
        t = {"x": _acts(g, c["m"], c["k"], c["dtype"]), "w": weights(c["n"], c["k"])}
        if kind == "grad":
            t["dy"] = _grads(g, c["m"], c["n"], c["dtype"])
        return t
    t = {"x": _acts(g, c["t"], c["h"], c["dtype"])}
    if kind == "experts" or c["routes"] == "given":
        t["idx"], t["weight"] = _routes(g, c["t"], c["e"], c["top_k"])
    else:
        t["router"] = weights(c["e"], c["h"]).to(DT[c["dtype"]])
    if kind == "experts":
        t["w"] = weights(c["e"], c["n"], c["h"])
    else:
        t["gate"], t["up"] = weights(c["e"], c["i"], c["h"]), weights(c["e"], c["i"], c["h"])
        t["down"] = weights(c["e"], c["h"], c["i"])
    return t


def _up(n, m):
    return -(-n // m) * m


# ---- the plain forms: elementary operations in 32 bits --------------------------------------------------------------

def _table():
    v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
    return torch.cat([v, -v])


def _plain_codes(x):
    """Packed codes [.., k / 2] and scales' bytes [.., blocks] of blocks of 32 along the last axis, k up to a multiple
    of 32, the blocks up to one of 4."""
    x = x.float()
    k = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, _up(k, 128) - k)).unflatten(-1, (-1, 32))
    byte = torch.clamp_min(b.abs().amax(dim=-1).view(torch.int32) >> 23, 2) - 2
    v = b * ((254 - byte) << 23).view(torch.float32)[..., None]
    m = v.abs()
    code = (m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5)
    code = code + 8 * torch.signbit(v).to(torch.uint8)
    q = code[..., 0::2] + 16 * code[..., 1::2]
    return q.flatten(-2)[..., :_up(k, 32) // 2].contiguous(), byte.to(torch.uint8)


def _plain_values(q, s):
    """The values that codes and their scales stand for, in f32."""
    v = _table()[torch.stack([q & 15, q >> 4], dim=-1).int()].flatten(-2)
    n = v.shape[-1] // 32
    return (v.unflatten(-1, (n, 32)) * torch.exp2(s[..., :n].float() - 127)[..., None]).flatten(-2)


def _plain_rounded(x):
    """x as its codes hold it, with the axis up to a multiple of 32."""
    return _plain_values(*_plain_codes(x))


def _plain_product(a, b):
    """a [.., m, k] times b [.., n, k] transposed."""
    return torch.matmul(a, b.transpose(-1, -2).contiguous())


def _plain_sort(c, idx):
    """The row of each slot, the slot of each row (-1 for none), and the expert of each row (e for none)."""
    e = c["e"]
    flat = idx.reshape(-1).long()
    key, order = torch.sort(torch.where(flat < 0, e, flat), stable=True)
    rows = torch.arange(len(key), device=DEV)
    live = key < e
    row_of = torch.empty_like(rows)
    row_of[order] = torch.where(live, rows, -1)
    return row_of.view(idx.shape), torch.where(live, order, -1), key


def _plain_route(x, router, top_k):
    """The experts of the largest logits (ties to the lowest index) and the softmax over them."""
    logits = x.float() @ router.float().t()
    val, idx = torch.sort(logits, dim=1, descending=True, stable=True)
    return idx[:, :top_k].int(), torch.softmax(val[:, :top_k], dim=1)


def _plain(s):
    c, t = s["case"], s["in"]
    kind, dt = c["kind"], DT[c["dtype"]]
    if kind == "quantize":
        x = t["x"].t() if c["mode"] == "cols" else t["x"]
        return {"y": _plain_rounded(x)[:, :x.shape[1]].to(dt)}
    if kind == "linear":
        return {"y": _plain_product(_plain_rounded(t["x"]), _plain_values(*t["wq"])).to(dt)}
    if kind == "grad":
        dx = _plain_product(_plain_rounded(t["dy"]), _plain_values(*t["wtq"]))
        dw = _plain_product(_plain_rounded(t["dy"].t()), _plain_rounded(t["x"].t()))
        return {"dx": dx.to(dt), "dw": dw}
    if kind == "experts":
        e, k = c["e"], c["top_k"]
        row_of, slot_of, expert = _plain_sort(c, t["idx"])
        live = expert < e
        place = torch.where(live, torch.arange(len(expert), device=DEV) + expert * s["most"], e * s["most"])
        first = torch.searchsorted(expert, torch.arange(e, device=DEV))
        place = torch.where(live, place - first[torch.where(live, expert, 0)], place)
        xs = torch.zeros((e * s["most"] + 1, c["h"]), device=DEV)
        xs[place] = torch.where(live[:, None], _plain_rounded(t["x"])[torch.clamp_min(slot_of, 0) // k], 0.0)
        ys = _plain_product(xs[:-1].view(e, s["most"], -1), _plain_values(*t["wq"])).flatten(0, 1)
        ys = ys[torch.where(live, place, 0)].to(dt).float()
        weight = torch.where(row_of >= 0, t["weight"], 0.0)
        return {"y": (ys[torch.clamp_min(row_of, 0)] * weight[:, :, None]).sum(1).to(dt)}
    if c["routes"] == "given":
        idx, weight = t["idx"], t["weight"]
    else:
        idx, weight = _plain_route(t["x"], t["router"], c["top_k"])
    x, e = t["x"].float(), c["e"]
    share = ((idx[:, :, None] == torch.arange(e, device=DEV)) * weight[:, :, None]).sum(1)
    gate = _plain_product(x, _plain_values(*t["gate"]).flatten(0, 1))
    up = _plain_product(x, _plain_values(*t["up"]).flatten(0, 1))
    h = gate / (1 + torch.exp(-gate)) * up * share.repeat_interleave(c["i"], dim=1)
    y = (h @ _plain_values(*t["down"]).transpose(1, 2).flatten(0, 1)).to(dt)
    return {"y": y} if c["routes"] == "given" else {"y": y, "idx": idx, "weight": weight}


# ---- the framework's calls ------------------------------------------------------------------------------------------

def _own(s):
    import ferrisres_amd as frx

    c, t, o, k = s["case"], s["in"], s["out"], s["kept"]
    kind = c["kind"]
    global _ctx
    if _ctx is None:
        _ctx = frx.Context(0)
    ctx = _ctx
    if kind == "quantize":
        ctx.fp4_quantize(t["x"], frx.FP4_COLS if c["mode"] == "cols" else frx.FP4_ROWS, *k["xq"])
        ctx.fp4_dequantize(*k["xq"], o["y"])
        return o
    if kind == "linear":
        ctx.fp4_linear_act(t["x"], *t["wq"], o["y"])
        return o
    if kind == "grad":
        ctx.fp4_quantize(t["dy"], frx.FP4_ROWS, *k["dyq"])
        ctx.fp4_linear(*k["dyq"], *t["wtq"], o["dx"])
        ctx.fp4_quantize(t["dy"], frx.FP4_COLS, *k["dytq"])
        ctx.fp4_quantize(t["x"], frx.FP4_COLS, *k["xtq"])
        ctx.fp4_linear(*k["dytq"], *k["xtq"], o["dw"])
        return o
    if kind == "experts":
        if "rows" not in k:
            k["rows"] = frx.MoeRows(c["e"], 1, *k["plan"])
        rows = k["rows"]
        ctx.moe_sort(t["idx"], rows)
        ctx.fp4_quantize(t["x"], frx.FP4_ROWS, *k["xq"])
        ctx.moe_dispatch(k["xq"][0], rows, k["aq"][0])
        ctx.moe_dispatch(k["xq"][1], rows, k["aq"][1])
        ctx.fp4_linear_grouped(*k["aq"], *t["wq"], rows.offsets, k["ys"])
        ctx.moe_combine(k["ys"], rows, t["weight"], o["y"])
        return o
    weights = (*t["gate"], *t["up"], *t["down"])
    if c["routes"] == "given":
        ctx.fp4_moe_ffn(t["x"], None, *weights, o["y"], t["idx"], t["weight"])
    else:
        ctx.fp4_moe_ffn(t["x"], t["router"], *weights, o["y"], o["idx"], o["weight"])
    return o


def prepare(case, seed):
    c, t = case, _inputs(case, seed)
    kind, dt = c["kind"], DT[c["dtype"]]
    s = {"case": c, "in": t, "out": {}, "kept": {}}
    o, k = s["out"], s["kept"]
    new = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device=DEV)  # noqa: E731
    codes = lambda m, n: (new(m, _up(n, 32) // 2, dtype=torch.uint8), new(m, _up(n, 128) // 32, dtype=torch.uint8))  # noqa: E731
    if kind == "quantize":
        m, n = (c["k"], c["m"]) if c["mode"] == "cols" else (c["m"], c["k"])
        o["y"], k["xq"] = new(m, n, dtype=dt), codes(m, n)
        return s
    if kind == "grad":  # a program that serves or trains keeps its weights as codes
        t["wtq"] = _plain_codes(t.pop("w").t())
        m, n, h = c["m"], c["n"], c["k"]
        o["dx"], o["dw"] = new(m, h, dtype=dt), new(n, h)
        k["dyq"], k["dytq"], k["xtq"] = codes(m, n), codes(n, m), codes(h, m)
        return s
    if kind in ("linear", "experts"):
        t["wq"] = _plain_codes(t.pop("w"))
    if kind == "linear":
        o["y"] = new(c["m"], c["n"], dtype=dt)
        return s
    tok, h, e, j = c["t"], c["h"], c["e"], c["top_k"]
    whole = lambda *shape: new(*shape, dtype=torch.int32)  # noqa: E731
    if kind == "experts":
        s["most"] = max(1, int((t["idx"].reshape(-1, 1) == torch.arange(e, device=DEV)).sum(0).max()))  # rows of the fullest expert, what the plain form pads the others to
        k["plan"] = whole(e + 1), whole(tok, j), whole(tok * j)
        k["xq"], k["aq"] = codes(tok, h), codes(tok * j, h)
        k["ys"], o["y"] = new(tok * j, c["n"], dtype=dt), new(tok, c["n"], dtype=dt)
        return s
    for name in ("gate", "up", "down"):
        t[name] = _plain_codes(t.pop(name))
    o["y"] = new(tok, h, dtype=dt)
    if c["routes"] == "router":
        o["idx"], o["weight"] = whole(tok, j), new(tok, j)
    return s


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass has to move and to compute -------------------------------------------------------------------------

def _expected_experts(c):
    """Experts that at least one of the tokens reaches when each takes top_k of e at random."""
    return c["e"] * (1 - (1 - c["top_k"] / c["e"]) ** c["t"])


def work(case):
    c = case
    kind, width = c["kind"], 2 if c["dtype"] == "bf16" else 4
    code = 1 / 2 + 1 / 32  # bytes of a value
    if kind == "quantize":
        # x in, codes and scales out; the same back
        return {"bytes": 2 * c["m"] * c["k"] * (width + code), "flops": 3 * c["m"] * c["k"]}
    if kind in ("linear", "grad"):
        m, n, k = c["m"], c["n"], c["k"]
        if kind == "linear":
            return {"bytes": n * k * code + (m * k + m * n) * width, "flops": 2 * m * n * k}
        return {"bytes": n * k * (code + 4) + (2 * m * k + m * n) * width, "flops": 4 * m * n * k}
    t, h, j, experts = c["t"], c["h"], c["top_k"], _expected_experts(c)
    if kind == "experts":
        n = c["n"]
        return {"bytes": experts * n * h * code + t * (h + n) * width + 8 * t * j, "flops": 2 * t * j * n * (h + 1)}
    i = c["i"]
    route = {"bytes": 8 * t * j, "flops": 0}
    if c["routes"] == "router":
        route = {"bytes": c["e"] * h * width + 8 * t * j, "flops": 2 * t * c["e"] * h}
    return {"bytes": experts * 3 * h * i * code + 2 * t * h * width + route["bytes"],
            "flops": t * j * 6 * h * i + route["flops"]}


# ---- the same outputs in 64 bits ------------------------------------------------------------------------------------

def _exact_values(x):
    """What the codes of blocks of 32 along the last axis stand for, in f64."""
    x = x.double()
    n = x.shape[-1]
    where = torch.arange(n, device=DEV) // 32
    top = torch.zeros((*x.shape[:-1], _up(n, 32) // 32), dtype=torch.float64, device=DEV)
    top.scatter_reduce_(-1, where.expand(x.shape), x.abs(), "amax")
    e = torch.clamp(torch.frexp(top)[1].long() - 3, -127, 127)  # frexp's mantissa lies in [1/2, 1)
    e = torch.where(top > 0, e, -127)
    scale = ((e + 1023) << 52).view(torch.float64)[..., where]
    v = x / scale
    step = ((torch.clamp_min(torch.frexp(v)[1].long() - 1, 0) - 1 + 1023) << 52).view(torch.float64)
    return torch.clamp(torch.round(v / step) * step, -6, 6) * scale


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    kind, dt = c["kind"], DT[c["dtype"]]
    if kind == "quantize":
        return {"y": _exact_values(t["x"].t() if c["mode"] == "cols" else t["x"])}
    if kind == "linear":
        return {"y": _exact_values(t["x"]) @ _exact_values(t["w"]).t()}
    if kind == "grad":
        return {"dx": _exact_values(t["dy"]) @ _exact_values(t["w"].t()).t(),
                "dw": _exact_values(t["dy"].t()) @ _exact_values(t["x"].t()).t()}
    tokens, x = c["t"], t["x"].double()
    if kind == "moe" and c["routes"] == "router":
        logits = x @ t["router"].double().t()
        val, idx = torch.topk(logits, c["top_k"], dim=1)
        weight = torch.exp(val - val[:, :1])
        weight = weight / weight.sum(1, keepdim=True)
    else:
        idx, weight = t["idx"], t["weight"].double()
    y = torch.zeros((tokens, c["n"] if kind == "experts" else c["h"]), dtype=torch.float64, device=DEV)
    if kind == "experts":
        x = _exact_values(x)
    for e in range(c["e"]):
        tok, j = torch.nonzero(idx == e, as_tuple=True)
        if not len(tok):
            continue
        if kind == "experts":
            out = (x[tok] @ _exact_values(t["w"][e]).t()).to(dt).double()
        else:
            gate, up = x[tok] @ _exact_values(t["gate"][e]).t(), x[tok] @ _exact_values(t["up"][e]).t()
            out = (gate * torch.sigmoid(gate) * up) @ _exact_values(t["down"][e]).t()
        y.index_add_(0, tok, weight[tok, j, None] * out)
    return {"y": y} if kind == "experts" or c["routes"] == "given" else {"y": y, "idx": None, "weight": weight}
