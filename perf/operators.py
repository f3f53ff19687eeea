"""What the 8-bit floating-point linears and the expert sort are timed on: the product with a scale for each block of
128, its quantiser, and the exchange of tokens between their own order and the experts', forward and backward, through
the entry points of ferrisres_amd.Context.

Widths are those of the benchmark and the tests: 2048 x 2048 (the reference's single linear), hidden 2048 / inner 5632,
4096 / 11008 and 5120 / 13824, and 16 experts of which each token takes two.

Conventions. A block of 128 values shares one f32 scale s = max(amax * f32(1 / top), 2^-126), top = 448 (e4m3) or 57344
(e5m2); a value's code is its f32 product with the f32 reciprocal of s, rounded to nearest even. Activations and gradients are
quantised along the axis that the product sums over, one row at a time; weights in tiles of 128 x 128.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
TOP = {E4M3: 448.0, E5M2: 57344.0}
TINY = 2.0 ** -126
MOST_MACS = 2048 * 4096 * 11008  # of a linear's product
_ctx = None


def listed():
    return [
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
        # activations of a prompt, codes along the rows
        {"name": "quantize_rows_bf16", "kind": "quantize", "m": 2048, "k": 5632, "dtype": "bf16", "mode": "rows"},
        # a layer's f32 weights after an optimiser step: tiles, for the forward product and (transposed) for dx
        {"name": "quantize_weights_f32", "kind": "quantize", "m": 11008, "k": 4096, "dtype": "f32", "mode": "tiles"},
        # a decode batch through one linear of each expert: sort, quantise, dispatch, product, combine
        {"name": "experts_8tok_bf16", "kind": "experts", "t": 8, "h": 2048, "n": 5632, "e": 16, "top_k": 2,
         "dtype": "bf16"},
        # a prompt chunk through the same
        {"name": "experts_512tok_bf16", "kind": "experts", "t": 512, "h": 2048, "n": 5632, "e": 16, "top_k": 2,
         "dtype": "bf16"},
        # the same chunk's backward pass: gradients of the weights of the combination, of the experts and of x
        {"name": "experts_grad_512tok_bf16", "kind": "experts_grad", "t": 512, "h": 2048, "n": 5632, "e": 16,
         "top_k": 2, "dtype": "bf16"},
        # the exchange alone, there and back, forward and backward: a small f32 batch and a long bf16 one
        {"name": "exchange_33tok_f32", "kind": "exchange", "t": 33, "h": 2048, "e": 8, "top_k": 4, "dtype": "f32"},
        {"name": "exchange_8192tok_bf16", "kind": "exchange", "t": 8192, "h": 4096, "e": 64, "top_k": 2,
         "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, step):
    return max(step, _log_int(rng, lo, hi) // step * step)


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear", "grad", "quantize", "experts", "experts_grad", "exchange"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    step = 16 if rng.random() < 0.3 else 128  # widths that leave a block unfilled among them
    if kind in ("linear", "grad"):
        m = _log_int(rng, 1, 4096) if kind == "linear" else _log_int(rng, 64, 2048)
        while True:
            k, n = _width(rng, 1024, 14336, step), _width(rng, 1024, 14336, step)
            if m * k * n <= MOST_MACS:
                return {"kind": kind, "m": m, "k": k, "n": n, "dtype": dtype}
    if kind == "quantize":
        while True:
            m, k = _log_int(rng, 16, 16384), _width(rng, 512, 14336, step)
            if m * k <= 11008 * 4096:
                return {"kind": kind, "m": m, "k": k, "dtype": dtype, "mode": rng.choice(("rows", "cols", "tiles"))}
    top_k = rng.choice((1, 2, 2, 4))
    if kind == "exchange":
        while True:
            t, h = _log_int(rng, 1, 16384), _width(rng, 512, 8192, step)
            if t * top_k * h * (2 if dtype == "f32" else 1) <= 8192 * 2 * 4096:
                return {"kind": kind, "t": t, "h": h, "e": rng.choice((8, 16, 64)), "top_k": top_k, "dtype": dtype}
    while True:
        h, n, e = _width(rng, 1024, 4096, step), _width(rng, 1024, 5632, step), rng.choice((8, 16, 32))
        t = _log_int(rng, 1, 1024) if kind == "experts" else _log_int(rng, 32, 512)
        if h * n * e <= 2048 * 5632 * 16 and t * top_k * h * n <= 2048 * 2048 * 5632:
            return {"kind": kind, "t": t, "h": h, "n": n, "e": e, "top_k": top_k, "dtype": dtype}


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
    """The tensors a user's program has: activations, gradients, routes, and weights in f32."""
    g = _gen(seed)
    kind = c["kind"]
    if kind == "quantize":
        return {"x": (0.02 * torch.randn((c["m"], c["k"]), generator=g, device=DEV)).to(DT[c["dtype"]])
                if c["mode"] == "tiles" else _acts(g, c["m"], c["k"], c["dtype"])}
    if kind in ("linear", "grad"):
        t = {"x": _acts(g, c["m"], c["k"], c["dtype"]),
             "w": 0.02 * torch.randn((1, c["n"], c["k"]), generator=g, device=DEV)}
        if kind == "grad":
            t["dy"] = _grads(g, c["m"], c["n"], c["dtype"])
        return t
    t = {"x": _acts(g, c["t"], c["h"], c["dtype"])}
    t["idx"], t["weight"] = _routes(g, c["t"], c["e"], c["top_k"])
    n = c.get("n", c["h"])
    if kind != "exchange":
        t["w"] = 0.02 * torch.randn((c["e"], n, c["h"]), generator=g, device=DEV)
    if kind != "experts":
        t["dy"] = _grads(g, c["t"], n, c["dtype"])
        t["ys"] = torch.randn((_capacity(c), n), generator=g, device=DEV).to(DT[c["dtype"]])
    return t


def _up(n, m):
    return -(-n // m) * m


def _align(c):
    """Rows an expert's segment is a multiple of: whole blocks of 128 where weights' gradients sum over them."""
    return 128 if c["kind"] == "experts_grad" else 1


def _capacity(c):
    a = _align(c)
    return _up(c["t"] * c["top_k"] + c["e"] * (a - 1), a)


# ---- the plain forms: elementary operations in 32 bits --------------------------------------------------------------

def _codes(x, amax, code):
    s = torch.clamp_min(amax * (1.0 / TOP[code]), TINY)
    return s, (x * torch.reciprocal(s)).to(code)


def _plain_rows(x, code):
    """Codes [.., m, k up to a multiple of 16] and scales [.., m, blocks] of blocks of 128 along the rows."""
    x = x.float()
    k = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, _up(k, 128) - k)).unflatten(-1, (-1, 128))
    s, q = _codes(b, b.abs().amax(dim=-1, keepdim=True), code)
    return q.flatten(-2)[..., :_up(k, 16)].contiguous(), s.squeeze(-1)


def _plain_tiles(w):
    """Codes [e, n, k up to a multiple of 16] and scales [e, n blocks, k blocks] of tiles of 128 x 128."""
    w = w.float()
    e, n, k = w.shape
    t = torch.nn.functional.pad(w, (0, _up(k, 128) - k, 0, _up(n, 128) - n)).view(e, _up(n, 128) // 128, 128, -1, 128)
    s, q = _codes(t, t.abs().amax(dim=(2, 4), keepdim=True), E4M3)
    q = q.reshape(e, _up(n, 128), _up(k, 128))[:, :n, :_up(k, 16)].contiguous()
    return q, s.reshape(e, _up(n, 128) // 128, -1)


def _spread(s, n):
    """A scale for each of n values from one for each block of 128."""
    return s.repeat_interleave(128, dim=-1)[..., :n]


def _plain_deq(q, s):
    """The values that codes with scales along the rows stand for."""
    return q.float() * _spread(s, q.shape[-1])


def _plain_deq_tiles(q, s):
    return q.float() * _spread(_spread(s.transpose(-1, -2), q.shape[-2]).transpose(-1, -2), q.shape[-1])


def _plain_sort(c, idx):
    """offsets [e + 1], the row of each slot, the slot of each row; -1 for none."""
    e, a, rows = c["e"], _align(c), _capacity(c)
    flat = idx.reshape(-1).long()
    key, order = torch.sort(torch.where(flat < 0, e, flat), stable=True)
    counts = (key[:, None] == torch.arange(e, device=DEV)).sum(0)
    offsets = torch.zeros((e + 1,), dtype=torch.int64, device=DEV)
    offsets[1:] = torch.cumsum((counts + a - 1) // a * a, 0)
    start = torch.cumsum(counts, 0) - counts
    live = key < e
    safe = torch.where(live, key, 0)
    row = torch.where(live, offsets[safe] + torch.arange(len(key), device=DEV) - start[safe], rows)
    row_of = torch.empty((len(key),), dtype=torch.int64, device=DEV)
    row_of[order] = torch.where(live, row, -1)
    slot_of = torch.full((rows + 1,), -1, dtype=torch.int64, device=DEV)
    slot_of[row] = order
    return offsets.int(), row_of.view(idx.shape).int(), slot_of[:rows].int()


def _plain_dispatch(x, slot_of, top_k):
    """Each row's token; rows of no token are zero."""
    xs = x[torch.clamp_min(slot_of, 0).long() // top_k]
    return torch.where((slot_of >= 0)[:, None], xs.float(), 0.0).to(x.dtype)


def _plain_combine(ys, row_of, weight):
    rows = ys[torch.clamp_min(row_of, 0).long()].float()
    weight = torch.where(row_of >= 0, 1.0 if weight is None else weight, 0.0)
    return (rows * weight[:, :, None]).sum(1).to(ys.dtype)


def _plain_combine_backward(dy, ys, row_of, slot_of, weight):
    top_k = row_of.shape[1]
    slot = torch.clamp_min(slot_of, 0).long()
    dys = dy[slot // top_k].float() * weight.reshape(-1)[slot][:, None]
    dys = torch.where((slot_of >= 0)[:, None], dys, 0.0).to(dy.dtype)
    dots = (ys[torch.clamp_min(row_of, 0).long()].float() * dy.float()[:, None]).sum(2)
    return dys, torch.where(row_of >= 0, dots, 0.0)


def _plain_by_expert(c, a, offsets, most):
    """The rows of a as [experts, most, columns], and where each row is in it."""
    rows = torch.arange(a.shape[0], device=DEV)
    expert = (rows[:, None] >= offsets[1:-1].long()).sum(1)
    place = expert * most + rows - offsets.long()[expert]
    inside = rows < offsets[-1]
    place = torch.where(inside, place, c["e"] * most)
    out = torch.zeros((c["e"] * most + 1, a.shape[1]), device=DEV)
    out[place] = a * inside[:, None]
    return out[:-1].view(c["e"], most, -1), place, inside


def _plain(s):
    c, t = s["case"], s["in"]
    kind = c["kind"]
    if kind == "quantize":
        if c["mode"] == "tiles":
            q, sc = _plain_tiles(t["x"][None])
            qt, st = _plain_tiles(t["x"].t()[None])
            return {"q": q[0], "scale": sc[0], "qt": qt[0], "scale_t": st[0]}
        q, sc = _plain_rows(t["x"].t() if c["mode"] == "cols" else t["x"], E4M3)
        return {"q": q, "scale": sc}
    if kind == "linear":
        y = _plain_deq(*_plain_rows(t["x"], E4M3)) @ _plain_deq_tiles(t["wq"][0], t["ws"][0]).t()
        return {"y": y.to(DT[c["dtype"]])}
    if kind == "grad":
        m, n, k = c["m"], c["n"], c["k"]
        dx = _plain_deq(*_plain_rows(t["dy"], E5M2)) @ _plain_deq_tiles(t["wtq"][0], t["wts"][0]).t()
        dw = _plain_deq(*_plain_rows(t["dy"].t(), E5M2)) @ _plain_deq(*_plain_rows(t["x"].t(), E4M3)).t()
        return {"dx": dx.to(DT[c["dtype"]]), "dw": dw}
    if kind == "exchange":
        offsets, row_of, slot_of = _plain_sort(c, t["idx"])
        xs = _plain_dispatch(t["x"], slot_of, c["top_k"])
        y = _plain_combine(t["ys"], row_of, t["weight"])
        dys, dweight = _plain_combine_backward(t["dy"], t["ys"], row_of, slot_of, t["weight"])
        dx = _plain_combine(dys, row_of, None)
        return {"offsets": offsets, "row_of": row_of, "xs": xs, "y": y, "dys": dys, "dweight": dweight, "dx": dx}
    if kind == "experts":
        offsets, row_of, slot_of = _plain_sort(c, t["idx"])
        q, sc = _plain_rows(t["x"], E4M3)
        a = _plain_dispatch(_plain_deq(q, sc), slot_of, c["top_k"])
        a, place, inside = _plain_by_expert(c, a, offsets, s["most"])
        ys = torch.bmm(a, _plain_deq_tiles(t["wq"], t["ws"]).transpose(1, 2).contiguous())
        ys = torch.where(inside[:, None], ys.flatten(0, 1)[torch.where(inside, place, 0)], 0.0).to(DT[c["dtype"]])
        return {"y": _plain_combine(ys, row_of, t["weight"])}
    offsets, row_of, slot_of = s["plan"]
    dys, dweight = _plain_combine_backward(t["dy"], t["ys"], row_of, slot_of, t["weight"])
    a, place, inside = _plain_by_expert(c, _plain_deq(*_plain_rows(dys, E5M2)), offsets, s["most"])
    dxs = torch.bmm(a, _plain_deq_tiles(t["wtq"], t["wts"]).transpose(1, 2).contiguous())
    dxs = torch.where(inside[:, None], dxs.flatten(0, 1)[torch.where(inside, place, 0)], 0.0).to(DT[c["dtype"]])
    # the sums over an expert's rows go by blocks of 128 of them: whole blocks, as its segment is aligned
    da, _, _ = _plain_by_expert(c, _plain_deq(*_plain_rows(dys.t(), E5M2)).t(), offsets, s["most"])
    xa, _, _ = _plain_by_expert(c, _plain_deq(*_plain_rows(t["xs"].t(), E4M3)).t(), offsets, s["most"])
    dw = torch.bmm(da.transpose(1, 2).contiguous(), xa)
    return {"dweight": dweight, "dx": _plain_combine(dxs, row_of, None), "dw": dw}


# ---- the framework's calls ------------------------------------------------------------------------------------------

def _own(s):
    import ferrisres_amd as frx

    c, t, o = s["case"], s["in"], s["out"]
    kind = c["kind"]
    global _ctx
    if _ctx is None:
        _ctx = frx.Context(0)
    ctx = _ctx
    if kind == "quantize":
        if c["mode"] == "tiles":
            ctx.fp8_quantize(t["x"], frx.FP8_TILES, o["q"], o["scale"])
            ctx.fp8_quantize(t["x"], frx.FP8_TILES_T, o["qt"], o["scale_t"])
        else:
            ctx.fp8_quantize(t["x"], frx.FP8_COLS if c["mode"] == "cols" else frx.FP8_ROWS, o["q"], o["scale"])
        return o
    if kind == "linear":
        ctx.fp8_linear_act(t["x"], t["wq"][0], t["ws"][0], o["y"])
        return o
    k = s["kept"]
    if kind == "grad":
        ctx.fp8_quantize(t["dy"], frx.FP8_ROWS, k["dyq"], k["dys"])
        ctx.fp8_linear(k["dyq"], k["dys"], t["wtq"][0], t["wts"][0], o["dx"])
        ctx.fp8_quantize(t["dy"], frx.FP8_COLS, k["dytq"], k["dyts"])
        ctx.fp8_quantize(t["x"], frx.FP8_COLS, k["xtq"], k["xts"])
        ctx.fp8_linear(k["dytq"], k["dyts"], k["xtq"], k["xts"], o["dw"])
        return o
    if "rows" not in k:
        plan = s["plan"] if kind == "experts_grad" else (o["offsets"], o["row_of"], k["slot_of"])
        k["rows"] = frx.MoeRows(c["e"], _align(c), *plan)
    rows = k["rows"]
    if kind == "exchange":
        ctx.moe_sort(t["idx"], rows)
        ctx.moe_dispatch(t["x"], rows, o["xs"])
        ctx.moe_combine(t["ys"], rows, t["weight"], o["y"])
        ctx.moe_combine_backward(t["dy"], t["ys"], rows, t["weight"], o["dys"], o["dweight"])
        ctx.moe_combine(o["dys"], rows, None, o["dx"])
        return o
    if kind == "experts":
        ctx.moe_sort(t["idx"], rows)
        ctx.fp8_quantize(t["x"], frx.FP8_ROWS, k["xq"], k["xqs"])
        ctx.moe_dispatch(k["xq"], rows, k["aq"])
        ctx.moe_dispatch(k["xqs"], rows, k["as"])
        ctx.fp8_linear_grouped(k["aq"], k["as"], t["wq"], t["ws"], rows.offsets, k["ys"])
        ctx.moe_combine(k["ys"], rows, t["weight"], o["y"])
        return {"y": o["y"]}
    ctx.moe_combine_backward(t["dy"], t["ys"], rows, t["weight"], k["dys"], o["dweight"])
    ctx.fp8_quantize(k["dys"], frx.FP8_ROWS, k["dyq"], k["dyqs"])
    ctx.fp8_linear_grouped(k["dyq"], k["dyqs"], t["wtq"], t["wts"], rows.offsets, k["dxs"])
    ctx.moe_combine(k["dxs"], rows, None, o["dx"])
    ctx.fp8_quantize(k["dys"], frx.FP8_COLS, k["dytq"], k["dyts"])
    ctx.fp8_quantize(t["xs"], frx.FP8_COLS, k["xtq"], k["xts"])
    ctx.fp8_grad_weight_grouped(k["dytq"], k["dyts"], k["xtq"], k["xts"], rows.offsets, o["dw"])
    return o


def _blocks(n):
    return _up(n, 128) // 128


def prepare(case, seed):
    c, t = case, _inputs(case, seed)
    kind, dt = c["kind"], DT[c["dtype"]]
    s = {"case": c, "in": t, "out": {}, "kept": {}}
    o, k = s["out"], s["kept"]
    new = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device=DEV)  # noqa: E731
    codes = lambda m, n, code=E4M3: (new(m, _up(n, 16), dtype=code), new(m, _blocks(n)))  # noqa: E731
    if kind == "quantize":
        m, n = c["m"], c["k"]
        if c["mode"] == "tiles":
            o["q"], o["scale"] = new(m, _up(n, 16), dtype=E4M3), new(_blocks(m), _blocks(n))
            o["qt"], o["scale_t"] = new(n, _up(m, 16), dtype=E4M3), new(_blocks(n), _blocks(m))
        else:
            o["q"], o["scale"] = codes(n, m) if c["mode"] == "cols" else codes(m, n)
        return s
    if "w" in t:  # a program that serves or trains keeps its weights as codes
        w = t.pop("w")
        if kind in ("grad", "experts_grad"):
            t["wtq"], t["wts"] = _plain_tiles(w.transpose(1, 2))
        else:
            t["wq"], t["ws"] = _plain_tiles(w)
        del w
    if kind == "linear":
        o["y"] = new(c["m"], c["n"], dtype=dt)
        return s
    if kind == "grad":
        m, n, h = c["m"], c["n"], c["k"]
        o["dx"], o["dw"] = new(m, h, dtype=dt), new(n, h)
        k["dyq"], k["dys"] = codes(m, n, E5M2)
        k["dytq"], k["dyts"] = codes(n, m, E5M2)
        k["xtq"], k["xts"] = codes(h, m)
        return s
    tok, h, e, rows = c["t"], c["h"], c["e"], _capacity(c)
    n = c.get("n", h)
    whole = lambda *shape: new(*shape, dtype=torch.int32)  # noqa: E731
    if kind == "experts_grad":
        s["plan"] = _plain_sort(c, t["idx"])
        t["xs"] = _plain_dispatch(t["x"], s["plan"][2], c["top_k"])
        o["dweight"], o["dx"], o["dw"] = new(tok, c["top_k"]), new(tok, h, dtype=dt), new(e, n, h)
        k["dys"], k["dxs"] = new(rows, n, dtype=dt), new(rows, h, dtype=dt)
        k["dyq"], k["dyqs"] = codes(rows, n, E5M2)
        k["dytq"], k["dyts"] = codes(n, rows, E5M2)
        k["xtq"], k["xts"] = codes(h, rows)
        sizes = s["plan"][0].long().diff()
    else:
        o["offsets"], o["row_of"], k["slot_of"] = whole(e + 1), whole(tok, c["top_k"]), whole(rows)
        sizes = (t["idx"].reshape(-1, 1) == torch.arange(e, device=DEV)).sum(0)
    s["most"] = max(1, int(sizes.max()))  # rows of the fullest expert, what the plain form pads the others to
    if kind == "exchange":
        o["xs"], o["y"], o["dx"] = new(rows, h, dtype=dt), new(tok, h, dtype=dt), new(tok, h, dtype=dt)
        o["dys"], o["dweight"] = new(rows, h, dtype=dt), new(tok, c["top_k"])
    elif kind == "experts":
        o["y"], k["ys"] = new(tok, n, dtype=dt), new(rows, n, dtype=dt)
        k["xq"], k["xqs"] = codes(tok, h)
        k["aq"], k["as"] = codes(rows, h)
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
    if kind == "quantize":
        m, k = c["m"], c["k"]
        if c["mode"] == "tiles":
            return {"bytes": m * k * (width + 2) + m * k / 2048, "flops": 4 * m * k}
        return {"bytes": m * k * (width + 1) + m * k / 32, "flops": 3 * m * k}
    if kind in ("linear", "grad"):
        m, n, k = c["m"], c["n"], c["k"]
        if kind == "linear":
            return {"bytes": n * k + n * k / 4096 + (m * k + m * n) * width, "flops": 2 * m * n * k}
        return {"bytes": n * k + n * k / 4096 + (2 * m * k + m * n) * width + 4 * n * k, "flops": 4 * m * n * k}
    t, h, j = c["t"], c["h"], c["top_k"]
    n, slots = c.get("n", h), t * j
    if kind == "exchange":
        # x, ys, dy and the routes in; xs, y, dys, dx, the weights' gradient and the plan out
        return {"bytes": (4 * t + 3 * slots) * h * width + 16 * slots + 4 * c["e"], "flops": 6 * slots * h}
    experts = _expected_experts(c)
    if kind == "experts":
        return {"bytes": experts * n * h + t * (h + n) * width + 8 * slots, "flops": 2 * slots * n * h + 2 * slots * n}
    return {"bytes": experts * n * h + c["e"] * 4 * n * h + (t * (n + h) + slots * (n + h)) * width + 12 * slots,
            "flops": 4 * slots * n * h + 4 * slots * n}


# ---- the same outputs in 64 bits ------------------------------------------------------------------------------------

def _round8(v, code):
    """v (f64) to the nearest value of an 8-bit format, ties to even: 3 or 2 bits behind the leading one, the smallest
    exponent -6 or -14."""
    bits, low = (3, -6) if code == E4M3 else (2, -14)
    exponent = torch.clamp_min(torch.frexp(v)[1] - 1, low)
    step = ((exponent.long() - bits + 1023) << 52).view(torch.float64)  # 2 ** (exponent - bits)
    return torch.round(v / step) * step


def _scale64(amax, code):
    """A block's scale and its reciprocal: f32 numbers by definition, as the codes' rounding goes by them."""
    part = torch.tensor(1.0 / TOP[code], dtype=torch.float32).double().item()
    s = torch.clamp_min((amax * part).float().double(), TINY)
    return s, (1.0 / s).float().double()


def _cut(n):
    return torch.arange(n, device=DEV) // 128


def _block_amax(x, dim):
    """The largest magnitude of each block of 128 along dim."""
    where = _cut(x.shape[dim])
    shape = list(x.shape)
    shape[dim] = _blocks(x.shape[dim])
    where = where.view([-1 if d == dim else 1 for d in range(x.dim())]).expand(x.shape)
    return torch.zeros(shape, dtype=x.dtype, device=DEV).scatter_reduce(dim, where, x.abs(), "amax")


def _quant64(x, dim, code):
    """(codes' values, scales, the values they stand for) of x [m, k] in blocks of 128 along dim."""
    x = x.double()
    s, inv = _scale64(_block_amax(x, dim), code)
    at = _cut(x.shape[dim])
    q = _round8((x * inv.index_select(dim, at)).float().double(), code)
    return q, s, q * s.index_select(dim, at)


def _quant64_tiles(w):
    w = w.double()
    s, inv = _scale64(_block_amax(_block_amax(w, 0), 1), E4M3)
    a, b = _cut(w.shape[0]), _cut(w.shape[1])
    q = _round8((w * inv[a][:, b]).float().double(), E4M3)
    return q, s, q * s[a][:, b]


def _padded(q, dim):
    """q with zeros up to a multiple of 16 along dim, as f32 (its values are exact there)."""
    shape = list(q.shape)
    shape[dim] = _up(shape[dim], 16)
    out = torch.zeros(shape, device=DEV)
    out.narrow(dim, 0, q.shape[dim]).copy_(q)
    return out


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    kind, dt = c["kind"], DT[c["dtype"]]
    if kind == "quantize":
        if c["mode"] == "tiles":
            q, s, _ = _quant64_tiles(t["x"])
            return {"q": _padded(q, 1), "scale": s, "qt": _padded(q, 0).t(), "scale_t": s.t()}
        q, s, _ = _quant64(t["x"], 0 if c["mode"] == "cols" else 1, E4M3)
        return {"q": _padded(q, 0).t(), "scale": s.t()} if c["mode"] == "cols" else {"q": _padded(q, 1), "scale": s}
    if kind in ("linear", "grad"):
        w = _quant64_tiles(t["w"][0])[2]
        if kind == "linear":
            return {"y": _quant64(t["x"], 1, E4M3)[2] @ w.t()}
        return {"dx": _quant64(t["dy"], 1, E5M2)[2] @ w,
                "dw": _quant64(t["dy"], 0, E5M2)[2].t() @ _quant64(t["x"], 0, E4M3)[2]}
    # the rows of each expert, slot by slot in its order
    idx, weight, j = t["idx"].flatten(), t["weight"].double().flatten(), c["top_k"]
    slots = [torch.nonzero(idx == e).flatten() for e in range(c["e"])]
    tokens, rows, first = c["t"], _capacity(c), 0
    n = c.get("n", c["h"])
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=DEV)  # noqa: E731
    if kind == "experts":
        x, y = _quant64(t["x"], 1, E4M3)[2], zeros(tokens, n)
        for e, at in enumerate(slots):
            if len(at):
                ys = (x[at // j] @ _quant64_tiles(t["w"][e])[2].t()).to(dt).double()
                y.index_add_(0, at // j, weight[at, None] * ys)
        return {"y": y}
    ys, dy = t["ys"].double(), t["dy"].double()
    dweight, dx = zeros(tokens * j), zeros(tokens, c["h"])
    y, xs, dys = zeros(tokens, n), zeros(rows, c["h"]), zeros(rows, n)
    dw = None if kind == "exchange" else zeros(c["e"], n, c["h"])
    for e, at in enumerate(slots):
        size = _up(len(at), _align(c))
        mine = slice(first, first + len(at))
        whole = slice(first, first + size)
        first += size
        if not len(at):
            continue
        y.index_add_(0, at // j, weight[at, None] * ys[mine])
        dweight[at] = (ys[mine] * dy[at // j]).sum(1)
        xs[mine] = t["x"][at // j].double()
        dys[mine] = (weight[at, None] * dy[at // j]).to(dt).double()
        if kind == "exchange":
            dx.index_add_(0, at // j, dys[mine])
            continue
        w = _quant64_tiles(t["w"][e])[2]
        dxs = (_quant64(dys[mine], 1, E5M2)[2] @ w).to(dt).double()
        dx.index_add_(0, at // j, dxs)
        dw[e] = _quant64(dys[whole], 0, E5M2)[2].t() @ _quant64(xs[whole], 0, E4M3)[2]
    dweight = dweight.view(tokens, j)
    if kind == "exchange":
        return {"offsets": None, "row_of": None, "xs": xs, "y": y, "dys": dys, "dweight": dweight, "dx": dx}
    return {"dweight": dweight, "dx": dx, "dw": dw}
