"""Cases of the FP8 block-scaled products and of the routed expert products around them, with plain forms.

Layouts are the library's (column-major); a torch row-major tensor [cols, rows] is a column-major rows x cols
matrix. A block-scaled operand is FP8 values with one f32 scale per 128 elements along K ("vec": scale [K/128, I]
in torch terms, I the non-K index) or per 128 x 128 block ("blk": stored as the operand is). The three products of
a linear layer Y = X W^T with X [tokens, in], W [out, in]:
  fwd   : m = out, n = tokens, k = in;     A = W   op T blk, B = X  op N vec
  dgrad : m = in,  n = tokens, k = out;    A = W   op N blk, B = dY op N vec
  wgrad : m = in,  n = out,    k = tokens; A = X   op N vec, B = dY op T vec
"""
import math
import os
import sys

import numpy as np
import torch

own = False

FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FLOAT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _cdiv(a, b):
    return (a + b - 1) // b


def _up(a, b):
    return _cdiv(a, b) * b


def listed():
    return [
        # A serving step: a few dozen tokens choose 4 of 64 experts; one launch, latency counts.
        {"name": "route-decode", "op": "route", "tokens": 48, "experts": 64, "top_k": 4, "score": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "renorm": True, "scale": 1.0, "dtype": "bf16", "align": 1},
        # A prompt batch with balance bias and group-limited choice.
        {"name": "route-prefill", "op": "route", "tokens": 16384, "experts": 256, "top_k": 8, "score": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "renorm": True, "scale": 2.5, "dtype": "f32", "align": 128},
        # Gradient of the routing weights for a training batch of an odd length.
        {"name": "route-backward", "op": "route_bwd", "tokens": 16383, "experts": 160, "top_k": 6, "score": "softmax",
         "renorm": False, "scale": 1.0, "dtype": "f32"},
        # Activations of a prompt batch, gathered into expert order while they are cast (each token to 4 experts).
        {"name": "quantize-gather", "op": "quant", "mode": "vec", "axis": 0, "rows": 4096, "cols": 16384, "src_cols": 4096,
         "div": 4, "gather": True, "src": "bf16", "dst": "e4m3"},
        # A weight matrix cast to 128 x 128 blocks after an optimizer step.
        {"name": "quantize-weights", "op": "quant", "mode": "blk", "axis": 0, "rows": 8192, "cols": 8192, "src_cols": 8192,
         "div": 1, "gather": False, "src": "f32", "dst": "e4m3"},
        # One serving step of 16 tokens through a linear layer: bound by reading the weights once.
        {"name": "gemm-decode", "op": "gemm", "kind": "fwd", "m": 4096, "n": 16, "k": 4096, "a": "e4m3", "b": "e4m3",
         "c": "bf16"},
        # The repository's headline size in FP8.
        {"name": "gemm-8192", "op": "gemm", "kind": "fwd", "m": 8192, "n": 8192, "k": 8192, "a": "e4m3", "b": "e4m3",
         "c": "bf16"},
        # The experts' products of a serving step: few rows per expert, some experts empty.
        {"name": "experts-decode", "op": "grouped", "kind": "fwd", "groups": 64, "m": 2048, "k": 2048, "rows": 128,
         "align": 1, "a": "e4m3", "b": "e4m3", "c": "bf16"},
        # The experts' products of a prompt batch, ragged.
        {"name": "experts-prefill", "op": "grouped", "kind": "fwd", "groups": 32, "m": 4096, "k": 2048, "rows": 32768,
         "align": 1, "a": "e4m3", "b": "e4m3", "c": "bf16"},
        # The experts' weight gradients: each expert's tokens are the contracted axis.
        {"name": "experts-wgrad", "op": "grouped", "kind": "wgrad", "groups": 16, "m": 2048, "n": 2048, "rows": 16384,
         "align": 128, "a": "e4m3", "b": "e5m2", "c": "f32"},
        # The experts' outputs summed back to their tokens, and its gradient.
        {"name": "combine", "op": "combine", "tokens": 8192, "top_k": 8, "hidden": 4096, "dtype": "bf16", "align": 1},
        {"name": "combine-backward", "op": "combine_bwd", "tokens": 4096, "top_k": 4, "hidden": 4096, "dtype": "bf16",
         "align": 128},
    ]


def _pow2(e, dtype):
    """2 ** e for whole e in the normal range, by its bits."""
    if dtype == torch.float32:
        return ((e.to(torch.int32) + 127) << 23).view(torch.float32)
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "route_bwd", "quant", "gemm", "gemm", "grouped", "grouped", "combine", "combine_bwd"])
    if op in ("route", "route_bwd"):
        c = {"op": op, "tokens": _log(rng, 1, 16384), "score": rng.choice(["softmax", "sigmoid"]),
             "renorm": rng.random() < 0.5, "scale": rng.choice([1.0, 2.5]), "dtype": rng.choice(["f32", "bf16", "f16"])}
        if op == "route":
            groups = rng.choice([1, 1, 4, 8])
            per = _log(rng, 4, 32)
            c.update(groups=groups, top_groups=rng.randint(1, groups), bias=rng.random() < 0.5,
                     experts=groups * per if groups > 1 else _log(rng, 4, 256), align=rng.choice([1, 16, 128]))
            pool = c["experts"] // groups * c["top_groups"]
        else:
            c["experts"] = pool = _log(rng, 4, 256)
        # one renormalised weight is constant: it has no gradient
        c["top_k"] = rng.randint(1 if op == "route" else 2, min(8, pool))
        return c
    if op == "quant":
        mode = rng.choice(["vec", "vec", "blk"])
        rows, cols = _log(rng, 16, 8192), _log(rng, 1, 8192)
        gather = mode == "vec" and rng.random() < 0.5
        return {"op": op, "mode": mode, "axis": rng.choice([0, 1]) if mode == "vec" else 0, "rows": rows, "cols": cols,
                "src_cols": _log(rng, 1, cols) if gather else cols, "div": 1, "gather": gather,
                "src": rng.choice(["bf16", "f16", "f32"]), "dst": rng.choice(["e4m3", "e5m2"])}
    if op == "gemm":
        kind = rng.choice(["fwd", "fwd", "dgrad", "wgrad"])
        m, k = _log(rng, 128, 8192), _log(rng, 128, 8192)
        n = _log(rng, 1, 8192) if kind != "wgrad" else _log(rng, 128, 8192)
        if kind == "wgrad":
            k = _log(rng, 1, 8192)
        return {"op": op, "kind": kind, "m": m, "n": n, "k": k, "a": "e4m3", "b": rng.choice(["e4m3", "e5m2"]),
                "c": rng.choice(["bf16", "f16", "f32"])}
    if op == "grouped":
        kind = rng.choice(["fwd", "fwd", "dgrad", "wgrad"])
        groups, rows = _log(rng, 1, 128), _log(rng, 1, 16384)
        c = {"op": op, "kind": kind, "groups": groups, "m": _log(rng, 128, 2048), "rows": rows,
             "align": 128 if kind == "wgrad" else rng.choice([1, 16]), "a": "e4m3", "b": rng.choice(["e4m3", "e5m2"]),
             "c": rng.choice(["bf16", "f32"])}
        c["n" if kind == "wgrad" else "k"] = _log(rng, 128, 2048)
        return c
    return {"op": op, "tokens": _log(rng, 1, 4096), "top_k": rng.randint(1, 8), "hidden": _log(rng, 16, 4096),
            "dtype": rng.choice(["bf16", "f16", "f32"]), "align": rng.choice([1, 128])}


# ---- inputs -----------------------------------------------------------------

_kept = {}


def _lib():
    """The binding and the handle that a program keeps."""
    if "gs" not in _kept:
        sys.path.insert(0, os.path.join(os.getcwd(), "slang-gemm_b200"))
        import gemm_sm100 as gs
        _kept["gs"] = gs
        _kept["handle"] = gs.Handle()
    gs, h = _kept["gs"], _kept["handle"]
    h.set_stream(torch.cuda.current_stream())
    return gs, h


def _type(gs, t):
    return {torch.float32: gs.R_32F, torch.bfloat16: gs.R_16BF, torch.float16: gs.R_16F, torch.float8_e4m3fn: gs.R_8F_E4M3,
            torch.float8_e5m2: gs.R_8F_E5M2}[t.dtype]


def _fp8(gen, outer, inner, kind, batch=1):
    """[batch, outer, inner] FP8 values as a cast of normal data leaves them, rows padded to 16 bytes."""
    ld = _up(max(inner, 1), 16)
    t = torch.empty(batch, max(outer, 1), ld, dtype=torch.float32, device="cuda")
    t.normal_(0.0, 100.0 if kind == "e4m3" else 8000.0, generator=gen)
    top = 448.0 if kind == "e4m3" else 57344.0
    return t.clamp_(-top, top).to(FP8[kind])[:, :max(outer, 1), :inner]


def _scales(gen, *shape):
    """f32 scales: about 1e-3, spread over a factor of a few."""
    return torch.randn(*shape, generator=gen, device="cuda").mul_(0.5).exp_().mul_(1e-3)


def _split(gen, rows, groups, align):
    """Ragged groups of `rows` rows in all (some small, some empty), each start aligned; the offsets as a list."""
    p = torch.rand(groups, generator=gen, device="cuda").square_()
    p = (p / p.sum()).cumsum(0).mul_(rows).round_().long().tolist()
    p[-1] = rows
    off = [0]
    for e in range(groups):
        n = p[e] - (p[e - 1] if e else 0)
        off.append(off[-1] + _up(n, align))
    return off


def _plan(gen, tokens, top_k, align, experts=64):
    """slot_row [tokens, top_k] and row_slot [rows] of a random choice of distinct experts, as the router lays them out."""
    experts = max(experts, top_k)
    ids = torch.rand(tokens, experts, generator=gen, device="cuda").argsort(1)[:, :top_k].reshape(-1)
    order = ids.argsort(stable=True)
    counts = torch.zeros(experts, dtype=torch.int64, device="cuda").index_add_(0, ids, torch.ones_like(ids))
    padded = (counts + align - 1) // align * align
    start = padded.cumsum(0) - padded
    first = counts.cumsum(0) - counts
    sorted_ids = ids[order]
    row = start[sorted_ids] + torch.arange(tokens * top_k, device="cuda") - first[sorted_ids]
    rows = tokens * top_k + min(experts, tokens * top_k) * (align - 1)
    slot_row = torch.empty(tokens * top_k, dtype=torch.int32, device="cuda")
    slot_row[order] = row.int()
    row_slot = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    row_slot[row] = order.int()
    return slot_row.view(tokens, top_k), row_slot


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    op = case["op"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if op in ("route", "route_bwd"):
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        s["logits"] = randn(t, e).mul_(2.0).to(FLOAT[case["dtype"]])
        if op == "route":
            s["bias"] = randn(e).mul_(0.05) if case["bias"] else None
            s["rows"] = t * k + min(e, t * k) * (case["align"] - 1)
            s["ids"] = torch.empty(t, k, dtype=torch.int32, device="cuda")
            s["weights"] = torch.empty(t, k, device="cuda")
            s["offsets"] = torch.empty(e + 1, dtype=torch.int32, device="cuda")
            s["slot_row"] = torch.empty(t, k, dtype=torch.int32, device="cuda")
            s["row_slot"] = torch.empty(s["rows"], dtype=torch.int32, device="cuda")
            if own:
                gs, _ = _lib()
                s["workspace"] = torch.empty(max(1, gs.moe_route_workspace(t, e, k)), dtype=torch.uint8, device="cuda")
        else:
            s["ids"] = s["logits"].double().topk(k, 1).indices.int()
            s["dweights"] = randn(t, k)
            s["dlogits"] = torch.empty_like(s["logits"])
    elif op == "quant":
        r, c = case["rows"], case["cols"]
        ld = _up(r, 8)
        x = randn(case["src_cols"], ld)
        # rows of very different size, as activations and gradients have them
        x.mul_(randn(case["src_cols"], 1).exp_())
        s["src"] = x.to(FLOAT[case["src"]])[:, :r]
        s["index"] = None
        if case["gather"]:
            hi = case["src_cols"] * case["div"]
            s["index"] = torch.randint(0, hi, (c,), generator=gen, device="cuda", dtype=torch.int32)
            s["index"][torch.rand(c, generator=gen, device="cuda") < 0.02] = -1  # padding rows of the experts
        s["dst"] = torch.zeros(c, _up(r, 16), dtype=torch.uint8, device="cuda").view(FP8[case["dst"]])
        rb, cb = _cdiv(r, 128), _cdiv(c, 128)
        s["scale"] = torch.zeros((cb, rb) if case["mode"] == "blk" else (rb, c) if case["axis"] == 0 else (cb, r), device="cuda")
    elif op == "gemm":
        m, n, k, kind = case["m"], case["n"], case["k"], case["kind"]
        mb, kb = _cdiv(m, 128), _cdiv(k, 128)
        s["A"] = _fp8(gen, m if kind == "fwd" else k, k if kind == "fwd" else m, case["a"])[0]
        s["B"] = _fp8(gen, k if kind == "wgrad" else n, n if kind == "wgrad" else k, case["b"])[0]
        s["sA"] = _scales(gen, *((mb, kb) if kind == "fwd" else (kb, mb) if kind == "dgrad" else (kb, m)))
        s["sB"] = _scales(gen, kb, n)
        s["C"] = torch.empty(n, m, dtype=FLOAT[case["c"]], device="cuda")
    elif op == "grouped":
        g, m, kind = case["groups"], case["m"], case["kind"]
        s["host_offsets"] = off = _split(gen, case["rows"], g, case["align"])
        s["offsets"] = torch.tensor(off, dtype=torch.int32, device="cuda")
        rows = off[-1]
        mb = _cdiv(m, 128)
        if kind == "wgrad":
            n, kb = case["n"], _cdiv(rows, 128)
            s["A"], s["B"] = _fp8(gen, rows, m, case["a"])[0], _fp8(gen, rows, n, case["b"])[0]
            s["sA"], s["sB"] = _scales(gen, kb, m), _scales(gen, kb, n)
            s["C"] = torch.empty(g, n, m, dtype=FLOAT[case["c"]], device="cuda")
        else:
            k, kb = case["k"], _cdiv(case["k"], 128)
            s["A"] = _fp8(gen, m if kind == "fwd" else k, k if kind == "fwd" else m, case["a"], g)
            s["B"] = _fp8(gen, rows, k, case["b"])[0]
            s["sA"] = _scales(gen, g, *((mb, kb) if kind == "fwd" else (kb, mb)))
            s["sB"] = _scales(gen, kb, rows)
            s["C"] = torch.empty(rows, m, dtype=FLOAT[case["c"]], device="cuda")
    else:
        t, k, hid = case["tokens"], case["top_k"], case["hidden"]
        s["slot_row"], s["row_slot"] = _plan(gen, t, k, case["align"])
        rows = s["row_slot"].numel()
        s["y"] = randn(rows, hid).to(FLOAT[case["dtype"]])
        s["weights"] = randn(t, k).softmax(1)
        if op == "combine":
            s["out"] = torch.empty(t, hid, dtype=s["y"].dtype, device="cuda")
        else:
            s["dout"] = randn(t, hid).to(s["y"].dtype)
            s["dy"] = torch.empty_like(s["y"])
            s["dweights"] = torch.empty(t, k, device="cuda")
    return s


# ---- one pass ---------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    return (_own if own else _plain)[op](s)


def _ld(t):
    """Leading dimension of a row-major view (its outer stride), also where the view has one row."""
    return t.stride(-2)


def _own_route(s):
    gs, h = _lib()
    c = s["case"]
    h.moe_route(c["tokens"], c["experts"], c["top_k"], s["logits"], _type(gs, s["logits"]), c["experts"], s["ids"], s["weights"],
                bias=s["bias"], score=gs.ROUTE_SIGMOID if c["score"] == "sigmoid" else gs.ROUTE_SOFTMAX, groups=c["groups"],
                top_groups=c["top_groups"], renormalize=c["renorm"], scale=c["scale"], align=c["align"], offsets=s["offsets"],
                slot_row=s["slot_row"], row_slot=s["row_slot"], rows=s["rows"], workspace=s["workspace"],
                workspace_bytes=s["workspace"].numel())
    return {"ids": s["ids"], "weights": s["weights"], "offsets": s["offsets"], "slot_row": s["slot_row"], "row_slot": s["row_slot"]}


def _own_route_bwd(s):
    gs, h = _lib()
    c = s["case"]
    h.moe_route_backward(c["tokens"], c["experts"], c["top_k"], s["logits"], _type(gs, s["logits"]), c["experts"], s["ids"],
                         s["dweights"], s["dlogits"], _type(gs, s["dlogits"]), c["experts"],
                         score=gs.ROUTE_SIGMOID if c["score"] == "sigmoid" else gs.ROUTE_SOFTMAX, renormalize=c["renorm"],
                         scale=c["scale"])
    return s["dlogits"]


def _own_quant(s):
    gs, h = _lib()
    c = s["case"]
    mode = gs.SCALE_BLK128 if c["mode"] == "blk" else gs.SCALE_VEC128
    h.fp8_quantize(mode, c["axis"], c["rows"], c["cols"], s["src"], _type(gs, s["src"]), _ld(s["src"]), s["dst"],
                   _type(gs, s["dst"]), _ld(s["dst"]), s["scale"], _ld(s["scale"]), index=s["index"], index_div=c["div"],
                   src_cols=c["src_cols"])
    return {"q": s["dst"][:, :c["rows"]], "scale": s["scale"]}


def _own_gemm(s):
    gs, h = _lib()
    c, kind = s["case"], s["case"]["kind"]
    h.gemm_fp8(gs.OP_T if kind == "fwd" else gs.OP_N, gs.OP_T if kind == "wgrad" else gs.OP_N, c["m"], c["n"], c["k"], 1.0,
               s["A"], _type(gs, s["A"]), _ld(s["A"]), s["sA"], gs.SCALE_VEC128 if kind == "wgrad" else gs.SCALE_BLK128,
               _ld(s["sA"]), s["B"], _type(gs, s["B"]), _ld(s["B"]), s["sB"], gs.SCALE_VEC128, _ld(s["sB"]), 0.0, s["C"],
               _type(gs, s["C"]), c["m"])
    return s["C"]


def _own_grouped(s):
    gs, h = _lib()
    c, kind = s["case"], s["case"]["kind"]
    rows = s["host_offsets"][-1]
    if kind == "wgrad":
        h.gemm_fp8_grouped(gs.GROUP_K, gs.OP_N, gs.OP_T, c["m"], c["n"], rows, c["groups"], s["offsets"], 1.0, s["A"],
                           _type(gs, s["A"]), _ld(s["A"]), 0, s["sA"], gs.SCALE_VEC128, _ld(s["sA"]), 0, s["B"],
                           _type(gs, s["B"]), _ld(s["B"]), s["sB"], gs.SCALE_VEC128, _ld(s["sB"]), 0.0, s["C"],
                           _type(gs, s["C"]), c["m"], s["C"].stride(0))
    else:
        h.gemm_fp8_grouped(gs.GROUP_N, gs.OP_T if kind == "fwd" else gs.OP_N, gs.OP_N, c["m"], rows, c["k"], c["groups"],
                           s["offsets"], 1.0, s["A"], _type(gs, s["A"]), _ld(s["A"]), s["A"].stride(0), s["sA"],
                           gs.SCALE_BLK128, _ld(s["sA"]), s["sA"].stride(0), s["B"], _type(gs, s["B"]), _ld(s["B"]),
                           s["sB"], gs.SCALE_VEC128, _ld(s["sB"]), 0.0, s["C"], _type(gs, s["C"]), c["m"], 0)
    return s["C"]


def _own_combine(s):
    gs, h = _lib()
    c = s["case"]
    h.moe_combine(c["tokens"], c["top_k"], c["hidden"], s["y"], _type(gs, s["y"]), c["hidden"], s["row_slot"].numel(),
                  s["slot_row"], s["weights"], s["out"], _type(gs, s["out"]), c["hidden"])
    return s["out"]


def _own_combine_bwd(s):
    gs, h = _lib()
    c = s["case"]
    h.moe_combine_backward(c["tokens"], c["top_k"], c["hidden"], s["y"], _type(gs, s["y"]), c["hidden"], s["row_slot"].numel(),
                           s["slot_row"], s["row_slot"], s["weights"], s["dout"], _type(gs, s["dout"]), c["hidden"], s["dy"],
                           c["hidden"], s["dweights"])
    return {"dy": s["dy"], "dweights": s["dweights"]}


def _scores(logits, score):
    l = logits.double()
    l = torch.where(torch.isnan(l), -math.inf, l).clamp(max=torch.finfo(torch.float32).max)
    if score == "sigmoid":
        return l, 1 / (1 + torch.exp(-l))
    top = l.amax(1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    x = torch.exp(l - top)
    total = x.sum(1, keepdim=True)
    return l, torch.where(total > 0, x / total, 0.0)


def _plain_route(s):
    c = s["case"]
    t, e, k, g = c["tokens"], c["experts"], c["top_k"], c["groups"]
    l, sc = _scores(s["logits"], c["score"])
    choice = sc if s["bias"] is None else sc + s["bias"].double()
    dead = torch.isneginf(l) | torch.isnan(choice)
    choice = torch.where(dead, -math.inf, choice)
    # without a bias the scores' order is the logits' order, also where scores round together
    key = torch.where(dead, -math.inf, l) if s["bias"] is None else choice
    if g > 1:
        two = choice.view(t, g, e // g).sort(dim=2, descending=True).values[:, :, :2]
        first = two[:, :, 0]
        both = torch.where(torch.isneginf(two), 0.0, two).sum(2)
        gscore = torch.where(torch.isneginf(first), -math.inf, both)
        kept = gscore.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        keep = torch.zeros(t, g, dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        key = torch.where(keep.repeat_interleave(e // g, 1), key, -math.inf)
    best = key.sort(dim=1, descending=True, stable=True)
    ids, live = best.indices[:, :k], ~torch.isneginf(best.values[:, :k])
    w = torch.where(live, sc.gather(1, ids), 0.0)
    if c["renorm"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    w = (w * c["scale"]).float()
    ids = torch.where(live, ids, -1)
    flat = torch.where(live, ids, e).reshape(-1)
    counts = (flat[:, None] == torch.arange(e, device="cuda")).sum(0)
    padded = (counts + c["align"] - 1) // c["align"] * c["align"]
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), padded.cumsum(0)])
    order = flat.argsort(stable=True)
    first = torch.cat([counts.cumsum(0) - counts, counts.sum()[None]])
    start = torch.cat([offsets[:e], torch.zeros(1, dtype=torch.int64, device="cuda")])
    sorted_ids = flat[order]
    row = start[sorted_ids] + torch.arange(t * k, device="cuda") - first[sorted_ids]
    row = torch.where(sorted_ids == e, -1, row)
    slot_row = torch.empty_like(row)
    slot_row[order] = row
    row_slot = torch.full((s["rows"] + 1,), -1, dtype=torch.int64, device="cuda")
    row_slot[torch.where(row < 0, s["rows"], row)] = order
    return {"ids": ids.int(), "weights": w, "offsets": offsets.int(), "slot_row": slot_row.int().view(t, k),
            "row_slot": row_slot[:-1].int()}


def _plain_route_bwd(s):
    c = s["case"]
    _, sc = _scores(s["logits"], c["score"])
    ids, g = s["ids"].long(), s["dweights"].double() * c["scale"]
    w = sc.gather(1, ids)
    if c["renorm"]:
        total = w.sum(1, keepdim=True)
        g = (g - (g * w).sum(1, keepdim=True) / total) / total
    ds = torch.zeros_like(sc).scatter_(1, ids, g)
    d = ds * sc * (1 - sc) if c["score"] == "sigmoid" else sc * (ds - (ds * sc).sum(1, keepdim=True))
    return d.to(s["logits"].dtype)


def _blocks(x, mode, axis):
    """amax of |finite x| of each block, spread over its elements, and the blocks' own layout; x is [cols, rows]."""
    c, r = x.shape
    pr, pc = _up(r, 128) - r, _up(c, 128) - c
    a = torch.nn.functional.pad(torch.where(torch.isfinite(x), x.abs(), 0.0), (0, pr, 0, pc))
    if mode == "blk":
        return a.view((c + pc) // 128, 128, (r + pr) // 128, 128).amax((1, 3))
    if axis == 0:
        return a[:c].view(c, -1, 128).amax(2).t()
    return a[:, :r].reshape(-1, 128, r).amax(1)


def _plain_quant(s):
    c = s["case"]
    x = s["src"].float()
    if s["index"] is not None:
        i = s["index"].long()
        x = torch.where((i >= 0)[:, None], x[(i.clamp(min=0) // c["div"])], 0.0)
    amax = _blocks(x, c["mode"], c["axis"])
    mant, exp = torch.frexp(amax)
    exp = (exp + (mant > 0.875) - (9 if c["dst"] == "e4m3" else 16)).clamp(min=-126)
    scale = torch.where(amax > 0, _pow2(exp, torch.float32), 1.0)
    n, r = x.shape
    if c["mode"] == "blk":
        full = scale.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :r]
    else:
        full = scale.t().repeat_interleave(128, 1)[:, :r] if c["axis"] == 0 else scale.repeat_interleave(128, 0)[:n]
    return {"q": (x / full).to(FP8[c["dst"]]), "scale": scale.contiguous()}


def _spread(s, vec, k_first, i, k):
    """Scales [i, k] of every element: vec [K/128, I]; blk as stored, its K blocks first or second."""
    if vec:
        return s.t().repeat_interleave(128, 1)[:i, :k]
    return (s.t() if k_first else s).repeat_interleave(128, 0)[:i].repeat_interleave(128, 1)[:, :k]


def _plain_gemm(s):
    c, kind = s["case"], s["case"]["kind"]
    m, n, k = c["m"], c["n"], c["k"]
    a = s["A"].float() if kind == "fwd" else s["A"].float().t()
    b = s["B"].float().t() if kind == "wgrad" else s["B"].float()
    a = a * _spread(s["sA"], kind == "wgrad", kind == "dgrad", m, k)
    b = b * _spread(s["sB"], True, False, n, k)
    return (b @ a.t()).to(s["C"].dtype)


def _plain_grouped(s):
    c, kind, off = s["case"], s["case"]["kind"], s["host_offsets"]
    m, out = c["m"], []
    for e in range(c["groups"]):
        lo, hi = off[e], off[e + 1]
        if kind == "wgrad":
            a = s["A"][lo:hi].float().t() * _spread(s["sA"][lo // 128:_cdiv(hi, 128)], True, False, m, hi - lo)
            b = s["B"][lo:hi].float().t() * _spread(s["sB"][lo // 128:_cdiv(hi, 128)], True, False, c["n"], hi - lo)
            out.append((b @ a.t()).to(s["C"].dtype))
        elif hi > lo:
            a = s["A"][e].float() if kind == "fwd" else s["A"][e].float().t()
            a = a * _spread(s["sA"][e], False, kind == "dgrad", m, c["k"])
            b = s["B"][lo:hi].float() * _spread(s["sB"][:, lo:hi], True, False, hi - lo, c["k"])
            out.append((b @ a.t()).to(s["C"].dtype))
    if kind == "wgrad":
        return torch.stack(out)
    return torch.cat(out) if out else torch.empty(0, m, dtype=s["C"].dtype, device="cuda")


def _plain_combine(s):
    rows = s["slot_row"].long()
    y = torch.where((rows >= 0)[:, :, None], s["y"][rows.clamp(min=0)].float(), 0.0)
    return (y * s["weights"][:, :, None]).sum(1).to(s["y"].dtype)


def _plain_combine_bwd(s):
    k = s["case"]["top_k"]
    slot, rows = s["row_slot"].long(), s["slot_row"].long()
    live = (slot >= 0)[:, None]
    slot = slot.clamp(min=0)
    d = s["dout"].float()
    dy = torch.where(live, d[slot // k] * s["weights"].reshape(-1)[slot][:, None], 0.0)
    dw = (s["y"][rows.clamp(min=0)].float() * d[:, None, :]).sum(2)
    return {"dy": dy.to(s["y"].dtype), "dweights": torch.where(rows >= 0, dw, 0.0)}


_own = {"route": _own_route, "route_bwd": _own_route_bwd, "quant": _own_quant, "gemm": _own_gemm, "grouped": _own_grouped,
        "combine": _own_combine, "combine_bwd": _own_combine_bwd}
_plain = {"route": _plain_route, "route_bwd": _plain_route_bwd, "quant": _plain_quant, "gemm": _plain_gemm,
          "grouped": _plain_grouped, "combine": _plain_combine, "combine_bwd": _plain_combine_bwd}


# ---- from the definitions, in 64 bits ----------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "route_bwd": _exact_route_bwd, "quant": _exact_quant, "gemm": _exact_gemm,
            "grouped": _exact_grouped, "combine": _exact_combine, "combine_bwd": _exact_combine_bwd}[case["op"]](s, case)


def _np_scores(logits, score):
    x = logits.double().cpu().numpy().copy()
    x[np.isnan(x)] = -np.inf
    x = np.minimum(x, np.finfo(np.float32).max)
    if score == "sigmoid":
        with np.errstate(over="ignore"):
            return x, np.where(x >= 0, 1 / (1 + np.exp(-x)), np.exp(np.minimum(x, 0)) / (1 + np.exp(np.minimum(x, 0))))
    p = np.exp(x - np.maximum(x.max(1, keepdims=True), np.finfo(np.float32).min))
    z = p.sum(1, keepdims=True)
    return x, np.divide(p, z, out=np.zeros_like(p), where=z > 0)


def _exact_route(s, c):
    x, p = _np_scores(s["logits"], c["score"])
    t, e = x.shape
    k, g = c["top_k"], c["groups"]
    v = p + s["bias"].double().cpu().numpy() if c["bias"] else p.copy()
    v[np.isneginf(x) | np.isnan(v)] = -np.inf
    key = v if c["bias"] else np.where(np.isneginf(v), -np.inf, x)
    if g > 1:
        top = -np.sort(-v.reshape(t, g, e // g), axis=2)[:, :, :2]
        total = np.where(np.isneginf(top), 0, top).sum(2)
        total[np.isneginf(top[:, :, 0])] = -np.inf
        rank = np.argsort(np.argsort(-total, axis=1, kind="stable"), axis=1, kind="stable")
        key = np.where(np.repeat(rank < c["top_groups"], e // g, axis=1), key, -np.inf)
    ids = np.argsort(-key, axis=1, kind="stable")[:, :k]
    live = ~np.isneginf(np.take_along_axis(key, ids, 1))
    w = np.take_along_axis(p, ids, 1) * live
    if c["renorm"]:
        z = w.sum(1, keepdims=True)
        w = np.divide(w, z, out=np.zeros_like(w), where=z > 0)
    ids = np.where(live, ids, -1)
    flat, a = ids.reshape(-1), c["align"]
    offsets, slot_row, row_slot = [0], np.full(t * k, -1), np.full(s["rows"], -1)
    for i in range(e):
        slots = np.nonzero(flat == i)[0]
        at = offsets[-1] + np.arange(len(slots))
        slot_row[slots] = at
        row_slot[at] = slots
        offsets.append(offsets[-1] + _up(len(slots), a))
    return {"ids": ids.astype(np.int32), "weights": w * c["scale"], "offsets": np.array(offsets, np.int32),
            "slot_row": slot_row.reshape(t, k).astype(np.int32), "row_slot": row_slot.astype(np.int32)}


def _exact_route_bwd(s, c):
    _, p = _np_scores(s["logits"], c["score"])
    ids, g = s["ids"].long().cpu().numpy(), s["dweights"].double().cpu().numpy()
    t = np.arange(p.shape[0])[:, None]
    chosen = p[t, ids]
    # dL/dlogit = sum_j g_j dw_j/dlogit, from log-derivatives: dw_j = w_j (dlog s_j - dlog of the norm)
    if c["score"] == "sigmoid":
        out, one = np.zeros_like(p), 1 - chosen
        if c["renorm"]:
            w = chosen / chosen.sum(1, keepdims=True)
            out[t, ids] = c["scale"] * w * one * (g - (g * w).sum(1, keepdims=True))
        else:
            out[t, ids] = c["scale"] * g * chosen * one
        return out
    if c["renorm"]:  # a softmax over the chosen ones alone
        w = chosen / chosen.sum(1, keepdims=True)
        out = np.zeros_like(p)
        out[t, ids] = c["scale"] * w * (g - (g * w).sum(1, keepdims=True))
        return out
    out = -p * (g * chosen).sum(1, keepdims=True)
    out[t, ids] += g * chosen
    return out * c["scale"]


def _exact_quant(s, c):
    x = s["src"].double()
    if s["index"] is not None:
        x = torch.cat([x, torch.zeros_like(x[:1])])[torch.where(s["index"] < 0, x.shape[0], s["index"] // c["div"]).long()]
    top, low, bits = (448.0, -6, 3) if c["dst"] == "e4m3" else (57344.0, -14, 2)
    n, r = x.shape
    scale = torch.empty(s["scale"].shape, dtype=torch.float64, device="cuda")
    q = torch.empty_like(x)
    bc = 128 if c["mode"] == "blk" or c["axis"] == 1 else n
    br = 128 if c["mode"] == "blk" or c["axis"] == 0 else r
    for j in range(0, n, bc):
        for i in range(0, r, br):
            part = x[j:j + bc, i:i + br].abs()
            amax = part.amax() if c["mode"] == "blk" else part.amax(1) if c["axis"] == 0 else part.amax(0)
            most = torch.full_like(amax, top)
            f, e = torch.frexp(torch.where(amax > 0, amax, most) / most)
            e = (e - (f == 0.5).int()).clamp(min=-126)  # the whole number at or above log2(amax / most)
            step = _pow2(e, torch.float64)
            if c["mode"] == "blk":
                scale[j // 128, i // 128] = step
                q[j:j + bc, i:i + br] = x[j:j + bc, i:i + br] / step
            elif c["axis"] == 0:
                scale[i // 128] = step
                q[j:j + bc, i:i + br] = x[j:j + bc, i:i + br] / step[:, None]
            else:
                scale[j // 128] = step
                q[j:j + bc, i:i + br] = x[j:j + bc, i:i + br] / step
    grid = _pow2(torch.frexp(q.abs().clamp(min=2.0 ** low)).exponent - 1 - bits, torch.float64)
    return {"q": torch.round(q / grid) * grid, "scale": scale}


def _wide(q, scale, vec, k_outer, k, i):
    """[i, k] float64 values of an operand stored [i, k] or (k_outer) [k, i], each 128 of K times its scale."""
    x = q.double().t().clone() if k_outer else q.double()
    for b in range(0, k, 128):
        if vec:
            x[:, b:b + 128] *= scale[b // 128].double()[:, None]
        else:
            f = scale[b // 128] if k_outer else scale[:, b // 128]
            x[:, b:b + 128] *= f.double().repeat_interleave(128)[:i, None]
    return x


def _exact_gemm(s, c):
    wgrad = c["kind"] == "wgrad"
    a = _wide(s["A"], s["sA"], wgrad, c["kind"] != "fwd", c["k"], c["m"])
    return _wide(s["B"], s["sB"], True, wgrad, c["k"], c["n"]) @ a.t()


def _exact_grouped(s, c):
    off, kind = s["host_offsets"], c["kind"]
    if kind == "wgrad":
        out = torch.zeros(c["groups"], c["n"], c["m"], dtype=torch.float64, device="cuda")
        for e in range(c["groups"]):
            for b in range(off[e], off[e + 1], 128):
                f = s["sB"][b // 128].double()[:, None] * s["sA"][b // 128].double()
                h = min(b + 128, off[e + 1])
                out[e] += f * (s["B"][b:h].double().t() @ s["A"][b:h].double())
        return out
    out = torch.zeros(off[-1], c["m"], dtype=torch.float64, device="cuda")
    for e in range(c["groups"]):
        lo, hi = off[e], off[e + 1]
        if hi > lo:
            a = _wide(s["A"][e], s["sA"][e], False, kind == "dgrad", c["k"], c["m"])
            out[lo:hi] = _wide(s["B"][lo:hi], s["sB"][:, lo:hi], True, False, c["k"], hi - lo) @ a.t()
    return out


def _exact_combine(s, c):
    out = torch.zeros(c["tokens"], c["hidden"], dtype=torch.float64, device="cuda")
    for j in range(c["top_k"]):
        out += s["weights"][:, j].double()[:, None] * s["y"][s["slot_row"][:, j].long()].double()
    return out


def _exact_combine_bwd(s, c):
    dy = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
    dw = torch.zeros(c["tokens"], c["top_k"], dtype=torch.float64, device="cuda")
    d = s["dout"].double()
    for j in range(c["top_k"]):
        at = s["slot_row"][:, j].long()
        dy[at] = s["weights"][:, j].double()[:, None] * d
        dw[:, j] = (s["y"][at].double() * d).sum(1)
    return {"dy": dy, "dweights": dw}


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    op = case["op"]
    es = {"f32": 4, "bf16": 2, "f16": 2}
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        rows = t * k + min(e, t * k) * (case["align"] - 1)
        return {"bytes": t * e * es[case["dtype"]] + t * k * 12 + rows * 4 + (e + 1) * 4 + (e * 4 if case["bias"] else 0),
                "flops": 4 * t * e}
    if op == "route_bwd":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        return {"bytes": 2 * t * e * es[case["dtype"]] + t * k * 8, "flops": 6 * t * e}
    if op == "quant":
        r, c = case["rows"], case["cols"]
        blocks = _cdiv(r, 128) * _cdiv(c, 128) if case["mode"] == "blk" else _cdiv(r, 128) * c if case["axis"] == 0 else r * _cdiv(c, 128)
        read = min(case["src_cols"], c) * r * es[case["src"]] + (4 * c if case["gather"] else 0)
        return {"bytes": read + r * c + 4 * blocks, "flops": 2 * r * c}
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        sa = _cdiv(k, 128) * (m if case["kind"] == "wgrad" else _cdiv(m, 128))
        return {"bytes": (m + n) * k + m * n * es[case["c"]] + 4 * (sa + _cdiv(k, 128) * n), "flops": 2 * m * n * k}
    if op == "grouped":
        g, m, rows = case["groups"], case["m"], case["rows"]
        if case["kind"] == "wgrad":
            n = case["n"]
            return {"bytes": (m + n) * rows + g * m * n * es[case["c"]] + 4 * _cdiv(rows, 128) * (m + n) + 4 * (g + 1),
                    "flops": 2 * m * n * rows}
        k = case["k"]
        used = min(g, rows)
        return {"bytes": used * (m * k + 4 * _cdiv(m, 128) * _cdiv(k, 128)) + rows * (k + 4 * _cdiv(k, 128)) + rows * m * es[case["c"]],
                "flops": 2 * m * k * rows}
    t, k, hid, b = case["tokens"], case["top_k"], case["hidden"], es[case["dtype"]]
    if op == "combine":
        return {"bytes": t * k * hid * b + t * hid * b + t * k * 8, "flops": 2 * t * k * hid}
    rows = t * k + min(64, t * k) * (case["align"] - 1)
    return {"bytes": t * k * hid * b + t * hid * b + rows * hid * b + t * k * 12 + rows * 4, "flops": 3 * t * k * hid}
