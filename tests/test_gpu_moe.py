"""GPU tests of the expert routing, its gradient, the row plan, the combine and
its gradient against plain float64 forms, and of a whole routed FP8 layer:
route -> gather and quantise -> grouped product -> combine, and its backward."""
import math

import pytest
import torch

import gemm_sm100 as gs
from fp8_util import FLOAT
from routed_experts import RoutedExperts

pytestmark = pytest.mark.gpu
TYPE = {v: k for k, v in FLOAT.items()}
SIGMOID, SOFTMAX = gs.ROUTE_SIGMOID, gs.ROUTE_SOFTMAX
TOP = torch.finfo(torch.float32).max


def plain_scores(logits, score):
    l = logits.double()
    l = torch.where(l.isnan(), -math.inf, l).clamp(max=TOP)
    if score == SIGMOID:
        return l, 1 / (1 + torch.exp(-l))
    p = torch.exp(l - l.amax(1, keepdim=True).clamp(min=-TOP))
    z = p.sum(1, keepdim=True)
    return l, torch.where(z > 0, p / z, 0.0)


def plain_route(logits, k, score, bias, groups, top_groups, renorm, scale, count=None):
    """ids and weights, token by token."""
    l, s = plain_scores(logits, score)
    t, e = s.shape
    ids, weights = torch.full((t, k), -1), torch.zeros(t, k, dtype=torch.float64)
    for i in range(t if count is None else min(t, count)):
        c = s[i] if bias is None else s[i] + bias.double()
        c = torch.where(l[i].isneginf() | c.isnan(), -math.inf, c)
        key = c if bias is not None else torch.where(c.isneginf(), -math.inf, l[i])
        alive = list(range(groups))
        if groups > 1:
            best = []
            for g in range(groups):
                two = [v for v in c[g * (e // groups):(g + 1) * (e // groups)].sort(descending=True).values[:2].tolist()
                       if v > -math.inf]
                best.append(sum(two) if two else -math.inf)
            alive = sorted(range(groups), key=lambda g: (-best[g], g))[:top_groups]
        pool = [x for x in range(e) if x // (e // groups) in alive and key[x] > -math.inf]
        pool = sorted(pool, key=lambda x: (-float(key[x]), x))[:k]
        w = s[i][pool]
        if renorm:
            w = w / w.sum() if len(pool) and float(w.sum()) > 0 else torch.zeros_like(w)
        ids[i, :len(pool)] = torch.tensor(pool, dtype=torch.int64)
        weights[i, :len(pool)] = w * scale
    return ids, weights


def plain_plan(ids, experts, align, rows):
    flat = ids.reshape(-1).tolist()
    offsets, slot_row, row_slot = [0], [-1] * len(flat), [-1] * rows
    for e in range(experts):
        at = offsets[-1]
        for s, x in enumerate(flat):
            if x == e:
                slot_row[s], row_slot[at] = at, s
                at += 1
        offsets.append(offsets[-1] + (at - offsets[-1] + align - 1) // align * align)
    return offsets, slot_row, row_slot


def run_route(h, logits, k, score=SOFTMAX, bias=None, groups=1, top_groups=1, renorm=False, scale=1.0, count=None, align=1,
              pad=0, plan=True, extra=5):
    t, e = logits.shape
    buf = torch.full((t, e + pad), math.nan, dtype=logits.dtype, device="cuda")
    buf[:, :e] = logits.cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    out = dict(ids=torch.full((t, k), 99, **i32), weights=torch.full((t, k), math.nan, device="cuda"))
    kw = {}
    if plan:
        rows = gs.moe_rows(t, e, k, align) + extra
        ws = gs.moe_route_workspace(t, e, k)
        out.update(offsets=torch.full((e + 1,), 99, **i32), slot_row=torch.full((t, k), 99, **i32),
                   row_slot=torch.full((rows,), 99, **i32))
        kw = dict(offsets=out["offsets"], slot_row=out["slot_row"], row_slot=out["row_slot"], rows=rows,
                  workspace=torch.full((max(ws, 4),), 0xEE, dtype=torch.uint8, device="cuda"), workspace_bytes=ws)
    h.moe_route(t, e, k, buf, TYPE[logits.dtype], e + pad, out["ids"], out["weights"], bias=None if bias is None else bias.cuda(),
                score=score, groups=groups, top_groups=top_groups, renormalize=renorm, scale=scale,
                token_count=None if count is None else torch.tensor([count], **i32), align=align, **kw)
    torch.cuda.synchronize()
    assert h.last_kernels() == gs.KERNEL_ROUTE
    return {n: v.cpu() for n, v in out.items()}


def check_route(got, logits, k, score, bias, groups, top_groups, renorm, scale, count, align):
    ids, w = plain_route(logits, k, score, bias, groups, top_groups, renorm, scale, count)
    assert torch.equal(got["ids"].long(), ids)
    # f32: the exponent's argument rounds by |l - max| <= 64 halves of 2^-23 at most, expf by 2 ulp, a sum of up to 1024
    # terms in 37 steps, two divisions and a product
    assert bool(((got["weights"].double() - w).abs() <= (64 + 4 + 37 + 4) * 2.0 ** -24 * w.abs() + 1e-44).all())
    if "offsets" in got:
        rows = got["row_slot"].numel()
        offsets, slot_row, row_slot = plain_plan(ids, logits.shape[1], align, rows)
        assert got["offsets"].tolist() == offsets
        assert got["slot_row"].reshape(-1).tolist() == slot_row
        assert got["row_slot"].tolist() == row_slot


@pytest.mark.parametrize("t,e,k,score,with_bias,groups,top_groups,renorm,scale,align,dtype", [
    (1, 1, 1, SOFTMAX, False, 1, 1, False, 1.0, 1, torch.float32),
    (1, 64, 4, SOFTMAX, False, 1, 1, True, 1.0, 1, torch.bfloat16),
    (48, 64, 4, SOFTMAX, False, 1, 1, True, 1.0, 128, torch.bfloat16),
    (17, 33, 3, SIGMOID, True, 1, 1, False, 2.5, 16, torch.float16),
    (100, 128, 8, SIGMOID, True, 8, 3, True, 2.5, 1, torch.float32),
    (130, 160, 6, SOFTMAX, True, 5, 2, False, 1.0, 128, torch.float32),
    (300, 256, 8, SIGMOID, True, 8, 4, True, 2.5, 128, torch.float32),
    (257, 512, 4, SOFTMAX, False, 4, 2, True, 1.0, 1, torch.bfloat16),
    (70, 1024, 32, SOFTMAX, False, 32, 4, False, 1.0, 4, torch.float32),
    (2000, 8, 2, SOFTMAX, False, 1, 1, True, 1.0, 128, torch.float16),
    (700, 6, 6, SIGMOID, False, 3, 3, False, 1.0, 1, torch.float32),
    (1100, 45, 4, SOFTMAX, True, 9, 4, True, 1.0, 16, torch.float32),
    (400, 1000, 3, SIGMOID, True, 1, 1, True, 1.0, 1, torch.float16),
])
def test_route(handle, t, e, k, score, with_bias, groups, top_groups, renorm, scale, align, dtype):
    gen = torch.Generator().manual_seed(t + e + k)
    logits = (torch.randn(t, e, generator=gen) * 2).to(dtype)
    bias = torch.randn(e, generator=gen) * 0.1 if with_bias else None
    for pad in (0, 3):
        got = run_route(handle, logits, k, score, bias, groups, top_groups, renorm, scale, None, align, pad)
        check_route(got, logits, k, score, bias, groups, top_groups, renorm, scale, None, align)


@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_route_ties_go_to_the_lowest_expert(handle, score, with_bias, groups, top_groups):
    gen = torch.Generator().manual_seed(6)
    logits = torch.randint(-2, 3, (200, 64), generator=gen).float()
    logits[0] = 0.0
    logits[1, ::2], logits[1, 1::2] = 0.0, -0.0
    bias = torch.randint(0, 2, (64,), generator=gen).float() * 0.25 if with_bias else None
    got = run_route(handle, logits, 5, score, bias, groups, top_groups, True)
    check_route(got, logits, 5, score, bias, groups, top_groups, True, 1.0, None, 1)


@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
def test_route_decides_near_ties_as_64_bits_do(handle, score):
    """Scores closer together than f32 can tell apart, in both orders."""
    gen = torch.Generator().manual_seed(7)
    t, e = 400, 64
    logits = torch.randn(t, e, generator=gen)
    bias = torch.zeros(e)
    bias[1::2] = 2.0 ** -30   # neighbours differ by this alone
    logits[:, 1::2] = logits[:, ::2]
    got = run_route(handle, logits, 7, score, bias, 4, 2, True)
    check_route(got, logits, 7, score, bias, 4, 2, True, 1.0, None, 1)


@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_route_masks(handle, score, groups, top_groups, with_bias):
    """Rows with masked experts, down to one and none, NaN, infinities and the type's lowest value."""
    gen = torch.Generator().manual_seed(8)
    logits = torch.randn(64, 32, generator=gen)
    bias = torch.randn(32, generator=gen) * 0.1 if with_bias else None
    if with_bias:
        bias[3], bias[4] = -math.inf, math.nan
    logits[0] = -math.inf
    logits[1] = math.nan
    logits[2, 1:] = -math.inf
    logits[3, 2:] = -math.inf
    logits[4, ::2] = -math.inf
    logits[5, 5] = math.inf
    logits[6, 5:8] = math.inf
    logits[7] = -TOP
    logits[8, 4:] = -TOP
    logits[9, 7] = math.nan
    logits[10] = torch.where(torch.arange(32) % 8 == 0, logits[10], -math.inf)  # one expert in each group
    got = run_route(handle, logits, 4, score, bias, groups, top_groups, True, align=4)
    check_route(got, logits, 4, score, bias, groups, top_groups, True, 1.0, None, 4)


@pytest.mark.parametrize("many", [2, 12, 50])
def test_route_infinite_biases_come_first(handle, many):
    """Experts with a bias of +inf tie at the top, in their order."""
    gen = torch.Generator().manual_seed(many)
    logits = torch.randn(100, 64, generator=gen)
    bias = torch.randn(64, generator=gen) * 0.1
    bias[torch.randperm(64, generator=gen)[:many]] = math.inf
    got = run_route(handle, logits, 6, SIGMOID, bias, renorm=True)
    check_route(got, logits, 6, SIGMOID, bias, 1, 1, True, 1.0, None, 1)


@pytest.mark.parametrize("t,count", [(40, 0), (40, 7), (40, 400), (3000, 1234)])
def test_route_leaves_out_padded_tokens(handle, t, count):
    gen = torch.Generator().manual_seed(t + count)
    logits = torch.randn(t, 16, generator=gen)
    got = run_route(handle, logits, 2, renorm=True, count=count, align=8)
    check_route(got, logits, 2, SOFTMAX, None, 1, 1, True, 1.0, count, 8)


def test_route_without_tokens_or_plan(handle):
    got = run_route(handle, torch.empty(0, 16), 2, align=8)
    assert got["offsets"].tolist() == [0] * 17 and set(got["row_slot"].tolist()) == {-1}
    logits = torch.randn(900, 16, generator=torch.Generator().manual_seed(1))
    got = run_route(handle, logits, 3, plan=False)
    check_route(got, logits, 3, SOFTMAX, None, 1, 1, False, 1.0, None, 1)


def test_route_one_expert_takes_all(handle):
    logits = torch.zeros(1500, 40)
    logits[:, 17] = 1.0
    got = run_route(handle, logits, 1, align=128)
    check_route(got, logits, 1, SOFTMAX, None, 1, 1, False, 1.0, None, 128)


def weights_of(logits, ids, score, renorm, scale):
    """Differentiable float64 weights of a given choice."""
    s = torch.sigmoid(logits) if score == SIGMOID else torch.softmax(logits, 1)
    w = s.gather(1, ids.clamp(min=0)) * (ids >= 0)
    if renorm:
        w = w / w.sum(1, keepdim=True)
    return w * scale


@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("t,e,k,dtype", [(1, 4, 2, torch.float32), (33, 64, 4, torch.float32), (50, 100, 8, torch.bfloat16),
                                         (9, 1024, 32, torch.float16), (2500, 16, 2, torch.float32)])
def test_route_backward(handle, score, renorm, t, e, k, dtype):
    gen = torch.Generator().manual_seed(t + e)
    logits = (torch.randn(t, e, generator=gen) * 2).to(dtype)
    ids = logits.double().topk(k, 1).indices
    if t > 30:
        ids[3, 1:] = -1
        ids[4, 0] = e + 5 if not renorm else ids[4, 0]  # outside: takes no part
    dw = torch.randn(t, k, generator=gen)
    leaf = logits.double().requires_grad_()
    live = torch.where(ids < e, ids, -1)
    (weights_of(leaf, live, score, renorm, 1.5) * dw.double()).sum().backward()
    for dt in {dtype, torch.float32}:
        out = torch.full((t, e + 2), 7.0, dtype=dt, device="cuda")
        handle.moe_route_backward(t, e, k, logits.cuda(), TYPE[dtype], e, ids.int().cuda(), dw.cuda(), out, TYPE[dt], e + 2,
                                  score=score, renormalize=renorm, scale=1.5)
        torch.cuda.synchronize()
        ref = leaf.grad
        # f32 terms: a score off by the same share as in the forward pass, times the spread of dw, a sum of k terms
        size = 1.5 * dw.abs().amax(1, keepdim=True).double() * (1 + k)
        tol = 128 * 2.0 ** -24 * size * torch.softmax(leaf.detach(), 1).clamp(min=1e-3 if score == SIGMOID else 0) \
            if score == SOFTMAX and not renorm else 128 * 2.0 ** -24 * size
        half = torch.finfo(dt).eps / 2
        tiny = 2.0 ** -25 if dt == torch.float16 else 1e-40
        err = (out[:, :e].double().cpu() - ref).abs()
        assert bool((err <= tol * (1 + half) + ref.abs() * (half + 128 * 2.0 ** -24) + tiny).all())
        assert bool((out[:, e:] == 7).all())
        if renorm or score == SIGMOID:
            assert bool((out[:, :e].cpu()[ref == 0] == 0).all())  # experts that were not chosen


def test_route_backward_against_differences(handle):
    """The kernel's gradient against central differences of its own forward weights."""
    gen = torch.Generator().manual_seed(3)
    t, e, k, step = 6, 12, 3, 2.0 ** -7
    logits = torch.randn(t, e, generator=gen)
    dw = torch.randn(t, k, generator=gen)
    for score in (SOFTMAX, SIGMOID):
        for renorm in (False, True):
            base = run_route(handle, logits, k, score, renorm=renorm, plan=False)
            out = torch.empty(t, e, device="cuda")
            handle.moe_route_backward(t, e, k, logits.cuda(), gs.R_32F, e, base["ids"].cuda(), dw.cuda(), out, gs.R_32F, e,
                                      score=score, renormalize=renorm)
            grad = out.cpu().double()
            for x in range(e):
                side = []
                for sign in (1, -1):
                    moved = logits.clone()
                    moved[:, x] += sign * step
                    got = run_route(handle, moved, k, score, renorm=renorm, plan=False)
                    w = torch.zeros(t, e, dtype=torch.float64).scatter_(1, got["ids"].long(), got["weights"].double())
                    same = (got["ids"].sort(1).values == base["ids"].sort(1).values).all(1)
                    side.append(((w.gather(1, base["ids"].long()) * dw.double()).sum(1), same))
                keep = side[0][1] & side[1][1]  # rows whose choice the step left alone
                diff = (side[0][0] - side[1][0]) / (2 * step)
                # third derivatives of these weights are below 1: step^2 / 6 each of k terms; f32 weights over the step
                tol = dw.abs().sum(1).double() * (step ** 2 / 6 + 128 * 2.0 ** -24 / step)
                assert bool(((diff - grad[:, x]).abs() <= tol)[keep].all())


def make_plan(gen, t, k, align, experts=9):
    ids = torch.rand(t, experts, generator=gen).argsort(1)[:, :k] if t else torch.empty(0, k, dtype=torch.int64)
    rows = gs.moe_rows(t, experts, k, align) + 3
    _, slot_row, row_slot = plain_plan(ids, experts, align, rows)
    return torch.tensor(slot_row, dtype=torch.int32).view(t, k), torch.tensor(row_slot, dtype=torch.int32), rows


COMBINE = [(1, 1, 1, torch.float32, 0), (5, 3, 64, torch.bfloat16, 0), (33, 4, 100, torch.float16, 0),
           (64, 8, 1000, torch.bfloat16, 5), (17, 2, 4096, torch.float32, 0), (3, 8, 2056, torch.bfloat16, 8)]


@pytest.mark.parametrize("t,k,hidden,dtype,pad", COMBINE)
@pytest.mark.parametrize("weighted", [True, False])
def test_combine(handle, t, k, hidden, dtype, pad, weighted):
    gen = torch.Generator().manual_seed(hidden)
    slot_row, _, rows = make_plan(gen, t, k, 4)
    if t > 4:
        slot_row[2, 1] = -1   # a slot without a row
        slot_row[3] = -1      # a token without any
        slot_row[4, 0] = rows + 7
    y = torch.randn(rows, hidden + pad, generator=gen).to(dtype)
    y[:, hidden:] = math.nan
    w = torch.rand(t, k, generator=gen) if weighted else None
    live = (slot_row >= 0) & (slot_row < rows)
    picked = torch.where(live[:, :, None], y[:, :hidden].double()[slot_row.clamp(0, rows - 1).long()], 0.0)
    terms = picked * (w.double() if weighted else torch.ones(t, k, dtype=torch.float64))[:, :, None]
    ref, mag = terms.sum(1), terms.abs().sum(1)
    for ot in (dtype, torch.float32):
        out = torch.full((t, hidden + pad), 7.0, dtype=ot, device="cuda")
        handle.moe_combine(t, k, hidden, y.cuda(), TYPE[dtype], hidden + pad, rows, slot_row.cuda(),
                           None if w is None else w.cuda(), out, TYPE[ot], hidden + pad)
        torch.cuda.synchronize()
        tol = k * 2.0 ** -24 * mag + ref.abs() * torch.finfo(ot).eps / 2 * (1 + 1e-3) + (2.0 ** -25 if ot == torch.float16 else 0)
        assert bool(((out[:, :hidden].double().cpu() - ref).abs() <= tol).all())
        assert bool((out[:, hidden:] == 7).all())


@pytest.mark.parametrize("t,k,hidden,dtype,pad", COMBINE)
def test_combine_backward(handle, t, k, hidden, dtype, pad):
    gen = torch.Generator().manual_seed(hidden + 1)
    slot_row, row_slot, rows = make_plan(gen, t, k, 4)
    if t > 4:
        for s in (2 * k + 1, 3 * k):
            r = int(slot_row.view(-1)[s])
            slot_row.view(-1)[s], row_slot[r] = -1, -1
    y, dout = (torch.randn(n, hidden + pad, generator=gen).to(dtype) for n in (rows, t))
    w = torch.rand(t, k, generator=gen)
    dy = torch.full((rows, hidden + pad), 7.0, dtype=dtype, device="cuda")
    dw = torch.full((t, k), 7.0, device="cuda")
    handle.moe_combine_backward(t, k, hidden, y.cuda(), TYPE[dtype], hidden + pad, rows, slot_row.cuda(), row_slot.cuda(),
                                w.cuda(), dout.cuda(), TYPE[dtype], hidden + pad, dy, hidden + pad, dw)
    torch.cuda.synchronize()
    # from the forward pass by autograd in 64 bits
    ly, lw = y[:, :hidden].double().requires_grad_(), w.double().requires_grad_()
    live = slot_row >= 0
    out = (torch.where(live[:, :, None], ly[slot_row.clamp(min=0).long()], 0.0) * lw[:, :, None]).sum(1)
    (out * dout[:, :hidden].double()).sum().backward()
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0
    err = (dy[:, :hidden].double().cpu() - ly.grad).abs()
    assert bool((err <= ly.grad.abs() * (half * (1 + 1e-3) + 2.0 ** -24) + tiny).all())
    assert bool((dy[:, hidden:] == 7).all())
    mag = (torch.where(live[:, :, None], y[:, :hidden].double()[slot_row.clamp(min=0).long()], 0.0).abs() *
           dout[:, None, :hidden].double().abs()).sum(2)
    # a lane's chain of fused multiply-adds (8 of every 256 columns, rounded up), then 5 shuffles, each half a step of at
    # most the sum of magnitudes
    terms = -(-hidden // 256) * 8 + 5
    assert bool(((dw.double().cpu() - lw.grad).abs() <= terms * 2.0 ** -24 * mag).all())


def test_combine_without_tokens_or_rows(handle):
    empty = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    dy = torch.full((3, 8), 7.0, device="cuda")
    handle.moe_combine_backward(0, 2, 8, dy, gs.R_32F, 8, 3, empty, torch.full((3,), -1, dtype=torch.int32, device="cuda"),
                                None, None, gs.R_32F, 8, dy, 8, None)
    out, dw = torch.full((2, 8), 7.0, device="cuda"), torch.full((2, 2), 7.0, device="cuda")
    none = torch.full((2, 2), -1, dtype=torch.int32, device="cuda")
    handle.moe_combine(2, 2, 8, None, gs.R_32F, 8, 0, none, None, out, gs.R_32F, 8)
    handle.moe_combine_backward(2, 2, 8, None, gs.R_32F, 8, 0, none, None, dw, out, gs.R_32F, 8, None, 8, dw)
    torch.cuda.synchronize()
    assert bool((dy == 0).all()) and bool((out == 0).all()) and bool((dw == 0).all())


def reference_layer(layer, w, x, logits, dout):
    """The layer in float64 with the same choice, without any cast: values and gradients."""
    xs, ls, ws = (v.double().clone().requires_grad_() for v in (x, logits, w))
    p = weights_of(ls, layer.ids.long(), SOFTMAX, True, 1.0)
    out = sum(p[:, j, None] * torch.einsum("ti,toi->to", xs, ws[layer.ids[:, j].long()]) for j in range(layer.top_k))
    (out * dout.double()).sum().backward()
    return out.detach(), xs.grad, ls.grad, ws.grad


def off(a, b):
    return float((a.double() - b).norm() / b.norm())


def make_layer(h, tokens=200, experts=6, top_k=2, d_in=256, d_out=384, align=128, seed=21, **kw):
    gen = torch.Generator().manual_seed(seed)
    layer = RoutedExperts(h, tokens, experts, top_k, d_in, d_out, align, **kw)
    w = (torch.randn(experts, d_out, d_in, generator=gen) * d_in ** -0.5).cuda()
    layer.set_weights(w)
    x = torch.randn(tokens, d_in, generator=gen).to(torch.bfloat16).cuda()
    logits = torch.randn(tokens, experts, generator=gen).cuda()
    dout = torch.randn(tokens, d_out, generator=gen).to(torch.bfloat16).cuda()
    return layer, w, x, logits, dout


def check_layer(layer, w, x, logits, dout):
    out, dx, dl, dw = reference_layer(layer, w, x, logits, dout)
    b = layer._grad
    # Every product has two operands rounded to FP8: at most 2^-4 of a value each (E4M3), 2^-3 (E5M2), and independent
    # between terms, so the norm of a long sum is off by less than the two shares added; bf16 adds 2^-8 per store.
    assert off(layer.out, out) < 2 * 2.0 ** -4 + 2 * 2.0 ** -8
    assert off(b["dx"], dx) < 2.0 ** -4 + 2.0 ** -3 + 3 * 2.0 ** -8
    assert off(b["dw"], dw) < 2.0 ** -4 + 2.0 ** -3 + 2.0 ** -8
    assert off(b["dlogits"], dl) < 2 * 2.0 ** -4 + 2 * 2.0 ** -8


def test_a_routed_layer_and_its_gradients(handle):
    layer, w, x, logits, dout = make_layer(handle)
    layer.forward(x, logits)
    layer.backward(x, logits, dout)
    torch.cuda.synchronize()
    assert handle.device_error() == 0
    check_layer(layer, w, x, logits, dout)


def test_a_routed_layer_captured_and_replayed_on_new_inputs(cuda):
    stream = torch.cuda.Stream()
    with gs.Handle(stream) as h:
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            layer, w, x, logits, dout = make_layer(h, tokens=700)
            layer.forward(x, logits)
            layer.backward(x, logits, dout)
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            layer.forward(x, logits)
            layer.backward(x, logits, dout)
        x.copy_(x.flip(0) * 0.5)
        logits.copy_(torch.randn_like(logits))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
        torch.cuda.synchronize()
        assert h.device_error() == 0
        check_layer(layer, w, x, logits, dout)
        del g


@pytest.mark.parametrize("tokens", [1, 3])
def test_a_routed_layer_for_single_tokens(handle, tokens):
    layer, w, x, logits, dout = make_layer(handle, tokens, 16, 4, 512, 256, align=1, seed=tokens)
    layer.forward(x, logits)
    torch.cuda.synchronize()
    out, _, _, _ = reference_layer(layer, w, x, logits, dout)
    assert off(layer.out, out) < 2 * 2.0 ** -4 + 2 * 2.0 ** -8
    with pytest.raises(ValueError):
        layer.backward(x, logits, dout)  # its plan is not aligned


def test_a_routed_layer_with_a_padded_batch(handle):
    """Tokens past token_count (padding of a captured batch, here NaN) reach no expert and leave no trace in the others."""
    count = torch.tensor([150], dtype=torch.int32, device="cuda")
    layer, w, x, logits, dout = make_layer(handle, token_count=count)
    x[150:], logits[150:], dout[150:] = math.nan, math.nan, 0.0
    layer.forward(x, logits)
    layer.backward(x, logits, dout)
    torch.cuda.synchronize()
    assert bool((layer.out[150:] == 0).all()) and bool((layer._grad["dx"][150:] == 0).all())
    out, dx, _, dw = reference_layer_of(layer, w, x[:150], logits[:150], dout[:150])
    assert off(layer.out[:150], out) < 2 * 2.0 ** -4 + 2 * 2.0 ** -8
    assert off(layer._grad["dx"][:150], dx) < 2.0 ** -4 + 2.0 ** -3 + 3 * 2.0 ** -8
    assert off(layer._grad["dw"], dw) < 2.0 ** -4 + 2.0 ** -3 + 2.0 ** -8


def reference_layer_of(layer, w, x, logits, dout):
    class Part:
        ids, top_k = layer.ids[:x.shape[0]], layer.top_k

    return reference_layer(Part, w, x, logits, dout)


def test_two_layers_on_two_streams_at_once(cuda):
    """An instance and a handle to each stream, sharing the weight blocks."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    with gs.Handle(streams[0]) as h0, gs.Handle(streams[1]) as h1:
        with torch.cuda.stream(streams[0]):
            layer, w, x, logits, dout = make_layer(h0, tokens=900)
        torch.cuda.synchronize()
        other = RoutedExperts(h1, 900, 6, 2, 256, 384, weights_of=layer)
        for _ in range(3):
            for l, s in ((layer, streams[0]), (other, streams[1])):
                with torch.cuda.stream(s):
                    l.forward(x, logits)
                    l.backward(x, logits, dout)
        torch.cuda.synchronize()
        check_layer(layer, w, x, logits, dout)
        for name in ("dx", "dlogits", "dw"):
            assert torch.equal(layer._grad[name], other._grad[name])
        assert torch.equal(layer.out, other.out)
