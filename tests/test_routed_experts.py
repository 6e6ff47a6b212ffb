"""CPU tests of RoutedExperts' own part: where its buffers are, what it hands to the library and what it refuses. The
handle is a stand-in that records the calls; nothing is launched."""
import pytest
import torch

import gemm_sm100 as gs
from routed_experts import RoutedExperts


class FakeHandle:
    device = "cpu"
    stream = 0

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args, **kw: self.calls.append((name, args, kw))


def layer(handle=None, tokens=5, experts=4, top_k=2, d_in=32, d_out=48, **kw):
    return RoutedExperts(handle or FakeHandle(), tokens, experts, top_k, d_in, d_out, **kw)


def tensors(obj):
    for v in vars(obj).values():
        if isinstance(v, torch.Tensor):
            yield v
        elif isinstance(v, dict):
            yield from (t for t in v.values() if isinstance(t, torch.Tensor))


def test_buffers_are_on_the_handles_device():
    """Not on the current device, which may be another by now."""
    l = layer()
    l.prepare_backward()
    assert {t.device for t in tensors(l)} == {torch.device("cpu")}


@pytest.mark.gpu
def test_a_handle_names_its_device(cuda):
    with gs.Handle() as h:
        assert h.device == "cuda:0"
        l = layer(h)
        assert {t.device for t in tensors(l)} == {torch.device("cuda", 0)}


def inputs(tokens=5, experts=4, d_in=32, d_out=48):
    return (torch.zeros(tokens, d_in, dtype=torch.bfloat16), torch.zeros(tokens, experts),
            torch.zeros(tokens, d_out, dtype=torch.bfloat16))


X = {
    "f32": lambda x: x.float(), "f16": lambda x: x.half(), "short": lambda x: x[:4], "long": lambda x: torch.cat([x, x]),
    "narrow": lambda x: x[:, :-1], "flat": lambda x: x.reshape(-1), "transposed": lambda x: x.t().contiguous().t(),
    "expanded": lambda x: x[:1].expand_as(x), "every second column": lambda x: torch.cat([x, x], 1)[:, ::2],
    "overlapping rows": lambda x: torch.as_strided(x, x.shape, (1, 1)), "another device": lambda x: x.to("meta"),
    "none": lambda x: None, "nested list": lambda x: x.tolist(),
}


@pytest.mark.parametrize("change", [k for k in X])
@pytest.mark.parametrize("which", ["x", "logits", "dout"])
def test_inputs_that_the_kernels_would_read_wrongly_are_refused(which, change):
    h = FakeHandle()
    l = layer(h)
    good = dict(zip(("x", "logits", "dout"), inputs()))
    l.forward(good["x"], good["logits"])
    l.backward(**good)
    if which == "logits" and change == "f32":
        change = "f16"
    bad = dict(good, **{which: X[change](good[which])})
    h.calls.clear()
    if which != "dout":
        with pytest.raises(ValueError, match=which):
            l.forward(bad["x"], bad["logits"])
    with pytest.raises(ValueError, match=which):
        l.backward(**bad)
    assert not h.calls  # refused before anything is launched


def test_rows_may_lie_apart():
    """A slice of a wider tensor: its leading dimension reaches the library."""
    h = FakeHandle()
    l = layer(h)
    wide = [torch.zeros(5, n, dtype=t)[:, 8:] for n, t in ((32 + 8, torch.bfloat16), (4 + 8, torch.float32), (48 + 8, torch.bfloat16))]
    l.forward(*wide[:2])
    l.backward(*wide)
    calls = {}
    for name, args, _ in h.calls:
        calls.setdefault(name, []).append(args)
    for args in calls["moe_route"] + calls["moe_route_backward"]:
        assert args[3] is wide[1] and args[5] == 12
    casts = [args for args in calls["fp8_quantize"] if args[4] is wide[0]]
    assert len(casts) == 2 and all(args[6] == 40 for args in casts)
    (args,) = calls["moe_combine_backward"]
    assert args[10] is wide[2] and args[12] == 56


def test_rows_may_have_more_than_one_axis():
    """[batch, sequence, features] without a gap is as many rows."""
    l = layer(tokens=6)
    x, logits, dout = (t.view(2, 3, -1) for t in inputs(6))
    l.forward(x, logits)
    l.backward(x, logits, dout)
    assert [args[5] for name, args, _ in l.h.calls if name == "moe_route"] == [4]
    with pytest.raises(ValueError, match="x"):
        l.forward(torch.cat([x, x], 2)[..., :32], logits)


def test_one_token_may_have_any_row_stride():
    l = layer(tokens=1)
    x, logits, dout = (torch.as_strided(t, t.shape, (1, 1)) for t in inputs(1))
    l.forward(x, logits)
    l.backward(x, logits, dout)
    assert [args[5] for name, args, _ in l.h.calls if name == "moe_route"] == [4]


@pytest.mark.gpu
def test_slices_of_wider_tensors_give_the_same_results(cuda):
    gen = torch.Generator().manual_seed(4)
    x, logits, dout = (torch.randn(150, n, generator=gen).to(t).cuda()
                       for n, t in ((256, torch.bfloat16), (6, torch.float32), (384, torch.bfloat16)))
    with gs.Handle() as h:
        l = layer(h, 150, 6, 2, 256, 384)
        l.set_weights(torch.randn(6, 384, 256, generator=gen).cuda())

        def outputs(*args):
            out = l.forward(*args[:2]).clone()
            grads = [g.clone() for g in l.backward(*args)]
            torch.cuda.synchronize()
            assert h.device_error() == 0
            return [out, *grads]

        whole = outputs(x, logits, dout)
        for left, right in ((8, 8), (3, 2)):  # 16-byte aligned rows, and odd ones
            wide = [torch.cat([t.new_full((150, left), 7), t, t.new_full((150, right), 7)], 1)[:, left:-right] for t in (x, logits, dout)]
            for a, b in zip(whole, outputs(*wide)):
                assert torch.equal(a, b)


W = {
    "f64": lambda w: w.double(), "fp8": lambda w: w.to(torch.float8_e4m3fn), "transposed": lambda w: w.transpose(1, 2).contiguous().transpose(1, 2),
    "[in, out]": lambda w: w.transpose(1, 2), "short": lambda w: w[:3], "long": lambda w: torch.cat([w, w]),
    "wide": lambda w: torch.cat([w, w], 2), "expanded rows": lambda w: w[:, :1].expand_as(w), "flat": lambda w: w.reshape(-1),
    "another device": lambda w: w.to("meta"), "list": lambda w: list(w),
}


@pytest.mark.parametrize("change", [k for k in W])
def test_weights_that_would_be_read_wrongly_are_refused(change):
    l = layer()
    with pytest.raises(ValueError, match="w"):
        l.set_weights(W[change](torch.zeros(4, 48, 32)))
    assert not l.h.calls


@pytest.mark.parametrize("dtype,code", [(torch.float32, gs.R_32F), (torch.float16, gs.R_16F), (torch.bfloat16, gs.R_16BF)])
def test_weights_may_lie_apart(dtype, code):
    l = layer()
    w = torch.zeros(8, 50, 40, dtype=dtype)[::2, 1:49, 8:]
    l.set_weights(w)
    assert [(args[4].data_ptr(), args[5], args[6]) for _, args, _ in l.h.calls] == [(w[e].data_ptr(), code, 40) for e in range(4)]


@pytest.mark.parametrize("sizes", [dict(experts=5), dict(d_in=48), dict(d_out=32)])
def test_weights_of_another_size_are_refused(sizes):
    other = layer(**sizes)
    with pytest.raises(ValueError, match="weights_of"):
        layer(weights_of=other)


def test_weights_of_another_device_are_refused():
    class Elsewhere(FakeHandle):
        device = "meta"

    with pytest.raises(ValueError, match="weights_of"):
        layer(weights_of=layer(Elsewhere()))


def test_weights_can_be_shared_by_layers_of_other_batches():
    first = layer()
    second = layer(tokens=9, top_k=1, align=1, weights_of=first)
    assert second.wq is first.wq and second.w_scale is first.w_scale


@pytest.mark.parametrize("name,value", [
    ("bias", torch.zeros(5)), ("bias", torch.zeros(4, dtype=torch.bfloat16)), ("bias", torch.zeros(8)[::2]),
    ("bias", torch.zeros(4, 2)), ("bias", torch.zeros(4, device="meta")), ("bias", [0.0] * 4),
    ("token_count", torch.tensor([3])), ("token_count", torch.tensor([3.0])), ("token_count", torch.tensor([], dtype=torch.int32)),
    ("token_count", torch.tensor([3, 4], dtype=torch.int32)), ("token_count", torch.tensor([3], dtype=torch.int32, device="meta")),
    ("token_count", 3),
])
def test_routing_tensors_that_would_be_read_wrongly_are_refused(name, value):
    with pytest.raises(ValueError, match=name):
        layer(**{name: value})


def test_routing_tensors_that_fit():
    layer(bias=torch.zeros(4), token_count=torch.tensor([3], dtype=torch.int32))
    layer(bias=torch.zeros(1, 4), token_count=torch.tensor(3, dtype=torch.int32))


@pytest.mark.parametrize("sizes", [dict(tokens=0), dict(tokens=-1), dict(d_in=0), dict(d_out=-16), dict(d_in=24), dict(d_out=40)])
def test_sizes_that_no_call_takes_are_refused(sizes):
    with pytest.raises(ValueError):
        layer(**sizes)


def test_backward_needs_a_forward():
    l = layer()
    x, logits, dout = inputs()
    with pytest.raises(RuntimeError, match="forward"):
        l.backward(x, logits, dout)
    assert not l.h.calls
    with pytest.raises(ValueError):
        layer(align=1).backward(x, logits, dout)  # the plan can never serve one


def test_nothing_is_allocated_after_prepare_backward(monkeypatch):
    l = layer()
    l.prepare_backward()
    buffers = [t.data_ptr() for t in tensors(l)]

    def never(*args, **kw):
        raise AssertionError("allocated")

    for name in ("empty", "zeros", "empty_like", "zeros_like", "full", "tensor"):
        monkeypatch.setattr(torch, name, never)
    x, logits, dout = (t.clone() for t in inputs_made_before)
    l.forward(x, logits)
    l.backward(x, logits, dout)
    l.prepare_backward()
    assert buffers == [t.data_ptr() for t in tensors(l)]


inputs_made_before = inputs()


def test_no_buffer_is_filled():
    """A fill would run on torch's stream, and the layer's kernels on the handle's."""
    seen = []

    class Fills(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(getattr(func, "__name__", str(func)))
            return func(*args, **(kwargs or {}))

    with Fills():
        layer().prepare_backward()
    assert not [n for n in seen if "zero" in n or "fill" in n or "full" in n or "ones" in n], seen


@pytest.mark.gpu
def test_a_layer_made_on_another_stream_than_its_handles(cuda):
    """Its memory was used by work that is still under way on torch's stream; the layer waits for that once."""
    gen = torch.Generator().manual_seed(5)
    x, logits, dout = (torch.randn(300, n, generator=gen).to(t).cuda()
                       for n, t in ((256, torch.bfloat16), (6, torch.float32), (384, torch.bfloat16)))
    w = torch.randn(6, 384, 256, generator=gen).cuda()
    torch.cuda.synchronize()

    def outputs(h):
        l = layer(h, 300, 6, 2, 256, 384)
        l.set_weights(w)
        out = l.forward(x, logits)
        grads = l.backward(x, logits, dout)
        torch.cuda.synchronize()
        assert h.device_error() == 0
        return [t.clone() for t in (out, *grads)]

    with gs.Handle() as h:
        want = outputs(h)
    with gs.Handle(torch.cuda.Stream()) as h:
        for _ in range(5):
            junk = [torch.full((3, 2 ** 20), 1e9, device="cuda") for _ in range(8)]
            for _ in range(20):
                for t in junk:
                    t.mul_(1.000001)  # keeps torch's stream busy while the memory changes hands
            del junk, t
            for a, b in zip(want, outputs(h)):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_first_backward_under_capture(cuda):
    """With prepare_backward, and without: the buffers are then the graph's memory."""
    gen = torch.Generator().manual_seed(6)
    x, logits, dout = (torch.randn(300, n, generator=gen).to(t).cuda()
                       for n, t in ((256, torch.bfloat16), (6, torch.float32), (384, torch.bfloat16)))
    w = torch.randn(6, 384, 256, generator=gen).cuda()
    torch.cuda.synchronize()
    stream, results = torch.cuda.Stream(), []
    with gs.Handle(stream) as h:
        for prepare in (True, False):
            with torch.cuda.stream(stream):
                l = layer(h, 300, 6, 2, 256, 384)
                l.set_weights(w)
                l.forward(x, logits)  # the kernels are loaded before the capture
                if prepare:
                    l.prepare_backward()
            stream.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                l.forward(x, logits)
                l.backward(x, logits, dout)
            with torch.cuda.stream(stream):
                for _ in range(3):
                    g.replay()
            torch.cuda.synchronize()
            assert h.device_error() == 0
            results.append([t.clone() for t in (l.out, *(l._grad[n] for n in ("dx", "dlogits", "dw")))])
            del l, g
    for a, b in zip(*results):
        assert torch.equal(a, b)
