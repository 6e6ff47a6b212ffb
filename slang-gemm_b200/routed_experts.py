"""A routed FP8 expert layer on the library's calls, with its gradients.

    y[t] = sum over the top_k experts e chosen for token t of p[t, e] * W_e x[t]

`RoutedExperts` holds what a program keeps between steps: the experts' weights as
FP8 blocks, the plan's index arrays and the buffers of the products. `forward` is
moe_route -> fp8_quantize (gathering the tokens into expert order) ->
gemm_fp8_grouped -> moe_combine; `backward` runs their gradients: the input
gradient is the grouped product with the same weight blocks read the other way,
the weight gradient the grouped product over each expert's tokens, both operands
cast in vectors along the tokens.

The buffers are made by the constructor and, the gradients' larger ones, by
`prepare_backward` (or else the first backward): torch allocates them, and where
torch's current stream is not the handle's, the call waits for that stream, which
may still use the memory. After that nothing synchronises or allocates, so both
directions can be captured into a CUDA graph.

All kernels run on the handle's stream: the caller orders the inputs' making before
them and the outputs' use, or the layer's end, after them. An instance serves one
stream at a time; concurrent use needs an instance each (the weight blocks can be
shared by passing `weights_of`).
"""
from __future__ import annotations

import torch

import gemm_sm100 as gs


def _blocks(n: int) -> int:
    return (n + 127) // 128


def _rows(name, t, dtype, rows, cols, device):
    """The leading dimension of t, a rows x cols matrix as the kernels read it (or a contiguous [..., cols] of as many rows);
    ValueError if it is another. Looks at no value, so it may run under capture."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {dtype} [{rows}, {cols}] on {device}, not {_describe(t)}")
    if t.shape != (rows, cols):
        if t.dim() > 2 and t.shape[-1] == cols and t.numel() == rows * cols and t.is_contiguous():
            return cols
        raise ValueError(f"{name} must be {dtype} [{rows}, {cols}] on {device}, not {_describe(t)}")
    ld, step = t.stride()
    if (step != 1 and cols > 1) or (ld < cols and rows > 1):
        raise ValueError(f"{name}'s rows must be contiguous and must not overlap; its strides are {t.stride()}")
    return ld if rows > 1 else cols


def _describe(t) -> str:
    return f"{t.dtype} {list(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__


def _vector(name, t, dtype, n, device):
    """ValueError unless t is None or n contiguous elements."""
    if t is not None and not (isinstance(t, torch.Tensor) and t.dtype == dtype and t.numel() == n and t.device == device and
                              t.is_contiguous()):
        raise ValueError(f"{name} must be {dtype} [{n}] on {device}, contiguous, not {_describe(t)}")


class RoutedExperts:
    """tokens, experts, top_k: the routing's sizes; d_in, d_out: the experts' (multiples of 16). align 128 is what the
    weight gradient needs; 1 wastes no rows and is for serving (no backward). score, bias, groups, top_groups and scale
    are moe_route's. The buffers are on the handle's device."""

    def __init__(self, handle, tokens, experts, top_k, d_in, d_out, align=128, score=gs.ROUTE_SOFTMAX, bias=None,
                 groups=1, top_groups=1, renormalize=True, scale=1.0, token_count=None, weights_of=None):
        if tokens < 1 or d_in < 1 or d_out < 1:
            raise ValueError("tokens, d_in and d_out must be positive")
        if d_in % 16 or d_out % 16:
            raise ValueError("d_in and d_out must be multiples of 16 (16-byte aligned FP8 rows)")
        self.h, self.tokens, self.experts, self.top_k = handle, tokens, experts, top_k
        self.d_in, self.d_out, self.align = d_in, d_out, align
        self.routing = dict(bias=bias, score=score, groups=groups, top_groups=top_groups, renormalize=renormalize,
                            scale=scale, token_count=token_count)
        self.rows = rows = gs.moe_rows(tokens, experts, top_k, align)
        self.device = torch.device(handle.device)
        _vector("bias", bias, torch.float32, experts, self.device)
        _vector("token_count", token_count, torch.int32, 1, self.device)
        i32, u8, f32, bf16 = (dict(dtype=t, device=self.device)
                              for t in (torch.int32, torch.uint8, torch.float32, torch.bfloat16))
        self.ids, self.p = torch.empty(tokens, top_k, **i32), torch.empty(tokens, top_k, **f32)
        self.slot_row, self.row_slot = torch.empty(tokens, top_k, **i32), torch.empty(rows, **i32)
        self.offsets = torch.empty(experts + 1, **i32)
        self._ws_bytes = gs.moe_route_workspace(tokens, experts, top_k)
        self._ws = torch.empty(max(self._ws_bytes, 4), **u8)
        ki, ko = _blocks(d_in), _blocks(d_out)
        if weights_of is not None and ((weights_of.experts, weights_of.d_in, weights_of.d_out, weights_of.device) !=
                                       (experts, d_in, d_out, self.device)):
            raise ValueError("weights_of must be a layer with the same experts, d_in and d_out on the same device")
        if weights_of is None:
            self.wq, self.w_scale = torch.empty(experts, d_out, d_in, **u8), torch.empty(experts, ko, ki, **f32)
        else:
            self.wq, self.w_scale = weights_of.wq, weights_of.w_scale
        self.xq, self.x_scale = torch.empty(rows, d_in, **u8), torch.empty(ki, rows, **f32)
        self.y = torch.empty(rows, d_out, **bf16)  # rows behind the last expert's are neither written nor read
        self.out = torch.empty(tokens, d_out, **bf16)
        self._grad = None
        self._ran = False
        self._settle()

    def _settle(self):
        """New memory may still be in use on the stream it was allocated on; the kernels that write it are on the handle's."""
        if self.device.type != "cuda" or torch.cuda.is_current_stream_capturing():
            return
        current = torch.cuda.current_stream(self.device)
        if current.cuda_stream != self.h.stream:
            current.synchronize()

    def prepare_backward(self):
        """Makes the gradients' buffers, if they are not there: to be called before a capture, or a time that counts."""
        if self.align % 128:
            raise ValueError("backward needs a plan aligned to 128 rows")
        if self._grad is None:
            f32, u8, bf16 = (dict(dtype=t, device=self.device) for t in (torch.float32, torch.uint8, torch.bfloat16))
            r, rb = self.rows, _blocks(self.rows)
            self._grad = dict(
                dy=torch.empty_like(self.y), dp=torch.empty_like(self.p),
                dlogits=torch.empty(self.tokens, self.experts, **f32),
                gq=torch.empty(r, self.d_out, **u8), g_scale=torch.empty(_blocks(self.d_out), r, **f32),
                gtq=torch.empty(r, self.d_out, **u8), gt_scale=torch.empty(rb, self.d_out, **f32),
                xtq=torch.empty(r, self.d_in, **u8), xt_scale=torch.empty(rb, self.d_in, **f32),
                dx_rows=torch.empty(r, self.d_in, **bf16), dx=torch.empty(self.tokens, self.d_in, **bf16),
                dw=torch.empty(self.experts, self.d_out, self.d_in, **f32))
            self._settle()

    def set_weights(self, w):
        """w: [experts, d_out, d_in] f32, f16 or bf16 with contiguous rows (which may lie apart); cast to FP8 blocks."""
        types = {torch.float32: gs.R_32F, torch.float16: gs.R_16F, torch.bfloat16: gs.R_16BF}
        if (not isinstance(w, torch.Tensor) or w.dtype not in types or w.shape != (self.experts, self.d_out, self.d_in) or
                w.device != self.device):
            raise ValueError(f"w must be f32, f16 or bf16 [{self.experts}, {self.d_out}, {self.d_in}] on {self.device}, "
                             f"not {_describe(w)}")
        if w.stride(2) != 1 or w.stride(1) < self.d_in:
            raise ValueError(f"w's rows must be contiguous and must not overlap; its strides are {w.stride()}")
        wt = types[w.dtype]
        for e in range(self.experts):
            self.h.fp8_quantize(gs.SCALE_BLK128, 0, self.d_in, self.d_out, w[e], wt, w.stride(1), self.wq[e],
                                gs.R_8F_E4M3, self.d_in, self.w_scale[e], _blocks(self.d_in))

    def forward(self, x, logits):
        """x: [tokens, d_in] bf16, logits: [tokens, experts] f32, each with contiguous rows (which may lie apart); a batch of
        fewer tokens is padded to `tokens` rows and counted by token_count. Returns out [tokens, d_out] bf16 (the layer's
        buffer)."""
        h, i, o, rows = self.h, self.d_in, self.d_out, self.rows
        ldx = _rows("x", x, torch.bfloat16, self.tokens, i, self.device)
        ldl = _rows("logits", logits, torch.float32, self.tokens, self.experts, self.device)
        h.moe_route(self.tokens, self.experts, self.top_k, logits, gs.R_32F, ldl, self.ids, self.p,
                    align=self.align, offsets=self.offsets, slot_row=self.slot_row, row_slot=self.row_slot, rows=rows,
                    workspace=self._ws, workspace_bytes=self._ws_bytes, **self.routing)
        h.fp8_quantize(gs.SCALE_VEC128, 0, i, rows, x, gs.R_16BF, ldx, self.xq, gs.R_8F_E4M3, i, self.x_scale, rows,
                       index=self.row_slot, index_div=self.top_k, src_cols=self.tokens)
        h.gemm_fp8_grouped(gs.GROUP_N, gs.OP_T, gs.OP_N, o, rows, i, self.experts, self.offsets, 1.0, self.wq,
                           gs.R_8F_E4M3, i, o * i, self.w_scale, gs.SCALE_BLK128, _blocks(i), _blocks(i) * _blocks(o),
                           self.xq, gs.R_8F_E4M3, i, self.x_scale, gs.SCALE_VEC128, rows, 0.0, self.y, gs.R_16BF, o, 0)
        h.moe_combine(self.tokens, self.top_k, o, self.y, gs.R_16BF, o, rows, self.slot_row, self.p, self.out,
                      gs.R_16BF, o)
        self._ran = True
        return self.out

    def backward(self, x, logits, dout):
        """Gradients of the last forward, for its x and logits and dout [tokens, d_out] bf16: dx [tokens, d_in] bf16, dlogits
        f32, dw [experts, d_out, d_in] f32 (buffers of the layer)."""
        h, i, o, rows = self.h, self.d_in, self.d_out, self.rows
        ldx = _rows("x", x, torch.bfloat16, self.tokens, i, self.device)
        ldl = _rows("logits", logits, torch.float32, self.tokens, self.experts, self.device)
        ldg = _rows("dout", dout, torch.bfloat16, self.tokens, o, self.device)
        self.prepare_backward()
        if not self._ran:
            raise RuntimeError("backward without a forward: the choice and the experts' outputs are its")
        b = self._grad
        h.moe_combine_backward(self.tokens, self.top_k, o, self.y, gs.R_16BF, o, rows, self.slot_row, self.row_slot,
                               self.p, dout, gs.R_16BF, ldg, b["dy"], o, b["dp"])
        h.moe_route_backward(self.tokens, self.experts, self.top_k, logits, gs.R_32F, ldl, self.ids, b["dp"],
                             b["dlogits"], gs.R_32F, self.experts, score=self.routing["score"],
                             renormalize=self.routing["renormalize"], scale=self.routing["scale"])
        h.fp8_quantize(gs.SCALE_VEC128, 0, o, rows, b["dy"], gs.R_16BF, o, b["gq"], gs.R_8F_E5M2, o, b["g_scale"], rows)
        h.fp8_quantize(gs.SCALE_VEC128, 1, o, rows, b["dy"], gs.R_16BF, o, b["gtq"], gs.R_8F_E5M2, o, b["gt_scale"], o)
        h.fp8_quantize(gs.SCALE_VEC128, 1, i, rows, x, gs.R_16BF, ldx, b["xtq"], gs.R_8F_E4M3, i, b["xt_scale"], i,
                       index=self.row_slot, index_div=self.top_k, src_cols=self.tokens)
        h.gemm_fp8_grouped(gs.GROUP_N, gs.OP_N, gs.OP_N, i, rows, o, self.experts, self.offsets, 1.0, self.wq,
                           gs.R_8F_E4M3, i, o * i, self.w_scale, gs.SCALE_BLK128, _blocks(i), _blocks(i) * _blocks(o),
                           b["gq"], gs.R_8F_E5M2, o, b["g_scale"], gs.SCALE_VEC128, rows, 0.0, b["dx_rows"], gs.R_16BF,
                           i, 0)
        h.moe_combine(self.tokens, self.top_k, i, b["dx_rows"], gs.R_16BF, i, rows, self.slot_row, None, b["dx"],
                      gs.R_16BF, i)
        h.gemm_fp8_grouped(gs.GROUP_K, gs.OP_N, gs.OP_T, i, o, rows, self.experts, self.offsets, 1.0, b["xtq"],
                           gs.R_8F_E4M3, i, 0, b["xt_scale"], gs.SCALE_VEC128, i, 0, b["gtq"], gs.R_8F_E5M2, o,
                           b["gt_scale"], gs.SCALE_VEC128, o, 0.0, b["dw"], gs.R_32F, i, o * i)
        return b["dx"], b["dlogits"], b["dw"]
