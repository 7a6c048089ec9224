"""RMSNorm with optional fused residual add: h = x + res; y = h * rsqrt(mean(h²)+eps) * w. And the norms behind and
in front of a block in one kernel, with the block's gate and a scaled residual (`sandwich_norm`).

Reference counterpart: HF RMSNorm modules and TE `LayerNormLinear(normalization="RMSNorm")`
(dllm_parallel/core/models/backbones/nemotron/model.py:3866-3960).
"""
from __future__ import annotations

import torch

from ..kernels import native
from ._util import (MAX_ROWS, dtype_code, grad_sink, mark_grad_written, on_device, ptr, refuse_tangents, refuse_twice, scratch,
                    stream, stream_of, use_native)


native.register_signatures({
    "tdllm_sandwich_norm_fwd": (native.c_int, [native.c_void_p] * 8 + [native.c_ll] * 3 + [native.c_int] * 4
                                + [native.c_float] * 2 + [native.c_void_p]),
    "tdllm_sandwich_norm_parts": (native.c_int, [native.c_int] * 2),
    "tdllm_sandwich_norm_bwd": (native.c_int, [native.c_void_p] * 14 + [native.c_int] * 6 + [native.c_void_p]
                                + [native.c_ll] * 3 + [native.c_int] * 4 + [native.c_float, native.c_void_p]),
})

SANDWICH_MAX_WIDTH = 16384


def rmsnorm_reference(x, w, eps, res=None):
    h = x if res is None else x + res
    hf = h.float()
    rstd = torch.rsqrt(hf.pow(2).mean(-1, keepdim=True) + eps)
    return (hf * rstd * w.float()).to(x.dtype), h


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, res, w, eps):
        H = x.shape[-1]
        x2 = x.reshape(-1, H)
        rows = x2.shape[0]
        has_res = res is not None
        y = torch.empty_like(x2)
        h = torch.empty_like(x2) if has_res else x2
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        native.check(native.lib().tdllm_rmsnorm_fwd(
            ptr(x2), ptr(res.reshape(-1, H)) if has_res else None, ptr(w), ptr(y),
            ptr(h) if has_res else None, ptr(rstd), rows, H, eps, stream()), "rmsnorm_fwd")
        ctx.save_for_backward(h, w, rstd)
        ctx.wref = w
        ctx.has_res = has_res
        ctx.shape = x.shape
        if has_res:
            return (y, h) if x.dim() == 2 else (y.view(x.shape), h.view(x.shape))
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy, dh=None):
        h, w, rstd = ctx.saved_tensors
        rows, H = h.shape
        dy2 = dy.contiguous().reshape(rows, H)
        # gradient flowing into the residual stream output (h) adds to dx
        dres = dh.contiguous().reshape(rows, H) if dh is not None else None
        dx = torch.empty_like(h)
        parts = native.lib().tdllm_rmsnorm_bwd_parts()
        scr = scratch(h.device, parts * H)
        sink, acc = grad_sink(ctx.wref)
        if sink is None:
            dw = torch.empty_like(w)
            target, tfp32, tacc = dw, False, False
        else:
            dw = None
            target, tfp32, tacc = sink, sink.dtype == torch.float32, acc
        native.check(native.lib().tdllm_rmsnorm_bwd(
            ptr(dy2), ptr(h), ptr(w), ptr(rstd), ptr(dres), ptr(dx), ptr(target), int(tfp32),
            int(tacc), ptr(scr), rows, H, stream()), "rmsnorm_bwd")
        if sink is not None:
            mark_grad_written(ctx.wref)
        dx = dx.view(ctx.shape)
        return dx, (dx if ctx.has_res else None), dw, None


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float = 1e-6,
            res: torch.Tensor | None = None):
    """Returns (y, h) where h = x + res is the updated residual stream (h is x when res is None)."""
    if not use_native(x):
        return rmsnorm_reference(x, w, eps, res)
    if res is None:
        return _RMSNorm.apply(x, None, w, eps), x
    y, h = _RMSNorm.apply(x, res, w, eps)
    return y, h


def sandwich_norm_reference(x, res, w_post, w_pre, gate=None, res_scale: float = 1.0, eps: float = 1e-6):
    """(y, h) of `sandwich_norm` in fp32 (64 bits for double inputs), each rounded once; y is formed from the unrounded h."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    xf = x.to(wide)
    b = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w_post.to(wide)
    if gate is not None:
        b = b * gate.to(wide)
    h = res_scale * res.to(wide) + b
    y = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + eps) * w_pre.to(wide)
    return y.to(x.dtype), h.to(x.dtype)


GATE_NONE, GATE_CHANNEL, GATE_FULL = 0, 1, 2
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _rows2d(t: torch.Tensor) -> torch.Tensor:
    """[rows, H] with unit inner stride, rows that start on 16 bytes and lie H values plus whole 16 bytes apart: what the
    kernels ask of every row operand. A view where the tensor is like that, else a copy."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.is_contiguous():
        return t if t.data_ptr() % 16 == 0 else t.clone()
    H = t.shape[1]
    if (t.stride(1) == 1 or H == 1) and t.data_ptr() % 16 == 0 and (t.stride(0) - H) * t.element_size() % 16 == 0 \
            and (t.stride(0) >= H or H * t.element_size() % 16 == 0):      # (rows that overlap have no line of their own)
        return t
    return t.contiguous()


def _sandwich_forward(x, res, w_post, w_pre, gate, res_scale, eps, want_stats):
    kind = GATE_NONE if gate is None else GATE_CHANNEL if gate.dim() == 1 else GATE_FULL
    rows, H = x.shape
    dtype, dev = x.dtype, x.device
    y, h = torch.empty((rows, H), dtype=dtype, device=dev), torch.empty((rows, H), dtype=dtype, device=dev)
    stats = torch.empty((2, rows), dtype=torch.float32, device=dev) if want_stats else None
    with on_device(x):
        native.check(native.lib().tdllm_sandwich_norm_fwd(
            x.data_ptr(), res.data_ptr(), w_post.data_ptr(), w_pre.data_ptr(), ptr(gate), y.data_ptr(), h.data_ptr(), ptr(stats),
            _row_stride(x), _row_stride(res), _row_stride(gate) if kind == GATE_FULL else H, rows, H, kind, _DTYPES[dtype],
            res_scale, eps, stream_of(x)), "sandwich_norm_fwd")
    return y, h, stats


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]      # (a single row's stride may be anything)


def _packed(t: torch.Tensor, rows: int, H: int) -> torch.Tensor:
    if t.dim() != 2:
        t = t.reshape(rows, H)
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _SandwichNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, res, w_post, w_pre, gate, res_scale, eps):
        x2, res2 = _rows2d(x), _rows2d(res)
        gate2 = gate if gate is None or gate.dim() == 1 else _rows2d(gate)
        y, h, stats = _sandwich_forward(x2, res2, w_post, w_pre, gate2, res_scale, eps, True)
        ctx.save_for_backward(x2, res2, w_post, w_pre, gate2, stats)
        ctx.refs = (w_post, w_pre, gate if gate is not None and gate.dim() == 1 else None)
        ctx.meta = (res_scale, x.shape)
        ctx.set_materialize_grads(False)
        return (y, h) if x.dim() == 2 else (y.view(x.shape), h.view(x.shape))

    @staticmethod
    def backward(ctx, dy, dh):
        refuse_twice("sandwich_norm")
        x, res, w_post, w_pre, gate, stats = ctx.saved_tensors
        res_scale, shape = ctx.meta
        rows, H = x.shape
        kind = GATE_NONE if gate is None else GATE_CHANNEL if gate.dim() == 1 else GATE_FULL
        dy = None if dy is None else _packed(dy, rows, H)
        dh = None if dh is None else _packed(dh, rows, H)
        dtype, dev = x.dtype, x.device
        dx, dres = torch.empty((rows, H), dtype=dtype, device=dev), torch.empty((rows, H), dtype=dtype, device=dev)
        dgate = torch.empty((rows, H), dtype=dtype, device=dev) if kind == GATE_FULL else None
        # vectors that own a slice of the flat gradient buffer are written (or added) there, the others are returned
        targets, flags, returned, written, again = [], [], [], [], []
        for vec, ref, need in zip((w_post, w_pre, gate if kind == GATE_CHANNEL else None), ctx.refs, ctx.needs_input_grad[2:5]):
            sink, acc = (None, False) if vec is None or not need else grad_sink(ref)
            if sink is not None and sink.dtype not in (torch.float32, x.dtype):
                raise native.NativeKernelError(f"gradient buffer of {sink.dtype} for a {x.dtype} parameter")
            if sink is not None and any(ref is r for r in written):   # one parameter in two places: added behind the kernel
                again.append((sink, torch.empty_like(sink)))
                sink, acc = again[-1][1], False
            grad = torch.empty_like(vec) if vec is not None and need and sink is None else None
            to = sink if sink is not None else grad
            targets.append(to)
            flags += [int(to is not None and to.dtype == torch.float32), int(acc)]
            returned.append(grad)
            if sink is not None:
                written.append(ref)
        with on_device(x):
            lib = native.lib()
            # (allocated per call: streams and captured graphs do not share it)
            part = torch.empty((lib.tdllm_sandwich_norm_parts(rows, H) * 2 * H,), dtype=torch.float32, device=dev)
            native.check(lib.tdllm_sandwich_norm_bwd(
                x.data_ptr(), res.data_ptr(), w_post.data_ptr(), w_pre.data_ptr(), ptr(gate), ptr(dy), ptr(dh),
                stats.data_ptr(), dx.data_ptr(), dres.data_ptr(), ptr(dgate), *(ptr(t) for t in targets), *flags, ptr(part),
                _row_stride(x), _row_stride(res), _row_stride(gate) if kind == GATE_FULL else H, rows, H, kind, _DTYPES[dtype], res_scale, stream_of(x)),
                "sandwich_norm_bwd")
        for sink, more in again:
            sink.add_(more)
        for ref in written:
            mark_grad_written(ref)
        if kind != GATE_FULL:
            dgate = returned[2]
        if len(shape) != 2:
            dx, dres = dx.view(shape), dres.view(shape)
            dgate = dgate.view(shape) if kind == GATE_FULL else dgate
        return dx, dres, returned[0], returned[1], dgate, None, None


def sandwich_norm(x: torch.Tensor, res: torch.Tensor, w_post: torch.Tensor, w_pre: torch.Tensor, *,
                  gate: torch.Tensor | None = None, res_scale: float = 1.0, eps: float = 1e-6):
    """The norm behind a block and the norm in front of the next one, around the residual stream:

        h = res_scale * res + gate * rmsnorm(x, w_post)        y = rmsnorm(h, w_pre)

    x (the block's output) and res [..., H]; w_post, w_pre [H]; gate None, [H] (one learned value per channel) or x's
    shape. Returns (y, h): the next block's input and the updated residual stream. CUDA tensors of bf16, fp16 and fp32 with
    H <= 16384 run `csrc/sandwich_norm.cu`; y is formed from h before h is rounded. Others take `sandwich_norm_reference`."""
    H = x.shape[-1] if x.dim() else 0
    if x.dim() < 1 or H < 1 or res.shape != x.shape:
        raise ValueError(f"x and res need one shape [..., H], got {tuple(x.shape)} and {tuple(res.shape)}")
    if w_post.shape != (H,) or w_pre.shape != (H,):
        raise ValueError(f"w_post and w_pre must be vectors of {H} values")
    if gate is not None and gate.shape != (H,) and gate.shape != x.shape:
        raise ValueError(f"gate must be a vector of {H} values or have x's shape, got {tuple(gate.shape)}")
    if x.numel() // H > MAX_ROWS:
        raise ValueError(f"sandwich_norm takes up to {MAX_ROWS} rows, got {x.numel() // H}")
    dtype, dev, grad = x.dtype, x.device, x.requires_grad
    for t in (res, w_post, w_pre) if gate is None else (res, w_post, w_pre, gate):
        if t.dtype != dtype or t.device != dev:
            raise ValueError("x, res, the weights and the gate must share dtype and device")
        grad = grad or t.requires_grad
    if dtype_code(x) is None:
        return sandwich_norm_reference(x, res, w_post, w_pre, gate, res_scale, eps)
    refuse_tangents("sandwich_norm", x, res, w_post, w_pre, gate)
    if H > SANDWICH_MAX_WIDTH:
        raise native.NativeKernelError(f"sandwich_norm kernels take widths up to {SANDWICH_MAX_WIDTH}, got {H}")
    w_post, w_pre = w_post.contiguous(), w_pre.contiguous()
    if gate is not None and gate.dim() == 1:
        gate = gate.contiguous()
    if grad and torch.is_grad_enabled():
        return _SandwichNorm.apply(x, res, w_post, w_pre, gate, float(res_scale), float(eps))
    g2 = gate if gate is None or gate.dim() == 1 else _rows2d(gate)
    y, h, _ = _sandwich_forward(_rows2d(x), _rows2d(res), w_post, w_pre, g2, float(res_scale), float(eps), False)
    return (y, h) if x.dim() == 2 else (y.view(x.shape), h.view(x.shape))
