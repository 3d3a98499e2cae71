"""RMSNorm (optionally fused with the residual add) — ``csrc/norm.cu`` on CUDA, torch on CPU.

Mirrors the behaviour of the reference RMSNorm module
(src/xorl/models/layers/normalization.py:628-799): ``y = x * rsqrt(mean(x^2) + eps) * w`` with an
optional pre-norm residual add that also returns the updated residual stream, and the
zero-centred ``(1 + w)`` variant.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .grad_sink import deliver_param_grad, grad_target, mark_written

_launches = 0


def launch_count() -> int:
    return _launches


def _rmsnorm_ref(x, w, eps, zero_centered):
    xf = x.float()
    rstd = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    wf = w.float() + 1.0 if zero_centered else w.float()
    return (xf * rstd * wf).to(x.dtype)


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, w, eps, zero_centered):
        global _launches
        shape = x.shape
        H = shape[-1]
        x2 = x.reshape(-1, H)
        if not x2.is_contiguous():
            x2 = x2.contiguous()
        T = x2.shape[0]
        y = torch.empty_like(x2)
        rstd = torch.empty(T, device=x.device, dtype=torch.float32)
        res2 = res_out = None
        if residual is not None:
            res2 = residual.reshape(-1, H)
            if not res2.is_contiguous():
                res2 = res2.contiguous()
            res_out = torch.empty_like(x2)
        lib = _lib.cuda_lib()
        _lib.check(lib.xb_rmsnorm_fwd(x2.data_ptr(), _lib.ptr(res2), w.data_ptr(), y.data_ptr(),
                                      _lib.ptr(res_out), rstd.data_ptr(), T, H, float(eps),
                                      int(zero_centered), _lib.stream_ptr()), "xb_rmsnorm_fwd")
        _launches += 1
        h = res_out if residual is not None else x2
        ctx.save_for_backward(h, rstd)
        ctx.w = w
        ctx.zero_centered = zero_centered
        ctx.shape = shape
        ctx.has_res = residual is not None
        if residual is not None:
            return y.reshape(shape), res_out.reshape(shape)
        return y.reshape(shape), None

    @staticmethod
    def backward(ctx, dy, dh):
        global _launches
        h, rstd = ctx.saved_tensors
        w = ctx.w
        T, H = h.shape
        dy2 = dy.reshape(T, H)
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        dres = None
        if ctx.has_res and dh is not None:
            dres = dh.reshape(T, H)
            if not dres.is_contiguous():
                dres = dres.contiguous()
        lib = _lib.cuda_lib()
        rows = lib.xb_rmsnorm_bwd_partial_rows(T)
        partial = torch.empty(rows * H, device=h.device, dtype=torch.float32)
        dx = torch.empty_like(h)
        # the reduction over the partial rows writes, or adds, straight into an engine's fp32 gradient buffer
        tgt, fresh = grad_target(w) if ctx.needs_input_grad[2] else (None, False)
        direct = tgt is not None and tgt.dtype == torch.float32 and tgt.is_contiguous() and T > 0
        dw = tgt if direct else torch.empty(H, device=h.device, dtype=torch.float32)
        _lib.check(lib.xb_rmsnorm_bwd(dy2.data_ptr(), h.data_ptr(), w.data_ptr(), rstd.data_ptr(),
                                      _lib.ptr(dres), dx.data_ptr(), partial.data_ptr(), None,
                                      dw.data_ptr(), int(direct and not fresh), T, H, int(ctx.zero_centered),
                                      _lib.stream_ptr()), "xb_rmsnorm_bwd")
        _launches += 2
        dx = dx.reshape(ctx.shape)
        dwg = None
        if direct:
            mark_written(w)
        elif ctx.needs_input_grad[2]:
            dwg = deliver_param_grad(w, dw)
        return dx, (dx if ctx.has_res else None), dwg, None, None


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float = 1e-6,
            residual: torch.Tensor | None = None, zero_centered: bool = False):
    """Returns ``y`` or, when ``residual`` is given, ``(y, x + residual)``."""
    if not x.is_cuda:
        if residual is not None:
            h = x + residual
            return _rmsnorm_ref(h, w, eps, zero_centered), h
        return _rmsnorm_ref(x, w, eps, zero_centered)
    if x.dtype != torch.bfloat16 or x.shape[-1] % 8 or x.shape[-1] > 16384:
        if residual is not None:
            h = x + residual
            return _rmsnorm_ref(h, w, eps, zero_centered), h
        return _rmsnorm_ref(x, w, eps, zero_centered)
    y, h = _lib.apply(_RMSNorm, x, residual, w, eps, zero_centered)
    if residual is not None:
        return y, h
    return y


def _gated_rms_norm_ref(x, gate, weight, group_size, eps, norm_first):
    act = torch.nn.functional.silu(gate.float())
    h = x.float() if norm_first else x.float() * act
    h = h.unflatten(-1, (-1, group_size))
    h = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + eps) * weight.float().view(-1, group_size)
    h = h.flatten(-2)
    return (h * act if norm_first else h).to(x.dtype)


def _norm_rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` [T, W] with rows that suit 16-byte loads: itself or a copy."""
    if t.stride(1) != 1 or t.stride(0) % 8 or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format)
    return t


@functools.lru_cache(maxsize=256)
def _gated_norm_partial(T: int, groups: int, group_size: int, shared: int, device: int) -> int:
    """Size of the weight gradient's partial sums: a matter of the device's SMs, so of the device."""
    with torch.cuda.device(device):
        return max(_lib.cuda_lib().xb_gated_norm_partial(T, groups, group_size, shared), 1)


class _GatedRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, w, group_size, eps, norm_first):
        global _launches
        shape = x.shape
        W = shape[-1]
        x2, z2 = (x, gate) if x.dim() == 2 else (x.reshape(-1, W), gate.reshape(-1, W))
        x2, z2 = _norm_rows(x2), _norm_rows(z2)
        wc = w if w.is_contiguous() else w.contiguous()
        T, groups, dev = x2.shape[0], W // group_size, x.device
        y = torch.empty_like(x2, memory_format=torch.contiguous_format)
        rstd = torch.empty((T, groups), dtype=torch.float32, device=dev) if True in ctx.needs_input_grad else None
        shared, wide = int(w.numel() == group_size), int(w.dtype == torch.float32)
        _lib.call_on(dev, "xb_gated_norm_fwd", x2.data_ptr(), x2.stride(0), z2.data_ptr(), z2.stride(0), wc.data_ptr(), wide,
                     shared, y.data_ptr(), _lib.ptr(rstd), T, groups, group_size, eps, norm_first)
        _launches += 1
        ctx.save_for_backward(x2, z2, wc, rstd)
        ctx.w, ctx.conf = w, (group_size, norm_first, shape, groups, shared, wide)
        return y if len(shape) == 2 else y.reshape(shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        global _launches
        x, z, wc, rstd = ctx.saved_tensors
        group_size, norm_first, shape, groups, shared, wide = ctx.conf
        T, W = x.shape
        dev = x.device
        dy = _norm_rows(dy if dy.dim() == 2 else dy.reshape(T, W))
        dx, dz = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (x, z))
        part = dw = None
        want, sink, out_wide = ctx.needs_input_grad[2], False, 0
        if want:
            part = torch.empty(_gated_norm_partial(T, groups, group_size, shared, dev.index), dtype=torch.float32, device=dev)
            # an engine's buffer takes fp32 sums; a gradient that autograd gets is rounded where it is summed
            sink = grad_target(ctx.w)[0] is not None
            dw = torch.empty_like(wc, dtype=torch.float32) if sink else torch.empty_like(wc)
            out_wide = int(sink or wide)
        _lib.call_on(dev, "xb_gated_norm_bwd", dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), z.data_ptr(), z.stride(0),
                     wc.data_ptr(), wide, shared, rstd.data_ptr(), dx.data_ptr(), dz.data_ptr(), _lib.ptr(part),
                     0 if part is None else part.numel(), _lib.ptr(dw), out_wide, T, groups, group_size, norm_first)
        _launches += 1 + int(want)
        if len(shape) != 2:
            dx, dz = dx.reshape(shape), dz.reshape(shape)
        return dx, dz, deliver_param_grad(ctx.w, dw) if sink else dw, None, None, None


GATED_NORM_MAX_GROUP = 8192


def gated_rms_norm(x: torch.Tensor, gate: torch.Tensor, weight: torch.Tensor, group_size: int, eps: float = 1e-6,
                   norm_first: bool = True) -> torch.Tensor:
    """RMS norm over groups of ``group_size`` columns with a SiLU gate, statistics in fp32, rounded once.

    ``norm_first``: ``rms(x) * weight * silu(gate)`` (the GatedDeltaNet output norm), else
    ``rms(x * silu(gate)) * weight`` (the Mamba2 one, src/xorl/ops/ssm/modules/gated_norm.py).  x and gate are [..., W]
    of one shape and type, any row stride; weight has W elements or ``group_size`` that all groups share.  The CUDA
    kernels (``csrc/gated_norm.cu``) take bf16 rows with a bf16 or fp32 weight and groups of a multiple of 8 columns,
    8192 at most; elsewhere the same arithmetic runs as tensor ops."""
    W = x.shape[-1]
    if gate.shape != x.shape or gate.device != x.device or weight.device != x.device:
        raise ValueError(f"gated_rms_norm: x and gate have one shape on one device with the weight (got {tuple(x.shape)} "
                         f"on {x.device}, {tuple(gate.shape)} on {gate.device}, weight on {weight.device})")
    if group_size <= 0 or W == 0 or W % group_size:
        raise ValueError(f"gated_rms_norm: groups of {group_size} columns do not divide rows of {W}")
    if weight.numel() not in (group_size, W):
        raise ValueError(f"gated_rms_norm: weight has {weight.numel()} elements, expected {group_size} or {W}")
    if (not x.is_cuda or x.dtype != torch.bfloat16 or gate.dtype != torch.bfloat16 or group_size % 8
            or weight.dtype not in (torch.bfloat16, torch.float32) or group_size > GATED_NORM_MAX_GROUP
            or W // group_size > 65535):
        return _gated_rms_norm_ref(x, gate, weight, group_size, eps, norm_first)
    return _lib.apply(_GatedRMSNorm, x, gate, weight, group_size, eps, bool(norm_first))
