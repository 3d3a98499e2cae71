"""Gated linear recurrences over packed documents, forward and backward (``csrc/recurrence.cu``).

``gated_delta_rule``  the recurrence of the GatedDeltaNet layers
(src/xorl/ops/linear_attention/ops/gated_delta_rule/chunk.py), ``ssd_scan`` the one of the Mamba2 layers
(src/xorl/ops/ssm/layers/mamba2_mixer.py).  Both carry one matrix state per head from token to token, restart it at
every document of ``cu_seqlens`` (int32 or int64 [documents + 1] on the inputs' device, ascending; read on the device
only), can take the states that enter the documents and return those that leave them, and are differentiable in every
floating input.

On a GPU with bf16 inputs whose head dims are multiples of 8 (state rows at most 128) the CUDA kernels run; they keep
every computed value in 32 bits and round outputs once.  Elsewhere the same arithmetic runs as tensor ops.  The kernels
read strided inputs in place when the last dimension is contiguous and rows start on 16-byte boundaries, and copy
others.  A call allocates its workspace; it does not synchronise and may be captured into a CUDA graph."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_launches = 0

CHUNK = 64              # tokens of a chunk of the kernels (csrc/recurrence.cu)
SLICE = 32              # columns of the state in one operand tile
TILE = 16384            # bytes of an operand tile of the state
MAX_STATE_ROWS = 128
# The states of all chunks are kept for the backward pass up to this size (4096 tokens of 32 heads of 128 x 128: 207 MB);
# a longer call makes them again, which is the forward pass without its outputs once more.
KEEP_BYTES = 1 << 30
OPERANDS = 32768        # bytes of the operand tile that the delta rule prepares per chunk and head


def launch_count() -> int:
    return _launches


class _Args(ctypes.Structure):
    """``XbRecArgs`` of csrc/recurrence.h."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "dy")]
                + [(n, ctypes.c_longlong) for n in ("q_t", "q_h", "k_t", "k_h", "v_t", "v_h", "dy_t", "dy_h")]
                + [(n, ctypes.c_void_p) for n in ("g", "b")]
                + [(n, ctypes.c_longlong) for n in ("g_t", "g_h", "b_t", "b_h")]
                + [(n, ctypes.c_void_p) for n in ("A", "D", "cu", "s_in", "s_out", "ds_out", "ds_in")]
                + [(n, ctypes.c_longlong) for n in ("s_k", "s_v")]
                + [(n, ctypes.c_void_p) for n in ("o", "dq", "dk_out", "dv_out", "dg", "db", "dA", "dD", "chunks",
                                                  "doc_off", "hd", "rqk", "qk", "kk", "pt", "s_tiles", "ds_tiles",
                                                  "u_tiles", "dr_tiles", "part", "status")]
                + [(n, ctypes.c_int) for n in ("T", "n_docs", "Hk", "Hv", "dk", "dv", "dkp", "dvp", "nc_max", "l2norm")]
                + [("scale", ctypes.c_float)])


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` [T, heads, dim] as the kernels read it: itself, or a copy where its strides do not suit 16-byte loads."""
    if x.stride(2) != 1 or x.stride(0) % 8 or x.stride(1) % 8 or x.stride(0) <= 0 or x.stride(1) <= 0 or x.data_ptr() % 16:
        return x.contiguous() if not x.is_contiguous() else x.clone()
    return x


def _pieces(sizes):
    """Byte offsets of buffers of ``sizes`` in one allocation, and its size."""
    at, out = 0, []
    for s in sizes:
        out.append(at)
        at += (s + 255) // 256 * 256
    return out, at


def _tiles(a: _Args, delta: bool):
    """(field, bytes) of the operand tiles that the gradients read: one set from the forward pass, one from the backward."""
    n = a.nc_max * a.Hv * (a.dvp // SLICE) * TILE
    return [("s_tiles", n)] + ([("u_tiles", n // 2)] if delta else []), [("ds_tiles", n)] + (
        [("dr_tiles", n // 2)] if delta else [("part", a.nc_max * a.Hv * 2 * 4)])


def _place(a: _Args, fields, device) -> torch.Tensor:
    offs, total = _pieces([n for _, n in fields])
    buf = torch.empty(total, dtype=torch.uint8, device=device)
    for (name, _), off in zip(fields, offs):
        setattr(a, name, buf.data_ptr() + off)
    return buf


def _fill(a: _Args, q, k, v, g, b, A, D, cu, s_in, ws, keep: bool, delta: bool, scale: float, l2norm: bool) -> torch.Tensor:
    """Inputs, sizes and the kept workspace (allocated if ``ws`` is None), which is returned."""
    T, Hk, dk = q.shape
    Hv, dv = v.shape[1], v.shape[2]
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_t, a.q_h, a.k_t, a.k_h, a.v_t, a.v_h = (q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0),
                                                v.stride(1))
    a.b, a.b_t, a.b_h = b.data_ptr(), b.stride(0), b.stride(1)
    if delta:
        a.g, a.g_t, a.g_h = g.data_ptr(), g.stride(0), g.stride(1)
        a.s_k, a.s_v = dv, 1
    else:
        a.A, a.D = A.data_ptr(), D.data_ptr()
        a.s_k, a.s_v = 1, dk
    a.cu, a.s_in = cu.data_ptr(), _lib.ptr(s_in)
    a.T, a.n_docs, a.Hk, a.Hv, a.dk, a.dv = T, cu.numel() - 1, Hk, Hv, dk, dv
    a.dkp, a.dvp = 64 if dk <= 64 else 128, -(-dv // 64) * 64
    a.nc_max = T // CHUNK + cu.numel() + 1
    a.l2norm, a.scale = int(l2norm), scale
    nc = a.nc_max
    sizes = [("chunks", nc * 16), ("doc_off", (cu.numel() + 2) * 4), ("hd", nc * Hv * 3 * CHUNK * 4),
             ("rqk", nc * Hk * 2 * CHUNK * 4)]
    if delta:
        sizes.append(("pt", nc * Hv * OPERANDS))
    if keep or not delta:
        sizes.append(("qk", nc * Hk * CHUNK * CHUNK * 4))
    if keep and delta:
        sizes.append(("kk", nc * Hk * CHUNK * CHUNK * 4))
    offs, total = _pieces([n for _, n in sizes])
    if ws is None:
        ws = torch.empty(total, dtype=torch.uint8, device=q.device)
    for (name, _), off in zip(sizes, offs):
        setattr(a, name, ws.data_ptr() + off)
    return ws


class _Recurrence(torch.autograd.Function):
    """q, k, v [T, heads, dim] bf16; g (delta) or A, D (scan), b fp32; s_in fp32 or None."""

    @staticmethod
    def forward(ctx, q, k, v, g, b, A, D, s_in, cu, delta, scale, l2norm, final):
        global _launches
        q, k, v = _rows(q), _rows(k), _rows(v)
        T, Hv, dv = v.shape
        a = _Args()
        with _lib.on_device(q):
            keep = any(ctx.needs_input_grad)
            ws = _fill(a, q, k, v, g, b, A, D, cu, s_in, None, keep, delta, scale, l2norm)
            o = torch.empty((T, Hv, dv), dtype=v.dtype, device=v.device)
            shape = (cu.numel() - 1, Hv) + ((q.shape[2], dv) if delta else (dv, q.shape[2]))
            s_out = torch.empty(shape, dtype=torch.float32, device=v.device) if final else None
            a.o, a.s_out = o.data_ptr(), _lib.ptr(s_out)
            tiles = None
            if keep and sum(n for _, n in _tiles(a, delta)[0]) <= KEEP_BYTES:
                tiles = _place(a, _tiles(a, delta)[0], v.device)
            _lib.check(_lib.cuda_lib().xb_recurrence_fwd(ctypes.byref(a), int(delta), _lib.stream_ptr()),
                       "xb_recurrence_fwd")
        _launches += 3
        ctx.save_for_backward(q, k, v, g, b, A, D, s_in, cu, ws, tiles)
        ctx.conf = (delta, scale, l2norm)
        ctx.set_materialize_grads(False)
        return o, s_out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds_out):
        global _launches
        q, k, v, g, b, A, D, s_in, cu, ws, tiles = ctx.saved_tensors
        delta, scale, l2norm = ctx.conf
        T, Hk, dk = q.shape
        Hv, dv = v.shape[1], v.shape[2]
        dev = q.device
        a = _Args()
        with _lib.on_device(q):
            dy = torch.zeros((T, Hv, dv), dtype=v.dtype, device=dev) if dy is None else _rows(dy)
            _fill(a, q, k, v, g, b, A, D, cu, s_in, ws, True, delta, scale, l2norm)
            a.dy, a.dy_t, a.dy_h = dy.data_ptr(), dy.stride(0), dy.stride(1)
            ds_out = None if ds_out is None else ds_out.contiguous()
            ds_in = torch.empty_like(s_in) if ctx.needs_input_grad[7] else None
            a.ds_out, a.ds_in = _lib.ptr(ds_out), _lib.ptr(ds_in)
            dq = torch.empty((T, Hk, dk), dtype=q.dtype, device=dev)
            dkk = torch.empty((T, Hk, dk), dtype=q.dtype, device=dev)
            dvv = torch.empty((T, Hv, dv), dtype=v.dtype, device=dev)
            db = torch.empty((T, Hv), dtype=torch.float32, device=dev)
            dg = torch.empty((T, Hv), dtype=torch.float32, device=dev) if delta else None
            dA = None if delta else torch.empty(Hv, dtype=torch.float32, device=dev)
            dD = None if delta else torch.empty(Hv, dtype=torch.float32, device=dev)
            a.dq, a.dk_out, a.dv_out, a.db = dq.data_ptr(), dkk.data_ptr(), dvv.data_ptr(), db.data_ptr()
            a.dg, a.dA, a.dD = _lib.ptr(dg), _lib.ptr(dA), _lib.ptr(dD)
            first, second = _tiles(a, delta)
            if tiles is None:
                tmp = _place(a, first + second, dev)
            else:
                tmp = _place(a, second, dev)
                for (name, _), off in zip(first, _pieces([n for _, n in first])[0]):
                    setattr(a, name, tiles.data_ptr() + off)
            _lib.check(_lib.cuda_lib().xb_recurrence_bwd(ctypes.byref(a), int(delta), int(tiles is not None), _lib.stream_ptr()),
                       "xb_recurrence_bwd")
        del tmp
        _launches += (2 if delta else 3) + int(tiles is None)
        return dq, dkk, dvv, dg, db, dA, dD, ds_in, None, None, None, None, None


def _check(what: str, q, k, v, per_head, cu, s_in, state_shape, names) -> None:
    if q.dim() != 3 or k.shape != q.shape or v.dim() != 3 or v.shape[0] != q.shape[0]:
        raise ValueError(f"{what}: {names[0]} and {names[1]} are [T, heads, dim] of one shape and {names[2]} is "
                         f"[T, heads, dim] with the same T (got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)})")
    if q.shape[1] == 0 or v.shape[1] % q.shape[1] or not (q.shape[2] and v.shape[2] and v.shape[1]):
        raise ValueError(f"{what}: {v.shape[1]} heads of {names[2]} cannot share {q.shape[1]} heads of {names[0]}")
    for name, t, shape in per_head:
        if tuple(t.shape) != shape:
            raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {shape}")
    if cu.dim() != 1 or cu.numel() < 1 or cu.is_floating_point():
        raise ValueError(f"{what}: cu_seqlens is a vector of integers, one more than there are documents")
    if s_in is not None and tuple(s_in.shape) != state_shape:
        raise ValueError(f"{what}: initial_state has shape {tuple(s_in.shape)}, expected {state_shape}")
    for t in [q, k, v] + [t for _, t, _ in per_head] + ([s_in] if s_in is not None else []):
        if t.device != q.device:
            raise ValueError(f"{what}: inputs on different devices ({q.device} and {t.device})")


def _kernel_ok(q, k, v) -> bool:
    return (q.is_cuda and q.dtype == k.dtype == v.dtype == torch.bfloat16 and q.shape[2] % 8 == 0
            and q.shape[2] <= MAX_STATE_ROWS and v.shape[2] % 8 == 0)


def _boundaries(cu: torch.Tensor, device) -> torch.Tensor:
    return cu.to(device=device, dtype=torch.int32).contiguous()


def gated_delta_rule_reference(q, k, v, g, beta, cu_seqlens, *, scale: float = 1.0, qk_l2norm: bool = False,
                               initial_state=None, return_final_state: bool = False):
    """Tensor-op form of ``gated_delta_rule``, in fp32 chunks."""
    from ..models.gated_deltanet import gated_delta_rule_chunked
    qf, kf = q.float(), k.float()
    if qk_l2norm:
        qf, kf = torch.nn.functional.normalize(qf, dim=-1), torch.nn.functional.normalize(kf, dim=-1)
    rep = v.shape[1] // q.shape[1]
    qf, kf = (qf * scale).repeat_interleave(rep, 1), kf.repeat_interleave(rep, 1)
    out = gated_delta_rule_chunked(qf, kf, v, g.float(), beta.float(), cu_seqlens, initial_state=initial_state,
                                   return_final_state="all" if return_final_state else False)
    if not return_final_state:
        return out
    return out[0], out[1][:cu_seqlens.numel() - 1]


def gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     cu_seqlens: torch.Tensor, *, scale: float = 1.0, qk_l2norm: bool = False,
                     initial_state: Optional[torch.Tensor] = None, return_final_state: bool = False):
    """S_t = e^{g_t} S_{t-1} + k_t (x) beta_t (v_t - (e^{g_t} S_{t-1})^T k_t);  o_t = S_t^T (scale q_t).

    q, k [T, Hk, dk], v [T, Hv, dv], g (log decay) and beta [T, Hv]; head h of v reads head h // (Hv / Hk) of q and k,
    which ``qk_l2norm`` normalises per head first.  Returns o [T, Hv, dv] in v's type, with ``return_final_state``
    also the states [documents, Hv, dk, dv] (fp32) that leave the documents; ``initial_state`` of the same shape
    enters them (zeros if None).  Rows outside every document give zeros."""
    T, Hv = v.shape[0], v.shape[1] if v.dim() == 3 else 0
    _check("gated_delta_rule", q, k, v, [("g", g, (T, Hv)), ("beta", beta, (T, Hv))], cu_seqlens, initial_state,
           (cu_seqlens.numel() - 1, Hv, q.shape[-1], v.shape[-1]), ("q", "k", "v"))
    scale = float(scale)
    if not 0 < abs(scale) < float("inf"):
        raise ValueError(f"gated_delta_rule: scale is a finite number other than 0 (got {scale})")
    if not _kernel_ok(q, k, v):
        return gated_delta_rule_reference(q, k, v, g, beta, cu_seqlens, scale=scale, qk_l2norm=qk_l2norm,
                                          initial_state=initial_state, return_final_state=return_final_state)
    s_in = None if initial_state is None else initial_state.float().contiguous()
    o, s = _lib.apply(_Recurrence, q, k, v, g.float(), beta.float(), None, None, s_in,
                      _boundaries(cu_seqlens, q.device), True, scale, bool(qk_l2norm), bool(return_final_state))
    return (o, s) if return_final_state else o


def ssd_scan_reference(x, dt, A, B, C, D, cu_seqlens, *, initial_state=None, return_final_state: bool = False,
                       chunk: int = 128):
    """Tensor-op form of ``ssd_scan``, in fp32 chunks; the entering states are added behind the scan from zero."""
    from ..models.mamba2 import segment_ids, ssd_chunked
    T, H, P = x.shape
    if T == 0:
        y = x.float()
    else:
        seg = segment_ids(cu_seqlens.to(x.device), T)
        y = ssd_chunked(x, dt, A, B, C, D, seg, chunk)
    n, rep = cu_seqlens.numel() - 1, H // B.shape[1]
    if initial_state is None and not return_final_state:
        return y.to(x.dtype)
    la = dt.float() * A.float()
    Bh, Ch = B.float().repeat_interleave(rep, 1), C.float().repeat_interleave(rep, 1)
    cuts = cu_seqlens.tolist()
    add, finals = [], []
    for d in range(n):
        s, e = cuts[d], max(cuts[d], cuts[d + 1])
        inc = la[s:e].cumsum(0)
        total = la[s:e].sum(0)
        S0 = x.new_zeros(H, P, B.shape[2], dtype=torch.float32) if initial_state is None else initial_state[d].float()
        add.append(torch.exp(inc).unsqueeze(-1) * torch.einsum("hpn,thn->thp", S0, Ch[s:e]))
        w = torch.exp(total - inc) * dt[s:e].float()
        finals.append(torch.exp(total).view(H, 1, 1) * S0
                      + torch.einsum("thp,thn->hpn", w.unsqueeze(-1) * x[s:e].float(), Bh[s:e]))
    if n and T:
        head, tail = y[:cuts[0]], y[max(cuts[0], cuts[-1]):]
        y = torch.cat([head, y[cuts[0]:max(cuts[0], cuts[-1])] + torch.cat(add, 0), tail], 0)
    y = y.to(x.dtype)
    if not return_final_state:
        return y
    return y, torch.stack(finals, 0) if finals else x.new_zeros(0, H, P, B.shape[2], dtype=torch.float32)


def ssd_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: torch.Tensor,
             cu_seqlens: torch.Tensor, *, initial_state: Optional[torch.Tensor] = None,
             return_final_state: bool = False, chunk: int = 128):
    """S_t = e^{dt_t A} S_{t-1} + dt_t x_t (x) B_t;  y_t = S_t C_t + D x_t.

    x [T, H, P], dt [T, H] (behind softplus and clamp), A, D [H], B, C [T, G, N] shared by the H / G heads of a group.
    Returns y [T, H, P] in x's type, with ``return_final_state`` also the states [documents, H, P, N] (fp32) that
    leave the documents; ``initial_state`` of the same shape enters them (zeros if None).  Rows before the first and
    behind the last boundary are documents of their own, without states.  ``chunk``: chunk length of the tensor-op form."""
    T, H = x.shape[0], x.shape[1] if x.dim() == 3 else 0
    _check("ssd_scan", B, C, x, [("dt", dt, (T, H)), ("A", A, (H,)), ("D", D, (H,))], cu_seqlens, initial_state,
           (cu_seqlens.numel() - 1, H, x.shape[-1], B.shape[-1]), ("B", "C", "x"))
    if not _kernel_ok(B, C, x):
        return ssd_scan_reference(x, dt, A, B, C, D, cu_seqlens, initial_state=initial_state,
                                  return_final_state=return_final_state, chunk=chunk)
    s_in = None if initial_state is None else initial_state.float().contiguous()
    y, s = _lib.apply(_Recurrence, C, B, x, None, dt.float(), A.float().contiguous(), D.float().contiguous(), s_in,
                      _boundaries(cu_seqlens, x.device), False, 1.0, False, bool(return_final_state))
    return (y, s) if return_final_state else y
