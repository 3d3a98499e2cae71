"""Gated linear recurrences over packed documents, forward and backward (``csrc/recurrence.cu``).

``gated_delta_rule``  the recurrence of the GatedDeltaNet layers
(src/xorl/ops/linear_attention/ops/gated_delta_rule/chunk.py), ``ssd_scan`` the one of the Mamba2 layers
(src/xorl/ops/ssm/layers/mamba2_mixer.py).  Both carry one matrix state per head from token to token, restart it at
every document of ``cu_seqlens`` (int32 or int64 [documents + 1] on the inputs' device, ascending within the rows; read on
the device only, where other boundaries are clamped and reported: ``_lib.raise_on_status``), can take the states that
enter the documents and return those that leave them, and are differentiable in every floating input.

On a GPU with bf16 inputs whose head dims are multiples of 8 (state rows at most 128) the CUDA kernels run.  They add up
states, sums and gradients in 32 bits and round outputs once; a computed value that enters a product of the tensor cores
(states, U, P and their gradients) does so with 17 bits, with 24 where ``csrc/recurrence.cu`` says so, which leaves fp32
outputs off by up to 7e-6 of their norm.  Elsewhere, and in the ``_reference`` forms for who wants fp32 throughout, the same
arithmetic runs as tensor ops.  Outputs have the same bits with and without gradients, so that a recomputed pass repeats the
first one.  The kernels read strided inputs in place when the last dimension is contiguous and rows start on 16-byte
boundaries, and copy others.  A call allocates its workspace; it does not synchronise and may be captured into a CUDA
graph (a backward pass: while no graph of the same leaves that was built outside the capture is alive, since torch would
wait for its stream and end the process)."""
from __future__ import annotations

import functools
import struct
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_launches = 0

CHUNK = 64              # tokens of a chunk of the kernels (csrc/recurrence.cu)
TILE = 16384            # bytes of an operand tile of the state
MAX_STATE_ROWS = 128
# What a call may keep from its forward pass for its backward pass besides its inputs, in bytes; a program may set it.  It keeps
# the operands and the state tiles of all chunks if both fit (4096 tokens of 32 heads of 128 x 128: 0.4 GB), or the operands
# alone, and makes the rest again: the tiles are the forward pass without its outputs once more, the operands its prepare
# kernel.  Forward and backward, kept, operands alone, nothing: 4096 tokens of such heads 0.52, 0.61, 0.67 ms; 16384 tokens (1.6
# GB) 1.92, 2.27, 2.43 ms; the scan of 128 heads of 64 x 128, 4096 tokens (0.6 GB) 0.64, 0.72, 0.74 ms.  The bound is about a
# hundredth of the GPU's memory, so that some tens of such layers which recompute nothing leave room for the rest.
KEEP_BYTES = 3 << 29
# With at most so many tokens per document on average, documents of at most so many go token by token
# (csrc/recurrence_step.cu, which gives the times of both ways), the others through the chunked kernels.  The same with and
# without gradients, so that a forward pass that is run again for its gradients has the bits of the first one.  A backward
# pass works on chunks: where their tiles may be kept all documents go through the chunked kernels too, else the backward
# pass makes what it needs.
STEP = 16
OPERANDS = 40960        # bytes of the operand tile that the delta rule prepares per chunk and head


def launch_count() -> int:
    return _launches


_pack = struct.Struct("57q").pack      # the fields of XbRecArgs (csrc/recurrence.cu)
_CONTIGUOUS = torch.contiguous_format


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` [T, heads, dim] as the kernels read it: itself, or a copy where its strides do not suit 16-byte loads."""
    t, h, d = x.stride()
    if d != 1 or t % 8 or h % 8 or t <= 0 or h <= 0 or x.data_ptr() % 16:
        return x.clone(memory_format=_CONTIGUOUS)
    return x


def _state(x: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """A state as the kernels read it: contiguous, on a 16-byte boundary."""
    if x is None or (x.is_contiguous() and x.data_ptr() % 16 == 0):
        return x
    return x.clone(memory_format=_CONTIGUOUS)


@functools.lru_cache(maxsize=256)
def _layout(T: int, docs: int, Hk: int, Hv: int, dk: int, dv: int, delta: bool, train: bool, step: int, limit: int = 0):
    """Where the workspaces of a call of these sizes lie: (chunks, bytes of the forward pass's, bytes of the backward pass's,
    what is kept in between (2: operands and state tiles, 1: operands, 0: nothing), offsets of chunks .. pt and of the tiles
    among them, of the backward pass's buffers).  ``step``: of the forward pass; a backward pass's own layout has none."""
    nc = T // CHUNK + (T // (step + 1) if step else docs + 2)
    square = nc * CHUNK * CHUNK * 4
    work = [nc * 16, 2 * (docs + 3) * 4, nc * Hv * 3 * CHUNK * 4, nc * Hk * 2 * CHUNK * 4,
            Hk * square if train or not delta else 0, Hk * square if train and delta else 0, nc * Hv * OPERANDS if delta else 0]
    tiles = nc * Hv * (-(-dv // 64) * 2) * TILE
    first = [tiles, tiles // 2 if delta else 0, tiles // 2 if delta else tiles]
    second = [tiles, tiles // 2 if delta else 0, nc * Hv * (-(-dv // 64) * 4 * CHUNK if delta else 2) * 4]

    def place(sizes):
        at, out = 0, []
        for s in sizes:
            out.append(at if s else -1)                  # -1: no such buffer
            at += (s + 255) // 256 * 256
        return out, at

    kept, kept_bytes = place(work + first)
    if train and kept_bytes <= limit:
        later, later_bytes = place(second)
        return nc, kept_bytes, later_bytes, 2, tuple(kept), tuple(later)
    kept, kept_bytes = place(work)
    later, later_bytes = place(second + (first if train else [0, 0, 0]))
    return nc, kept_bytes, later_bytes, int(train and kept_bytes <= limit), tuple(kept), tuple(later)


def _words(q, k, v, g, b, A, D, cu, s_in, s_out, ds_out, ds_in, dy, outs, ws, tmp, lay, delta, l2norm, step=0, docs=None):
    """The arguments of the C entry points; ``docs`` where there are no boundaries."""
    T, Hk, dk = q.shape
    _, Hv, dv = v.shape
    qs, ks, vs, bs = q.stride(), k.stride(), v.stride(), b.stride()
    nc, _, _, keep, kept, later = lay
    base = ws.data_ptr()
    work = [base + o if o >= 0 else 0 for o in kept]
    back = [0] * 6
    if tmp is not None:
        base = tmp.data_ptr()
        back = [base + o if o >= 0 else 0 for o in later]
    # state tiles (U and third parts with them) come from the forward pass or are made again; dS and dR tiles and partial sums are the backward's
    work += back[:3] if keep == 2 else back[3:] + back[:3]
    return _pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if dy is None else dy.data_ptr(), qs[0], qs[1], ks[0], ks[1],
                  vs[0], vs[1], *((0, 0) if dy is None else dy.stride()[:2]),
                  0 if g is None else g.data_ptr(), b.data_ptr(), *((0, 0) if g is None else g.stride()), bs[0], bs[1],
                  _ptr(A), _ptr(D), _ptr(cu), _ptr(s_in), _ptr(s_out), _ptr(ds_out), _ptr(ds_in),
                  *((dv, 1) if delta else (1, dk)), *outs, *work,
                  T, cu.shape[0] - 1 if docs is None else docs, Hk, Hv, dk, dv, nc, l2norm, step)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


class _Recurrence(torch.autograd.Function):
    """q, k, v [T, heads, dim] bf16; g (delta) or A, D (scan), b fp32; s_in fp32 or None."""

    @staticmethod
    def forward(ctx, q, k, v, g, b, A, D, s_in, cu, delta, scale, l2norm, final):
        global _launches
        q, k, v, s_in = _rows(q), _rows(k), _rows(v), _state(s_in)
        T, Hk, dk = q.shape
        _, Hv, dv = v.shape
        dev = v.device
        docs = cu.shape[0] - 1
        train = True in ctx.needs_input_grad
        step = STEP if T <= STEP * max(docs, 1) else 0
        lay = _layout(T, docs, Hk, Hv, dk, dv, delta, train, 0, KEEP_BYTES)
        if step and lay[3] < 2:
            lay = _layout(T, docs, Hk, Hv, dk, dv, delta, False, step)
        ws = torch.empty(lay[1], dtype=torch.uint8, device=dev)
        o = torch.empty_like(v, memory_format=_CONTIGUOUS)
        s_out = torch.empty((docs, Hv, dk, dv) if delta else (docs, Hv, dv, dk), dtype=torch.float32, device=dev) if final else None
        _lib.call_on(dev, "xb_recurrence_fwd", _words(q, k, v, g, b, A, D, cu, s_in, s_out, None, None, None,
                                                      (o.data_ptr(), 0, 0, 0, 0, 0, 0, 0), ws, None, lay, delta, l2norm, step),
                     scale, delta)
        _launches += 3 if not step else 4 if T > step or lay[3] else 1
        # boundaries are read again only where the plan is made again, from a copy: the caller's may hold the next batch's by then
        ctx.save_for_backward(q, k, v, g, b, A, D, s_in, cu.clone() if train and not lay[3] else None, ws if lay[3] else None)
        ctx.conf = (delta, scale, l2norm, docs, lay)
        ctx.set_materialize_grads(False)
        return o, s_out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds_out):
        global _launches
        q, k, v, g, b, A, D, s_in, cu, ws = ctx.saved_tensors
        delta, scale, l2norm, docs, lay = ctx.conf
        dev = q.device
        kept = lay[3]
        if not kept:
            lay = _layout(q.shape[0], docs, q.shape[1], v.shape[1], q.shape[2], v.shape[2], delta, True, 0)
            ws = torch.empty(lay[1], dtype=torch.uint8, device=dev)
        dy = torch.zeros_like(v, memory_format=_CONTIGUOUS) if dy is None else _rows(dy)
        ds_out = _state(ds_out)
        ds_in = torch.empty_like(s_in) if ctx.needs_input_grad[7] else None
        dq, dkk, dvv = (torch.empty_like(t, memory_format=_CONTIGUOUS) for t in (q, k, v))
        db = torch.empty_like(b, memory_format=_CONTIGUOUS)
        if delta:
            dg, dA, dD = torch.empty_like(b, memory_format=_CONTIGUOUS), None, None
        else:
            dg, dA, dD = None, torch.empty_like(A), torch.empty_like(D)
        tmp = torch.empty(lay[2], dtype=torch.uint8, device=dev)
        _lib.call_on(dev, "xb_recurrence_bwd", _words(q, k, v, g, b, A, D, cu, s_in, None, ds_out, ds_in, dy,
                                               (0, dq.data_ptr(), dkk.data_ptr(), dvv.data_ptr(), _ptr(dg), db.data_ptr(),
                                                _ptr(dA), _ptr(dD)), ws, tmp, lay, delta, l2norm, docs=docs),
              scale, delta, kept)
        _launches += (2 if delta else 3) + (kept < 2) + 2 * (kept == 0)
        return dq, dkk, dvv, dg, db, dA, dD, ds_in, None, None, None, None, None


def _check(what: str, q, k, v, per_head, cu, s_in, state_shape, names) -> None:
    if q.dim() != 3 or k.shape != q.shape or v.dim() != 3 or v.shape[0] != q.shape[0]:
        raise ValueError(f"{what}: {names[0]} and {names[1]} are [T, heads, dim] of one shape and {names[2]} is "
                         f"[T, heads, dim] with the same T (got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)})")
    if q.shape[1] == 0 or v.shape[1] % q.shape[1] or not (q.shape[2] and v.shape[2] and v.shape[1]):
        raise ValueError(f"{what}: {v.shape[1]} heads of {names[2]} cannot share {q.shape[1]} heads of {names[0]}")
    if cu.dim() != 1 or cu.shape[0] < 1 or cu.is_floating_point():
        raise ValueError(f"{what}: cu_seqlens is a vector of integers, one more than there are documents")
    dev = q.device
    if k.device != dev or v.device != dev:
        raise ValueError(f"{what}: inputs on different devices")
    for name, t, shape in per_head:
        if t.shape != shape:
            raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {shape}")
        if t.device != dev:
            raise ValueError(f"{what}: {name} is on {t.device}, {names[0]} on {dev}")
    if s_in is not None and (s_in.shape != state_shape or s_in.device != dev):
        raise ValueError(f"{what}: initial_state is {tuple(s_in.shape)} on {s_in.device}, expected {state_shape} on {dev}")


def _kernel_ok(q, k, v) -> bool:
    return (q.is_cuda and q.dtype == k.dtype == v.dtype == torch.bfloat16 and q.shape[2] % 8 == 0
            and q.shape[2] <= MAX_STATE_ROWS and v.shape[2] % 8 == 0)


def _boundaries(cu: torch.Tensor, device) -> torch.Tensor:
    return cu.to(device=device, dtype=torch.int32).contiguous()


def gated_delta_rule_reference(q, k, v, g, beta, cu_seqlens, *, scale: float = 1.0, qk_l2norm: bool = False,
                               initial_state=None, return_final_state: bool = False):
    """Tensor-op form of ``gated_delta_rule``, in fp32 chunks."""
    from ..models.gated_deltanet import gated_delta_rule_chunked
    if v.shape[0] == 0:                                          # no rows: the states pass through
        S = initial_state.float().clone() if initial_state is not None else v.new_zeros(
            cu_seqlens.numel() - 1, v.shape[1], q.shape[2], v.shape[2], dtype=torch.float32)
        return (v.clone(), S) if return_final_state else v.clone()
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
    s_in = None if initial_state is None else initial_state.float()
    o, s = _lib.apply(_Recurrence, q, k, v, g.float(), beta.float(), None, None, s_in,
                      _boundaries(cu_seqlens, q.device), True, scale, bool(qk_l2norm), return_final_state)
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
    s_in = None if initial_state is None else initial_state.float()
    y, s = _lib.apply(_Recurrence, C, B, x, None, dt.float(), A.float().contiguous(), D.float().contiguous(), s_in,
                      _boundaries(cu_seqlens, x.device), False, 1.0, False, return_final_state)
    return (y, s) if return_final_state else y
