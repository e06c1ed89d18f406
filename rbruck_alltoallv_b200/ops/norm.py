"""The norms around a transformer block, fused with the block's gate, the residual scale and the residual sum
(``csrc/kernels/block_norm.cu``).  The reference library has no compute kernels; this stands next to the MoE layer, whose
input and output these norms are.

With a block ``f`` between them, a layer of the network is::

    _, u = block_norm(residual, pre_weight=w_in)                              # norm in front of the first block
    residual, u = block_norm(residual, f(u), w_post, gate=g, scale=s, pre_weight=w_next)
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from .. import _native
from .._cuda_decl import BlockNorm

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_GATES = {"none": 0, "channel": 1, "token": 2, "full": 3}
MAX_HIDDEN = 16384


def _ptr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None else None


def _rows(t: Optional[torch.Tensor], H: int):
    """``t`` as rows of H packed elements, and the distance between the rows."""
    if t is None:
        return None, 0
    if t.dim() != 2:
        t = t.reshape(-1, H)
    if t.stride(1) != 1 and H > 1:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else H


def _fill(residual, branch, post_weight, gate, kind, scale, pre_weight, eps):
    """The call's argument block without its outputs, and the tensors that it points into."""
    H = residual.shape[-1]
    r, r_ld = _rows(residual, H)
    z, z_ld = _rows(branch, H)
    g, g_ld = _rows(gate, H) if kind == "full" else (gate.contiguous() if gate is not None else None, 0)
    w1 = post_weight.contiguous() if post_weight is not None else None
    w2 = pre_weight.contiguous() if pre_weight is not None else None
    ztype = (branch if branch is not None else residual).dtype
    f32 = torch.float32
    a = BlockNorm(T=r.shape[0], H=H, z_type=_TYPES[ztype], r_type=_TYPES[residual.dtype], gate_kind=_GATES[kind],
                  w1_f32=w1 is not None and w1.dtype == f32, w2_f32=w2 is not None and w2.dtype == f32,
                  gate_f32=g is not None and g.dtype == f32, scale=scale, eps=eps, z=_ptr(z), r=_ptr(r), w1=_ptr(w1),
                  gate=_ptr(g), w2=_ptr(w2), z_ld=z_ld, r_ld=r_ld, gate_ld=g_ld)
    return a, (r, z, g, w1, w2)


def _forward(residual, branch, post_weight, gate, kind, scale, pre_weight, eps, stats):
    a, held = _fill(residual, branch, post_weight, gate, kind, scale, pre_weight, eps)
    dev = residual.device
    r2 = torch.empty(residual.shape, dtype=residual.dtype, device=dev) if branch is not None else None
    u = None
    if pre_weight is not None:
        u = torch.empty(residual.shape, dtype=residual.dtype if branch is None else branch.dtype, device=dev)
    rstd = torch.empty(2, a.T, dtype=torch.float32, device=dev) if stats else None
    a.r2, a.u = _ptr(r2), _ptr(u)
    if stats:
        a.rstd1, a.rstd2 = rstd.data_ptr(), rstd.data_ptr() + 4 * a.T
    if a.T:
        lib = _native.cuda_lib()
        with _native.on_device(dev.index):
            rc = lib.rbv_block_norm(C.byref(a), _native.current_stream(dev.index))
        if rc:
            raise RuntimeError(f"block norm launch failed (CUDA error {rc})")
    del held
    return r2, u, rstd


class _BlockNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, branch, post_weight, gate, pre_weight, kind, scale, eps):
        r2, u, rstd = _forward(residual, branch, post_weight, gate, kind, scale, pre_weight, eps, True)
        ctx.save_for_backward(residual, branch, post_weight, gate, pre_weight, rstd)
        ctx.call = (kind, scale, eps)
        ctx.set_materialize_grads(False)
        return r2, u

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_r2, d_u):
        residual, branch, post_weight, gate, pre_weight, rstd = ctx.saved_tensors
        kind, scale, eps = ctx.call
        if d_r2 is None and d_u is None:
            return (None,) * 8
        a, held = _fill(residual, branch, post_weight, gate, kind, scale, pre_weight, eps)
        T, H, dev = a.T, a.H, residual.device
        dr2, a.dr2_ld = _rows(d_r2, H)
        du, a.du_ld = _rows(d_u, H)
        a.dr2, a.du = _ptr(dr2), _ptr(du)
        a.rstd1, a.rstd2 = rstd.data_ptr(), rstd.data_ptr() + 4 * T
        need_r, need_z, need_w1, need_gate, need_w2 = ctx.needs_input_grad[:5]

        def grad(t, needed):
            return (torch.empty if T else torch.zeros)(t.shape, dtype=t.dtype, device=dev) if needed and t is not None else None
        dr, dz = grad(residual, need_r), grad(branch, need_z)
        dw1, dgate, dw2 = grad(post_weight, need_w1), grad(gate, need_gate), grad(pre_weight, need_w2 and d_u is not None)
        a.dr, a.dz, a.dw1, a.dgate, a.dw2 = _ptr(dr), _ptr(dz), _ptr(dw1), _ptr(dgate), _ptr(dw2)
        if T == 0:
            return dr, dz, dw1, dgate, dw2, None, None, None
        lib = _native.cuda_lib()
        with _native.on_device(dev.index):
            if dw1 is not None or dw2 is not None or (dgate is not None and kind == "channel"):
                partial = torch.empty(lib.rbv_block_norm_parts(T, H, a.z_type), 2, H, dtype=torch.float32, device=dev)
                a.partial = partial.data_ptr()
            rc = lib.rbv_block_norm_backward(C.byref(a), _native.current_stream(dev.index))
        if rc:
            raise RuntimeError(f"block norm backward launch failed (CUDA error {rc})")
        del held
        return dr, dz, dw1, dgate, dw2, None, None, None


def _check(residual, branch, post_weight, gate, scale, pre_weight, eps):
    if not isinstance(residual, torch.Tensor) or residual.dim() < 1:
        raise ValueError("the residual must be a tensor [..., hidden]")
    if residual.dtype not in _TYPES:
        raise ValueError(f"the residual must be bf16, fp16 or fp32, not {residual.dtype}")
    H = residual.shape[-1]
    if not 1 <= H <= MAX_HIDDEN:
        raise ValueError(f"hidden sizes of 1 to {MAX_HIDDEN} are supported, not {H}")
    if branch is None and pre_weight is None:
        raise ValueError("neither a block output nor the weight of a norm in front of the next block: nothing to do")
    if branch is None and (post_weight is not None or gate is not None):
        raise ValueError("post_weight and gate belong to a block output")
    if branch is not None and post_weight is None:
        raise ValueError("a block output needs its norm's weight (post_weight)")
    kind = residual.dtype
    if branch is not None:
        kind = branch.dtype
        if branch.shape != residual.shape:
            raise ValueError(f"block output {tuple(branch.shape)} and residual {tuple(residual.shape)} differ in shape")
        if kind not in _TYPES or residual.dtype not in (kind, torch.float32):
            raise ValueError(f"the residual must have the block output's type ({kind}) or fp32, not {residual.dtype}")
    for name, w in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if w is not None and (w.shape != (H,) or w.dtype not in (kind, torch.float32)):
            raise ValueError(f"{name} must be [{H}] in {kind} or fp32, not {tuple(w.shape)} in {w.dtype}")
    if gate is not None and gate.dtype not in (kind, torch.float32):
        raise ValueError(f"the gate must be {kind} or fp32, not {gate.dtype}")
    for t in (branch, post_weight, gate, pre_weight):
        if t is not None and t.device != residual.device:
            raise ValueError("all tensors must be on one device")
    if gate is not None:
        try:
            fits = torch.broadcast_shapes(gate.shape, residual.shape) == residual.shape
        except RuntimeError:
            fits = False
        if not fits:
            raise ValueError(f"a gate {tuple(gate.shape)} does not broadcast to {tuple(residual.shape)}")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    if not residual.is_cuda:
        raise ValueError("block_norm runs on a GPU: the tensors are on the host")


def block_norm(residual: torch.Tensor, branch: Optional[torch.Tensor] = None, post_weight: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, scale: float = 1.0, pre_weight: Optional[torch.Tensor] = None,
               eps: float = 1e-6) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(residual_out, normed)`` with ``residual_out = residual + scale * gate * rms_norm(branch) * post_weight`` and
    ``normed = rms_norm(residual_out) * pre_weight``, where ``rms_norm(v) = v / sqrt(mean(v ** 2) + eps)`` over the last
    dimension; one kernel, differentiable (once) in all five tensors.

    ``branch`` (the block's output) and ``residual`` are ``[..., hidden]``, in bf16, fp16 or fp32; the residual may be fp32
    next to a 16-bit branch.  Without a branch ``residual_out`` is the residual itself; without ``pre_weight`` ``normed`` is
    None.  The weights ``[hidden]`` and the gate are in the branch's type or fp32.  ``gate`` is one value per channel
    ``[hidden]``, per token ``[..., 1]`` or per element; any other shape that broadcasts to the residual's is expanded first.
    ``normed`` has the branch's type and is made from the sum before that is rounded to the residual's type.  Rows may be
    strided (elements of a row packed).  Launched on the current stream of the tensors' device."""
    _check(residual, branch, post_weight, gate, scale, pre_weight, eps)
    kind = "none"
    if gate is not None:
        shape, lead = gate.shape, residual.shape[:-1]
        if shape == residual.shape[-1:]:
            kind = "channel"
        elif shape == lead + (1,):
            kind = "token"
        else:
            kind = "full"
            if shape != residual.shape:
                gate = gate.expand(residual.shape)
    scale, eps = float(scale), float(eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (residual, branch, post_weight, gate, pre_weight)):
        r2, u = _BlockNormFunction.apply(residual, branch, post_weight, gate, pre_weight, kind, scale, eps)
    else:
        r2, u, _ = _forward(residual, branch, post_weight, gate, kind, scale, pre_weight, eps, False)
    return (residual if branch is None else r2), u
