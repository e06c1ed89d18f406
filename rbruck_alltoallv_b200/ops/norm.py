"""The norms around a transformer block, fused with the block's gate, the residual scale and the residual sum
(``csrc/kernels/block_norm.cu``).  The reference library has no compute kernels; this stands next to the MoE layer, whose
input and output these norms are.

With a block ``f`` between them, a layer of the network is::

    _, u = block_norm(residual, pre_weight=w_in)                              # norm in front of the first block
    residual, u = block_norm(residual, f(u), w_post, gate=g, scale=s, pre_weight=w_next)
"""
from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch

from .. import _native

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_GATES = {"none": 0, "channel": 1, "token": 2, "full": 3}
MAX_HIDDEN = 16384


# rbv_norm_t as the C compiler lays it out.  (Packing it in one call takes a fraction of the time of a ctypes.Structure with
# thirty fields; a call on a few tokens takes no longer on the GPU than its launch on the host.)
_pack = struct.Struct("@q7i2f5P3q6P2q6P").pack


def _ptr(t: Optional[torch.Tensor]) -> int:
    return t.data_ptr() if t is not None else 0


def _rows(t: torch.Tensor, H: int):
    """``t`` as rows of H packed elements, and the distance between the rows."""
    if t.is_contiguous():
        return t, H
    if t.dim() != 2:
        t = t.reshape(-1, H)
    if t.stride(1) != 1 and H > 1:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else H


def _inputs(residual, branch, post_weight, gate, kind, pre_weight):
    """The argument block's fields up to its scale, and from z to the row distances; the tensors that they point into."""
    H = residual.shape[-1]
    f32 = torch.float32
    r, r_ld = _rows(residual, H)
    z, z_ld = _rows(branch, H) if branch is not None else (None, 0)
    g, g_ld = (None, 0) if gate is None else _rows(gate, H) if kind == 3 else (gate.contiguous(), 0)
    w1 = post_weight.contiguous() if post_weight is not None else None
    w2 = pre_weight.contiguous() if pre_weight is not None else None
    head = (residual.numel() // H, H, _TYPES[residual.dtype if z is None else z.dtype], _TYPES[residual.dtype], kind,
            w1 is not None and w1.dtype is f32, w2 is not None and w2.dtype is f32, g is not None and g.dtype is f32)
    return head, (_ptr(z), r.data_ptr(), _ptr(w1), _ptr(g), _ptr(w2), z_ld, r_ld, g_ld), (r, z, g, w1, w2)


def _launch(entry, call, device, what):
    index = device.index
    if torch.cuda.current_device() == index:
        rc = entry(call, _native.current_stream(index))
    else:
        with torch.cuda.device(index):
            rc = entry(call, _native.current_stream(index))
    if rc:
        raise RuntimeError(f"{what} launch failed (CUDA error {rc})")


def _forward(residual, branch, post_weight, gate, kind, scale, pre_weight, eps, stats):
    head, body, held = _inputs(residual, branch, post_weight, gate, kind, pre_weight)
    T = head[0]
    r2 = residual.new_empty(residual.shape) if branch is not None else None
    u = (residual if branch is None else branch).new_empty(residual.shape) if pre_weight is not None else None
    rstd, at = None, 0
    if stats:
        rstd = torch.empty(2 * T, dtype=torch.float32, device=residual.device)
        at = rstd.data_ptr()
    if T:
        call = _pack(*head, scale, eps, *body, at, at + 4 * T if stats else 0, _ptr(r2), _ptr(u), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
        _launch(_native.cuda_lib().rbv_block_norm, call, residual.device, "block norm")
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
        need_r, need_z, need_w1, need_gate, need_w2 = ctx.needs_input_grad[:5]
        head, body, held = _inputs(residual, branch, post_weight, gate, kind, pre_weight)
        T, H = head[:2]

        def grad(t, needed):
            return (t.new_empty if T else t.new_zeros)(t.shape) if needed else None
        dr, dz, dw1 = grad(residual, need_r), grad(branch, need_z), grad(post_weight, need_w1)
        dgate, dw2 = grad(gate, need_gate), grad(pre_weight, need_w2 and d_u is not None)
        if T:
            dr2, dr2_ld = _rows(d_r2, H) if d_r2 is not None else (None, 0)
            du, du_ld = _rows(d_u, H) if d_u is not None else (None, 0)
            lib, partial = _native.cuda_lib(), None
            if dw1 is not None or dw2 is not None or (dgate is not None and kind == _GATES["channel"]):
                partial = rstd.new_empty(2 * H * lib.rbv_block_norm_parts(T, H, head[2]))
            at = rstd.data_ptr()
            call = _pack(*head, scale, eps, *body, at, at + 4 * T, 0, 0, _ptr(dr2), _ptr(du), dr2_ld, du_ld, _ptr(dz), _ptr(dr),
                         _ptr(dgate), _ptr(dw1), _ptr(dw2), _ptr(partial))
            _launch(lib.rbv_block_norm_backward, call, residual.device, "block norm backward")
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
        g = gate.shape
        if len(g) > residual.dim() or any(n != 1 and n != m for n, m in zip(reversed(g), reversed(residual.shape))):
            raise ValueError(f"a gate {tuple(g)} does not broadcast to {tuple(residual.shape)}")
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
        shape, full = gate.shape, residual.shape
        if shape == full[-1:]:
            kind = "channel"
        elif shape == full[:-1] + (1,):
            kind = "token"
        else:
            kind = "full"
            if shape != full:
                gate = gate.expand(full)
    kind, scale, eps = _GATES[kind], float(scale), float(eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (residual, branch, post_weight, gate, pre_weight)):
        r2, u = _BlockNormFunction.apply(residual, branch, post_weight, gate, pre_weight, kind, scale, eps)
    else:
        r2, u, _ = _forward(residual, branch, post_weight, gate, kind, scale, pre_weight, eps, False)
    return (residual if branch is None else r2), u
