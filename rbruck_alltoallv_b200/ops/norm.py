"""The norms around a transformer block, fused with the block's gate, the residual scale and the residual sum
(``csrc/kernels/block_norm.cu``, bound in ``csrc/api/torch_ops.cpp``).  The reference library has no compute kernels; this
stands next to the MoE layer, whose input and output these norms are.

With a block ``f`` between them, a layer of the network is::

    _, u = block_norm(residual, pre_weight=w_in)                              # norm in front of the first block
    residual, u = block_norm(residual, f(u), w_post, gate=g, scale=s, pre_weight=w_next)
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _native

MAX_HIDDEN = 16384


def block_norm(residual: torch.Tensor, branch: Optional[torch.Tensor] = None, post_weight: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, scale: float = 1.0, pre_weight: Optional[torch.Tensor] = None,
               eps: float = 1e-6) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(residual_out, normed)`` with ``residual_out = residual + scale * gate * rms_norm(branch) * post_weight`` and
    ``normed = rms_norm(residual_out) * pre_weight``, where ``rms_norm(v) = v / sqrt(mean(v ** 2) + eps)`` over the last
    dimension; one kernel, differentiable (once, in reverse mode) in all five tensors.

    ``branch`` (the block's output) and ``residual`` are ``[..., hidden]``, in bf16, fp16 or fp32; the residual may be fp32
    next to a 16-bit branch.  Without a branch ``residual_out`` is the residual itself; without ``pre_weight`` ``normed`` is
    None.  The weights ``[hidden]`` and the gate are in the branch's type or fp32.  ``gate`` is one value per channel
    ``[hidden]``, per token ``[..., 1]`` or per element; any other shape that broadcasts to the residual's is expanded first.
    ``normed`` has the branch's type and is made from the sum before that is rounded to the residual's type.  Rows may be
    strided (elements of a row packed).  Launched on the current stream of the tensors' device; both passes can be captured into a
    graph, the backward pass while no graph of an earlier, eager pass through the same leaves is alive (torch would accumulate into
    them on that pass's stream, which a capture does not survive)."""
    if type(scale) is not float and isinstance(scale, torch.Tensor) and scale.requires_grad and torch.is_grad_enabled():
        raise ValueError("scale is a number: one that is learned goes into the gate")
    return _native.torch_ops().block_norm(residual, branch, post_weight, gate, scale, pre_weight, eps)
