"""MoE FFN layer as a user-facing module, plus the smoke routine used by the repository entry point."""
from __future__ import annotations

import torch

from ..ops.moe import MoEExpertParallel, linear_int8, quantize_weight_int8, reference_forward
from ..ops.norm import block_norm


class MoELayer:
    """Top-2 routed SwiGLU FFN with experts sharded over the communicator's ranks.

    ``router_weight`` [E, H] (optional): when given, logits are ``x @ router_weight.T`` in fp32; otherwise the
    caller passes logits to :meth:`forward`.
    """

    def __init__(self, comm, num_experts, hidden, inter, tokens, router_weight=None, **kw):
        self.ep = MoEExpertParallel(comm, num_experts, hidden, inter, tokens, **kw)
        self.router_weight = router_weight

    def _logits(self, x, logits):
        if logits is None:
            if self.router_weight is None:
                raise ValueError("either logits or a router weight is needed")
            logits = (x.float() @ self.router_weight.float().t()).contiguous()
        return logits

    def forward(self, x, logits=None):
        return self.ep.forward(x, self._logits(x, logits))

    def decode(self, x, logits=None):
        """The same layer for a few decoded tokens, however many (see :meth:`MoEExpertParallel.decode`)."""
        return self.ep.decode(x, self._logits(x, logits))

    __call__ = forward


class MoEBlock:
    """The FFN block of a transformer around a :class:`MoELayer` with a router weight: RMS norm in front of the experts, RMS norm
    of their output, a gate and a residual scale (``residual + scale * gate * norm(experts(norm(residual)))``), and the norm in
    front of the next block where ``next_weight`` is given.

    ``pre_weight``, ``post_weight``, ``next_weight`` [H] and ``gate`` (per channel, token or element; optional) as
    :func:`~rbruck_alltoallv_b200.ops.norm.block_norm` takes them; the residual is bf16 or fp32.  The experts and their router
    have no backward pass: a call that would need one (the normed input, the router or the experts' weights require a gradient) is refused."""

    def __init__(self, layer: MoELayer, pre_weight, post_weight, gate=None, scale=1.0, next_weight=None, eps=1e-6):
        if layer.router_weight is None:
            raise ValueError("the block's layer needs a router weight")
        self.layer, self.pre_weight, self.post_weight, self.gate = layer, pre_weight, post_weight, gate
        self.scale, self.next_weight, self.eps = scale, next_weight, eps

    def forward(self, residual, normed=None, decode=False):
        """``(residual, normed)`` behind the block from those in front of it; ``normed`` may be left out for the first block.
        ``decode``: any number of tokens up to 64, through the layer's :meth:`~MoELayer.decode`."""
        if normed is None:                     # (with no block's output in 16 bits the weight has the residual's type or is fp32)
            weight = self.pre_weight.float() if residual.dtype == torch.float32 else self.pre_weight
            _, normed = block_norm(residual, pre_weight=weight, eps=self.eps)
        ep = self.layer.ep
        if torch.is_grad_enabled() and any(t.requires_grad for t in (normed, self.layer.router_weight, ep.w13, ep.w2)):
            raise ValueError("the experts have no backward pass: call the block under torch.no_grad(), or with an input norm, a router "
                             "and experts that want no gradient")
        normed = normed.to(torch.bfloat16)
        out = self.layer.decode(normed) if decode else self.layer(normed)
        return block_norm(residual, out, self.post_weight, self.gate, self.scale, self.next_weight, self.eps)

    __call__ = forward


def smoke_moe(comm=None):
    """Tiny single-GPU forward checked against the fp32 reference."""
    from ..parallel.comm import Communicator
    own = Communicator(nranks=1, heap_bytes=256 << 20, arena_bytes=1 << 20)
    try:
        T, H, I, E = 256, 256, 512, 8
        layer = MoELayer(own, E, H, I, T, seed=1)
        g = torch.Generator(device="cuda")
        g.manual_seed(7)
        x = torch.randn(T, H, device="cuda", generator=g).to(torch.bfloat16)
        logits = torch.randn(T, E, device="cuda", generator=g)
        out = layer(x, logits)
        layer.ep.check()
        ref, _, _ = reference_forward(x, logits, layer.ep.w13, layer.ep.w2)
        err = (out.float() - ref).abs().max().item()
        scale = ref.abs().max().item()
        assert err <= 0.02 * scale + 1e-3, f"MoE smoke mismatch: max err {err} vs scale {scale}"
        # the same layer with MXFP8 expert GEMMs (hardware block scaling, fused SwiGLU + quantiser epilogue)
        mx = MoELayer(own, E, H, I, T, seed=1, fp8="mx")
        out = mx(x, logits)
        mx.ep.check()
        rel = (out.float() - ref).norm().item() / ref.norm().item()
        assert rel < 0.08, f"MXFP8 MoE smoke deviates {rel:.3f} from the fp32 reference"
        # a few decoded tokens, int8 experts, an int8 projection, and the block around the layer, forward and backward of its norms
        few = layer.decode(x[:5], logits[:5])
        assert (few.float() - ref[:5]).abs().max().item() <= 0.02 * scale + 1e-3, "few-token MoE smoke mismatch"
        i8 = MoELayer(own, E, H, I, T, seed=1, fp8="int8")
        rel = (i8(x, logits).float() - ref).norm().item() / ref.norm().item()
        i8.ep.check()
        assert rel < 0.08, f"int8 MoE smoke deviates {rel:.3f} from the fp32 reference"
        w = torch.randn(I, H, device="cuda", generator=g)
        y, want = linear_int8(x[:3], *quantize_weight_int8(w)).float(), x[:3].float() @ w.t()
        assert (y - want).norm() < 0.03 * want.norm(), "int8 linear smoke mismatch"
        layer.router_weight = torch.randn(E, H, device="cuda", generator=g)
        ones = torch.ones(H, device="cuda")
        r, u = MoEBlock(layer, ones, ones, scale=0.5, next_weight=ones)(x)
        layer.ep.check()
        assert r.shape == u.shape == x.shape and u.isfinite().all()
        z = torch.randn(T, H, device="cuda", generator=g).requires_grad_()
        (dz,) = torch.autograd.grad(block_norm(r.float(), z, ones)[0].sum(), z)
        # (a norm does not change with its input's length: its gradient has no part along it, but for eps)
        assert ((dz * z).sum(-1).abs() <= 1e-4 * dz.norm(dim=-1) * z.norm(dim=-1)).all()
    finally:
        own.close()
