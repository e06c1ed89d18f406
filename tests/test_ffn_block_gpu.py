"""The operators of an FFN block together, as a model uses them: norm, experts (many tokens, a few, bf16 and int8), norm with gate
and residual; an int8 projection behind it; and a training step through the norms around a torch FFN."""
import pytest
import torch

import norm_oracle

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
H, I, E, T = 256, 512, 8, 64


@pytest.fixture
def comm():
    from rbruck_alltoallv_b200.parallel.comm import Communicator
    c = Communicator(nranks=1, heap_bytes=64 << 20, arena_bytes=1 << 20)
    yield c
    c.close()


def _weights(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [1 + 0.2 * torch.randn(H, device="cuda", generator=g) for _ in range(4)] + [torch.randn(E, H, device="cuda", generator=g) * 0.1]


def _experts(layer, u):
    """The layer in 64 bits from its bf16 weights; the choice from the same 32-bit logits."""
    ep = layer.ep
    p, which = torch.topk(torch.softmax((u.float() @ layer.router_weight.t()).double(), -1), 2, dim=-1)
    p = p / p.sum(-1, keepdim=True)
    out = torch.zeros(u.shape, dtype=torch.float64, device="cuda")
    for e in range(E):
        rows, k = (which == e).nonzero(as_tuple=True)
        gu = u[rows].double() @ ep.w13[e].double().t()
        out.index_add_(0, rows, p[rows, k, None] * ((torch.nn.functional.silu(gu[:, 0::2]) * gu[:, 1::2]) @ ep.w2[e].double().t()))
    return out


@pytest.mark.parametrize("res", [BF, F32])
@pytest.mark.parametrize("experts,decode,n", [(False, False, T), (False, True, 5), (False, True, T), ("int8", False, T)])
def test_two_blocks(comm, res, experts, decode, n):
    """Bit for bit the calls of its parts; and in 64 bits from the block's own input norm on: roundings to bf16 of the experts'
    intermediate and result and of the output (2^-8 each, 2^-6 together); with int8 experts two quantisations of operands, each
    half a step of 1/127 of the largest at most, some 0.6 % of the norm each for normal values (5 % are allowed)."""
    from rbruck_alltoallv_b200.models.moe_layer import MoEBlock, MoELayer
    from rbruck_alltoallv_b200.ops.moe import linear_int8, quantize_weight_int8
    from rbruck_alltoallv_b200.ops.norm import block_norm
    w_in, w_post, w_next, gate, router = _weights()
    layer = MoELayer(comm, E, H, I, T, seed=5, router_weight=router, fp8=experts, init_std=0.05)
    first = MoEBlock(layer, w_in, w_post, gate, 0.5, w_next, eps=1e-5)
    last = MoEBlock(layer, w_next, w_post, None, 1.0, None)
    x = torch.randn(n, H, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(res)
    r1, u1 = first(x, decode=decode)
    r2, none = last(r1, u1, decode=decode)
    layer.ep.check()
    assert none is None and r1.dtype == r2.dtype == res and u1.dtype == BF
    run = layer.decode if decode else layer
    u0 = block_norm(x, pre_weight=w_in, eps=1e-5)[1].to(BF)
    z = run(u0)
    a, b = block_norm(x, z, w_post, gate, 0.5, w_next, 1e-5)
    assert torch.equal(a, r1) and torch.equal(b, u1)
    assert torch.equal(block_norm(r1, run(u1), w_post)[0], r2)
    want = norm_oracle.forward(x.double(), _experts(layer, u0), w_post.double(), gate.double(), 0.5, w_next.double(), 1e-5)
    limit = 0.05 if experts else 2.0 ** -6
    for got, name in ((r1, "residual"), (u1, "normed")):
        assert (got.double() - want[name][0]).norm() <= limit * want[name][0].norm(), name
    head = torch.randn(72, H, device="cuda") * 0.05
    q, s = quantize_weight_int8(head)
    y, exact = linear_int8(u1, q, s).double(), u1.double() @ head.double().t()
    assert (y - exact).norm() <= 0.03 * exact.norm()


def test_decode_of_a_block_wants_bf16_experts(comm):
    from rbruck_alltoallv_b200.models.moe_layer import MoEBlock, MoELayer
    w = _weights()
    layer = MoELayer(comm, E, H, I, T, router_weight=w[4], fp8="int8")
    with pytest.raises(ValueError, match="bf16 experts"):
        MoEBlock(layer, w[0], w[1])(torch.zeros(4, H, dtype=BF, device="cuda"), decode=True)
    with pytest.raises(ValueError, match="router weight"):
        MoEBlock(MoELayer(comm, E, H, I, T), w[0], w[1])


@pytest.mark.parametrize("kind,res", [(F32, F32), (BF, F32)])
def test_training_step(kind, res):
    """Two blocks with a torch FFN between the norms, against the same network in 64 bits: the gradients agree to the roundings
    on the way: in 32 bits 2^-16 of a gradient's norm, with bf16 activations some ten roundings of 2^-8 on the longest path (0.04)."""
    from rbruck_alltoallv_b200.ops.norm import block_norm
    gen = torch.Generator(device="cuda").manual_seed(3)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, device="cuda", generator=gen) * std + mean
    n, h = 96, 160
    params = {"w_in": normal(h, std=0.1, mean=1.0)}
    for i in range(2):
        params.update({f"up{i}": normal(2 * h, h, std=h ** -0.5), f"down{i}": normal(h, h, std=h ** -0.5), f"post{i}": normal(h, std=0.1, mean=1.0),
                       f"gate{i}": normal(h, std=0.3) if i else normal(n, 1, std=0.3), f"pre{i}": normal(h, std=0.1, mean=1.0)})
    x, target = normal(n, h), normal(n, h)

    def ffn(u, up, down):
        a, b = (u @ up.t()).chunk(2, dim=-1)
        return (torch.nn.functional.silu(a) * b) @ down.t()

    def network(p, x, norm, cast):
        r, u = norm(x, None, None, None, 1.0, p["w_in"])
        for i in range(2):
            r, u = norm(r, ffn(cast(u), cast(p[f"up{i}"]), cast(p[f"down{i}"])), p[f"post{i}"], p[f"gate{i}"], 0.5, p[f"pre{i}"])
        return r, u

    def plain(r, z, w1, g, s, w2):
        if z is not None:
            r = r + s * g * w1 * z * torch.rsqrt(z.square().mean(-1, keepdim=True) + 1e-6)
        return r, r * torch.rsqrt(r.square().mean(-1, keepdim=True) + 1e-6) * w2
    leaves = {k: v.clone().requires_grad_() for k, v in params.items()}
    r, u = network(leaves, x.to(res), block_norm, lambda t: t.to(kind))
    loss = (r.float() * target).sum() + u.float().square().mean() * n
    loss.backward()
    exact = {k: v.double().requires_grad_() for k, v in params.items()}
    r, u = network(exact, x.double(), plain, lambda t: t)
    ((r * target.double()).sum() + u.square().mean() * n).backward()
    limit = 2.0 ** -16 if kind == F32 else 0.04
    for k in params:
        assert (leaves[k].grad.double() - exact[k].grad).norm() <= limit * exact[k].grad.norm(), k


@pytest.mark.parametrize("decode", [False, True])
def test_a_block_that_would_lose_a_gradient_is_refused(comm, decode):
    from rbruck_alltoallv_b200.models.moe_layer import MoEBlock, MoELayer
    w_in, w_post, w_next, gate, router = _weights()
    layer = MoELayer(comm, E, H, I, T, router_weight=router)
    x = torch.randn(T, H, device="cuda")
    for leaf in (w_in, x):
        leaf.requires_grad_()
        with pytest.raises(ValueError, match="no backward pass"):
            MoEBlock(layer, w_in, w_post, gate, 0.5, w_next)(x, decode=decode)
        with torch.no_grad():
            assert not MoEBlock(layer, w_in, w_post, gate, 0.5, w_next)(x, decode=decode)[0].requires_grad
        leaf.requires_grad_(False)
    w_post.requires_grad_()                              # behind the experts
    r, u = MoEBlock(layer, w_in, w_post, gate, 0.5, w_next)(x, decode=decode)
    (r.sum() + u.sum()).backward()
    layer.ep.check()
    assert w_post.grad.isfinite().all() and (w_post.grad != 0).any()


@pytest.mark.parametrize("decode", [False, True])
def test_weights_in_16_bits_next_to_a_residual_in_32(comm, decode):
    """Bit for bit the block with the same weights in 32 bits."""
    from rbruck_alltoallv_b200.models.moe_layer import MoEBlock, MoELayer
    *weights, router = [w.to(BF) for w in _weights()]
    layer = MoELayer(comm, E, H, I, T, router_weight=router)
    x = torch.randn(T, H, device="cuda")
    w_in, w_post, w_next, gate = weights
    got = MoEBlock(layer, w_in, w_post, gate, 0.5, w_next)(x, decode=decode)
    w_in, w_post, w_next, gate = [w.float() for w in weights]
    want = MoEBlock(layer, w_in, w_post, gate, 0.5, w_next)(x, decode=decode)
    layer.ep.check()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0].dtype == F32 and got[1].dtype == BF
