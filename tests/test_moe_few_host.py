"""The few-token MoE layer without a GPU: what is refused."""
import pytest
import torch

from rbruck_alltoallv_b200.ops.moe import moe_few_tokens

BF = torch.bfloat16


def _args(T=3, H=16, I=24, E=4):
    return dict(x=torch.zeros(T, H, dtype=BF), logits=torch.zeros(T, E), w13=torch.zeros(E, 2 * I, H, dtype=BF),
                w2=torch.zeros(E, H, I, dtype=BF))


@pytest.mark.parametrize("change,words", [
    (dict(x=torch.zeros(16, dtype=BF)), "are wanted"),
    (dict(x=torch.zeros(3, 16)), "must be bf16"),
    (dict(logits=torch.zeros(3, 4, dtype=BF)), "logits fp32"),
    (dict(logits=torch.zeros(3, 5)), "do not fit"),
    (dict(w13=torch.zeros(4, 24, 16, dtype=BF)), "do not fit"),
    (dict(w2=torch.zeros(4, 8, 24, dtype=BF)), "do not fit"),
    (_args(T=65), "at most 64"),
    (_args(H=12), "multiples of 8"),
    (_args(I=20), "multiples of 8"),
    (_args(E=257), "at most 256"),
    (dict(top_k=0), "top_k"),
    (dict(top_k=5), "top_k"),
    ({**_args(E=16), "top_k": 9}, "top_k"),
    (dict(w2=torch.zeros(4, 24, 16, dtype=BF).transpose(1, 2)), "contiguous"),
    (dict(w13=torch.zeros(4 * 48 * 16 + 1, dtype=BF)[1:].view(4, 48, 16)), "16-byte aligned"),
    (dict(x=torch.zeros(3, 16, dtype=BF, requires_grad=True)), "no backward pass"),
    (dict(logits=torch.zeros(3, 4, requires_grad=True)), "no backward pass"),
    (dict(), "on one GPU"),
])
def test_refusals(change, words):
    with pytest.raises(ValueError, match=words):
        moe_few_tokens(**{**_args(), **change})


@pytest.mark.parametrize("name", ["w13", "w2"])
def test_weights_that_want_a_gradient_are_refused(name):
    args = _args()
    args[name].requires_grad_()
    with pytest.raises(ValueError, match="no backward pass"):
        moe_few_tokens(**args)
    with torch.no_grad(), pytest.raises(ValueError, match="on one GPU"):
        moe_few_tokens(**args)


@pytest.mark.parametrize("name", ["x", "logits", "w13", "w2"])
def test_tangents_are_refused(name):
    """There is no forward-mode derivative: a dual number's tangent must not be dropped."""
    import torch.autograd.forward_ad as fwd
    args = _args()
    with fwd.dual_level():
        args[name] = fwd.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(ValueError, match="forward-mode"):
            moe_few_tokens(**args)
        args[name] = fwd.unpack_dual(args[name]).primal
        with pytest.raises(ValueError, match="on one GPU"):
            moe_few_tokens(**args)
