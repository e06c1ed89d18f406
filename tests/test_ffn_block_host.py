"""The FFN block around a MoE layer without a GPU: what it refuses."""
from types import SimpleNamespace

import pytest
import torch

from rbruck_alltoallv_b200.models.moe_layer import MoEBlock

H = 16


class Layer:
    """Stands where the MoE layer does; a call that reaches it has not been refused."""

    def __init__(self, trainable=""):
        self.router_weight = torch.zeros(4, H, requires_grad=trainable == "router")
        self.ep = SimpleNamespace(w13=torch.zeros(4, 16, H, requires_grad=trainable == "up"),
                                  w2=torch.zeros(4, H, 8, requires_grad=trainable == "down"))

    def __call__(self, x):
        raise LookupError("reached")

    decode = __call__


def _ones(trainable=False):
    return torch.ones(H, requires_grad=trainable)


def _normed(trainable=False):
    return torch.zeros(3, H, dtype=torch.bfloat16, requires_grad=trainable)


@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("block,normed", [
    (lambda: MoEBlock(Layer("router"), _ones(), _ones()), lambda: _normed()),
    (lambda: MoEBlock(Layer("up"), _ones(), _ones()), lambda: _normed()),
    (lambda: MoEBlock(Layer("down"), _ones(), _ones()), lambda: _normed()),
    (lambda: MoEBlock(Layer(), _ones(), _ones()), lambda: _normed(trainable=True)),
])
def test_gradients_through_the_experts_are_refused(block, normed, decode):
    """The experts have no backward pass: what they would be asked for must not be lost without a word."""
    with pytest.raises(ValueError, match="no backward pass"):
        block()(torch.zeros(3, H), normed(), decode=decode)
    with torch.no_grad(), pytest.raises(LookupError):
        block()(torch.zeros(3, H), normed(), decode=decode)


def test_gradients_around_the_experts_are_not_refused():
    block = MoEBlock(Layer(), _ones(), _ones(trainable=True), gate=_ones(trainable=True), next_weight=_ones(trainable=True))
    with pytest.raises(LookupError):
        block(torch.zeros(3, H, requires_grad=True), _normed())


@pytest.mark.parametrize("weight", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [torch.bfloat16, torch.float32])
def test_the_first_norm_takes_weights_of_either_type(weight, residual):
    """(refused for the host's tensors, not for their types)"""
    block = MoEBlock(Layer(), _ones().to(weight), _ones().to(weight))
    with pytest.raises(ValueError, match="on the host"):
        block(torch.zeros(3, H, dtype=residual))
