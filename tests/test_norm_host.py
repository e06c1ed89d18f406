"""The norms around a block without a GPU: what is refused, and the oracle's gradients against differences."""
import pytest
import torch

import norm_oracle
from rbruck_alltoallv_b200.ops.norm import MAX_HIDDEN, block_norm


def _args(T=4, H=16, kind=torch.bfloat16):
    return dict(residual=torch.zeros(T, H, dtype=kind), branch=torch.zeros(T, H, dtype=kind),
                post_weight=torch.ones(H), pre_weight=torch.ones(H))


@pytest.mark.parametrize("change,words", [
    (dict(residual=torch.zeros(4, 16, dtype=torch.float64)), "bf16, fp16 or fp32"),
    (dict(residual=torch.zeros(4, 16, dtype=torch.int32)), "bf16, fp16 or fp32"),
    (dict(residual=torch.zeros(4, 16, dtype=torch.float16)), "block output's type"),
    (dict(residual=torch.zeros(4, 0, dtype=torch.bfloat16)), "hidden sizes"),
    (dict(residual=torch.zeros(1, MAX_HIDDEN + 1, dtype=torch.bfloat16)), "hidden sizes"),
    (dict(residual=torch.zeros(5, 16, dtype=torch.bfloat16)), "differ in shape"),
    (dict(branch=None), "belong to a block output"),
    (dict(branch=None, post_weight=None, pre_weight=None), "nothing to do"),
    (dict(post_weight=None), "needs its norm's weight"),
    (dict(post_weight=torch.ones(15)), "post_weight must be"),
    (dict(pre_weight=torch.ones(1, 16)), "pre_weight must be"),
    (dict(pre_weight=torch.ones(16, dtype=torch.float16)), "pre_weight must be"),
    (dict(gate=torch.ones(16, dtype=torch.float64)), "gate must be"),
    (dict(gate=torch.ones(3, 1)), "does not broadcast"),
    (dict(gate=torch.ones(2, 4, 16)), "does not broadcast"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(), "on the host"),
])
def test_refusals(change, words):
    with pytest.raises(ValueError, match=words):
        block_norm(**{**_args(), **change})


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
def test_oracle_gradients_against_differences(gate):
    """Central differences in 64 bits: the step 1e-5 leaves 1e-10 of curvature and 1e-11 of rounding, of values around 1."""
    gen = torch.Generator().manual_seed(5)
    T, H, s, eps = 5, 7, 0.7, 1e-3

    def normal(*shape):
        return torch.randn(*shape, generator=gen, dtype=torch.float64)
    v = {"residual": normal(T, H), "branch": normal(T, H), "post_weight": normal(H), "pre_weight": normal(H)}
    if gate != "none":
        v["gate"] = {"channel": normal(H), "token": normal(T, 1), "full": normal(T, H)}[gate]
    dr2, du = normal(T, H), normal(T, H)

    def loss(v):
        o = norm_oracle.forward(v["residual"], v["branch"], v["post_weight"], v.get("gate"), s, v["pre_weight"], eps)
        return ((o["residual"][0] * dr2).sum() + (o["normed"][0] * du).sum()).item()
    got = norm_oracle.backward(v["residual"], v["branch"], v["post_weight"], v.get("gate"), s, v["pre_weight"], eps, dr2, du)
    for name, t in v.items():
        assert got[name][0].shape == t.shape
        for i in range(t.numel()):
            at = {}
            for sign in (1, -1):
                moved = t.clone().view(-1)
                moved[i] += sign * 1e-5
                at[sign] = loss({**v, name: moved.view_as(t)})
            assert abs((at[1] - at[-1]) / 2e-5 - got[name][0].view(-1)[i].item()) < 1e-6, name


@pytest.mark.parametrize("name", ["residual", "branch", "post_weight", "gate", "pre_weight"])
def test_tangents_are_refused(name):
    """There is no forward-mode derivative: a dual number's tangent must not be dropped."""
    import torch.autograd.forward_ad as fwd
    args = {**_args(), "gate": torch.ones(16)}
    with fwd.dual_level():
        args[name] = fwd.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(ValueError, match="forward-mode"):
            block_norm(**args)
        args[name] = fwd.unpack_dual(args[name]).primal
        with pytest.raises(ValueError, match="on the host"):
            block_norm(**args)


def test_a_learnable_scale_is_refused():
    """``scale`` is a number: a tensor that wants a gradient must not become one without a word (it can be a gate of one element)."""
    scale = torch.tensor(0.5, requires_grad=True)
    with pytest.raises(ValueError, match="scale is a number"):
        block_norm(**{**_args(), "scale": scale})
    for number in (1, 0.5, scale.detach()):
        with pytest.raises(ValueError, match="on the host"):
            block_norm(**{**_args(), "scale": number})
