"""8-bit integer products without a GPU: what is refused, and the weight quantiser."""
import pytest
import torch

from rbruck_alltoallv_b200.ops.moe import (dequantize_int8, grouped_gemm_int8, linear_int8, quantize_rows_int8,
                                           quantize_weight_int8)

BF, I8, I32 = torch.bfloat16, torch.int8, torch.int32


def _linear(M=3, N=16, K=32):
    return dict(x=torch.zeros(M, K, dtype=BF), weight=torch.zeros(N, K, dtype=I8), scale=torch.ones(N))


@pytest.mark.parametrize("change,words", [
    (dict(x=torch.zeros(3, 32)), "bf16 matrix"),
    (dict(x=torch.zeros(32, dtype=BF)), "bf16 matrix"),
    (_linear(K=24), "steps of 16"),
    (_linear(K=131088), "131072"),
    (_linear(N=12), "steps of 8"),
    (dict(weight=torch.zeros(16, 32, dtype=torch.uint8)), "int8"),
    (dict(scale=torch.ones(15)), "one fp32 scale per channel"),
    (dict(scale=torch.ones(16, dtype=BF)), "one fp32 scale per channel"),
    (dict(weight=torch.zeros(32, 16, dtype=I8).t()), "contiguous"),
    (dict(weight=torch.zeros(16 * 32 + 1, dtype=I8)[1:].view(16, 32)), "16-byte aligned"),
    (dict(x=torch.zeros(3, 32, dtype=BF, requires_grad=True)), "no backward pass"),
    (dict(), "on a GPU"),
])
def test_linear_refusals(change, words):
    with pytest.raises(ValueError, match=words):
        linear_int8(**{**_linear(), **change})


def _grouped(M=5, G=2, N=16, K=32):
    return dict(Aq=torch.zeros(M, K, dtype=I8), a_scale=torch.ones(M), Bq=torch.zeros(G, N, K, dtype=I8), b_scale=torch.ones(G, N),
                group_start=torch.zeros(G, dtype=I32), group_rows=torch.zeros(G, dtype=I32))


@pytest.mark.parametrize("change,words", [
    (dict(Aq=torch.zeros(5, 16, dtype=I8)), "rows must be int8"),
    (dict(Aq=torch.zeros(5, 32, dtype=torch.uint8)), "rows must be int8"),
    (dict(a_scale=torch.ones(4)), "rows must be int8"),
    (dict(Aq=torch.zeros(32, 5, dtype=I8).t()), "contiguous"),
    (_grouped(N=20), "steps of 8"),
    (_grouped(K=40), "steps of 16"),
    (dict(group_rows=torch.zeros(2)), "int32"),
    (dict(group_start=torch.zeros(3, dtype=I32)), "int32"),
    (_grouped(G=65), "at most 64"),
    (dict(), "on one GPU"),
])
def test_grouped_refusals(change, words):
    with pytest.raises(ValueError, match=words):
        grouped_gemm_int8(**{**_grouped(), **change})


def test_rows_refusals():
    with pytest.raises(ValueError, match="bf16 matrix"):
        quantize_rows_int8(torch.zeros(2, 32, dtype=torch.float16))
    with pytest.raises(ValueError, match="on a GPU"):
        quantize_rows_int8(torch.zeros(2, 32, dtype=BF))


def test_weight_quantiser():
    """Half a step of the scale at most (the quotient and the product back, up to 127 steps, are rounded to 24 bits: 127 * 2^-23
    of a step more), the largest value exactly at 127, zero channels with the scale 1."""
    w = torch.randn(3, 8, 48, generator=torch.Generator().manual_seed(1)).to(BF)
    w[1, 4] = 0
    q, s = quantize_weight_int8(w)
    assert q.dtype == I8 and q.shape == w.shape and s.shape == (3, 8) and s[1, 4] == 1 and (q[1, 4] == 0).all()
    assert ((dequantize_int8(q, s) - w.float()).abs() <= s[..., None] * (0.5 + 127 * 2 ** -22)).all()
    top = q.abs().amax(-1)
    assert (top[s != 1] == 127).all()


@pytest.mark.parametrize("kind", [torch.float32, BF])
def test_weight_quantiser_of_bad_and_tiny_channels(kind):
    """As for rows: a channel with a NaN or an infinity gets the scale NaN, so that whatever is made of it is NaN, and one whose
    values are all below 2^-100 zeros and the scale 1; its neighbours are what they were."""
    w = torch.randn(2, 9, 32, generator=torch.Generator().manual_seed(2)).to(kind)
    want, ws = quantize_weight_int8(w)
    w[0, 1, 3], w[0, 2, 31], w[1, 3, 0] = float("nan"), float("inf"), -float("inf")
    w[1, 4], w[1, 5], w[1, 6] = 2.0 ** -120, 0.0, 2.0 ** -119
    q, s = quantize_weight_int8(w)
    for at in ((0, 1), (0, 2), (1, 3)):
        assert s[at].isnan() and (q[at] == 0).all() and dequantize_int8(q, s)[at].isnan().all()
    for at in ((1, 4), (1, 5)):
        assert s[at] == 1 and (q[at] == 0).all()
    assert (q[1, 6] == 127).all() and s[1, 6] == w[1, 6, 0].float() / 127.0
    rest = torch.ones(2, 9, dtype=torch.bool)
    for at in ((0, 1), (0, 2), (1, 3), (1, 4), (1, 5), (1, 6)):
        rest[at] = False
    assert torch.equal(q[rest], want[rest]) and torch.equal(s[rest], ws[rest])


def test_scales_that_want_a_gradient_are_refused():
    with pytest.raises(ValueError, match="no backward pass"):
        linear_int8(**{**_linear(), "scale": torch.ones(16, requires_grad=True)})
    for name, shape in (("a_scale", (5,)), ("b_scale", (2, 16))):
        with pytest.raises(ValueError, match="no backward pass"):
            grouped_gemm_int8(**{**_grouped(), name: torch.ones(shape, requires_grad=True)})
    with torch.no_grad(), pytest.raises(ValueError, match="on a GPU"):
        linear_int8(**{**_linear(), "scale": torch.ones(16, requires_grad=True)})
    q, s = quantize_weight_int8(torch.randn(16, 32, requires_grad=True))      # a trained weight, quantised for serving
    assert not s.requires_grad
    with pytest.raises(ValueError, match="on a GPU"):
        linear_int8(torch.zeros(3, 32, dtype=BF), q, s)


@pytest.mark.parametrize("name", ["x", "scale"])
def test_tangents_are_refused(name):
    """There is no forward-mode derivative: a dual number's tangent must not be dropped."""
    import torch.autograd.forward_ad as fwd
    args = _linear()
    with fwd.dual_level():
        args[name] = fwd.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(ValueError, match="forward-mode"):
            linear_int8(**args)
        args[name] = fwd.unpack_dual(args[name]).primal
        with pytest.raises(ValueError, match="on a GPU"):
            linear_int8(**args)


@pytest.mark.parametrize("channels", [2 ** 32 + 8, 2 ** 31 - 8])
def test_channels_beyond_an_int_are_refused(channels):
    """Channel numbers, and a tile beyond them, are 32-bit integers in the kernels: 2^32 + 8 channels must not become 8."""
    weight, scale = torch.zeros(1, 16, dtype=I8).expand(channels, 16), torch.ones(1).expand(channels)
    with pytest.raises(ValueError, match="at most 2147483392 channels"):
        linear_int8(torch.zeros(3, 16, dtype=BF), weight, scale)
    per_group = channels // 64 * 8
    with pytest.raises(ValueError, match="at most 2147483392 channels"):
        grouped_gemm_int8(**{**_grouped(G=8, K=16), "Bq": weight[:per_group].expand(8, per_group, 16),
                             "b_scale": scale[:per_group].expand(8, per_group)})
