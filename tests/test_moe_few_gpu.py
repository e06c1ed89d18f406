"""GPU tests of the few-token MoE layer against its definition in 64 bits (``moe_few_oracle``)."""
import math

import pytest
import torch

import moe_few_oracle

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _make(T, H, I, E, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=g) * std
    return (normal(T, H).to(BF), normal(T, E), normal(E, 2 * I, H, std=0.05).to(BF), normal(E, H, I, std=0.05).to(BF))


def _check(x, logits, w13, w2, top_k, got=None):
    from rbruck_alltoallv_b200.ops.moe import moe_few_tokens
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    if got is None:
        got = moe_few_tokens(x, logits, w13, w2, top_k, error=err)
    want, bound = moe_few_oracle.layer(x, logits, w13, w2, top_k)
    assert err.item() == 0 and got.shape == want.shape
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan)
    bad = ~((got.double() - want).abs() <= (want.abs() + bound) * 2.0 ** -8 + bound) & ~nan
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, first {bad.nonzero()[0].tolist()}"
    return got


@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 16, 17, 31, 32, 33, 64])
@pytest.mark.parametrize("H,I,E,k", [(256, 512, 8, 2), (8, 8, 2, 1), (72, 1000, 5, 3), (520, 264, 64, 6), (1024, 2816, 32, 8)])
def test_layer(T, H, I, E, k):
    _check(*_make(T, H, I, E, seed=T * 1000 + H), k)


def test_large_layers():
    _check(*_make(1, 2048, 1408, 64), 2)
    _check(*_make(40, 4096, 14336, 4), 2)
    _check(*_make(3, 5120, 1536, 160), 8)


def test_every_token_on_one_expert():
    for T in (5, 30, 50, 64):
        x, logits, w13, w2 = _make(T, 256, 192, 16, seed=T)
        logits[:, 11] = 9.0
        _check(x, logits, w13, w2, 1)
        _check(x, logits, w13, w2, 4)


def test_256_experts():
    x, logits, w13, w2 = _make(64, 64, 40, 256)
    logits[3, 255], logits[4, 0] = 50.0, 50.0
    _check(x, logits, w13, w2, 8)


def test_ties_go_to_the_lower_expert():
    x, logits, w13, w2 = _make(6, 64, 64, 40)
    logits[:] = 0.5
    logits[1, 7:] = 1.0
    logits[2, 3], logits[2, 30] = -0.0, 0.0
    logits[2, 4:30] = -1.0
    logits[2, :3] = logits[2, 31:] = -1.0
    logits[3] = -3.0e38
    logits[4] = torch.finfo(torch.float32).min
    for k in (1, 2, 5):
        _check(x, logits, w13, w2, k)


def test_masked_experts_and_empty_rows():
    x, logits, w13, w2 = _make(20, 128, 72, 12)
    logits[:, 4] = -math.inf
    w13[4] = math.nan                                    # an expert that nobody may take
    logits[3] = -math.inf                                # padded slots
    logits[19] = -math.inf
    x[3] = math.nan
    logits[7, 1:] = -math.inf                            # one choice left, two
    logits[8, 2:] = -math.inf
    logits[9, 5] = math.nan
    for k in (1, 2, 4):
        got = _check(x, logits, w13, w2, k)
        assert (got[3] == 0).all() and (got[19] == 0).all() and got[9].isnan().all()
    got = _check(x, torch.full_like(logits, -math.inf), w13, w2, 2)
    assert (got == 0).all()


def test_infinite_logits_and_results_in_place():
    from rbruck_alltoallv_b200.ops.moe import moe_few_tokens
    x, logits, w13, w2 = _make(18, 64, 40, 6)
    want = moe_few_tokens(x, logits, w13, w2)
    logits[4, 2] = math.inf
    got = moe_few_tokens(x, logits, w13, w2)
    others = [t for t in range(18) if t != 4]
    assert got[4].isnan().all() and torch.equal(got[others], want[others])
    y = x.clone()
    assert moe_few_tokens(y, logits, w13, w2, out=y) is not None and torch.equal(y[others], want[others])
    with pytest.raises(ValueError, match="error must be"):
        moe_few_tokens(x, logits, w13, w2, error=torch.zeros(1, dtype=torch.int32))


def test_a_bad_token_stays_alone():
    from rbruck_alltoallv_b200.ops.moe import moe_few_tokens
    x, logits, w13, w2 = _make(24, 256, 128, 4)
    clean = moe_few_tokens(x, logits, w13, w2)
    x[5, 17], x[6, 200] = math.nan, math.inf
    got = moe_few_tokens(x, logits, w13, w2)
    others = [t for t in range(24) if t not in (5, 6)]
    assert torch.equal(got[others], clean[others]) and got[5].isnan().all()


@pytest.mark.parametrize("T", [2, 9, 16, 30, 64])
def test_bad_tokens_stay_alone_in_every_size_of_batch(T):
    from rbruck_alltoallv_b200.ops.moe import moe_few_tokens
    x, logits, w13, w2 = _make(T, 264, 136, 5)
    logits[T - 1] = logits[0]                            # on the same experts
    logits[T // 2] = -math.inf                           # a padded slot with anything in it
    clean = moe_few_tokens(x, logits, w13, w2)
    x[0, 3], x[T // 2] = math.inf, math.nan
    got = moe_few_tokens(x, logits, w13, w2)
    assert not got[0].isfinite().all()
    assert torch.equal(got[1:], clean[1:]) and (got[T // 2] == 0).all()


def test_strides_out_and_no_tokens():
    from rbruck_alltoallv_b200.ops.moe import moe_few_tokens
    x, logits, w13, w2 = _make(10, 128, 64, 8)
    want = moe_few_tokens(x, logits, w13, w2)
    for off in (0, 8, 3):
        wide, wl = torch.zeros(10, 200, dtype=BF, device="cuda"), torch.zeros(10, 21, device="cuda")
        wide[:, off:off + 128], wl[:, off:off + 8] = x, logits
        out = torch.full((12, 128), 7.0, dtype=BF, device="cuda")
        got = moe_few_tokens(wide[:, off:off + 128], wl[:, off:off + 8], w13, w2, out=out[1:11])
        assert torch.equal(got, want) and torch.equal(out[1:11], want) and (out[0] == 7).all() and (out[11] == 7).all()
    assert torch.equal(moe_few_tokens(x.t().contiguous().t(), logits.t().contiguous().t(), w13, w2), want)
    assert torch.equal(moe_few_tokens(x[:1].expand(10, 128), logits[:1].expand(10, 8), w13, w2), want[:1].expand(10, 128))
    assert moe_few_tokens(x[:0], logits[:0], w13, w2).shape == (0, 128)


def test_results_do_not_depend_on_the_batch_or_the_run():
    """Sums are added in a fixed order: the same call gives the same bits, again and again."""
    from rbruck_alltoallv_b200.ops.moe import moe_few_tokens
    x, logits, w13, w2 = _make(33, 1024, 704, 16)
    want = moe_few_tokens(x, logits, w13, w2)
    for _ in range(50):
        assert torch.equal(moe_few_tokens(x, logits, w13, w2), want)


def test_streams_and_graphs():
    """Two streams at once, two captured graphs replayed at once on changed inputs: every call has its own workspace."""
    from rbruck_alltoallv_b200.ops.moe import moe_few_tokens
    x, logits, w13, w2 = _make(12, 512, 1024, 16)
    y, logits_y = x.flip(0).contiguous(), logits.flip(0).contiguous()
    want, want_y = moe_few_tokens(x, logits, w13, w2), moe_few_tokens(y, logits_y, w13, w2)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        with torch.cuda.stream(one):
            a = moe_few_tokens(x, logits, w13, w2)
        with torch.cuda.stream(two):
            b = moe_few_tokens(y, logits_y, w13, w2)
        got.append((a, b))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) and torch.equal(b, want_y) for a, b in got)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        a = moe_few_tokens(x, logits, w13, w2)
    with torch.cuda.graph(g2):
        b = moe_few_tokens(y, logits_y, w13, w2)
    x.neg_()
    logits.mul_(-0.5)
    want = moe_few_tokens(x, logits, w13, w2)
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(one):
            g1.replay()
        with torch.cuda.stream(two):
            g2.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want_y)


def test_layer_decode():
    """The layer's decode() takes any number of tokens and agrees with its forward() within both paths' roundings."""
    from rbruck_alltoallv_b200.models.moe_layer import MoELayer
    from rbruck_alltoallv_b200.parallel.comm import Communicator
    comm = Communicator(nranks=1, heap_bytes=64 << 20, arena_bytes=1 << 20)
    try:
        H, I, E = 256, 512, 8
        router = torch.randn(E, H, device="cuda") * 0.1
        layer = MoELayer(comm, E, H, I, 64, seed=3, router_weight=router)
        x = torch.randn(64, H, device="cuda").to(BF)
        whole = layer(x)
        for T in (1, 5, 64):
            logits = x[:T].float() @ router.t()
            got = layer.decode(x[:T])
            _check(x[:T], logits, layer.ep.w13, layer.ep.w2, 2, got)
            _check(x[:T], logits, layer.ep.w13, layer.ep.w2, 2, layer.decode(x[:T], logits))
            # forward() rounds the FFN's result once more and does not scale before rounding: three roundings of 2^-8 of the largest value on each side would be 2^-5.4, and they do not all add up
            assert (got.float() - whole[:T].float()).abs().max() <= 2 ** -5 * whole.float().abs().max()
        layer.ep.check()
        fp8 = MoELayer(comm, E, 256, 512, 8, seed=3, fp8=True)
        with pytest.raises(ValueError, match="bf16 experts on one rank"):
            fp8.decode(x[:4], torch.zeros(4, E, device="cuda"))
    finally:
        comm.close()


def test_results_over_operands_are_refused():
    from rbruck_alltoallv_b200.ops.moe import moe_few_tokens
    x, logits, w13, w2 = _make(5, 64, 40, 8)
    shared = torch.zeros(5 * 64, dtype=BF, device="cuda")
    over = shared[:80].view(torch.float32).view(5, 8)
    over.copy_(logits)
    for scores, out in ((over, shared), (logits, w2.view(-1)[64:64 + 5 * 64]), (logits, w13.view(-1)[:5 * 64])):
        with pytest.raises(ValueError, match="must not share memory"):
            moe_few_tokens(x, scores, w13, w2, out=out.view(5, 64))


def test_a_token_alone_and_in_a_batch():
    """The cut of the work depends on the batch, and with it the order of sums: a token agrees with itself within both bounds."""
    from rbruck_alltoallv_b200.ops.moe import moe_few_tokens
    x, logits, w13, w2 = _make(64, 512, 704, 16, seed=4)
    want, bound = moe_few_oracle.layer(x, logits, w13, w2, 2)
    limit = (want.abs() + bound) * 2.0 ** -8 + bound
    whole = moe_few_tokens(x, logits, w13, w2).double()
    for n in (1, 2, 9, 17, 33):
        part = moe_few_tokens(x[:n], logits[:n], w13, w2).double()
        assert ((part - whole[:n]).abs() <= 2 * limit[:n]).all()


def test_weights_beyond_32_bits():
    E, H, I = 24, 4096, 14336                                # 2.8e9 elements of w13
    w13, w2 = torch.zeros(E, 2 * I, H, dtype=BF, device="cuda"), torch.zeros(E, H, I, dtype=BF, device="cuda")
    x, logits, a, b = _make(5, H, I, 2)
    w13[22:], w2[22:] = a, b
    scores = torch.full((5, E), -1e4, device="cuda")
    scores[:, 22:] = logits
    for T in (1, 5):
        got = _check(x[:T], scores[:T], w13, w2, 2)
        assert (got != 0).any()
