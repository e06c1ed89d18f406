"""GPU tests of the 8-bit integer products.

The quantised values and scales are compared bit for bit with x / s in 32 bits.  The products' integer sums are exact, so
against 64 bits a result is off by its rounding to bf16 (2^-8 of it) and three roundings in 32 bits (of the sum, and of two
products; 2^-22 is allowed); with SwiGLU by what those do to gate and up (|silu'| <= 1.1) and 2^-20 for the exponential and
the division."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, I8, I32 = torch.bfloat16, torch.int8, torch.int32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _plain_rows(x):
    f = x.float()
    most = f.abs().amax(-1)
    # (a division of tensors: torch divides by a Python number by multiplying with its rounded reciprocal, which is not max / 127)
    s = torch.where(most > 0, most / torch.full_like(most, 127.0), torch.ones_like(most))
    return torch.round(f / s[:, None]).clamp(-127, 127).to(I8), s


def _rows(M, K, seed=0):
    g = _gen(seed)
    x = torch.randn(M, K, device="cuda", generator=g) * torch.exp(2 * torch.randn(M, 1, device="cuda", generator=g))
    return x.to(BF)


def _weight(shape, seed=1):
    g = _gen(seed)
    w = torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int16).to(I8)
    return w, (0.5 + torch.rand(shape[:-1], device="cuda", generator=g)) * 1e-3


def _want(q, s, w, c, swiglu=False):
    """(value, bound before the last rounding)"""
    y = (q.double() @ w.double().t()) * s.double()[:, None] * c.double()
    err = y.abs() * 2.0 ** -22
    if swiglu:
        gate, up = y[:, 0::2], y[:, 1::2]
        err = 1.1 * up.abs() * err[:, 0::2] + gate.abs() * err[:, 1::2]
        y = torch.nn.functional.silu(gate) * up
        err = err + y.abs() * 2.0 ** -20
    return y, err


def _check(got, want):
    y, err = want
    assert got.shape == y.shape
    bad = ~((got.double() - y).abs() <= (y.abs() + err) * 2.0 ** -8 + err + 1e-38)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, first {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("M,K", [(1, 16), (3, 256), (2, 272), (5, 4096), (700, 1408), (4, 8208), (3, 16384), (2, 20000), (1, 131072), (40000, 32)])
def test_rows_bit_for_bit(M, K):
    from rbruck_alltoallv_b200.ops.moe import quantize_rows_int8
    x = _rows(M, K, seed=K)
    q, s = quantize_rows_int8(x)
    want, ws = _plain_rows(x)
    assert torch.equal(s, ws) and torch.equal(q, want)


def test_rows_next_to_halves():
    """Values whose quotient is a half, or next to one: every bf16 in a binade against several maxima."""
    from rbruck_alltoallv_b200.ops.moe import quantize_rows_int8
    v = torch.arange(128, 256, device="cuda").float()
    values = torch.cat([v * 2.0 ** -p for p in range(0, 14)])
    values = torch.cat([values, -values, torch.zeros(64, device="cuda")])
    top = torch.arange(128, 256, device="cuda").float() * 2.0
    x = torch.cat([values.expand(128, -1), top[:, None].expand(128, 16)], dim=1).to(BF)
    x = torch.minimum(torch.maximum(x, -x[:, -1:]), x[:, -1:]).contiguous()
    q, s = quantize_rows_int8(x)
    want, ws = _plain_rows(x)
    assert torch.equal(s, ws) and torch.equal(q, want)


def test_rows_strides_used_and_odd_rows():
    from rbruck_alltoallv_b200.ops.moe import dequantize_int8, quantize_rows_int8
    x = _rows(20, 64)
    want, ws = _plain_rows(x)
    for off in (0, 8, 3):
        wide = torch.zeros(20, 100 + 4, dtype=BF, device="cuda")
        wide[:, off:off + 64] = x
        q, s = quantize_rows_int8(wide[:, off:off + 64])
        assert torch.equal(q, want) and torch.equal(s, ws)
    q, s = quantize_rows_int8(x.t().contiguous().t())
    assert torch.equal(q, want) and torch.equal(s, ws)
    q, s = quantize_rows_int8(x, torch.tensor([7], dtype=I32, device="cuda"))
    assert torch.equal(q[:7], want[:7]) and torch.equal(s[:7], ws[:7])
    x[0], x[1], x[2, 5], x[3, 6], x[4, 0] = 0, 2.0 ** -120, math.nan, math.inf, -math.inf
    x[5] = torch.finfo(BF).max
    q, s = quantize_rows_int8(x)
    assert (q[:2] == 0).all() and (s[:2] == 1).all() and s[2:5].isnan().all() and (q[5] == 127).all() and s[5].isfinite()
    assert torch.equal(q[6:], want[6:]) and dequantize_int8(q, s)[2:5].isnan().all()
    q, s = quantize_rows_int8(x[:0])
    assert q.shape == (0, 64) and s.shape == (0,)


LINEAR = [(8, 16), (256, 4096), (1000, 2816), (4096, 512), (264, 14336), (72, 1040), (28672, 256), (16, 131072)]


@pytest.mark.parametrize("M", [1, 2, 8, 9, 16, 17, 32, 33, 64, 65, 77, 300])
@pytest.mark.parametrize("N,K", LINEAR)
def test_linear(M, N, K):
    from rbruck_alltoallv_b200.ops.moe import linear_int8
    x, (w, c) = _rows(M, K, seed=M), _weight((N, K), seed=N)
    err = torch.zeros(1, dtype=I32, device="cuda")
    got = linear_int8(x, w, c, error=err)
    assert err.item() == 0
    _check(got, _want(*_plain_rows(x), w, c))


@pytest.mark.parametrize("M,K", [(1, 4096), (1, 16), (2, 2048), (3, 1360), (4, 1024), (5, 816), (8, 512), (8, 528), (7, 400), (1, 4112)])
def test_linear_rows_quantised_by_every_cta(M, K):
    from rbruck_alltoallv_b200.ops.moe import linear_int8
    wide = torch.zeros(M, K + 24, dtype=BF, device="cuda")
    x, (w, c) = wide[:, 8:8 + K], _weight((264, K), seed=K)
    x.copy_(_rows(M, K, seed=M))
    q, s = _plain_rows(x)
    _check(linear_int8(x, w, c), _want(q, s, w, c))
    x[0] = 0
    x[M - 1, K // 2] = float("nan") if M % 2 else float("inf")
    got = linear_int8(x, w, c)
    assert got[M - 1].isnan().all() and (M == 1 or (got[0] == 0).all())
    _check(got[1:M - 1], _want(q[1:M - 1], s[1:M - 1], w, c)) if M > 2 else None


def test_linear_right_behind_the_kernel_that_makes_its_weights():
    from rbruck_alltoallv_b200.ops.moe import linear_int8, quantize_rows_int8
    x, one, two = _rows(1, 4096, seed=1), _rows(4096, 4096, seed=2), _rows(4096, 4096, seed=3)
    wants = [linear_int8(x, *quantize_rows_int8(v)) for v in (one, two)]
    torch.cuda.synchronize()
    for v, want in [(one, wants[0]), (two, wants[1])] * 10:
        assert torch.equal(linear_int8(x, *quantize_rows_int8(v)), want)


@pytest.mark.parametrize("M,N,K", [(65, 1016, 11136), (96, 256, 8208), (160, 4096, 14336), (200, 264, 5120), (520, 520, 4096), (1300, 2048, 4096),
                                   (4700, 4096, 1024), (3, 28672, 4096), (40, 9608, 3600), (64, 14336, 1040)])
def test_linear_more_sizes(M, N, K):
    """Tiles that do not fill the SMs, or just more than fill them; twice, for what a call leaves behind."""
    from rbruck_alltoallv_b200.ops.moe import linear_int8
    x, (w, c) = _rows(M, K, seed=M), _weight((N, K), seed=N)
    want = _want(*_plain_rows(x), w, c)
    for _ in range(2):
        _check(linear_int8(x, w, c), want)


def test_linear_extremes_are_exact():
    """The largest sum of the largest depth, 131072 * 127 * 127, and its negative."""
    from rbruck_alltoallv_b200.ops.moe import linear_int8
    K = 131072
    w = torch.full((16, K), 127, dtype=I8, device="cuda")
    w[1] = -127
    for M in (1, 70):
        x = torch.ones(M, K, dtype=BF, device="cuda")
        got = linear_int8(x, w, torch.ones(16, device="cuda"))
        want = torch.full((M, 16), 127.0 * 127 * K * (1 / 127.0), device="cuda")
        want[:, 1] *= -1
        assert torch.equal(got, want.to(BF))


def test_linear_strides_out_and_bad_rows():
    from rbruck_alltoallv_b200.ops.moe import linear_int8
    w, c = _weight((48, 96))
    for M in (5, 80):
        x = _rows(M, 96)
        want = linear_int8(x, w, c)
        wide = torch.zeros(M, 160, dtype=BF, device="cuda")
        wide[:, 8:104] = x
        out = torch.full((M + 2, 48), 7.0, dtype=BF, device="cuda")
        assert torch.equal(linear_int8(wide[:, 8:104], w, c, out=out[1:M + 1]), want)
        assert (out[0] == 7).all() and (out[M + 1] == 7).all() and torch.equal(out[1:M + 1], want)
        wide[:, 3:99] = x
        assert torch.equal(linear_int8(wide[:, 3:99], w, c), want)
        assert torch.equal(linear_int8(x[:1].expand(M, 96), w, c), want[:1].expand(M, 48))
        x[2, 7] = math.inf
        got = linear_int8(x, w, c)
        rest = [r for r in range(M) if r != 2]
        assert got[2].isnan().all() and torch.equal(got[rest], want[rest])
    assert linear_int8(x[:0], w, c).shape == (0, 48)


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("rows,N,K", [([1], 256, 128), ([31, 32, 33], 512, 192), ([0, 255, 0, 256, 257], 264, 272), ([288, 1, 511], 1000, 16),
                                      ([513, 1025], 256, 1040), ([5] * 64, 72, 400), ([0, 0, 3], 8, 4096), ([64, 64], 2048, 2816),
                                      ([65, 2], 4096, 256)])
def test_grouped(rows, N, K, swiglu):
    from rbruck_alltoallv_b200.ops.moe import grouped_gemm_int8
    G, M = len(rows), sum(rows)
    q, s = _plain_rows(_rows(M + 3, K, seed=M))
    w, c = _weight((G, N, K), seed=N)
    if swiglu:
        c = c * 0.05
    start = [sum(rows[:g]) for g in range(G)]
    gs, gr = (torch.tensor(v, dtype=I32, device="cuda") for v in (start, rows))
    n_out = N // 2 if swiglu else N
    wide = torch.full((M + 3, n_out + 6), 7.0, dtype=BF, device="cuda")
    out = wide[:, 2:2 + n_out]
    err = torch.zeros(1, dtype=I32, device="cuda")
    grouped_gemm_int8(q, s, w, c, gs, gr, out=out, swiglu=swiglu, error=err)
    assert err.item() == 0
    assert (out[M:] == 7).all() and (wide[:, :2] == 7).all() and (wide[:, 2 + n_out:] == 7).all()
    for g, (at, n) in enumerate(zip(start, rows)):
        if n:
            _check(out[at:at + n], _want(q[at:at + n], s[at:at + n], w[g], c[g], swiglu))


def test_groups_beyond_the_rows_are_left_out():
    from rbruck_alltoallv_b200.ops.moe import grouped_gemm_int8
    q, s = _plain_rows(_rows(40, 64))
    w, c = _weight((2, 64, 64))
    gs, gr = torch.tensor([0, 30], dtype=I32, device="cuda"), torch.tensor([30, 50], dtype=I32, device="cuda")
    err = torch.zeros(1, dtype=I32, device="cuda")
    out = grouped_gemm_int8(q, s, w, c, gs, gr, error=err)
    _check(out[30:], _want(q[30:], s[30:], w[1], c[1]))
    assert err.item() == 6
    err.zero_()
    out = torch.full((40, 64), 7.0, dtype=BF, device="cuda")
    grouped_gemm_int8(q, s, w, c, torch.tensor([-5, 20], dtype=I32, device="cuda"), torch.tensor([10, 20], dtype=I32, device="cuda"),
                      out=out, error=err)
    assert err.item() == 6 and (out[:20] == 7).all()
    _check(out[20:], _want(q[20:], s[20:], w[1], c[1]))
    with pytest.raises(ValueError, match="error must be"):
        grouped_gemm_int8(q, s, w, c, gs, gr, error=torch.zeros(1, dtype=I32))


def test_streams_and_graphs():
    from rbruck_alltoallv_b200.ops.moe import linear_int8
    w, c = _weight((1024, 2048))
    for M in (3, 100):
        x, y = _rows(M, 2048, seed=1), _rows(M, 2048, seed=2)
        want, want_y = linear_int8(x, w, c), linear_int8(y, w, c)
        one, two = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        got = []
        for _ in range(20):
            with torch.cuda.stream(one):
                a = linear_int8(x, w, c)
            with torch.cuda.stream(two):
                b = linear_int8(y, w, c)
            got.append((a, b))
        torch.cuda.synchronize()
        assert all(torch.equal(a, want) and torch.equal(b, want_y) for a, b in got)
        g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g1):
            a = linear_int8(x, w, c)
        with torch.cuda.graph(g2):
            b = linear_int8(y, w, c)
        x.mul_(-3.0)
        want = linear_int8(x, w, c)
        torch.cuda.synchronize()
        for _ in range(5):
            with torch.cuda.stream(one):
                g1.replay()
            with torch.cuda.stream(two):
                g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want_y)


@pytest.mark.parametrize("T,H,I,E", [(64, 256, 512, 8), (33, 272, 1040, 4), (500, 512, 256, 16)])
def test_layer_with_int8_experts(T, H, I, E):
    """The layer against the same steps in 64 bits with the same quantisers: two roundings to bf16 (the FFN's intermediate, which
    may move a quantised value by one step of 1/127 of the row's largest, and the expert's result) before the last one."""
    from rbruck_alltoallv_b200.models.moe_layer import MoELayer
    from rbruck_alltoallv_b200.parallel.comm import Communicator
    comm = Communicator(nranks=1, heap_bytes=64 << 20, arena_bytes=1 << 20)
    try:
        layer = MoELayer(comm, E, H, I, T, seed=3, fp8="int8")
        ep = layer.ep
        x = torch.randn(T, H, device="cuda", generator=_gen(8)).to(BF)
        logits = torch.randn(T, E, device="cuda", generator=_gen(9))
        got = layer(x, logits)
        ep.check()
        p, which = torch.topk(torch.softmax(logits.double(), -1), 2, dim=-1)
        p = p / p.sum(-1, keepdim=True)
        want, bound = torch.zeros(T, H, dtype=torch.float64, device="cuda"), torch.zeros(T, H, dtype=torch.float64, device="cuda")
        for e in range(E):
            rows, k = (which == e).nonzero(as_tuple=True)
            if not len(rows):
                continue
            q, s = _plain_rows(x[rows])
            mid, _ = _want(q, s, ep.w13_q[e], ep.w13_s[e], True)
            hq, hs = _plain_rows(mid.to(BF))
            w2 = ep.w2_q[e].double()
            y = (hq.double() @ w2.t()) * hs.double()[:, None] * ep.w2_s[e].double()
            # every intermediate value off by one bf16 step at most (2^-7 of it) and so by that plus one quantisation step
            step = mid.abs() * 2.0 ** -7 + hs.double()[:, None] * 1.01
            off = ((step != 0) * step) @ w2.abs().t() * ep.w2_s[e].double()
            want.index_add_(0, rows, p[rows, k, None] * y)
            bound.index_add_(0, rows, p[rows, k, None] * (off + y.abs() * 2.0 ** -7))
        assert ((got.double() - want).abs() <= bound + want.abs() * 2.0 ** -7).all()
        # and far closer than that bound as a whole: hardly a value moves
        assert (got.double() - want).norm() <= 0.02 * want.norm()
    finally:
        comm.close()


@pytest.mark.parametrize("M,K", [(1, 4096), (2, 2048), (8, 512), (7, 528), (1, 4112), (40, 4096), (64, 1024), (80, 2048)])
def test_linear_in_place(M, K):
    """Results over the rows they are made of, wholly and in part, while another stream keeps SMs busy, so that CTAs start one after
    the other: nobody may read a row that somebody has written over."""
    from rbruck_alltoallv_b200.ops.moe import linear_int8
    w, c = _weight((K, K), seed=K)
    x = _rows(M, K, seed=M)
    want = linear_int8(x, w, c)
    big, side = torch.randn(4096, 4096, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(10):
        both = torch.zeros(M * K + 8 * K, dtype=BF, device="cuda")
        at = i % 2 * 8 * (K // 16)
        y, out = both[:M * K].view(M, K), both[at:at + M * K].view(M, K)
        y.copy_(x)
        with torch.cuda.stream(side):
            big @ big
        assert torch.equal(linear_int8(y, w, c, out=out), want)
    side.synchronize()


def test_results_over_operands_are_refused():
    from rbruck_alltoallv_b200.ops.moe import grouped_gemm_int8, linear_int8
    raw = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    as_bf = lambda at, *shape: raw[at:].view(BF)[:math.prod(shape)].view(shape)
    w, c = raw[:64 * 64].view(I8).view(64, 64), raw[4096:4096 + 256].view(torch.float32)
    for M in (4, 70):
        x = _rows(M, 64)
        for at in (0, 2048, 4096, 4096 + 240):
            with pytest.raises(ValueError, match="must not share memory"):
                linear_int8(x, w, c, out=as_bf(at, M, 64))
        linear_int8(x, w, c, out=as_bf(4096 + 256, M, 64))              # right behind them
    q, s = raw[8192:8192 + 70 * 64].view(I8).view(70, 64), torch.ones(70, device="cuda")
    gs, gr = torch.zeros(1, dtype=I32, device="cuda"), torch.full((1,), 70, dtype=I32, device="cuda")
    for at in (0, 4096, 8192, 8192 + 70 * 64 - 16):
        with pytest.raises(ValueError, match="must not share memory"):
            grouped_gemm_int8(q, s, w[None], c[None], gs, gr, out=as_bf(at, 70, 64))
    for at in (0, 16):
        with pytest.raises(ValueError, match="must not share memory"):
            grouped_gemm_int8(_plain_rows(_rows(70, 64))[0], raw[16384:16384 + 280].view(torch.float32), w[None].clone(), c[None].clone(), gs, gr,
                              out=as_bf(16384 + at, 70, 64))
    grouped_gemm_int8(q, s, w[None], c[None], gs, gr, out=as_bf(16384, 70, 64))


@pytest.mark.parametrize("M", [3, 70])
@pytest.mark.parametrize("which", ["linear", "grouped", "moe"])
def test_results_written_over_what_a_graph_has_saved(M, which):
    """Autograd has to learn that ``out`` was written: a gradient made from the new values would be wrong without a word."""
    from rbruck_alltoallv_b200.ops.moe import grouped_gemm_int8, linear_int8, moe_few_tokens
    from rbruck_alltoallv_b200.ops.norm import block_norm
    if which == "moe":
        M = min(M, 64)
    (w, c), x = _weight((64, 64)), _rows(M, 64)
    q, s = _plain_rows(x)
    gs, gr = torch.zeros(1, dtype=I32, device="cuda"), torch.full((1,), M, dtype=I32, device="cuda")
    w13, w2, logits = _rows(2 * 2 * 40, 64).view(2, 80, 64), _rows(2 * 64, 40).view(2, 64, 40), torch.zeros(M, 2, device="cuda")
    call = {"linear": lambda out: linear_int8(x, w, c, out=out), "grouped": lambda out: grouped_gemm_int8(q, s, w[None], c[None], gs, gr, out=out),
            "moe": lambda out: moe_few_tokens(x, logits, w13, w2, out=out)}[which]
    out, weight = torch.empty(M, 64, dtype=BF, device="cuda"), torch.ones(64, device="cuda", requires_grad=True)
    call(out)
    r, _ = block_norm(torch.zeros(M, 64, dtype=BF, device="cuda"), out, weight)
    call(out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.float().sum().backward()
    with pytest.raises(ValueError, match="no backward pass"):
        call(torch.empty(M, 64, dtype=BF, device="cuda", requires_grad=True))
    with torch.inference_mode():
        call(torch.empty(M, 64, dtype=BF, device="cuda"))


def test_offsets_beyond_32_bits():
    """Rows, weights and results of more than 2^31 elements each: their last parts, from 64 bits."""
    from rbruck_alltoallv_b200.ops.moe import grouped_gemm_int8, linear_int8, quantize_rows_int8
    K = 16384
    M = 2 ** 31 // K + 5
    x = torch.zeros(M, K, dtype=BF, device="cuda")
    x[-5:] = _rows(5, K)
    q, s = quantize_rows_int8(x)
    want, ws = _plain_rows(x[-5:])
    assert torch.equal(q[-5:], want) and torch.equal(s[-5:], ws) and (q[:-5] == 0).all()
    del x
    N = 2 ** 31 // K + 8                                     # the rows' integers as weights of as many channels
    w, c = torch.zeros(N, K, dtype=I8, device="cuda"), torch.ones(N, device="cuda")
    w[-16:], c[-16:] = _weight((16, K))
    for rows in (3, 70):
        y = _rows(rows, K, seed=rows)
        got = linear_int8(y, w, c)
        _check(got[:, -16:], _want(*_plain_rows(y), w[-16:], c[-16:]))
        assert (got[:, :-16] == 0).all()
    del w, q
    rows, N = 2 ** 31 // 32768 + 70, 32768                   # results
    (w, c), y = _weight((N, 16)), _rows(rows, 16)
    q, s = _plain_rows(y)
    gs, gr = torch.tensor([0, rows - 70], dtype=I32, device="cuda"), torch.tensor([rows - 70, 70], dtype=I32, device="cuda")
    got = grouped_gemm_int8(q, s, torch.stack([w, w]), torch.stack([c, c]), gs, gr)
    for at in (0, rows - 200, rows - 100):
        _check(got[at:at + 100], _want(q[at:at + 100], s[at:at + 100], w, c))
