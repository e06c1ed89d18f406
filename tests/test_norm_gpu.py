"""GPU tests of the norms around a block, against their definition in 64 bits.

Bounds: a result rounded to type t is off by eps(t) / 2 of its value; the 32-bit arithmetic before that adds up to
2^-17 of the magnitude (the sum of the terms' magnitudes) that the oracle returns: the longest chain are the sums over
tokens, at most 4000 / 148 + 148 / 8 + 8 < 64 additions in a row after some twenty roundings of each term, and two
units in the last place of the reciprocal square root."""
import pytest
import torch

import norm_oracle

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _close(name, got, pair):
    value, mag = pair
    assert got.shape == value.shape, name
    eps = torch.finfo(got.dtype)
    bound = value.abs() * (eps.eps / 2) * 1.01 + mag * 2.0 ** -17 + eps.smallest_normal * eps.eps
    bad = ~((got.double() - value).abs() <= bound)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()}, first {bad.nonzero()[0].tolist()}"


def _make(T, H, kind, res, wt, gate, seed=0, lead=None):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(*shape, device="cuda", generator=g) * std + mean
    v = {"residual": normal(T, H, std=2.0).to(res), "branch": normal(T, H, std=0.5).to(kind),
         "post_weight": normal(H, mean=1.0, std=0.3).to(wt), "pre_weight": normal(H, mean=1.0, std=0.3).to(wt)}
    v["gate"] = {"none": None, "channel": normal(H).to(wt), "token": normal(T, 1).to(wt), "full": normal(T, H).to(kind)}[gate]
    return v, normal(T, H).to(res), normal(T, H).to(kind)


def _double(v):
    return [None if v[n] is None else v[n].detach().double() for n in ("residual", "branch", "post_weight", "gate", "pre_weight")]


def _check(v, dr2, du, scale=0.7, eps=1e-5):
    from rbruck_alltoallv_b200.ops.norm import block_norm
    names = [n for n in v if v[n] is not None]
    for n in names:
        v[n] = v[n].detach().requires_grad_()
    args = dict(residual=v["residual"], branch=v["branch"], post_weight=v["post_weight"], gate=v["gate"], scale=scale,
                pre_weight=v["pre_weight"], eps=eps)
    with torch.no_grad():
        plain = block_norm(**args)
    out = block_norm(**args)
    r, z, w1, g, w2 = _double(v)
    want = norm_oracle.forward(r, z, w1, g, scale, w2, eps)
    for n, a, b in zip(("residual", "normed"), plain, out):
        if n in want:
            _close(n, a, want[n])
            assert torch.equal(a, b.detach()), "with and without gradients"
    keep = [(o, d) for o, d, w in ((out[0], dr2, v["branch"] is not None), (out[1], du, w2 is not None)) if w and d is not None]
    grads = torch.autograd.grad([o for o, _ in keep], [v[n] for n in names], [d for _, d in keep], allow_unused=True)
    want = norm_oracle.backward(r, z, w1, g, scale, w2, eps, None if dr2 is None or z is None else dr2.double(),
                                None if du is None or w2 is None else du.double())
    for n, a in zip(names, grads):
        if n in want:
            assert a.dtype == v[n].dtype
            _close("gradient of " + n, a, want[n])
        else:
            assert a is None


SHAPES = [(1, 1), (1, 4096), (3, 8), (5, 257), (7, 64), (2, 1001), (130, 256), (33, 264), (300, 4104), (9, 8192), (5, 8191),
          (3, 16384), (2, 16383), (1000, 40), (3999, 96)]


@pytest.mark.parametrize("T,H", SHAPES)
@pytest.mark.parametrize("kind,res,wt,gate", [(BF, BF, BF, "channel"), (BF, F32, F32, "token"), (HF, HF, F32, "full"),
                                              (F32, F32, F32, "channel"), (HF, F32, HF, "none")])
def test_both_passes(T, H, kind, res, wt, gate):
    _check(*_make(T, H, kind, res, wt, gate, seed=T + H))


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("kind,res", [(BF, BF), (BF, F32), (HF, HF), (F32, F32)])
def test_gates_and_types(kind, res, gate):
    _check(*_make(200, 520, kind, res, kind, gate, seed=3))
    _check(*_make(20, 5000, kind, res, F32, gate, seed=4))


@pytest.mark.parametrize("drop", ["pre", "post", "dr2", "du"])
@pytest.mark.parametrize("H", [128, 131])
def test_parts_of_the_operator(drop, H):
    v, dr2, du = _make(50, H, BF, BF, F32, "none" if drop == "post" else "channel")
    if drop == "pre":
        v["pre_weight"] = None
    elif drop == "post":
        v["branch"] = v["post_weight"] = None
    elif drop == "dr2":
        dr2 = None
    else:
        du = None
    _check(v, dr2, du)


def test_scale_and_eps():
    for scale, eps in ((0.0, 1e-6), (-2.0, 1.0), (1.0, 0.0)):
        v, dr2, du = _make(17, 72, F32, F32, F32, "channel", seed=9)
        _check(v, dr2, du, scale=scale, eps=eps)


def test_zero_rows():
    """A block output of zeros (a masked token) has no direction: its norm is zero and only eps keeps the gradient finite."""
    v, dr2, du = _make(6, 64, BF, F32, F32, "channel")
    v["branch"][2] = 0
    v["branch"][4], v["residual"][4] = 0, 0
    _check(v, dr2, du, eps=1e-2)


def test_no_tokens():
    from rbruck_alltoallv_b200.ops.norm import block_norm
    v, dr2, du = _make(0, 64, BF, BF, F32, "channel")
    for n in v:
        v[n] = v[n].requires_grad_()
    out = block_norm(v["residual"], v["branch"], v["post_weight"], v["gate"], 0.5, v["pre_weight"])
    assert out[0].shape == out[1].shape == (0, 64)
    grads = torch.autograd.grad(out, list(v.values()), (dr2, du))
    assert all((g == 0).all() for g in grads)


def test_one_bad_row_stays_alone():
    from rbruck_alltoallv_b200.ops.norm import block_norm
    v, _, _ = _make(40, 256, BF, BF, F32, "token")
    clean = block_norm(v["residual"], v["branch"], v["post_weight"], v["gate"], 0.5, v["pre_weight"])
    v["branch"][7, 3], v["residual"][9, 200] = float("inf"), float("nan")
    out = block_norm(v["residual"], v["branch"], v["post_weight"], v["gate"], 0.5, v["pre_weight"])
    others = [i for i in range(40) if i not in (7, 9)]
    for a, b in zip(clean, out):
        assert torch.equal(a[others], b[others])
    assert out[0][7, 3].isnan() and out[1][9].isnan().all()


def test_strides_and_shapes():
    """Rows of a wider tensor (aligned to vectors and not), more dimensions, a gate that broadcasts in another way, a
    transposed block output, gradients that arrive expanded."""
    from rbruck_alltoallv_b200.ops.norm import block_norm
    for off in (0, 8, 3):
        v, dr2, du = _make(31, 128, BF, F32, F32, "none")
        wide = torch.zeros(31, 200, dtype=BF, device="cuda")
        wide[:, off:off + 128] = v["branch"]
        resw = torch.zeros(31, 300, device="cuda")
        resw[:, off:off + 128] = v["residual"]
        want = block_norm(v["residual"], v["branch"], v["post_weight"], None, 1.0, v["pre_weight"])
        got = block_norm(resw[:, off:off + 128], wide[:, off:off + 128], v["post_weight"], None, 1.0, v["pre_weight"])
        for a, b in zip(want, got):
            assert (a.float() - b.float()).abs().max() <= 2 ** -7 * a.float().abs().max()
        _check({**v, "branch": wide[:, off:off + 128], "residual": resw[:, off:off + 128]}, dr2, du)
        _check({**v, "branch": v["branch"].t().contiguous().t()}, dr2[:1].expand(31, 128), du[:, :1].expand(31, 128))
    v, dr2, du = _make(24, 64, HF, HF, F32, "none")
    three = {n: (t.view(2, 12, 64) if t is not None and t.dim() == 2 else t) for n, t in v.items()}
    three["gate"] = torch.randn(2, 1, 64, device="cuda")                     # one gate per sequence and channel
    _check(three, dr2.view(2, 12, 64), du.view(2, 12, 64))
    three["gate"] = torch.randn(1, device="cuda")
    _check(three, dr2.view(2, 12, 64), du.view(2, 12, 64))
    three["gate"] = torch.randn(2, 12, 1, device="cuda")
    _check(three, dr2.view(2, 12, 64), du.view(2, 12, 64))


def test_gradient_against_differences():
    """Along a random direction in 32 bits: with a step of 2^-7 the curvature is below 2^-13 and the rounding of the two
    sums of 64 x 96 terms below 2^-24 * 80 / 2^-6, both of values around 80; a hundredth is allowed."""
    from rbruck_alltoallv_b200.ops.norm import block_norm
    v, dr2, du = _make(64, 96, F32, F32, F32, "channel", seed=21)
    for n in v:
        v[n].requires_grad_()
    out = block_norm(v["residual"], v["branch"], v["post_weight"], v["gate"], 0.5, v["pre_weight"])
    grads = torch.autograd.grad(out, list(v.values()), (dr2, du))
    gen = torch.Generator(device="cuda").manual_seed(2)
    for n, g in zip(v, grads):
        way = torch.randn(v[n].shape, device="cuda", generator=gen) * g.sign().abs() + 2 * g / g.abs().max()
        way = way / way.norm() * v[n].detach().norm() / 4

        def loss(s):
            w = {**{k: t.detach() for k, t in v.items()}, n: v[n].detach() + s * way}
            a, b = block_norm(w["residual"], w["branch"], w["post_weight"], w["gate"], 0.5, w["pre_weight"])
            return (a.double() * dr2).sum() + (b.double() * du).sum()
        h = 2.0 ** -7
        slope, want = (loss(h) - loss(-h)) / (2 * h), (g.double() * way).sum()
        assert abs(slope - want) <= 0.01 * (g.double().norm() * way.double().norm()) * 0.2 + 0.01 * abs(want), n


def test_streams_and_graphs():
    """The same results on another stream, and from a captured forward and backward pass replayed on new values."""
    from rbruck_alltoallv_b200.ops.norm import block_norm
    v, dr2, du = _make(300, 512, BF, F32, F32, "channel")
    for n in v:
        v[n].requires_grad_()

    def step():
        out = block_norm(v["residual"], v["branch"], v["post_weight"], v["gate"], 0.5, v["pre_weight"])
        return [t.detach() for t in out] + list(torch.autograd.grad(out, list(v.values()), (dr2, du)))
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.cuda.graph(two):
        second = step()
    with torch.no_grad():
        v["branch"].mul_(-1.5)
        dr2.add_(0.25)
    graph.replay()
    two.replay()
    fresh = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, fresh)) and all(torch.equal(a, b) for a, b in zip(second, fresh))
    assert not torch.equal(want[0], fresh[0])


def test_some_gradients_and_no_second_ones():
    """Gradients only for what asks for them; accumulated by backward(); a graph of the backward pass is refused when it is used."""
    from rbruck_alltoallv_b200.ops.norm import block_norm
    v, dr2, du = _make(30, 72, BF, F32, F32, "channel", seed=4)
    r, z, w1, g, w2 = _double(v)
    want = norm_oracle.backward(r, z, w1, g, 0.5, w2, 1e-6, dr2.double(), du.double())
    for asked in (["gate"], ["branch"], ["residual", "pre_weight"], ["post_weight", "branch"], []):
        leaves = {n: t.detach().clone().requires_grad_(n in asked) for n, t in v.items()}
        out = block_norm(leaves["residual"], leaves["branch"], leaves["post_weight"], leaves["gate"], 0.5, leaves["pre_weight"])
        assert all(o.requires_grad == bool(asked) for o in out)
        if asked:
            torch.autograd.backward(out, (dr2, du))
        for n, t in leaves.items():
            assert (t.grad is not None) == (n in asked)
            if n in asked:
                _close(n, t.grad, want[n])
    x = v["branch"].detach().clone().requires_grad_()
    out = block_norm(v["residual"], x, v["post_weight"], v["gate"], 0.5, v["pre_weight"])
    (first,) = torch.autograd.grad(out, x, (dr2, du), create_graph=True)
    _close("branch", first.detach(), want["branch"])
    with pytest.raises(RuntimeError):                 # (autograd itself finds that nothing leads from there to x)
        torch.autograd.grad(first.float().sum(), x)
    with pytest.raises(RuntimeError, match="differentiable once"):
        first.float().sum().backward()


@pytest.mark.parametrize("T", [149, 150, 152, 300, 1189])
@pytest.mark.parametrize("H", [1024, 1032, 2048, 4096, 6144, 8200, 16384])
@pytest.mark.parametrize("kind,res,gate", [(BF, BF, "channel"), (BF, F32, "full"), (F32, F32, "token"), (HF, HF, "none")])
def test_several_rows_per_cta(T, H, kind, res, gate):
    """More rows than SMs, of 2 KB and more: the kernels with several rows in work, at the ends of their shapes."""
    if H > 8192 and T > 160:
        T = 160
    _check(*_make(T, H, kind, res, F32, gate, seed=T + H))


@pytest.mark.parametrize("kind", [BF, HF])
@pytest.mark.parametrize("shape", [(2, 1, 72), (1, 300, 1), (300, 1), (1,), (2, 300, 1)])
def test_gradient_of_a_broadcast_gate_is_rounded_once(kind, shape):
    """A gate in 16 bits that is shared by many elements: its gradient is a sum of up to 43200 terms and rounded like any other, not
    term by term.  The sum over 600 or 72 x 600 terms is torch's, a tree of 32-bit additions: within 2^-17 of the magnitudes too."""
    v, dr2, du = _make(600, 72, kind, F32, F32, "none", seed=6)
    three = {n: (t.view(2, 300, 72) if t is not None and t.dim() == 2 else t) for n, t in v.items()}
    three["gate"] = torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8)).to(kind)
    _check(three, dr2.view(2, 300, 72), du.view(2, 300, 72))


@pytest.mark.parametrize("T", [149, 300, 4800, 9500])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
def test_rows_of_one_warp(T, gate):
    """512 elements in 32 bits are the shortest rows that go several to a CTA: a group is one warp, up to 32 of them.  9500 rows are
    65 in the CTA with most, 5 a group: the chains of additions stay below 64."""
    _check(*_make(T, 512, F32, F32, F32, gate, seed=T))


@pytest.mark.parametrize("H", [8200, 12288, 16384])
@pytest.mark.parametrize("gate", ["none", "full"])
def test_rows_of_more_than_sixteen_warps(H, gate):
    _check(*_make(310, H, BF, BF, BF, gate, seed=H))


@pytest.mark.parametrize("T", [300, 1189])
@pytest.mark.parametrize("H", [131, 1001, 4097, 8191])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("kind,res", [(F32, F32), (BF, F32), (HF, HF)])
def test_widths_that_are_not_whole_vectors_over_many_rows(T, H, gate, kind, res):
    """More rows than CTAs fit at once: a CTA of single elements goes on to its next row, and sums over several."""
    _check(*_make(T, H, kind, res, F32, gate, seed=T + H))


def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the last rows are those of a call on them alone, in both passes and with a gate per element.  (Both
    calls have more rows than SMs, so that they take the same kernels; the sums over the tokens are left out.)"""
    from rbruck_alltoallv_b200.ops.norm import block_norm
    H, tail = 4096, 300
    T = 2 ** 31 // H + tail
    v, dr2, du = _make(tail, H, BF, BF, F32, "full")
    rows = {n: t for n, t in v.items() if t.dim() == 2} | {"dr2": dr2, "du": du}
    big = {}
    for n, t in rows.items():
        big[n] = torch.zeros(T, H, dtype=BF, device="cuda")
        big[n][-tail:] = t
    for s in (rows, big):
        for n in ("residual", "branch", "gate"):
            s[n].requires_grad_()
    results = []
    for s in (rows, big):
        out = block_norm(s["residual"], s["branch"], v["post_weight"], s["gate"], 0.5, v["pre_weight"])
        grads = torch.autograd.grad(out, [s["residual"], s["branch"], s["gate"]], (s["dr2"], s["du"]))
        results.append([t.detach()[-tail:] for t in (*out, *grads)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
