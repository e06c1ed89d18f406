"""The norms around a block from their definition in 64 bits, with the magnitudes that bound what 32-bit arithmetic can lose.

Every function returns {name: (value, magnitude)}: the magnitude is the same expression with every difference replaced by the
sum of its terms' magnitudes, so that an error of k roundings is at most k * 2^-24 times it."""
import torch


def forward(r, z, w1, g, s, w2, eps):
    one = torch.ones((), dtype=torch.float64, device=r.device)
    out = {}
    r2, m2 = r, r.abs()
    if z is not None:
        i1 = 1 / torch.sqrt(z.square().mean(-1, keepdim=True) + eps)
        n = s * (one if g is None else g) * w1 * z * i1
        r2, m2 = r + n, r.abs() + n.abs()
        out["residual"] = (r2, m2)
    if w2 is not None:
        i2 = 1 / torch.sqrt(r2.square().mean(-1, keepdim=True) + eps)
        out["normed"] = (r2 * i2 * w2, m2 * i2 * w2.abs())
    return out


def _to(shape, v):
    return v.sum_to_size(shape)


def backward(r, z, w1, g, s, w2, eps, dr2, du):
    one = torch.ones((), dtype=torch.float64, device=r.device)
    gg = one if g is None else g
    r2, m2, zh = r, r.abs(), None
    if z is not None:
        i1 = 1 / torch.sqrt(z.square().mean(-1, keepdim=True) + eps)
        zh = z * i1
        r2, m2 = r + s * gg * w1 * zh, r.abs() + (s * gg * w1 * zh).abs()
    out = {}
    d = torch.zeros_like(r) if dr2 is None else dr2
    dm = d.abs()
    if w2 is not None and du is not None:
        i2 = 1 / torch.sqrt(r2.square().mean(-1, keepdim=True) + eps)
        xh, xm, a = r2 * i2, m2 * i2, du * w2
        d = d + i2 * (a - xh * (a * xh).mean(-1, keepdim=True))
        dm = dm + i2 * (a.abs() + xm * (a.abs() * xm).mean(-1, keepdim=True))
        out["pre_weight"] = (_to(w2.shape, du * xh), _to(w2.shape, du.abs() * xm))
    out["residual"] = (d, dm)
    if z is not None:
        f = s * gg * w1
        b, bm = f * d, f.abs() * dm
        out["branch"] = (i1 * (b - zh * (b * zh).mean(-1, keepdim=True)), i1 * (bm + zh.abs() * (bm * zh.abs()).mean(-1, keepdim=True)))
        full = torch.broadcast_to(s * gg, r.shape)
        out["post_weight"] = (_to(w1.shape, full * d * zh), _to(w1.shape, full.abs() * dm * zh.abs()))
        if g is not None:
            out["gate"] = (_to(g.shape, s * w1 * zh * d), _to(g.shape, (abs(s) * w1.abs() * zh.abs() * dm)))
    return out
