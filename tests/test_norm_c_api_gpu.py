"""The C entry of the norms around a block: tensors whose rows do not start at vectors, which the torch binding never makes."""
import ctypes as C

import pytest
import torch

import norm_oracle
from test_norm_gpu import BF, F32, HF, _close, _make

pytestmark = pytest.mark.gpu
TYPE = {BF: 0, HF: 1, F32: 2}
FULL = 3


class Norm(C.Structure):
    _fields_ = [("T", C.c_longlong)] + [(n, C.c_int) for n in "H z_type r_type gate_kind w1_f32 w2_f32 gate_f32".split()] + [
        ("scale", C.c_float), ("eps", C.c_float)] + [(n, C.c_void_p) for n in "z r w1 gate w2".split()] + [
        (n, C.c_longlong) for n in "z_ld r_ld gate_ld".split()] + [(n, C.c_void_p) for n in "rstd1 rstd2 r2 u dr2 du".split()] + [
        (n, C.c_longlong) for n in "dr2_ld du_ld".split()] + [(n, C.c_void_p) for n in "dz dr dgate dw1 dw2 partial".split()]


def _off(shape, kind, by):
    """A packed tensor `by` elements behind a 16-byte boundary."""
    n = 1
    for d in shape:
        n *= d
    return torch.full((n + 8,), 7.0, dtype=kind, device="cuda")[by:by + n].view(shape)


@pytest.mark.parametrize("which", ["dgate", "partial", "dz", "dr", "none"])
@pytest.mark.parametrize("kind", [BF, F32])
@pytest.mark.parametrize("T,H", [(300, 1024), (9, 256)])
def test_unaligned_results(T, H, kind, which):
    from rbruck_alltoallv_b200 import _native
    lib = _native.cuda_lib()
    lib.rbv_block_norm_parts.argtypes = [C.c_longlong, C.c_int, C.c_int]
    for f in (lib.rbv_block_norm, lib.rbv_block_norm_backward):
        f.argtypes, f.restype = [C.c_void_p, C.c_void_p], C.c_int
    v, dr2, du = _make(T, H, kind, F32, F32, "full", seed=T)
    keep = {"rstd1": torch.empty(T, device="cuda"), "rstd2": torch.empty(T, device="cuda"), "r2": torch.empty(T, H, device="cuda"),
            "u": torch.empty(T, H, dtype=kind, device="cuda"), "dr2": dr2, "du": du, "z": v["branch"], "r": v["residual"],
            "w1": v["post_weight"], "w2": v["pre_weight"], "gate": v["gate"]}
    parts = lib.rbv_block_norm_parts(T, H, TYPE[kind])
    for n, shape, t in (("dz", (T, H), kind), ("dr", (T, H), F32), ("dgate", (T, H), kind), ("dw1", (H,), F32), ("dw2", (H,), F32),
                        ("partial", (parts, 2, H), F32)):
        keep[n] = _off(shape, t, 1 if n == which else 0)
    call = Norm(T=T, H=H, z_type=TYPE[kind], r_type=2, gate_kind=FULL, w1_f32=1, w2_f32=1, gate_f32=kind == F32, scale=0.5, eps=1e-5,
                z_ld=H, r_ld=H, gate_ld=H, dr2_ld=H, du_ld=H, **{n: t.data_ptr() for n, t in keep.items()})
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.rbv_block_norm(C.byref(call), stream) == 0
    assert lib.rbv_block_norm_backward(C.byref(call), stream) == 0
    torch.cuda.synchronize()
    args = [v[n].double() for n in ("residual", "branch", "post_weight", "gate")]
    want = norm_oracle.backward(*args, 0.5, v["pre_weight"].double(), 1e-5, dr2.double(), du.double())
    for name, n in (("residual", "dr"), ("branch", "dz"), ("gate", "dgate"), ("post_weight", "dw1"), ("pre_weight", "dw2")):
        _close(name, keep[n], want[name])
    if which != "none":
        base = keep[which].untyped_storage()
        edge = torch.empty(0, dtype=keep[which].dtype, device="cuda").set_(base)
        assert edge[0] == 7 and (edge[keep[which].numel() + 1:] == 7).all()
