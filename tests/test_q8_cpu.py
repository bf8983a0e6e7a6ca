"""Refusals of the 8-bit linear layers' entry points, before any device work
(fake, aligned addresses that are never dereferenced; CPU tensors at the
Python layer), and the extension of their calls beside another torch than its own."""
import pytest
import torch

from llamamps_b200 import _lib
from llamamps_b200 import kernels as K

A = 1 << 20
INVALID, UNSUPPORTED = -1, -2


def _quantise(**kw):
    v = {**dict(x=A, ldx=64, codes=A, ldc=64, scales=A, values=None, ldv=0, rows=2, k=64), **kw}
    return _lib.lib().lmps_quantise_rows_q8(v["x"], v["ldx"], v["codes"], v["ldc"], v["scales"], v["values"], v["ldv"],
                                            v["rows"], v["k"], None)


def _norm(**kw):
    v = {**dict(x=A, ldx=64, r=None, ldr=0, s=None, lds=0, g=A, eps=1e-6, codes=A, ldc=64, scales=A, values=None, ldv=0,
                rows=2, k=64), **kw}
    return _lib.lib().lmps_rms_norm_q8(v["x"], v["ldx"], v["r"], v["ldr"], v["s"], v["lds"], v["g"], v["eps"],
                                       v["codes"], v["ldc"], v["scales"], v["values"], v["ldv"], v["rows"], v["k"], None)


def _gemm(**kw):
    v = {**dict(x=A, ldx=64, xs=A, w=A, ldw=64, ws=A, b=None, r=None, ldr=0, y=A, ldy=32, m=2, n=32, k=64, gated=0,
                err=A), **kw}
    return _lib.lib().lmps_w8a8_gemm(v["x"], v["ldx"], v["xs"], v["w"], v["ldw"], v["ws"], v["b"], v["r"], v["ldr"],
                                     v["y"], v["ldy"], v["m"], v["n"], v["k"], v["gated"], v["err"], None)


@pytest.mark.parametrize("call", [_quantise, _norm])
@pytest.mark.parametrize("kw", [
    dict(x=None), dict(codes=None), dict(scales=None), dict(rows=0), dict(k=0), dict(ldx=63), dict(ldc=63),
    dict(values=A, ldv=63), dict(x=A + 1), dict(scales=A + 2), dict(values=A + 1, ldv=64),
])
def test_row_refusals(call, kw):
    assert call(**kw) == INVALID


@pytest.mark.parametrize("call", [_quantise, _norm])
@pytest.mark.parametrize("k", [(1 << 30) + 1, (1 << 31) - 2049, (1 << 31) - 16, (1 << 31) - 1])
def test_rows_whose_positions_pass_32_bits_are_refused(call, k):
    """Positions are 32-bit numbers that step up to 2048 past the end of a row."""
    far = (1 << 31) - 1
    assert call(rows=1, k=k, ldx=far, ldc=far) == UNSUPPORTED
    assert call(rows=1, k=k, ldx=far, ldc=far, values=A, ldv=far) == UNSUPPORTED


@pytest.mark.parametrize("kw", [
    dict(g=None), dict(g=A + 1), dict(eps=-1e-6), dict(eps=float("nan")), dict(r=A, ldr=64), dict(s=A, lds=64),
    dict(r=A, ldr=63, s=A, lds=64), dict(r=A, ldr=64, s=A, lds=63), dict(r=A + 1, ldr=64, s=A, lds=64),
])
def test_norm_refusals(kw):
    assert _norm(**kw) == INVALID


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), INVALID), (dict(xs=None), INVALID), (dict(w=None), INVALID), (dict(ws=None), INVALID),
    (dict(y=None), INVALID), (dict(err=None), INVALID), (dict(m=0), INVALID), (dict(n=0), INVALID), (dict(k=0), INVALID),
    (dict(ldx=48), INVALID), (dict(ldx=72), INVALID), (dict(ldw=48), INVALID), (dict(ldw=72), INVALID),
    (dict(ldy=31), INVALID), (dict(r=A, ldr=31), INVALID), (dict(x=A + 8), INVALID), (dict(w=A + 8), INVALID),
    (dict(xs=A + 2), INVALID), (dict(y=A + 1), INVALID), (dict(b=A + 1), INVALID), (dict(gated=2), INVALID),
    (dict(gated=1, b=A), INVALID), (dict(gated=1, r=A, ldr=32), INVALID),
    (dict(k=131072, ldx=131072, ldw=131072), UNSUPPORTED), (dict(m=(1 << 29) + 1), UNSUPPORTED),
    (dict(n=(1 << 29) + 1, ldy=(1 << 29) + 1), UNSUPPORTED),
])
def test_gemm_refusals(kw, status):
    assert _gemm(**kw) == status


def test_python_layer_refuses_cpu_tensors():
    h, c = torch.zeros(2, 64, dtype=torch.float16), torch.zeros(2, 64, dtype=torch.int8)
    s = torch.ones(2)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.quantise_rows_q8(h)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.rms_norm_q8(h, h[0], residual=h)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.w8a8_gemm(c, s, c, s)
    with pytest.raises(TypeError, match="tensor"):
        K.w8a8_gemm([1], s, c, s)
    with pytest.raises(ValueError, match="shape"):
        K.quantise_rows_q8(h[:, :0])


def test_the_extension_is_built_for_this_torch(monkeypatch):
    monkeypatch.setattr(_lib, "_BIND_Q8", None)
    assert _lib.binding_q8().torch_version == torch.__version__
    monkeypatch.setattr(_lib, "_BIND_Q8", None)
    monkeypatch.setattr(torch, "__version__", "0.0.0")
    with pytest.warns(RuntimeWarning, match="built against"):
        assert _lib.binding_q8().gemm() is None
