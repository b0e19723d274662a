"""Microscaled (MX) operators without a GPU: the plain implementation against itself and differences, and every refusal of the C ABI
and of the Python entry points that comes before a launch."""
import ctypes

import numpy as np
import pytest
import torch

import vcsr_mc_b200 as vm
from tests import mx_ref as ref
from vcsr_mc_b200 import _lib


@pytest.mark.parametrize("kind", ["mxf8", "mxf4"])
def test_plain_quantize_is_nearest_and_unclipped(kind):
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((40, 77)) * np.exp2(rng.integers(-140, 120, (40, 1)))).astype(np.float32)
    codes, scales = ref.quantize(x, kind)
    got = ref.values(codes, scales, kind)
    full = np.repeat(scales, 32, 1)[:, :77].astype(float)
    step = np.exp2(full - 127) * (2.0 if kind == "mxf4" else 32.0)  # the widest gap of the element type
    assert np.all(np.abs(got - x.astype(np.float64)) <= step / 2)
    amax = np.abs(x[:, :32]).max(1).astype(np.float64)
    top = ref.LARGEST[kind] * np.exp2(scales[:, 0] - 127.0)
    assert np.all(amax <= top) and np.all((amax > top / 2) | (scales[:, 0] == 0))


def test_plain_backward_against_differences():
    rng = np.random.default_rng(2)
    x, r, w, G = rng.standard_normal((3, 9)), rng.standard_normal((3, 9)), rng.standard_normal(9), rng.standard_normal((3, 9))
    R = rng.standard_normal((3, 9))

    def loss(x, w):
        s = x + r
        return (ref.norm(s, w, 1e-3)[0] * G).sum() + (s * R).sum()

    s = x + r
    dx, dw, _, _ = ref.norm_backward(G, w, s, ref.norm(s, w, 1e-3)[1], R)
    h = 1e-5
    for i in range(3):
        for j in range(9):
            d = np.zeros((3, 9))
            d[i, j] = h
            assert abs((loss(x + d, w) - loss(x - d, w)) / (2 * h) - dx[i, j]) < 1e-7
    for j in range(9):
        d = np.zeros(9)
        d[j] = h
        assert abs((loss(x, w + d) - loss(x, w - d)) / (2 * h) - dw[j]) < 1e-7


# ---- refusals of the C ABI: every one is answered before a launch, so it needs no GPU -------------------
P = ctypes.c_void_p
OK_PTR = 1 << 20  # an aligned address that no refused call reads


def refused(name, *args):
    with pytest.raises(vm.VcsrmcError) as e:
        _lib.call(name, *args)
    assert e.value.status == _lib.INVALID_ARG
    return str(e.value)


QUANT = dict(X=OK_PTR, x=vm.F32, ldx=64, rows=4, O=64, q=vm.MXF8, Q=OK_PTR, ldq=64, S=OK_PTR, lds=2, st=None)


@pytest.mark.parametrize("bad", [dict(X=None), dict(x=vm.MXF8), dict(x=9), dict(ldx=63), dict(rows=-1), dict(O=0), dict(O=(1 << 30) + 1),
                                 dict(q=vm.F16), dict(Q=None), dict(S=None), dict(ldq=63), dict(lds=1), dict(q=vm.MXF4, ldq=31),
                                 dict(X=OK_PTR + 2), dict(x=vm.F16, X=OK_PTR + 1)])
def test_quantize_refusals(bad):
    refused("vcsrmc_mx_quantize", *{**QUANT, **bad}.values())
    a = {**QUANT, **bad}
    refused("vcsrmc_mx_dequantize", a["Q"], a["q"], a["ldq"], a["S"], a["lds"], a["rows"], a["O"], a["X"], a["x"], a["ldx"], None)


def test_product_refusals_without_a_handle():
    n = ctypes.c_int64()
    refused("vcsrmc_spmm_mx_workspace", None, 64, ctypes.byref(n))
    refused("vcsrmc_spmm_mx", None, OK_PTR, vm.MXF8, 64, OK_PTR, 2, 64, OK_PTR, 64, 0, None, 0, None)


NORM = dict(X=OK_PTR, x=vm.F32, ldx=64, res=OK_PTR, ldr=64, out=OK_PTR, ldo=64, r=vm.F16, w=OK_PTR, wt=vm.F32, eps=1e-6, rows=4, O=64,
            q=vm.MXF8, Q=OK_PTR, ldq=64, S=OK_PTR, lds=2, inv=OK_PTR, st=None)


@pytest.mark.parametrize("bad", [dict(X=None), dict(x=vm.MXF4), dict(x=vm.BF16), dict(ldx=1), dict(ldr=63), dict(ldo=63), dict(r=7),
                                 dict(w=None), dict(wt=vm.MXF8), dict(w=OK_PTR + 2), dict(eps=-1.0), dict(eps=float("nan")),
                                 dict(eps=float("inf")), dict(rows=-1), dict(O=0), dict(q=vm.F32), dict(Q=None), dict(S=None),
                                 dict(ldq=10), dict(lds=1), dict(inv=OK_PTR + 2), dict(res=OK_PTR + 1), dict(out=OK_PTR + 1)])
def test_norm_refusals(bad):
    refused("vcsrmc_add_rms_norm", *{**NORM, **bad}.values())


GRAD = dict(dY=OK_PTR, dy=vm.F32, lddy=64, dr=OK_PTR, lddr=64, h=OK_PTR, ldh=64, r=vm.F16, w=OK_PTR, wt=vm.F32, inv=OK_PTR, rows=4, O=64,
            dX=OK_PTR, lddx=64, dw=OK_PTR, ws=OK_PTR, n=1 << 20, st=None)


@pytest.mark.parametrize("bad", [dict(dY=None), dict(dy=vm.BF16), dict(lddy=63), dict(lddr=63), dict(h=None), dict(ldh=63), dict(r=5),
                                 dict(w=None), dict(wt=6), dict(inv=None), dict(rows=-1), dict(O=0), dict(dX=None), dict(lddx=63),
                                 dict(dw=None), dict(dw=OK_PTR + 1), dict(dX=OK_PTR + 1)])
def test_norm_backward_refusals(bad):
    refused("vcsrmc_add_rms_norm_backward", *{**GRAD, **bad}.values())


def test_python_refusals():
    u8, e8 = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    f8 = torch.zeros(4, 64, dtype=torch.float8_e4m3fn)
    assert vm.MXDense(u8, e8).shape == (4, 64) and vm.MXDense(u8, e8, cols=63).kind == vm.MXF4
    assert vm.MXDense(f8, e8.view(torch.float8_e8m0fnu)).kind == vm.MXF8
    for make in (lambda: vm.MXDense(u8.int(), e8), lambda: vm.MXDense(u8, e8.float()), lambda: vm.MXDense(u8, e8, cols=65),
                 lambda: vm.MXDense(f8, e8[:, :1]), lambda: vm.MXDense(f8, e8[:3]), lambda: vm.MXDense(f8.t(), e8),
                 lambda: vm.MXDense(u8[0], e8), lambda: vm.MXDense.empty(4, 4, vm.F16),
                 lambda: vm.mx_quantize(torch.zeros(4, 4)), lambda: vm.mx_dequantize(vm.MXDense(u8, e8)),
                 lambda: vm.add_rms_norm(torch.zeros(4, 4), torch.zeros(4)),
                 lambda: vm.add_rms_norm_backward(torch.zeros(4, 4), torch.zeros(4), torch.zeros(4, 4), torch.zeros(4))):
        with pytest.raises(vm.VcsrmcError):
            make()


def test_mx_matrix_is_what_was_checked():
    """The tensors and the shape of an MXDense stay those that its constructor checked."""
    Q = vm.MXDense(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), cols=63)
    assert (Q.rows, Q.cols, Q.shape, Q.kind, Q.device) == (4, 63, (4, 63), vm.MXF4, torch.device("cpu"))
    for name, value in (("data", torch.zeros(1, 1, dtype=torch.uint8)), ("scale", torch.zeros(1, 1, dtype=torch.uint8)), ("rows", 9), ("cols", 999),
                        ("kind", vm.MXF8), ("shape", (9, 9)), ("anything", 1)):
        with pytest.raises(AttributeError):
            setattr(Q, name, value)


@pytest.mark.parametrize("raw,want", [(0, "default"), (1, "default"), (2, 2), (0x7F0012345678, 0x7F0012345678)])
def test_raw_stream_handles(monkeypatch, raw, want):
    """A raw handle names the stream that CUDA means by it: 0 and 1 are the default stream (which torch itself gives as 0; an external
    stream made from it would be another one), any other is taken as it is."""
    from types import SimpleNamespace
    from vcsr_mc_b200 import api
    device = torch.device("cuda:0")
    monkeypatch.setattr(torch.cuda, "default_stream", lambda d: SimpleNamespace(which="default", device=d))
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda raw, device: SimpleNamespace(which=raw, device=device))
    monkeypatch.setattr(torch.cuda, "stream", lambda s: s)
    for given in (raw, SimpleNamespace(cuda_stream=raw)):
        guard = api._stream_guard(given, device)
        assert guard.which == want and guard.device == device
