"""What the block operators and gradient clipping refuse, without a device: the C entry points check
before they launch, the bindings check shapes and types before they look for a device."""
import ctypes
import math
import os

import pytest
import torch

from pointcloud_style_transfer_amd import _hip

pytestmark = pytest.mark.skipif(not os.path.exists(_hip.LIB_PATH), reason="library not built")

EINVAL, EUNSUPPORTED = 1001, 1002
BF, F32, E4 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def rc(name, *args):
    return getattr(_hip.lib(), name)(*args)


def error():
    return _hip.lib().pcst_last_error().decode()


def size(name, *args):
    sz = ctypes.c_size_t(123)
    return rc(name, *args, ctypes.byref(sz)), sz.value


@pytest.mark.parametrize("M,D,dt,wdt,want", [
    (4, 0, 1, 1, EINVAL), (-1, 8, 1, 1, EINVAL), (4, 16385, 1, 1, EUNSUPPORTED), (4, 8, 3, 3, EINVAL),
    (4, 8, 9, 0, EINVAL), (4, 8, 1, 2, EINVAL), (4, 8, 0, 1, EINVAL),
])
def test_norm_refusals(M, D, dt, wdt, want):
    one = ctypes.c_void_p(16)  # never read: the call is refused first
    assert rc("pcst_rms_norm", one, None, dt, M, D, one, wdt, 1e-6, one, None, None, None) == want
    assert "rms_norm" in error()
    assert rc("pcst_rms_norm_quant", one, None, dt, M, D, one, wdt, 1e-6, one, one, None, None) == want
    assert rc("pcst_rms_norm_bwd", one, dt, M, D, one, wdt, one, one, None, one, one, one, None) == want


def test_norm_null_pointers_and_no_rows():
    one = ctypes.c_void_p(16)
    assert rc("pcst_rms_norm", one, one, 1, 4, 8, one, 1, 1e-6, one, None, None, None) == EINVAL  # no place for s
    assert rc("pcst_rms_norm", None, None, 1, 4, 8, one, 1, 1e-6, one, None, None, None) == EINVAL
    assert rc("pcst_quant_rows", one, 1, 4, 8, one, None, None) == EINVAL
    assert rc("pcst_rms_norm_bwd", one, 1, 4, 8, one, 1, one, one, None, one, one, None, None) == EINVAL  # dw: workspace
    assert rc("pcst_rms_norm", None, None, 1, 0, 8, None, 1, 1e-6, None, None, None, None) == 0  # nothing to do
    assert size("pcst_rms_norm_bwd_workspace_size", 100000, 256) == (0, 2048 * 256 * 4)
    assert size("pcst_rms_norm_bwd_workspace_size", 100000, 4096) == (0, 512 * 4096 * 4)


@pytest.mark.parametrize("kw,want", [
    (dict(D=0), EINVAL), (dict(F=0), EINVAL), (dict(M=-1), EINVAL), (dict(D=1 << 20), EUNSUPPORTED),
    (dict(F=1 << 20), EUNSUPPORTED), (dict(M=1 << 31), EUNSUPPORTED), (dict(dt=4), EINVAL), (dict(act=3), EINVAL),
    (dict(out=2), EINVAL), (dict(dt=3, out=1), EINVAL), (dict(dt=3, out=0), EINVAL), (dict(bg=16), EINVAL), (dict(x=None), EINVAL),
    (dict(D=9, M=129), EINVAL), (dict(x=24, M=129), EINVAL),  # rows off 16-byte boundaries, and no workspace
    (dict(D=8192, M=129), EINVAL),  # a product that splits D, and no workspace
])
def test_gated_refusals(kw, want):
    a = dict(x=16, dt=1, M=4, D=8, F=8, bg=None, bu=None, act=0, out=1)
    a.update(kw)
    p = ctypes.c_void_p
    assert rc("pcst_gated_linear", p(a["x"]), a["dt"], a["M"], a["D"], p(16), p(16), a["F"], p(a["bg"]), p(a["bu"]), 0,
              a["act"], None, None, None, p(16), a["out"], None, None) == want
    assert "gated_linear" in error()


def test_gated_bwd_refusals():
    one = ctypes.c_void_p(16)

    def call(dt=1, M=4, ws=one, dh=one, bg=None):
        return rc("pcst_gated_linear_bwd", one, dt, M, 8, one, one, 8, bg, None, 0, 0, dh, one, one, one, 0, None,
                  None, ws, None)

    assert call(dt=3) == EINVAL and call(M=0) == EINVAL and call(ws=None) == EINVAL
    assert call(dh=None) == EINVAL and call(bg=one) == EINVAL
    assert size("pcst_gated_linear_bwd_workspace_size", 3, 4, 8, 8)[0] == EINVAL
    assert size("pcst_gated_linear_workspace_size", 1, 129, 64, 8, 1) == (0, 0)
    assert size("pcst_gated_linear_workspace_size", 1, 64, 63, 8, 0) == (0, 0)
    assert size("pcst_gated_linear_workspace_size", 1, 129, 64, 8, 0)[1] > 0
    assert size("pcst_gated_linear_workspace_size", 1, 129, 63, 8, 1)[1] > 0
    assert size("pcst_gated_linear_workspace_size", 1, 65, 8192, 8, 1)[1] > 0
    assert size("pcst_gated_linear_workspace_size", 1, 8192, 4096, 8192, 1) == (0, 0)


def test_clip_refusals():
    one = ctypes.c_void_p(16)
    I, U, P = ctypes.c_int64 * 1, ctypes.c_uint8 * 1, ctypes.c_void_p * 1

    def call(n=8, t=0, p=2, m=1.0, ptr=16, ws=one, norm=one, count=1):
        return rc("pcst_grad_clip", P(ptr), P(ptr), I(n), U(t), count, p, m, None, norm, ws, None)

    assert call(n=-1) == EINVAL and call(t=3) == EINVAL and call(t=1 | 2 << 4) == EINVAL
    assert call(p=3) == EINVAL and call(m=-1.0) == EINVAL and call(m=math.nan) == EINVAL
    assert call(ptr=None) == EINVAL and call(ws=None) == EINVAL and call(norm=None) == EINVAL
    assert call(count=-1) == EINVAL and call(n=1 << 41) == EINVAL
    for n, want in ((1, 8), (2048, 8), (2049, 16), (1 << 28, 1024 * 8)):
        assert size("pcst_grad_clip_workspace_size", I(n), 1) == (0, want)


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call,match", [
    (lambda: _hip.rms_norm(z(2, 8, dtype=torch.float64), z(8)), "float32, bfloat16 or float16"),
    (lambda: _hip.rms_norm(z(2, 8), z(7)), "weight is"),
    (lambda: _hip.rms_norm(z(2, 8), z(8, dtype=torch.float16)), "weight is"),
    (lambda: _hip.rms_norm(z(2, 8), z(8), z(1, 8)), "residual is"),
    (lambda: _hip.rms_norm(z(2, 8), z(8), z(2, 8, dtype=F32)), "residual is"),
    (lambda: _hip.rms_norm(z(2, 0), z(0)), "no values"),
    (lambda: _hip.rms_norm(z(2, 8), z(8)), "HIP device"),
    (lambda: _hip.quant_rows(z(2, 8)), "HIP device"),
    (lambda: _hip.gated_linear(z(2, 8), z(4, 8), z(5, 8)), "shapes are"),
    (lambda: _hip.gated_linear(z(2, 8), z(4, 7), z(4, 7)), "shapes are"),
    (lambda: _hip.gated_linear(z(2, 8), z(4, 8), z(4, 8, dtype=F32)), "one type"),
    (lambda: _hip.gated_linear(z(2, 8), z(4, 8), z(4, 8), z(4)), "both biases"),
    (lambda: _hip.gated_linear(z(2, 8), z(4, 8), z(4, 8), z(3), z(3)), "biases are"),
    (lambda: _hip.gated_linear(z(2, 8), z(4, 8), z(4, 8), act="tanh"), "act is"),
    (lambda: _hip.gated_linear(z(2, 8), z(4, 8), z(4, 8), out_dtype=F32), "no product"),
    (lambda: _hip.gated_linear(z(2, 8), z(4, 8), z(4, 8), scales=(1, 2, 3)), "scales"),
    (lambda: _hip.gated_linear(z(2, 8).to(E4), z(4, 8).to(E4), z(4, 8).to(E4), out_dtype=BF), "scales"),
    (lambda: _hip.gated_linear(z(2, 8), z(0, 8), z(0, 8)), "no features"),
    (lambda: _hip.gated_linear(z(2, 8), z(4, 8), z(4, 8)), "HIP device"),
    (lambda: _hip.gated_linear_bwd(z(2, 8).to(E4), z(4, 8).to(E4), z(4, 8).to(E4), z(2, 4)), "no gradients"),
    (lambda: _hip.grad_clip([z(4)], 1.0, 3.0), "norm_type"),
    (lambda: _hip.grad_clip([z(4)], -1.0), "max_norm"),
    (lambda: _hip.grad_clip([z(4)], math.nan), "max_norm"),
    (lambda: _hip.grad_clip([], 1.0), "no gradients"),
    (lambda: _hip.grad_clip([z(4)], 1.0, out=[]), "outputs for"),
    (lambda: _hip.grad_clip([z(4)], 1.0, out=[z(5)]), "an output has"),
    (lambda: _hip.grad_clip([z(4)], 1.0, out=[z(4, dtype=torch.float16)]), "an output has"),
    (lambda: _hip.grad_clip([z(4, 4)], 1.0, out=[z(4, 4).t()]), "an output has"),
    (lambda: _hip.grad_clip([z(4, 4).t()], 1.0, out=[z(4, 4)]), "an output has"),
    (lambda: _hip.grad_clip([z(4, 4).t()], 1.0, out=[z(2, 8).t()]), "an output has"),
    (lambda: _hip.grad_clip([z(4, dtype=torch.float64)], 1.0), "dense float32"),
    (lambda: _hip.grad_clip([z(4, 8)[:, ::2]], 1.0), "gaps"),
    (lambda: _hip.grad_clip([z(1, 8).expand(4, 8)], 1.0), "gaps"),
    (lambda: _hip.grad_clip([z(4, 8)], 1.0), "HIP device"),
])
def test_binding_refusals(call, match):
    with pytest.raises(RuntimeError, match=match):
        call()


def clip_rc(grads, out):
    """pcst_grad_clip on host addresses and without a workspace: refused for one or for the other."""
    n = len(grads)
    P, I, U = ctypes.c_void_p * n, ctypes.c_int64 * n, ctypes.c_uint8 * n
    code = lambda t: _hip._ELEM[t.dtype]  # noqa: E731
    outs = grads if out is None else out
    one = ctypes.c_void_p(16)
    lib_args = (P(*[t.data_ptr() for t in grads]), P(*[t.data_ptr() for t in outs]), I(*[t.numel() for t in grads]),
                U(*[code(g) | code(o) << 4 for g, o in zip(grads, outs)]), n, 2, 1.0, None, one, None, None)
    assert rc("pcst_grad_clip", *lib_args) == EINVAL
    return error()


def test_clip_refuses_overlap():
    a, f = z(32), z(32, dtype=F32)
    for grads, out in (([a, a], None), ([a[:20], a[16:]], None), ([a[:8]], [a[4:12]]), ([a[:8], a[8:16]], [z(8), a[:8]]),
                       ([f.view(BF)[:32]], [f])):
        assert "overlap" in clip_rc(grads, out)
    # neighbours in one buffer, a gradient onto itself and empty tensors are fine
    for grads, out in (([a[:16], a[16:]], None), ([a[:8]], [a[:8]]), ([a, a[:0], a[8:8]], None), ([a[:8]], [f[:8]])):
        assert "workspace" in clip_rc(grads, out)
    b = z(4, 6, 5).permute(2, 0, 1)  # dense, in another order
    for out in (None, [b], [torch.empty_like(b)]):
        with pytest.raises(RuntimeError, match="HIP device"):
            _hip.grad_clip([b], 1.0, out=out)


def test_eight_bits_carry_no_gradients():
    from pointcloud_style_transfer_amd.models import gated_linear_quant, quant_rows, rms_norm_quant

    w = z(8).requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        rms_norm_quant(z(2, 8), w)
    with pytest.raises(RuntimeError, match="no gradients"):
        quant_rows(w)
    q, s = z(4, 8).to(E4), z(4, dtype=F32)
    with pytest.raises(RuntimeError, match="no gradients"):
        gated_linear_quant(q, s, q, s, q, s, z(4).requires_grad_(), z(4))
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        gated_linear_quant(z(4, 8), s, q, s, q, s)


def test_empty_clip():
    from pointcloud_style_transfer_amd.utils import clip_grad_norm_, clip_grads

    assert float(clip_grads([], 1.0)) == 0.0
    assert float(clip_grad_norm_(torch.nn.Linear(2, 2).parameters(), 1.0)) == 0.0
