"""Refusals of the operators' entry points, before any device call (CPU only:
the pointers are never read)."""
import ctypes as C

import pytest
import torch

import garfield_amd as gf
from garfield_amd import _lib, operators

P = 0x10000   # a pointer that is aligned and never followed


def _mx(rows=8, K=128, codes=P, scales=P):
    return C.byref(_lib.MXRowsStruct(codes, scales, rows, K))


def _status(name, *args):
    return getattr(_lib.load(), name)(*args, None)


ARG, UNSUPPORTED = 1, 6


@pytest.mark.parametrize("args,status", [
    ((P, 3, 8, 128, 128, P, P), ARG),                 # element type
    ((P, 0, 8, 0, 128, P, P), ARG),                   # K = 0
    ((P, 0, 8, 128, 127, P, P), ARG),                 # rows overlap
    ((None, 0, 8, 128, 128, P, P), ARG),
    ((P, 0, 8, 128, 128, None, P), ARG),
    ((P, 0, 8, 128, 128, P, None), ARG),
    ((P + 2, 0, 8, 128, 128, P, P), ARG),             # not aligned to an element
    ((P, 0, 8, 128, 128, P + 8, P), ARG),             # codes not aligned to 16
    ((P, 0, 8, 128, 128, P, P + 2), ARG),
    ((P, 0, 1 << 32, 128, 128, P, P), UNSUPPORTED),
    ((P, 0, 8, 128, 1 << 62, P, P), ARG),             # offsets that pass 64 bits
])
def test_quantise_refuses(args, status):
    assert _status("gf_mx_quantise", *args) == status
    assert _lib.load().gf_last_error()


@pytest.mark.parametrize("args,status", [
    ((_mx(K=0), 0, P, 128), ARG), ((None, 0, P, 128), ARG), ((_mx(), 7, P, 128), ARG), ((_mx(), 0, None, 128), ARG),
    ((_mx(), 0, P, 100), ARG), ((_mx(codes=P + 4), 0, P, 128), ARG),
])
def test_dequantise_refuses(args, status):
    assert _status("gf_mx_dequantise", *args) == status


@pytest.mark.parametrize("name", ["gf_mx_product", "gf_mx_product_grad"])
@pytest.mark.parametrize("args,status", [
    ((P, 9, 4, 128, _mx(), 0, P, 128, None, 0), ARG), ((P, 0, 4, 128, _mx(), -1, P, 128, None, 0), ARG),
    ((P, 0, 4, 128, None, 0, P, 128, None, 0), ARG), ((P, 0, 4, 7, _mx(), 0, P, 128, None, 0), ARG),
    ((P, 0, 4, 128, _mx(), 0, P, 7, None, 0), ARG), ((None, 0, 4, 128, _mx(), 0, P, 128, None, 0), ARG),
    ((P, 0, 4, 128, _mx(), 0, None, 128, None, 0), ARG), ((P, 0, 4, 128, _mx(codes=None), 0, P, 128, None, 0), ARG),
    ((P + 1, 1, 4, 128, _mx(), 0, P, 128, None, 0), ARG), ((P, 0, 1 << 31, 128, _mx(), 0, P, 128, None, 0), UNSUPPORTED),
])
def test_products_refuse(name, args, status):
    assert _status(name, *args) == status


def test_product_mx_refuses():
    assert _status("gf_mx_product_mx", _mx(K=96), _mx(), 0, P, 8, None, 0) == ARG
    assert _status("gf_mx_product_mx", _mx(), _mx(), 5, P, 8, None, 0) == ARG
    assert _status("gf_mx_product_mx", _mx(), _mx(), 0, P, 7, None, 0) == ARG
    assert _status("gf_mx_product_mx", _mx(scales=None), _mx(), 0, P, 8, None, 0) == ARG


def test_more_workgroups_than_a_launch_has():
    """Refused on the host: 2^40 tiles."""
    far = 1 << 28
    assert _status("gf_mx_product_mx", _mx(far, 32), _mx(far, 32), 0, P, far, None, 0) == UNSUPPORTED
    n = C.c_size_t()
    assert _lib.load().gf_mx_product_workspace(0, 2, far, far, 64, C.byref(n)) == 0
    assert _status("gf_mx_product", P, 2, far, 64, _mx(far, 64), 0, P, far, P, n.value) == UNSUPPORTED


def test_workspace_is_checked():
    """A call whose workspace is too small, missing or misaligned is refused."""
    n = C.c_size_t()
    lib = _lib.load()
    found = 0
    for kind, call in ((0, lambda ws, b: _status("gf_mx_product", P, 0, 1, 1 << 20, _mx(16, 1 << 20), 0, P, 16, ws, b)),
                       (2, lambda ws, b: _status("gf_mx_product_grad", P, 0, 1, 1 << 20, _mx(1 << 20, 32), 0, P, 32, ws, b))):
        args = (kind, 0, 1, 16, 1 << 20) if kind == 0 else (kind, 0, 1, 1 << 20, 32)
        assert lib.gf_mx_product_workspace(*args, C.byref(n)) == 0
        if n.value:
            found += 1
            assert call(None, n.value) == ARG and call(P, n.value - 1) == ARG and call(P + 8, n.value) == ARG
    assert lib.gf_mx_product_workspace(3, 0, 1, 1, 1, C.byref(n)) == ARG
    assert lib.gf_mx_product_workspace(0, 3, 1, 1, 1, C.byref(n)) == ARG
    assert lib.gf_mx_product_workspace(0, 0, 1, 1, 0, C.byref(n)) == ARG
    assert lib.gf_mx_product_workspace(0, 0, 1, 1, 1, None) == ARG


def test_workspace_of_large_calls_is_bounded():
    """Beyond 4 GiB of planes the real side is split where it is used."""
    n = C.c_size_t()
    for dtype in (0, 1):
        assert _lib.load().gf_mx_product_workspace(0, dtype, 1 << 22, 8192, 4096, C.byref(n)) == 0
        assert n.value == 0
        assert _lib.load().gf_mx_product_workspace(0, dtype, 1 << 16, 8192, 4096, C.byref(n)) == 0
        assert 0 < n.value <= 4 << 30


def _opts(**kw):
    o = dict(k=4, score=0, groups=1, keep_groups=1, group_score=0, renormalise=1, scale=1.0)
    o.update(kw)
    return C.byref(_lib.RouteOpts(**o))


@pytest.mark.parametrize("opts,E,status", [
    (dict(k=0), 16, ARG), (dict(k=17), 16, ARG), (dict(k=65), 128, UNSUPPORTED), (dict(score=2), 16, ARG),
    (dict(groups=0), 16, ARG), (dict(groups=3), 16, ARG), (dict(groups=65, keep_groups=9), 650, UNSUPPORTED),
    (dict(groups=4, keep_groups=0), 16, ARG), (dict(groups=4, keep_groups=5), 16, ARG), (dict(group_score=2), 16, ARG),
    (dict(groups=8, keep_groups=1), 16, ARG),           # k beyond what the kept groups hold
    (dict(), 0, ARG), (dict(), 1025, UNSUPPORTED),
])
def test_route_refuses(opts, E, status):
    assert _status("gf_route", _opts(**opts), P, 0, 8, E, max(E, 1), None, P, P, None) == status


def test_route_refuses_pointers():
    ok = (_opts(), P, 0, 8, 16, 16, None, P, P, None)
    for i, bad in ((0, None), (1, None), (2, 5), (5, 15), (7, None), (8, None), (6, P + 2), (9, P + 1)):
        a = list(ok)
        a[i] = bad
        assert _status("gf_route", *a) == ARG, i
    ok = (_opts(), P, 0, 8, 16, 16, None, P, P, P, 16)
    for i, bad in ((0, None), (1, None), (2, 5), (5, 15), (7, None), (8, None), (9, None), (10, 15)):
        a = list(ok)
        a[i] = bad
        assert _status("gf_route_grad", *a) == ARG, i


def test_binding_refuses():
    """Host tensors, other types, shapes and strides, before the library is called."""
    x = torch.zeros(4, 32)
    with pytest.raises(ValueError, match="on the GPU"):
        gf.mx_quantise(x)
    with pytest.raises(ValueError, match="on the GPU"):
        gf.route(x, 2)
    with pytest.raises(ValueError, match="matrix"):
        gf.mx_quantise([[1.0]])
    with pytest.raises(ValueError, match="matrix"):
        gf.route(torch.zeros(4), 2)
    with pytest.raises(ValueError, match="MXRows"):
        gf.mx_product(x, x)
    with pytest.raises(ValueError, match="MXRows"):
        gf.mx_product_grad(x, x)
    with pytest.raises(ValueError, match="MXRows"):
        gf.mx_dequantise(x)
    with pytest.raises(ValueError, match="codes"):
        gf.MXRows(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 32)   # on the host
    with pytest.raises(ValueError, match="K must"):
        gf.MXRows(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 0)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        operators._type(torch.float64, "x")
    with pytest.raises(ValueError, match="softmax, sigmoid"):
        operators._choice(operators._SCORES, "relu", "score")
