"""A call's workspace is that of its own sizes (CPU: every call here is refused
before the device, its pointers are never read)."""
import ctypes as C

import pytest

from garfield_amd import _lib

P = 0x10000
ARG = 1


def _size(kind, dtype, M, rows, K):
    n = C.c_size_t()
    J = rows if kind == 2 else K
    assert _lib.load().gf_mx_product_workspace_at(kind, P, dtype, M, J, rows, K, C.byref(n)) == 0
    return n.value


def _refused(kind, dtype, M, rows, K, ws, size):
    w = C.byref(_lib.MXRowsStruct(P, P, rows, K))
    J, N = (rows, K) if kind == 2 else (K, rows)
    call = _lib.load().gf_mx_product_grad if kind == 2 else _lib.load().gf_mx_product
    return call(P, dtype, M, J, w, 0, P, N, ws, size, None) == ARG


# odd and even sizes; those between which the plan changes are found by bisection
def _sweep(kind, dtype, rows, K):
    sizes = {1, 16, 17, 31, 64, 100, 255, 256, 257, 500, 777, 1024, 2000, 4096, 5000, 9999, 20000, 65536}
    for a, b in zip(sorted(sizes), sorted(sizes)[1:]):
        if (_size(kind, dtype, a, rows, K) > 0) != (_size(kind, dtype, b, rows, K) > 0) \
                or _size(kind, dtype, a, rows, K) > _size(kind, dtype, b, rows, K):
            need = _size(kind, dtype, a, rows, K)
            while b - a > 1:
                m = (a + b) // 2
                got = _size(kind, dtype, m, rows, K)
                if (got > 0) == (need > 0) and got >= need:
                    a = m
                else:
                    b = m
            sizes |= {a, b}
    return sorted(sizes)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 2])
@pytest.mark.parametrize("rows,K", [(8192, 4096), (4096, 4096), (9376, 100), (53124, 1024)])
def test_every_size_is_checked_against_its_own(rows, K, kind, dtype):
    needs = 0
    for M in _sweep(kind, dtype, rows, K):
        n = _size(kind, dtype, M, rows, K)
        if n:
            needs += 1
            assert _refused(kind, dtype, M, rows, K, P, n - 1) and _refused(kind, dtype, M, rows, K, None, n)
            assert _refused(kind, dtype, M, rows, K, P + 8, n)
    assert needs or dtype == 2     # bfloat16 rows read in place may need none


def test_a_buffer_for_the_largest_is_too_small_for_others():
    """What the header says of the sizes: fewer queries may need more."""
    for M, more in ((4096, 4097), (1024, 1 << 20)):
        assert _size(0, 0, M, 8192, 4096) > _size(0, 0, more, 8192, 4096)
        assert _refused(0, 0, M, 8192, 4096, P, _size(0, 0, more, 8192, 4096))
