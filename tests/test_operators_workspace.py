"""Workspace of products with a real side: bounded, and none for rows that are
read where they lie (the queries run on the CPU, pointers are never read)."""
import ctypes as C

import pytest
import torch

import garfield_amd as gf
from garfield_amd import _lib, operators

P = 0x10000
ARG = 1
PARTS = 64 << 20     # partial sums, at most


def _any(kind, dtype, M, rows, K):
    n = C.c_size_t()
    assert _lib.load().gf_mx_product_workspace(kind, dtype, M, rows, K, C.byref(n)) == 0
    return n.value


def _at(kind, dtype, M, rows, K, ld=None, x=P):
    n = C.c_size_t()
    ld = (rows if kind == 2 else K) if ld is None else ld
    assert _lib.load().gf_mx_product_workspace_at(kind, x, dtype, M, ld, rows, K, C.byref(n)) == 0
    return n.value


SIZES = [(1 << 22, 8192, 4096), (1 << 22, 8192, 4095), (16384, 131072, 256), (16384, 131071, 256), (4096, 8192, 4096),
         (17, 53124, 1024), (300, 9376, 128), (1 << 30, 1 << 20, 1 << 16), (0x7FFFFF00, 0x7FFFFF00, 0x7FFFFF00)]


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("kind", [0, 2])
@pytest.mark.parametrize("M,rows,K", SIZES)
def test_bounded(M, rows, K, kind, dtype):
    J = rows if kind == 2 else K
    most = _any(kind, dtype, M, rows, K)
    assert most <= (4 << 30) + PARTS
    for ld, x in ((J, P), (J + 64, P), (J + 1, P), (J, P + 2 if dtype else P + 4), (1 << 30, P)):
        if ld >= J:
            assert _at(kind, dtype, M, rows, K, ld, x) <= most


@pytest.mark.parametrize("kind,M,rows,K", [(0, 1 << 22, 8192, 4096), (0, 4096, 8192, 4096), (2, 16384, 131072, 256),
                                           (2, 4096, 8192, 4096), (0, 100, 53124, 1024)])
def test_nothing_for_rows_read_in_place(kind, M, rows, K):
    """bfloat16 rows of whole steps, aligned: partial sums at most; the same rows
    moved by an element, or at an odd distance, need a copy or are split."""
    J = rows if kind == 2 else K
    N = K if kind == 2 else rows
    n = _at(kind, 2, M, rows, K)
    assert n % (4 * M * N) == 0 and n <= PARTS and n // (4 * M * N) != 1
    copy = 2 * M * J
    for ld, x in ((J, P + 2), (J + 4, P), (1 << 22, P)):
        n = _at(kind, 2, M, rows, K, ld, x)
        assert n <= PARTS or (copy <= 4 << 30 and copy <= n <= copy + PARTS)


def test_refusals():
    n = C.c_size_t()
    f = _lib.load().gf_mx_product_workspace_at
    assert f(3, P, 0, 1, 1, 1, 1, C.byref(n)) == ARG and f(-1, P, 0, 1, 1, 1, 1, C.byref(n)) == ARG
    assert f(0, P, 3, 1, 1, 1, 1, C.byref(n)) == ARG and f(0, P, 0, 1, 1, 1, 0, C.byref(n)) == ARG
    assert f(0, P, 0, 1 << 40, 1, 1, 1, C.byref(n)) == ARG and f(0, P, 0, 1, 1, 1, 1, None) == ARG


@pytest.mark.gpu
@pytest.mark.parametrize("shift,extra", [(0, 0), (0, 8), (1, 0), (0, 1), (8, 56)])
def test_products_by_alignment(shift, extra, monkeypatch):
    """bfloat16 rows of whole steps at every kind of address: exact products, and
    no memory but partial sums beside the result where they are read in place."""
    print("case alignment", shift, extra, flush=True)
    took, workspace = [], operators._workspace

    def spy(*a):
        got = workspace(*a)
        took.append(got[1])
        assert got[1] == 0 or got[0].numel() == got[1]
        return got

    monkeypatch.setattr(operators, "_workspace", spy)
    g = torch.Generator().manual_seed(5)
    M, N, K = 1030, 1216, 640
    w = gf.mx_quantise(torch.randint(-4, 5, (N, K), generator=g).float().cuda())
    wv = gf.mx_dequantise(w).double()
    for kind, J, cols in ((0, K, N), (2, N, K)):
        buf = torch.full((shift + M * (J + extra),), float("nan"), dtype=torch.bfloat16, device="cuda")
        x = buf[shift:].view(M, J + extra)[:, :J]
        x.copy_(torch.randint(-8, 9, (M, J), generator=g))
        call = gf.mx_product if kind == 0 else gf.mx_product_grad
        want = x.double() @ (wv.t().contiguous() if kind == 0 else wv)     # whole numbers below 2^20
        y = call(x, w, dtype=torch.float32)
        assert torch.equal(y.double(), want)
        bytes_ = took.pop()
        assert bytes_ == _at(kind, 2, M, N, K, J + extra, P + 2 * shift)
        if shift % 8 == 0 and extra % 8 == 0:
            assert bytes_ % (4 * M * cols) == 0
