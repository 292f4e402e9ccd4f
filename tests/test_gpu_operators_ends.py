"""The ends of the 4-bit rows' range: every scale byte in products with one value
a row, where nothing but the type's range can round."""
import numpy as np
import pytest
import torch

import garfield_amd as gf
import operators_oracle as orc

pytestmark = pytest.mark.gpu

N, K = 16 * 9, 64


def _rows(byte):
    """Row n: code n % 16 at position n // 16 (of nine), scale 2^(byte - 127)."""
    nib = np.zeros((N, 128), np.uint8)
    nib[np.arange(N), np.arange(N) // 16 * 7] = np.arange(N) % 16
    scales = np.zeros((N, 4), np.uint8)
    scales[:, :2] = byte
    codes = nib[:, 0::2] | nib[:, 1::2] << 4
    return gf.MXRows(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), K), orc.dequantise(codes, scales, K)


@pytest.mark.parametrize("byte", [0, 1, 2, 17, 127, 200, 250, 251, 252])
def test_products_at_every_scale(byte):
    print("case scale byte", byte, flush=True)
    w, wv = _rows(byte)
    with np.errstate(over="ignore"):
        assert np.array_equal(gf.mx_dequantise(w).cpu().numpy().astype(np.float64), wv)
    # results within the normal range of fp32: x of the opposite size (1 for
    # binary16, whose range ends at 2^15)
    for dtype, e in ((torch.float32, 127 - byte), (torch.bfloat16, 127 - byte), (torch.float16, max(-14, min(127 - byte, 15)))):
        xv = 2.0 ** min(e, 120) * (1 + 2.0 ** -6)
        for M in (1, 16, 40, 300):
            x = torch.full((M, K), xv, dtype=torch.float64).to(dtype)
            y = gf.mx_product(x.cuda(), w, dtype=torch.float32).double().cpu().numpy()
            want = x.double().numpy() @ wv.T
            normal = (np.abs(want) >= 2.0 ** -126) | (want == 0)
            assert np.array_equal(y[normal], want[normal]) and normal.mean() > 0.4, (dtype, M)
            # one row at a time in the gradient
            dy = torch.zeros(M, N, dtype=dtype)
            dy[:, 15 if M == 1 else 7] = xv
            dx = gf.mx_product_grad(dy.cuda(), w, dtype=torch.float32).double().cpu().numpy()
            want = dy.double().numpy() @ wv
            normal = (np.abs(want) >= 2.0 ** -126) | (want == 0)
            assert np.array_equal(dx[normal], want[normal]), (dtype, M)


@pytest.mark.parametrize("byte", [0, 1, 127, 252, 253, 254])
def test_both_sides_at_four_bits_take_every_scale(byte):
    print("case both scales", byte, flush=True)
    w, wv = _rows(byte)
    x, xv = _rows(254 - byte)
    for a, av in ((x[:1], xv[:1]), (x[:16], xv[:16]), (x, xv)):
        assert np.array_equal(gf.mx_product(a, w).double().cpu().numpy(), av @ wv.T)


def test_quantisation_stays_below_byte_253():
    x = torch.full((4, 64), torch.finfo(torch.float32).max)
    for dtype in (torch.float32, torch.bfloat16):
        w = gf.mx_quantise(x.to(dtype).clamp(max=torch.finfo(dtype).max).cuda())
        assert (w.scales[:, :2] == 252).all() and torch.isfinite(gf.mx_dequantise(w)).all()


def test_fp32_bits_that_enter():
    """Down to 2^-133 of a value, whatever its size."""
    print("case fp32 bits", flush=True)
    w, _ = _rows(227)                       # row 1: 0.5 * 2^100 at position 0
    for e in (-100, -109, -110):
        for M in (1, 40, 300):
            x = torch.zeros(M, K)
            x[:, 0] = 2.0 ** e * (1 + 2.0 ** -23)
            y = gf.mx_product(x.cuda(), w)
            assert (y[:, 1].double().cpu() == x[0, 0].double() * 2.0 ** 99).all(), (e, M)
