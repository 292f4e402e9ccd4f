"""Counts that the operators' binding hands to the library's 32 bits: what does
not fit or is no whole number is refused, not cut off."""
import numpy as np
import pytest
import torch

import garfield_amd as gf
from garfield_amd import operators

LIMIT = 0x7FFFFF00


def test_counts():
    operators._need_torch()
    for good in (0, 4, 4.0, np.int64(4), np.uint8(4), LIMIT):
        n = operators._count(good, "n")
        assert n == good and type(n) is int
    for bad in (-1, 2.5, 1 << 31, (1 << 32) + 4, float("nan"), float("inf"), "4", None, [4]):
        with pytest.raises(ValueError, match="whole number"):
            operators._count(bad, "n")


def test_columns_beyond_32_bits():
    x = torch.zeros(1, 1).expand(1, (1 << 32) + 8)
    with pytest.raises(ValueError, match="columns"):
        gf.mx_quantise(x)
    with pytest.raises(ValueError, match="columns"):
        gf.route(x, 4)
    with pytest.raises(ValueError, match="columns"):
        gf.route_grad(x, None, None)
    with pytest.raises(ValueError, match="whole number"):
        gf.MXRows(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), (1 << 32) + 32)


@pytest.mark.gpu
def test_route_arguments():
    print("case route arguments", flush=True)
    l = torch.randn(3, 16).cuda()
    for how in (dict(k=(1 << 32) + 4), dict(k=2.5), dict(k=4, groups=4, keep_groups=(1 << 32) + 1),
                dict(k=4, groups=(1 << 32) + 4), dict(k=-1), dict(k="4"), dict(k=4, bias=[0.0] * 16),
                dict(k=4, bias=np.zeros(16, np.float32))):
        with pytest.raises(ValueError):
            gf.route(l, **how)
    with pytest.raises(ValueError, match="ids"):
        gf.route_grad(l, [[0]], torch.ones(3, 1).cuda())
    with pytest.raises(ValueError, match="dweights"):
        gf.route_grad(l, torch.zeros(3, 1, dtype=torch.int32).cuda(), [[1.0]])
    with pytest.raises(gf.GarfieldError):
        gf.route(l, 65)
    assert torch.equal(gf.route(l, 4.0).ids, gf.route(l, np.int32(4)).ids)
