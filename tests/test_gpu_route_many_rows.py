"""Routing and its gradient at row counts that fill the chip: blocks of sixteen
waves that count the load together, and waves that take further rows after
their first, through the same LDS."""
import numpy as np
import pytest
import torch

import garfield_amd as gf
import route_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# Rows of up to 256 entries go four to a wave: sixteen waves a block from 8189
# rows on, second turns beyond 32,768 (the gradient at every width); longer rows
# have a wave each: 2048 and 8192.
CASES = [
    dict(T=8189, E=256, k=8, groups=16, keep_groups=4, dtype="f32"),
    dict(T=8200, E=256, k=8, groups=8, keep_groups=4, group_score="top2", bias=True, score="sigmoid", dtype="f32"),
    dict(T=8193, E=250, k=20, groups=5, keep_groups=2, group_score="top2", dtype="bf16"),
    dict(T=8190, E=128, k=3, bias=True, dtype="f16", renormalise=False),
    dict(T=33001, E=64, k=6, dtype="bf16", renormalise=False),
    dict(T=66003, E=16, k=2, bias=True, score="sigmoid", dtype="f32"),
    dict(T=40001, E=60, k=12, groups=4, keep_groups=3, group_score="top2", score="sigmoid", dtype="f16"),
    dict(T=2048, E=1024, k=16, dtype="bf16", renormalise=False),
    dict(T=2101, E=1024, k=64, groups=32, keep_groups=7, group_score="top2", bias=True, dtype="f32"),
    dict(T=8303, E=512, k=8, groups=8, keep_groups=3, bias=True, score="sigmoid", dtype="f32"),
    dict(T=9001, E=300, k=5, groups=3, keep_groups=2, dtype="f32", renormalise=False),
    dict(T=33017, E=320, k=10, groups=10, keep_groups=4, group_score="top2", bias=True, dtype="f32", renormalise=False),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_many_rows(i):
    c = dict(CASES[i])
    print("case many rows", i, c, flush=True)
    T, E, k, dtype = c.pop("T"), c.pop("E"), c.pop("k"), TYPES[c.pop("dtype")]
    score, renorm = c.pop("score", "softmax"), c.pop("renormalise", True)
    g = torch.Generator().manual_seed(100 + i)
    l = 2 * torch.randn(T, E, generator=g)
    l[1::5] = torch.round(2 * l[1::5]) / 2                          # ties
    l[2::5] = 1 + torch.randperm(E, generator=g) * 2.0 ** -22       # near ties: the pass in 64 bits
    l[3::7][torch.rand(l[3::7].shape, generator=g) < 0.5] = float("-inf")
    l[11::64] = float("-inf")
    l = l.to(dtype)
    # distinct, so that no two sums of different terms are equal but for their rounding
    bias = 0.05 * torch.randn(E, generator=g) if c.pop("bias", False) else None
    lv, bv = l.double().numpy(), None if bias is None else bias.double().numpy()
    bias = None if bias is None else bias.cuda()
    how = dict(score=score, renormalise=renorm, scale=2.5)
    r = gf.route(l.cuda(), k, bias=bias, **how, **c)
    ids, load = ref.choose(lv, k, bv, score=score, **c)
    assert np.array_equal(r.ids.cpu().numpy(), ids)
    assert np.array_equal(r.load.cpu().numpy(), load)
    w = ref.weights(lv, ids, bias=bv, **how)
    err = np.abs(r.weights.double().cpu().numpy() - w)
    assert (err <= ref.weight_bound(w, lv, ids, 2.5, bv)).all(), err.max()
    dw = torch.randn(T, k, generator=g)
    d = gf.route_grad(l.cuda(), r.ids, dw.cuda(), bias=bias, **how)
    want, mag = ref.gradient(lv, ids, dw.numpy(), bias=bv, **how)
    err = np.abs(d.double().cpu().numpy() - want)
    assert (err <= ref.gradient_bound(want, mag, lv, ids, dw.numpy(), 2.5, str(dtype)[6:], bv)).all(), err.max()
