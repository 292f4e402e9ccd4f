"""The routing's gradient entry by entry: each within a bound in proportion to
its own terms, those of entries that were not chosen (the softmax over all) among
them."""
import numpy as np
import pytest
import torch

import garfield_amd as gf
import route_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("score,renormalise", [("softmax", False), ("softmax", True), ("sigmoid", False), ("sigmoid", True)])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (5, 2, 1), (70, 16, 2), (33, 37, 17), (50, 100, 33), (40, 256, 8), (19, 255, 64),
                                   (23, 512, 16), (21, 1000, 49), (20, 1024, 64)])
def test_terms(T, E, k, score, renormalise, dtype):
    print("case gradient terms", T, E, k, score, renormalise, dtype, flush=True)
    g = torch.Generator().manual_seed(T * E + k)
    l = 2 * torch.randn(T, E, generator=g)
    if E > 4:
        l[3::5][torch.rand(l[3::5].shape, generator=g) < 0.7] = float("-inf")
        l[2::9] = float("-inf")
        l[4::11, 1] = float("inf")
        l[1::7, ::2] = float("nan")
    l = l.to(TYPES[dtype])
    bias = 0.1 * torch.randn(E, generator=g)
    if E > 4:
        bias[E // 2] = float("-inf")
    dw = torch.randn(T, k, generator=g)
    lv = l.double().numpy()
    for b in (None, bias):
        bv = None if b is None else b.double().numpy()
        ids, _ = ref.choose(lv, k, bv, score=score)
        how = dict(score=score, renormalise=renormalise, scale=1.5)
        d = gf.route_grad(l.cuda(), torch.from_numpy(ids).cuda(), dw.cuda(), bias=None if b is None else b.cuda(), **how)
        want, mag = ref.gradient(lv, ids, dw.numpy(), bias=bv, **how)
        err = np.abs(d.double().cpu().numpy() - want)
        assert (err <= ref.gradient_bound(want, mag, lv, ids, dw.numpy(), 1.5, str(d.dtype)[6:], bv)).all(), err.max()
