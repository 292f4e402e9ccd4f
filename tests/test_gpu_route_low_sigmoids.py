"""Sigmoid scores of very negative logits: weights that are shares of the chosen
scores, and their gradient, where the scores themselves are below fp32's range."""
import numpy as np
import pytest
import torch

import garfield_amd as gf
import operators_oracle as orc
import route_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def test_shares_by_hand():
    print("case low sigmoids by hand", flush=True)
    l = torch.tensor([[-100.0, -101.0], [-700.0, -700.0], [-5.0, -90.0], [float("-inf"), -200.0], [-1e38, -1e38]]).cuda()
    r = gf.route(l, 2, score="sigmoid", scale=2.0)
    w = r.weights.double().cpu().numpy()
    up = 1 / (1 + np.exp(-1))
    assert np.allclose(w[0], [2 * up, 2 - 2 * up], rtol=1e-5) and (w[1] == 1.0).all()
    assert w[2, 0] == 2.0 and np.isclose(w[2, 1], 2 * np.exp(-90.0) * (1 + np.exp(5.0)), rtol=1e-3)
    assert w[3].tolist() == [2.0, 0.0] and r.ids[3].tolist() == [1, -1]
    assert w[4].tolist() == [0.0, 0.0] and r.ids[4].tolist() == [0, 1]      # scores that count as 0


# the widths of the kernels' rows, each with the loop and both lists of choices
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("E,k", [(5, 2), (16, 9), (30, 5), (60, 20), (100, 8), (256, 8), (256, 3), (300, 12), (512, 64),
                                 (1024, 4), (1000, 2)])
def test_low_sigmoids(E, k, dtype):
    print("case low sigmoids", E, k, dtype, flush=True)
    tops = [3.0, -5.0, -16.9, -17.1, -40.0, -80.0, -87.0, -89.0, -100.0, -300.0, -700.0, -30000.0]
    g = torch.Generator().manual_seed(E + k)
    l = (torch.tensor(tops).repeat_interleave(9)[:, None] - 30 * torch.rand(9 * len(tops), E, generator=g) ** 2).to(TYPES[dtype])
    l[::4, ::3] = float("-inf")
    l[5] = float("-inf")
    l[7] = torch.finfo(l.dtype).min
    lv = l.double().numpy()
    dw = torch.randn(l.shape[0], k, generator=g)
    for scale in (1.0, 2.5):
        r = gf.route(l.cuda(), k, score="sigmoid", scale=scale)
        ids, _, load = orc.route(lv, k)
        assert np.array_equal(r.ids.cpu().numpy(), ids) and np.array_equal(r.load.cpu().numpy(), load)
        w = ref.weights(lv, ids, score="sigmoid", scale=scale)
        err = np.abs(r.weights.double().cpu().numpy() - w)
        assert (err <= ref.weight_bound(w, lv, ids, scale)).all(), err.max()
        d = gf.route_grad(l.cuda(), r.ids, dw.cuda(), score="sigmoid", scale=scale)
        want, mag = ref.gradient(lv, ids, dw.numpy(), score="sigmoid", scale=scale)
        err = np.abs(d.double().cpu().numpy() - want)
        bound = ref.gradient_bound(want, mag, lv, ids, dw.numpy(), scale, str(d.dtype)[6:])
        assert (err <= bound).all(), (err / bound).max()
