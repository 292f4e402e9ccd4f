"""The operators' 64-bit oracle against facts that do not come from it, on the
CPU: the grid and its ties, scale bytes at their limits, gradients against
differences, and small routings worked by hand."""
import numpy as np
import pytest

import operators_oracle as orc


def test_grid_and_ties():
    # 4 fixes the scale at 1 (floor(log2 4) - 2 = 0)
    x = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, 6.0, 7.9, -7.9, 0.26, 5.01]
    codes, scales = orc.quantise(np.array([x]))
    assert scales[0, 0] == 127
    v = orc.dequantise(codes, scales, len(x))[0]
    assert list(v) == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -0.0, -4.0, 6.0, 6.0, -6.0, 0.5, 6.0]


@pytest.mark.parametrize("top,byte", [(1.0, 125), (6.0, 127), (2.0 ** -126, 0), (2.0 ** -125, 0), (2.0 ** -124, 1),
                                      (2.0 ** 127, 252), (0.0, 0), (2.0 ** -149, 0), (np.inf, 255), (np.nan, 255)])
def test_scale_bytes(top, byte):
    _, scales = orc.quantise(np.array([[top, 0.0]]))
    assert scales[0, 0] == byte and list(scales[0, 1:]) == [0, 0, 0]


def test_values_are_nearest():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((20, 96)) * np.exp(rng.standard_normal((20, 1)))
    codes, scales = orc.quantise(x)
    v = orc.dequantise(codes, scales, 96)
    s = np.repeat(np.ldexp(1.0, scales[:, :3].astype(int) - 127), 32, axis=1)
    grid = np.concatenate([orc.MAGNITUDES, -orc.MAGNITUDES])
    best = np.abs(x[:, :, None] - s[:, :, None] * grid).min(2)
    assert np.array_equal(np.abs(x - v), best)


def test_route_by_hand():
    l = np.array([[1.0, 3.0, 3.0, 2.0], [-np.inf, np.nan, 0.0, -np.inf], [-np.inf] * 4, [np.inf, 0.0, 1.0, 2.0]])
    ids, w, load = orc.route(l, 2)
    assert ids.tolist() == [[1, 2], [2, -1], [-1, -1], [0, 3]]
    assert w.tolist() == [[0.5, 0.5], [1.0, 0.0], [0.0, 0.0], [1.0, 0.0]]
    assert load.tolist() == [1, 1, 2, 1]
    # groups {0, 1} and {2, 3}: the sum of two beats one large entry
    l = np.array([[2.0, -9.0, 1.0, 1.0]])
    for how, want in (("max", [0]), ("top2", [2])):
        ids, _, _ = orc.route(l, 1, groups=2, keep_groups=1, group_score=how, score="sigmoid")
        assert ids[0].tolist() == want
    # the bias chooses, the weights do not hold it
    ids, w, _ = orc.route(np.zeros((1, 3)), 1, bias=np.array([0.0, 0.1, -np.inf]), score="sigmoid", renormalise=False)
    assert ids[0, 0] == 1 and w[0, 0] == 0.5


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
def test_route_gradient_against_differences(score, renormalise):
    rng = np.random.default_rng(1)
    T, E, k = 5, 12, 4
    l = rng.standard_normal((T, E))
    l[0, :9] = -np.inf          # three entries left
    l[1] = -np.inf              # none
    bias = 0.1 * rng.standard_normal(E)
    bias[5] = -np.inf
    ids, _, _ = orc.route(l, k, bias=bias, score=score)
    g = rng.standard_normal((T, k))
    d = orc.route_grad(l, ids, g, bias=bias, score=score, renormalise=renormalise, scale=1.7)
    h = 1e-5
    for t in range(T):
        for e in range(E):
            if not np.isfinite(l[t, e]):
                assert d[t, e] == 0
                continue
            up, dn = l.copy(), l.copy()
            up[t, e] += h
            dn[t, e] -= h
            diff = sum((g * s * orc.weights_of(v, ids, score, renormalise, 1.7, bias)).sum()
                       for v, s in ((up, 1), (dn, -1))) / (2 * h)
            # second differences of functions bounded by 1.7: h^2 terms, and rounding / h
            assert abs(diff - d[t, e]) <= 1e-8
