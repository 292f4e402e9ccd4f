"""The reference of routing weights in logarithms: against the oracle where that
does not underflow, against differences, and what its bounds can see (CPU)."""
import numpy as np
import pytest

import operators_oracle as orc
import route_reference as ref


def _case(T, E, k, seed, low=0.0, masked=True):
    rng = np.random.default_rng(seed)
    l = (2 * rng.standard_normal((T, E)) + low).astype(np.float32).astype(np.float64)
    if masked:
        l[::7] = -np.inf
        l[1::5, ::3] = -np.inf
        l[2::9, 1] = np.inf
    ids, _, _ = orc.route(l, k)
    return l, ids, rng.standard_normal((T, k))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
def test_agrees_with_the_oracle(score, renormalise):
    l, ids, g = _case(40, 50, 6, 1)
    how = dict(score=score, renormalise=renormalise, scale=1.7)
    w = orc.weights_of(l, ids, score, renormalise, 1.7)
    assert np.allclose(ref.weights(l, ids, **how), w, rtol=1e-12, atol=1e-300)
    d, mag = ref.gradient(l, ids, g, **how)
    assert np.allclose(d, orc.route_grad(l, ids, g, **how), rtol=1e-11, atol=1e-14)
    assert (np.abs(d) <= mag * (1 + 1e-12) + 1e-300).all()


@pytest.mark.parametrize("low", [0.0, -30.0, -600.0])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gradient_against_differences(score, low):
    l, ids, g = _case(6, 12, 4, 2, low, masked=False)
    l[0, 3:] = -np.inf
    ids, _, _ = orc.route(l, 4)
    d, _ = ref.gradient(l, ids, g, score=score, scale=1.3)
    h = 1e-5
    for t in range(6):
        for e in range(12):
            if l[t, e] == -np.inf:
                assert d[t, e] == 0
                continue
            up, dn = l.copy(), l.copy()
            up[t, e] += h
            dn[t, e] -= h
            diff = sum((g * s * ref.weights(v, ids, score=score, scale=1.3)).sum() for v, s in ((up, 1), (dn, -1))) / (2 * h)
            assert abs(diff - d[t, e]) <= 1e-8      # h^2 terms of bounded functions, and rounding / h


def test_shares_of_low_sigmoids():
    w = ref.weights(np.array([[-100.0, -101.0]]), np.array([[0, 1]]), score="sigmoid")
    assert np.allclose(w, [[1 / (1 + np.exp(-1)), 1 / (1 + np.exp(1))]], rtol=1e-12)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep,rank", [(1, 1, "max"), (6, 2, "max"), (6, 2, "top2"), (12, 5, "top2"), (6, 6, "top2")])
def test_choice_agrees_with_the_oracle(groups, keep, rank, score):
    rng = np.random.default_rng(groups)
    l, _, _ = _case(60, 12, 4, 5)
    l[20:40] = np.round(l[20:40])
    for bias in (None, 0.1 * rng.standard_normal(12), np.array([0.25] * 11 + [-np.inf])):
        want = orc.route(l, 2, bias=bias, groups=groups, keep_groups=keep, group_score=rank, score=score)
        got = ref.choose(l, 2, bias, groups, keep, rank, score)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[2])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("E,k", [(16, 2), (64, 8), (256, 8), (1024, 16), (1024, 64)])
def test_gradient_bound_sees_a_lost_term(E, k, dtype):
    """Softmax over all entries: a gradient without the term of the entries that
    were not chosen, or with it a hundredth off, is outside the bound."""
    l, ids, g = _case(30, E, k, E + k, masked=False)
    how = dict(renormalise=False, scale=2.5)
    d, mag = ref.gradient(l, ids, g, **how)
    bound = ref.gradient_bound(d, mag, l, ids, g, 2.5, dtype)
    other = np.ones(l.shape, bool)
    np.put_along_axis(other, ids, False, 1)
    # what a type's own least value swallows cannot be seen in it
    seen = other & (np.abs(d) > 4 * orc.ROUNDING[dtype][1])
    assert seen.sum() > 0.9 * other.sum()
    # entries whose average of gradients nearly vanishes have little to lose
    assert (np.abs(d) > bound)[seen].mean() > 0.99
    if dtype == "float32":
        assert (np.abs(0.01 * d) > bound)[seen].mean() > 0.9
    # the bound that is absolute in the largest gradient lets the lost term pass at the largest size
    loose = orc.grad_bound(d, g, 2.5, dtype)
    if (E, k) == (1024, 64):
        assert (np.abs(d) <= loose)[other].all()
