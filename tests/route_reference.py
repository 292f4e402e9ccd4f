"""Weights and gradients of a routing in 64 bits from logarithms of the scores,
which no logit brings to zero, and bounds for the GPU's entry by entry.  numpy
only; the choice (ids) is an input."""
import numpy as np

from operators_oracle import FMAX, ROUNDING

LEAST_SIGMOID = np.float32(-708.39642)     # a smaller one counts as 0


def live_logits(logits, bias=None):
    """(logits with -inf where masked, +inf as fp32's largest; truth values)."""
    l = np.minimum(np.asarray(logits, np.float64), FMAX)
    live = l > -np.inf
    if bias is not None:
        live = live & (np.asarray(bias, np.float64) > -np.inf)[None]
    return np.where(live, l, -np.inf), live


def _shares(x):
    """The logarithm of exp(x) over its sum over a row."""
    top = x.max(1, keepdims=True)
    top = np.where(top > -np.inf, top, 0.0)
    x = x - top                             # first: a large top would swallow the sum's logarithm
    total = np.exp(x).sum(1, keepdims=True)
    return x - np.log(np.where(total > 0, total, 1.0))


def _chosen(logits, ids, score, renormalise, bias):
    """(logarithms of the weights at scale 1, of the sigmoids of the chosen or
    None, of the softmax over all entries or None)."""
    l, _ = live_logits(logits, bias)
    has = ids >= 0
    at = np.where(has, np.take_along_axis(l, np.maximum(ids, 0), 1), -np.inf)
    if score == "sigmoid":
        s = np.where(at >= LEAST_SIGMOID, -np.logaddexp(0.0, -at), -np.inf)
        return (_shares(s) if renormalise else s), s, None
    if renormalise:
        return _shares(at), None, None
    p = _shares(l)
    return np.where(has, np.take_along_axis(p, np.maximum(ids, 0), 1), -np.inf), None, p


def weights(logits, ids, score="softmax", renormalise=True, scale=1.0, bias=None):
    return scale * np.exp(_chosen(logits, ids, score, renormalise, bias)[0])


def gradient(logits, ids, dweights, score="softmax", renormalise=True, scale=1.0, bias=None):
    """(d (sum dweights * weights) / d logits, the same with every term's
    magnitude: what rounding errors are measured by)."""
    lw, ls, lp = _chosen(logits, ids, score, renormalise, bias)
    has, w = ids >= 0, np.exp(lw)
    g = np.where(has, np.asarray(dweights, np.float64), 0.0)
    T, E = np.shape(logits)
    d, mag = np.zeros((T, E)), np.zeros((T, E))
    mean, size = (g * w).sum(1, keepdims=True), (np.abs(g) * w).sum(1, keepdims=True)
    if score == "sigmoid":
        rest = np.where(has, -np.expm1(ls), 0.0)      # 1 - sigmoid
        c, m = (g - mean, np.abs(g) + size) if renormalise else (g, np.abs(g))
        c, m = c * w * rest, m * w
    elif renormalise:
        c, m = w * (g - mean), w * (np.abs(g) + size)
    else:
        p = np.exp(lp)
        d, mag = -p * mean, p * size
        c, m = w * g, w * np.abs(g)
    rows = np.broadcast_to(np.arange(T)[:, None], ids.shape)[has]
    np.add.at(d, (rows, ids[has]), c[has])
    np.add.at(mag, (rows, ids[has]), m[has])
    return scale * d, scale * mag


def relative_error(logits, ids, bias=None):
    """Of a weight, by row: a difference of logits is rounded by 2^-24 of itself,
    the exponential makes that its relative error and adds two units in the last
    place (2^-23), the sum of at most 1024 positive terms at most 16 more (16 or
    64 lanes of at most 64 terms, added as a tree, each term as far off as the
    weight: twice all of it), a division and two products three."""
    l, live = live_logits(logits, bias)
    with np.errstate(invalid="ignore"):
        span = np.where(live, l, l.max(1, keepdims=True)).max(1) - np.where(live, l, np.inf).min(1)
    span = np.minimum(np.where(live.any(1), span, 0.0), 120.0)        # beyond, e^-span is below 2^-149 anyway
    return (2 * (span * 2.0 ** -24 + 2 * 2.0 ** -23) + (16 + 3) * 2.0 ** -23)[:, None]


def weight_bound(ref, logits, ids, scale, bias=None):
    """A sigmoid or an exponential below 2^-126 is held in steps of 2^-149; a sum
    that it is divided by is not below 2^-25."""
    return relative_error(logits, ids, bias) * np.abs(ref) + scale * 2.0 ** -124


def gradient_bound(ref, mag, logits, ids, dweights, scale, out_type, bias=None):
    """Each term is a product of a weight, good to the relative error, with a
    gradient or an average of gradients by weights: twice that error and three
    roundings; then one to the type."""
    rel, least = ROUNDING[out_type]
    top = np.abs(np.where(ids >= 0, dweights, 0.0)).max(1, keepdims=True)
    return (2 * relative_error(logits, ids, bias) + 3 * 2.0 ** -23) * mag + rel * np.abs(ref) + least + scale * top * 2.0 ** -123
