"""A routing in 64 bits over whole arrays (numpy only): the choice by sorting;
weights and gradients of a choice from logarithms of the scores, which no logit
brings to zero; and bounds for the GPU's entry by entry."""
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


def choose(logits, k, bias=None, groups=1, keep_groups=None, group_score="max", score="softmax"):
    """(ids (T, k), load (E,)): ties to the lower index, -1 where fewer are live."""
    l, live = live_logits(logits, bias)
    T, E = l.shape
    key = l
    if bias is not None or (groups > 1 and group_score == "top2"):
        with np.errstate(over="ignore"):
            s = 1 / (1 + np.exp(-l)) if score == "sigmoid" else np.exp(_shares(l))
        key = np.where(live, s + (0.0 if bias is None else np.asarray(bias, np.float64)), -np.inf)
    if groups > 1:
        by = key.reshape(T, groups, E // groups)
        rank = by.max(2)
        if group_score == "top2" and E > groups:
            second = np.partition(by, -2, axis=2)[:, :, -2]
            rank = rank + np.where(second > -np.inf, second, 0.0)
        kept = np.argsort(-rank, axis=1, kind="stable")[:, :groups if keep_groups is None else keep_groups]
        keep = np.zeros((T, groups), bool)
        keep[np.arange(T)[:, None], kept] = True
        key = np.where(np.repeat(keep, E // groups, axis=1), key, -np.inf)
    ids = np.argsort(-key, axis=1, kind="stable")[:, :k]
    ids = np.where(np.take_along_axis(key, ids, 1) > -np.inf, ids, -1).astype(np.int32)
    return ids, np.bincount(ids[ids >= 0], minlength=E).astype(np.int32)


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
    """Of a weight, by row, in units of 2^-24 (half a unit in the last place): a
    difference v of logits, its product with a rounded log2 e and the exponential
    are off by at most 3 |v| + 4, in the term and again in the sum of its row;
    that sum is of at most 64 terms a lane, one after the other, and 6 exchanges;
    a division and two products make 4 more."""
    l, live = live_logits(logits, bias)
    low = np.where(live, l, np.inf).min(1)
    span = np.where(live.any(1), l.max(1), 0.0) - np.where(live.any(1), low, 0.0)
    span = np.minimum(span, 120.0)        # beyond, e^-span is below 2^-149 anyway
    return ((2 * (3 * span + 4) + 64 + 6 + 4) * 2.0 ** -24)[:, None]


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
