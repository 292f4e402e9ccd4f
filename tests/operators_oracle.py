"""The operators of learned retrieval in 64 bits on the CPU, from their
definitions: microscaled 4-bit rows, their products, routing and its gradient.

numpy only; a value's code is found by comparing it with all eight magnitudes,
the scale by integer exponents."""
import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
FMAX = float(np.finfo(np.float32).max)


def quantise(x):
    """(codes (n, 64 S) uint8, scales (n, 4 S) uint8) of x (n, K), float64."""
    x = np.asarray(x, np.float64)
    n, K = x.shape
    S = -(-K // 128)
    v = np.zeros((n, S * 128))
    v[:, :K] = x
    v = v.reshape(n, 4 * S, 32)
    bad = ~np.isfinite(v).all(2)
    top = np.abs(np.where(np.isfinite(v), v, 0.0)).max(2)
    exp = np.where(top > 0, np.frexp(top)[1] - 1, -10000)      # floor(log2 top)
    byte = np.clip(exp - 2 + 127, 0, 254)
    with np.errstate(invalid="ignore"):
        a = np.abs(np.ldexp(np.where(bad[:, :, None], 0.0, v), (127 - byte)[:, :, None]))
    dist = np.abs(a[..., None] - MAGNITUDES)
    code = dist.argmin(3)                                       # the lower of two at one distance
    up = np.minimum(code + 1, 7)
    tie = (code < 7) & (np.take_along_axis(dist, up[..., None], 3)[..., 0] == dist.min(3))
    code = np.where(tie & (code % 2 == 1), up, code)            # the middle goes to the even code
    code = np.where(a > 6, 7, code) + 8 * np.signbit(v)
    code = np.where(bad[:, :, None], 0, code).astype(np.uint8).reshape(n, -1)
    byte = np.where(bad, 255, byte).astype(np.uint8)
    return code[:, 0::2] | code[:, 1::2] << 4, byte


def dequantise(codes, scales, K):
    n = codes.shape[0]
    code = np.empty((n, codes.shape[1] * 2), np.uint8)
    code[:, 0::2], code[:, 1::2] = codes & 15, codes >> 4
    val = np.where(code & 8, -1.0, 1.0) * MAGNITUDES[code & 7]
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    with np.errstate(invalid="ignore"):
        return (val.reshape(n, -1, 32) * s[:, :, None]).reshape(n, -1)[:, :K]


def _live(logits, bias):
    l = np.minimum(np.asarray(logits, np.float64), FMAX)
    live = l > -np.inf
    if bias is not None:
        live = live & (np.asarray(bias, np.float64) > -np.inf)[None]
    return np.where(live, l, -np.inf), live


def scores(l, live, score):
    """Softmax over a row's live entries or sigmoids; 0 where not live."""
    with np.errstate(over="ignore", invalid="ignore"):
        if score == "sigmoid":
            return np.where(live, 1 / (1 + np.exp(-np.where(live, l, 0))), 0.0)
        top = l.max(1, keepdims=True)
        e = np.where(live, np.exp(np.where(live, l, 0) - np.where(top > -np.inf, top, 0)), 0.0)
        return e / np.where(e.sum(1, keepdims=True) > 0, e.sum(1, keepdims=True), 1)


def weights_of(logits, ids, score, renormalise, scale, bias=None):
    """The weights of a given choice (the function that route_grad differentiates)."""
    l, live = _live(logits, bias)
    has = ids >= 0
    at = np.maximum(ids, 0)
    if renormalise and score == "softmax":
        s = scores(np.where(has, np.take_along_axis(l, at, 1), -np.inf), has, "softmax")
    else:
        s = np.where(has, np.take_along_axis(scores(l, live, score), at, 1), 0.0)
    if renormalise:
        total = s.sum(1, keepdims=True)
        s = s / np.where(total > 0, total, 1)
    return scale * s


def route(logits, k, bias=None, groups=1, keep_groups=None, group_score="max", score="softmax", renormalise=True,
          scale=1.0):
    """(ids, weights, load), one row at a time by sorting tuples."""
    l, live = _live(logits, bias)
    T, E = l.shape
    keep_groups = groups if keep_groups is None else keep_groups
    by_score = bias is not None or (groups > 1 and group_score == "top2")
    key = scores(l, live, score) + (0 if bias is None else np.asarray(bias, np.float64)[None]) if by_score else l
    gs = E // groups
    ids = np.full((T, k), -1, np.int32)
    for t in range(T):
        cand = [e for e in range(E) if live[t, e]]
        if groups > 1:
            rank = []
            for g in range(groups):
                own = sorted((key[t, e] for e in cand if e // gs == g), reverse=True)[:2 if group_score == "top2" else 1]
                if own:
                    rank.append((-sum(own), g))
            kept = {g for _, g in sorted(rank)[:keep_groups]}
            cand = [e for e in cand if e // gs in kept]
        best = sorted(cand, key=lambda e: (-key[t, e], e))[:k]
        ids[t, :len(best)] = best
    load = np.bincount(ids[ids >= 0], minlength=E).astype(np.int32)
    return ids, weights_of(logits, ids, score, renormalise, scale, bias), load


def route_grad(logits, ids, dweights, bias=None, score="softmax", renormalise=True, scale=1.0):
    """d (sum dweights * weights) / d logits by the formulas."""
    l, live = _live(logits, bias)
    T, E = l.shape
    has = ids >= 0
    at = np.maximum(ids, 0)
    g = np.where(has, np.asarray(dweights, np.float64), 0.0)
    p = scores(l, live, score)
    d = np.zeros((T, E))
    if renormalise:
        w = weights_of(logits, ids, score, True, 1.0, bias)
        c = scale * w * (g - (g * w).sum(1, keepdims=True))
        if score == "sigmoid":
            c = c * (1 - np.take_along_axis(p, at, 1))
        np.add.at(d, (np.arange(T)[:, None], at), np.where(has, c, 0.0))
        return d
    np.add.at(d, (np.arange(T)[:, None], at), scale * g)
    if score == "sigmoid":
        return d * p * (1 - p)
    return p * (d - (d * p).sum(1, keepdims=True))


# ---- bounds that the GPU results are held to ------------------------------

# half a unit in the last place, relative, and half the least subnormal
ROUNDING = {"float32": (2.0 ** -24, 2.0 ** -150), "float16": (2.0 ** -11, 2.0 ** -25), "bfloat16": (2.0 ** -8, 2.0 ** -134)}


def product_bound(x, w, out_type):
    """What a product's fp32 sum and its final rounding may be off by: each of
    the J additions (and of the matrix instructions' internal ones) rounds by
    at most one unit in the last place, 2^-23, of a partial sum that the sum of
    magnitudes bounds."""
    J = x.shape[1]
    mag = np.abs(x) @ np.abs(w).T
    rel, least = ROUNDING[out_type]
    return (J + 8) * 2.0 ** -23 * mag * (1 + rel) + rel * np.abs(x @ w.T) + least + 2.0 ** -126 * J


# exp of a difference of fp32 logits within 64 of each other: the difference is
# rounded (64 * 2^-24), exp and the division by a sum of at most 1024 positive
# terms add a few units (8 * 2^-23); four times that for the products around it
WEIGHT_RTOL = 4 * (64 * 2.0 ** -24 + 8 * 2.0 ** -23)


def grad_bound(ref, dweights, scale, out_type):
    """The gradient's terms are differences of numbers up to scale * max|g| (an
    average of g among them), each good to WEIGHT_RTOL; then one rounding."""
    rel, least = ROUNDING[out_type]
    top = np.abs(np.asarray(dweights, np.float64)).max(1, keepdims=True)
    return 4 * WEIGHT_RTOL * scale * top * dweights.shape[1] + rel * np.abs(ref) + least
