"""The operators of learned retrieval whose speed is followed: embedding rows
at four bits with their products, and the routing of queries to cells.

A case is a dict of plain values.  Its "kind" says what one pass is:

- "quantise": rows to microscaled 4-bit floating point, and the values that
  the codes stand for.
- "product_mx": scores of queries, quantised in the call, against rows held at
  four bits.
- "product": scores of queries as they are (fp32, binary16, bfloat16) against
  rows held at four bits.
- "product_grad": the gradient of those scores with respect to the queries.
- "route": each query's k cells (experts, shards) from its logits, their
  weights and the load of every cell; with "train" also the gradient with
  respect to the logits.

The format: 32 consecutive values of a row share a scale 2^(byte - 127), byte
255 standing for NaN; a value is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6,
two codes a byte, the even element in the low half; rows are padded with
blocks of zeros to 128 values.
"""
import math

import numpy as np
import torch

own = False   # False: the operators in elementary torch operations; True: the framework's calls

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
FMAX = 3.4028234663852886e38


def listed():
    return [
        # The queries that a server has collected for one search, 768-d
        # embeddings: little data, launches count.
        dict(name="quantise_queries", kind="quantise", R=48, K=768, dtype="f32"),
        # All rows of the headline index (1M x 128), when it is built.
        dict(name="quantise_rows", kind="quantise", R=1_000_000, K=128, dtype="f32"),
        # One query against the 1000 cluster centres: the smallest call.
        dict(name="product_mx_one", kind="product_mx", M=1, N=1000, K=128, dtype="f32", out="f32"),
        # The headline batch of 10k queries against a whole cell of the 1M
        # index (16 cells): all scores written.
        dict(name="product_mx_cell", kind="product_mx", M=10_000, N=62_500, K=128, dtype="f32", out="bf16"),
        # A layer of a query encoder over a training batch's tokens, both
        # sides at four bits.
        dict(name="product_mx_layer", kind="product_mx", M=8192, N=8192, K=4096, dtype="bf16", out="bf16"),
        # The same layer for one token, the activations as they are.
        dict(name="product_token", kind="product", M=1, N=16_384, K=4096, dtype="bf16", out="bf16"),
        # Odd sizes: 777 fp32 queries of 100 dimensions against a cell of an
        # index of 150001 points.
        dict(name="product_ragged", kind="product", M=777, N=9376, K=100, dtype="f32", out="f32"),
        # An ordinary batch of bfloat16 activations against 4-bit rows.
        dict(name="product_batch", kind="product", M=4096, N=8192, K=4096, dtype="bf16", out="bf16"),
        # Its gradient: what trains an encoder in front of frozen 4-bit rows.
        dict(name="grad_batch", kind="product_grad", M=4096, N=8192, K=4096, dtype="bf16", out="bf16"),
        # The gradient at odd sizes, binary16, a long sum over a cell's rows
        # for few dimensions.
        dict(name="grad_ragged", kind="product_grad", M=777, N=9376, K=100, dtype="f16", out="f16"),
        # 10k queries to the cells of a 16 x 16 grid: the cells outside a
        # query's range masked, some ranges empty, no more than 4 of the 16
        # shards a query.
        dict(name="route_cells", kind="route", T=10_000, E=256, k=8, dtype="f32", score="softmax", bias=False,
             groups=16, keep=4, group="max", renorm=True, scale=1.0, mask=0.6, train=False),
        # A training step's tokens to 256 experts: sigmoid scores, a balance
        # bias, groups by their two best, the gradient too.
        dict(name="route_train", kind="route", T=16_384, E=256, k=8, dtype="f32", score="sigmoid", bias=True,
             groups=8, keep=4, group="top2", renorm=True, scale=2.5, mask=0.0, train=True),
    ]


def _log(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["quantise", "product_mx", "product_mx", "product", "product", "product_grad", "route", "route"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "quantise":
        while True:
            R, K = _log(rng, 1, 1_000_000), _log(rng, 1, 8192)
            if R * K <= 128_000_000:
                return dict(kind=kind, R=R, K=K, dtype=dtype)
    if kind != "route":
        while True:
            M, N, K = _log(rng, 1, 10_000), _log(rng, 1, 62_500), _log(rng, 1, 8192)
            if M * N * K <= 8192 * 8192 * 4096 // (1 if kind == "product_mx" else 4) and M * N <= 625_000_000:
                return dict(kind=kind, M=M, N=N, K=K, dtype=dtype, out=dtype)
    groups = rng.choice([1, 1, 2, 4, 8, 16])
    E = groups * _log(rng, 2, 1024 // groups)
    keep = rng.randint(1, groups)
    return dict(kind=kind, T=_log(rng, 1, 32_768), E=E, k=rng.randint(1, min(16, keep * (E // groups))), dtype=dtype,
                score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups, keep=keep,
                group=rng.choice(["max", "top2"]), renorm=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]),
                mask=rng.choice([0.0, 0.0, 0.6]), train=rng.random() < 0.5)


# ---- inputs ---------------------------------------------------------------

def _rows(g, n, d, dtype):
    """Embedding-like rows: Gaussian, some dimensions much larger than the
    others, row lengths that differ."""
    x = torch.randn(n, d, generator=g, device="cuda")
    wide = 1.0 + 7.0 * (torch.rand(d, generator=g, device="cuda") < 0.03).float()
    long = torch.exp(0.5 * torch.randn(n, 1, generator=g, device="cuda"))
    return (x.mul_(wide).mul_(long).mul_(1.0 / math.sqrt(d))).to(TYPES[dtype])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    st = dict(case=case)
    kind = case["kind"]
    if kind == "quantise":
        st["x"] = _rows(g, case["R"], case["K"], case["dtype"])
    elif kind == "route":
        T, E = case["T"], case["E"]
        logits = 1.5 * torch.randn(T, E, generator=g, device="cuda") + 0.5 * torch.randn(E, generator=g, device="cuda")
        if case["mask"]:
            # a query's own share of masked cells; one query in 64 has no cell left
            share = case["mask"] * 2.0 * torch.rand(T, 1, generator=g, device="cuda")
            drop = torch.rand(T, E, generator=g, device="cuda") < share
            drop |= torch.rand(T, 1, generator=g, device="cuda") < 1.0 / 64
            logits.masked_fill_(drop, -math.inf)
        st["logits"] = logits.to(TYPES[case["dtype"]])
        # the balance bias moves in steps of 0.001
        st["bias"] = (0.001 * torch.randint(-100, 101, (E,), generator=g, device="cuda").float()
                      if case["bias"] else None)
        if case["train"]:
            st["dweights"] = torch.randn(T, case["k"], generator=g, device="cuda")
    else:
        M, N, K = case["M"], case["N"], case["K"]
        codes, scales = _pack(_rows(g, N, K, "f32"))
        if own:
            import garfield_amd as gf
            st["w"] = gf.MXRows(codes, scales, K)
        else:
            st["codes"], st["scales"] = codes, scales
        if kind == "product_grad":
            st["dy"] = (torch.randn(M, N, generator=g, device="cuda") / math.sqrt(N)).to(TYPES[case["dtype"]])
        else:
            st["x"] = _rows(g, M, K, case["dtype"])
    return st


# ---- the plain form -------------------------------------------------------

def _blocks(x, width):
    """x in 32 bits, rows padded with zeros to a multiple of width, by blocks of 32."""
    n, d = x.shape
    p = torch.zeros(n, -(-d // width) * width, device=x.device)
    p[:, :d] = x
    return p.view(n, -1, 32)


def _codes(x, width):
    """Codes (0..15) and scale bytes of the rows' blocks."""
    v = _blocks(x, width)
    top = v.abs().amax(2, keepdim=True)
    # top = m * 2^e with m in [0.5, 1): floor(log2 top) = e - 1
    byte = torch.where(top == 0, torch.zeros_like(top), torch.frexp(top)[1].float() + (127 - 3)).clamp(0, 254)
    a = v.abs() / torch.exp2(byte - 127)
    # between two values the middle goes to the even code
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code + 8 * torch.signbit(v).to(torch.uint8)
    bad = ~torch.isfinite(v).all(2, keepdim=True)
    byte = torch.where(bad, torch.full_like(byte, 255.0), byte).to(torch.uint8)
    return torch.where(bad, torch.zeros_like(code), code), byte.squeeze(2)


def _pack(x):
    code, byte = _codes(x, 128)
    n = code.shape[0]
    pair = code.view(n, -1, 2)
    return (pair[:, :, 0] | (pair[:, :, 1] << 4)).contiguous(), byte.contiguous()


def _values(code, byte):
    """What codes (rows, blocks, 32) and scale bytes (rows, blocks) stand for."""
    table = torch.tensor(GRID + tuple(-v for v in GRID), device=code.device)
    scale = torch.exp2(byte.float() - 127)
    scale = torch.where(byte == 255, torch.full_like(scale, math.nan), scale)
    return (table[code.int()] * scale[:, :, None]).view(code.shape[0], -1)


def _unpack(codes, scales, K):
    n = codes.shape[0]
    code = torch.stack((codes & 15, codes >> 4), 2).view(n, -1, 32)
    return _values(code, scales)[:, :K]


def _scores(logits, score, live):
    """Softmax over the live entries, or the sigmoid, in the logits' precision."""
    if score == "sigmoid":
        s = 1 / (1 + torch.exp(-logits))
        return torch.where(live, s, torch.zeros_like(s))
    low = torch.where(live, logits, torch.full_like(logits, -math.inf))
    top = low.amax(1, keepdim=True)
    e = torch.where(live, torch.exp(low - torch.where(top == -math.inf, torch.zeros_like(top), top)),
                    torch.zeros_like(low))
    return e / torch.where(top == -math.inf, torch.ones_like(top), e.sum(1, keepdim=True))


def _select(c, logits, bias, live):
    """The chosen experts, best first, -1 where fewer than k are left.  The
    keys are in 64 bits where scores decide: which expert is chosen must not
    hang on the last bit of a 32-bit exponential."""
    T, E, G = logits.shape[0], c["E"], c["groups"]
    by_score = bias is not None or (G > 1 and c["group"] == "top2")
    key = _scores(logits.double(), c["score"], live) if by_score else logits.double()
    if bias is not None:
        key = key + bias.double()
    none = torch.full_like(key, -math.inf)
    key = torch.where(live, key, none)
    if G > 1:
        best = torch.sort(key.view(T, G, E // G), dim=2, descending=True)[0]
        rank = best[:, :, 0]
        if c["group"] == "top2" and E // G > 1:
            second = best[:, :, 1]
            rank = rank + torch.where(second == -math.inf, torch.zeros_like(second), second)
        kept = torch.sort(rank, dim=1, descending=True, stable=True)[1][:, :c["keep"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=key.device).scatter_(1, kept, True)
        key = torch.where(keep.repeat_interleave(E // G, 1), key, none)
    val, ids = torch.sort(key, dim=1, descending=True, stable=True)
    return torch.where(val[:, :c["k"]] > -math.inf, ids[:, :c["k"]], torch.full_like(ids[:, :c["k"]], -1))


def _route(c, raw, bias, dweights):
    logits = raw.float()
    live = (logits > -math.inf).expand_as(logits)      # NaN is masked too
    if bias is not None:
        live = live & (bias > -math.inf)
    logits = torch.where(live, logits, torch.zeros_like(logits)).clamp(-FMAX, FMAX)
    ids = _select(c, logits, bias, live)
    has = ids >= 0
    at = ids.clamp(min=0)
    zero = torch.zeros((), device=raw.device)
    scores = _scores(logits, c["score"], live)
    if c["renorm"] and c["score"] == "softmax":
        # the softmax over all entries cancels: the chosen logits alone
        s = _scores(logits.gather(1, at), "softmax", has)
    else:
        s = torch.where(has, scores.gather(1, at), zero)
    total = s.sum(1, keepdim=True)
    share = torch.where(total > 0, s / torch.where(total > 0, total, torch.ones_like(total)), zero)
    weights = c["scale"] * (share if c["renorm"] else s)
    load = torch.zeros(c["E"] + 1, dtype=torch.int32, device=raw.device)
    load.scatter_add_(0, torch.where(has, ids, torch.full_like(ids, c["E"])).flatten(),
                      torch.ones(ids.numel(), dtype=torch.int32, device=raw.device))
    out = [ids.int(), weights, load[:c["E"]]]
    if dweights is not None:
        g = torch.where(has, dweights, zero)
        if c["renorm"]:
            ds = c["scale"] * (g - (g * share).sum(1, keepdim=True))
            ds = ds * share if c["score"] == "softmax" else ds * share * (1 - s)
            d = torch.zeros_like(logits).scatter_add_(1, at, torch.where(has, ds, zero))
        else:
            d = torch.zeros_like(logits).scatter_add_(1, at, c["scale"] * g)
            if c["score"] == "softmax":
                d = scores * (d - (d * scores).sum(1, keepdim=True))
            else:
                d = d * scores * (1 - scores)
        out.append(d.to(raw.dtype))
    return out


def _plain(st):
    c = st["case"]
    if c["kind"] == "quantise":
        code, byte = _codes(st["x"], 32)
        return _values(code, byte)[:, :c["K"]].to(_kept(c)).contiguous()
    if c["kind"] == "route":
        return _route(c, st["logits"], st["bias"], st.get("dweights"))
    w = _unpack(st["codes"], st["scales"], c["K"])
    if c["kind"] == "product_grad":
        return (st["dy"].float() @ w).to(TYPES[c["out"]])
    x = st["x"].float()
    if c["kind"] == "product_mx":
        code, byte = _codes(x, 32)
        x = _values(code, byte)[:, :c["K"]]
    return (x @ w.t()).to(TYPES[c["out"]])


def _kept(c):
    """The type that holds quantised values exactly: bfloat16 does, binary16's range does not."""
    return torch.bfloat16 if c["dtype"] == "bf16" else torch.float32


def _framework(st):
    import garfield_amd as gf
    c = st["case"]
    if c["kind"] == "quantise":
        return gf.mx_dequantise(gf.mx_quantise(st["x"]), dtype=_kept(c))
    if c["kind"] == "product_mx":
        return gf.mx_product(gf.mx_quantise(st["x"]), st["w"], dtype=TYPES[c["out"]])
    if c["kind"] == "product":
        return gf.mx_product(st["x"], st["w"], dtype=TYPES[c["out"]])
    if c["kind"] == "product_grad":
        return gf.mx_product_grad(st["dy"], st["w"], dtype=TYPES[c["out"]])
    how = dict(score=c["score"], renormalise=c["renorm"], scale=c["scale"])
    r = gf.route(st["logits"], c["k"], bias=st["bias"], groups=c["groups"], keep_groups=c["keep"],
                 group_score=c["group"], **how)
    out = [r.ids, r.weights, r.load]
    if c["train"]:
        out.append(gf.route_grad(st["logits"], r.ids, st["dweights"], bias=st["bias"], **how))
    return out


def run(state):
    return _framework(state) if own else _plain(state)


# ---- what a pass has to move and compute ----------------------------------

def work(case):
    kind = case["kind"]
    if kind == "quantise":
        n = case["R"] * case["K"]
        return {"bytes": n * (SIZE[case["dtype"]] + (2 if case["dtype"] == "bf16" else 4)), "flops": 2 * n}
    if kind == "route":
        n, e = case["T"] * case["E"], SIZE[case["dtype"]]
        return {"bytes": n * e * (2 if case["train"] else 1) + case["T"] * case["k"] * (12 if case["train"] else 8)
                + case["E"] * 8, "flops": 8 * n}
    M, N, K = case["M"], case["N"], case["K"]
    w = N * -(-K // 32) * 17
    e, o = SIZE[case["dtype"]], SIZE[case["out"]]
    if kind == "product_grad":
        return {"bytes": M * N * e + w + M * K * o, "flops": 2 * M * N * K}
    return {"bytes": M * K * e + w + M * N * o, "flops": 2 * M * N * K}


# ---- the definitions in 64 bits -------------------------------------------

def _two_to(e):
    """2^e in 64 bits, e whole numbers in int64: the exponent field itself."""
    return ((e + 1023) << 52).view(torch.float64)


def _exact_mx(x):
    """The value that stands for each entry of x after quantisation, by the
    step of its binade."""
    n, d = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -d % 32)).reshape(n, -1, 32)
    top = v.abs().amax(2, keepdim=True)
    # floor(log2 top) is the exponent field (0 for top = 0, which the limit catches)
    s = _two_to(((top.contiguous().view(torch.int64) >> 52) - 1023 - 2).clamp(min=-127))
    v /= s
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0)).double()
    return ((torch.round(v / step) * step).clamp(-6, 6) * s).reshape(n, -1)[:, :d]


def _exact_route(c, raw, bias, dweights):
    l = np.minimum(raw.double().cpu().numpy(), FMAX)
    T, E, G, k = c["T"], c["E"], c["groups"], c["k"]
    b = np.zeros(E) if bias is None else bias.double().cpu().numpy()
    live = (l > -np.inf) & (b > -np.inf)[None]
    with np.errstate(all="ignore"):
        if c["score"] == "sigmoid":
            s = np.where(live, 1 / (1 + np.exp(-l)), 0.0)
        else:
            m = np.where(live, l, -np.inf).max(1, keepdims=True)
            s = np.where(live, np.exp(l - m), 0.0)
            s = s / np.maximum(s.sum(1, keepdims=True), 1e-300)
    by_score = bias is not None or (G > 1 and c["group"] == "top2")
    key = np.where(live, (s + b) if by_score else l, -np.inf)
    if G > 1:
        part = -np.sort(-key.reshape(T, G, -1), axis=2)
        rank = part[:, :, 0]
        if c["group"] == "top2" and part.shape[2] > 1:
            rank = rank + np.where(part[:, :, 1] > -np.inf, part[:, :, 1], 0.0)
        order = np.argsort(-rank, axis=1, kind="stable")
        place = np.empty_like(order)
        np.put_along_axis(place, order, np.broadcast_to(np.arange(G), (T, G)), 1)
        key = np.where(np.repeat(place < c["keep"], E // G, axis=1), key, -np.inf)
    ids = np.argsort(-key, axis=1, kind="stable")[:, :k]
    has = np.take_along_axis(key, ids, 1) > -np.inf
    if c["renorm"] and c["score"] == "softmax":
        # shares of the chosen logits: every other entry cancels
        z = np.where(has, np.take_along_axis(l, ids, 1), -np.inf)
        with np.errstate(all="ignore"):
            chosen = np.where(has, np.exp(z - z.max(1, keepdims=True)), 0.0)
    else:
        chosen = np.where(has, np.take_along_axis(s, ids, 1), 0.0)
    total = chosen.sum(1, keepdims=True)
    norm = np.where(total > 0, total, 1.0) if c["renorm"] else 1.0
    w = c["scale"] * chosen / norm
    load = np.bincount(ids[has], minlength=E).astype(np.int32)
    out = [np.where(has, ids, -1).astype(np.int32), w, load]
    if dweights is not None:
        g = np.where(has, dweights.double().cpu().numpy(), 0.0)
        if c["renorm"]:
            gs = c["scale"] * (g - (g * chosen / norm).sum(1, keepdims=True)) / norm
        else:
            gs = c["scale"] * g
        ds = np.zeros((T, E))
        np.put_along_axis(ds, ids, np.where(has, gs, 0.0), 1)
        if c["score"] == "sigmoid":
            d = ds * s * (1 - s)
        elif c["renorm"]:
            d = np.zeros((T, E))
            np.put_along_axis(d, ids, np.where(has, gs * chosen, 0.0), 1)
        else:
            d = s * (ds - (ds * s).sum(1, keepdims=True))
        out.append(d)
    return [torch.from_numpy(np.ascontiguousarray(o)) for o in out]


def exact(case, seed):
    global own
    kind = case["kind"]
    # the inputs of the plain form, whichever form is measured
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if kind == "quantise":
        return _exact_mx(st["x"])
    if kind == "route":
        return _exact_route(case, st["logits"], st["bias"], st.get("dweights"))
    # the rows that the codes stand for: a sign bit, then exponent and fraction
    # bits as the format defines them
    codes, scales, K = st["codes"], st["scales"], case["K"]
    code = torch.stack((codes % 16, codes // 16), 2).reshape(codes.shape[0], -1).double()
    sign = torch.where(code >= 8, -1.0, 1.0).double()
    mag = code - 8 * (code >= 8)
    ex, frac = torch.floor(mag / 2), mag % 2
    val = torch.where(ex == 0, 0.5 * frac, _two_to((ex - 1).long()) * (1 + 0.5 * frac))
    w = sign * val * _two_to(scales.long() - 127).repeat_interleave(32, 1)
    w = w[:, :K].contiguous()
    if kind == "product_grad":
        return st["dy"].double() @ w
    x = _exact_mx(st["x"]) if kind == "product_mx" else st["x"].double()
    return x @ w.t().contiguous()
