"""The operators of learned retrieval on the GPU against their 64-bit oracle.

Codes, scales, ids and loads are compared exactly; products within the bound
of fp32 sums (operators_oracle.product_bound), and exactly where the inputs
make every partial sum a multiple of 1/8 below 2^20; weights and gradients
within the bounds derived there."""
import numpy as np
import pytest
import torch

import garfield_amd as gf
import operators_oracle as orc

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _case(*a):
    print("case", *a, flush=True)


def _np(t):
    return t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _name(dtype):
    return str(dtype).split(".")[1]


def _strided(x, extra, fill=float("nan"), shift=0):
    """x's values in a matrix of a longer row distance, fill between the rows,
    starting shift elements into the allocation."""
    n, d = x.shape
    buf = torch.full((shift + n * (d + extra) + 8,), fill, dtype=x.dtype, device="cuda")
    v = buf[shift:shift + n * (d + extra)].view(n, d + extra)[:, :d]
    v.copy_(x)
    return v


def _rows(n, d, dtype, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g)
    if spread:
        x = x * torch.exp(2 * torch.randn(n, 1, generator=g))
    return x.to(dtype).cuda()


def _mx(n, d, seed):
    """MXRows of random rows and the 64-bit values that they stand for."""
    codes, scales = orc.quantise(_np(_rows(n, d, torch.float32, seed)))
    w = gf.MXRows(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), d)
    return w, orc.dequantise(codes, scales, d)


def _check_product(out, x, w, what):
    assert out.shape == (x.shape[0], w.shape[0])
    got, ref = _np(out), x @ w.T
    bound = orc.product_bound(x, w, _name(out.dtype))
    # what rounds beyond the type's largest value is an infinity of its sign
    top = float(torch.finfo(out.dtype).max) * (1 + orc.ROUNDING[_name(out.dtype)][0] / 2)
    over = np.isinf(got) & (np.sign(got) == np.sign(ref)) & (np.abs(ref) + bound >= top)
    err = np.where(over, 0.0, np.abs(np.where(over, ref, got) - ref))
    assert (err <= bound).all(), f"{what}: error up to {(err / np.maximum(bound, 1e-300)).max():.3g} of the bound"


# ---- quantisation ---------------------------------------------------------

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,d", [(1, 1), (1, 128), (3, 31), (5, 32), (2, 33), (7, 100), (4, 127), (2, 129), (33, 768),
                                 (300, 96), (1, 5000)])
def test_quantise_exact(n, d, dtype):
    _case("quantise", n, d, dtype)
    x = _rows(n, d, TYPES[dtype], n * 1000 + d)
    for v in (x, _strided(x, 3, shift=1), _strided(x, 32)):
        w = gf.mx_quantise(v)
        codes, scales = orc.quantise(_np(x))
        assert np.array_equal(_np(w.scales), scales)
        assert np.array_equal(_np(w.codes), codes)
        for out in TYPES.values():
            got = gf.mx_dequantise(w, out)
            ref = torch.from_numpy(orc.dequantise(codes, scales, d)).to(out)
            assert torch.equal(got.cpu(), ref)


def test_quantise_edges():
    """Ties, limits of the scale, zeros of both signs, infinities and NaN."""
    _case("quantise edges")
    x = np.zeros((16, 64), np.float32)
    x[0, :15] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, 6.0, 7.9, -7.9, 0.26, 5.01]
    x[1] = x[0, 0] * 2.0 ** -140
    x[2, :3] = [2.0 ** -149, -2.0 ** -127, 2.0 ** -126]
    x[3, :3] = [3.4028235e38, -3.4028235e38, 1e38]
    x[4, :2] = [np.inf, 1.0]
    x[5, 40] = np.nan
    x[5, 0] = 1.0
    x[6, 33] = -np.inf
    x[7] = -0.0
    x[8, ::2] = 2.0 ** -120
    for i in range(9, 16):
        x[i] = x[0, np.arange(64) % 15] * np.float32(2.0 ** (i * 20 - 250))
    w = gf.mx_quantise(torch.from_numpy(x).cuda())
    codes, scales = orc.quantise(x)
    assert np.array_equal(_np(w.scales), scales) and np.array_equal(_np(w.codes), codes)
    v = orc.dequantise(codes, scales, 64)
    assert np.array_equal(_np(gf.mx_dequantise(w)), v, equal_nan=True)
    assert np.isnan(v[5, 32:]).all() and not np.isnan(v[5, :32]).any()


def test_quantise_bits_of_every_kind():
    """Random bit patterns: all exponents, subnormals, NaN payloads."""
    _case("quantise bits")
    rng = np.random.default_rng(3)
    for dt, bits in (("f32", np.uint32), ("f16", np.uint16), ("bf16", np.uint16)):
        raw = rng.integers(0, np.iinfo(bits).max, (400, 64), dtype=np.int64).astype(bits)
        x = torch.from_numpy(raw.view(np.int32 if bits is np.uint32 else np.int16)).cuda().view(TYPES[dt])
        w = gf.mx_quantise(x)
        codes, scales = orc.quantise(_np(x))
        assert np.array_equal(_np(w.scales), scales) and np.array_equal(_np(w.codes), codes)


# ---- products -------------------------------------------------------------

SIZES = [(1, 1, 1), (1, 1000, 128), (2, 17, 33), (5, 64, 768), (15, 31, 100), (16, 16, 32), (17, 129, 127),
         (33, 300, 129), (64, 257, 96), (129, 130, 200), (300, 520, 160), (1, 40, 5000), (3, 5000, 64),
         (257, 255, 1030)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(M, N, K, dtype):
    _case("product", M, N, K, dtype)
    w, wv = _mx(N, K, N + K)
    x = _rows(M, K, TYPES[dtype], M + K)
    for v in (x, _strided(x, 5, shift=1), _strided(x, 64)):
        for out in (TYPES[dtype], torch.float32):
            _check_product(gf.mx_product(v, w, dtype=out), _np(x), wv, "product")


@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_mx(M, N, K):
    _case("product_mx", M, N, K)
    w, wv = _mx(N, K, N + K)
    x, xv = _mx(M, K, M + 7 * K)
    for out in TYPES.values():
        _check_product(gf.mx_product(x, w, dtype=out), xv, wv, "product_mx")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_grad(M, N, K, dtype):
    _case("product_grad", M, N, K, dtype)
    w, wv = _mx(N, K, N + K)
    dy = _rows(M, N, TYPES[dtype], M + N)
    for v in (dy, _strided(dy, 5, shift=1), _strided(dy, 64)):
        for out in (TYPES[dtype], torch.float32):
            _check_product(gf.mx_product_grad(v, w, dtype=out), _np(dy), np.ascontiguousarray(wv.T), "grad")


def _small_rows(n, d, seed):
    """Codes of every kind under scales 1/2, 1 and 2: multiples of 1/4 up to 12."""
    rng = np.random.default_rng(seed)
    S = -(-d // 128)
    nib = rng.integers(0, 16, (n, S * 128)).astype(np.uint8)
    nib[:, d:] = 0
    scales = rng.integers(126, 129, (n, 4 * S)).astype(np.uint8)
    scales[:, -(-d // 32):] = 0
    codes = nib[:, 0::2] | nib[:, 1::2] << 4
    return gf.MXRows(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), d), orc.dequantise(codes, scales, d)


@pytest.mark.parametrize("M,N,K", [(1, 1000, 128), (1, 70, 4096), (4, 333, 1024), (16, 500, 100), (31, 129, 768),
                                   (200, 300, 640), (513, 770, 96), (700, 260, 2000), (1030, 1100, 256),
                                   (3700, 3601, 640), (3850, 4001, 1060), (109, 33000, 130), (2100, 8200, 70),
                           (1900, 2050, 4000), (3, 50000, 100), (2, 49500, 700), (16, 13000, 1100), (5, 12500, 520),
                           (7, 4500, 1100), (5, 33000, 1100), (130, 1900, 2100), (300, 3001, 600), (26, 1931, 1000)])
def test_products_bit_for_bit(M, N, K):
    """Every product is a multiple of 1/16 and every partial sum below 2^20, so
    fp32 sums are exact in any order; a wrong element cannot hide."""
    _case("exact products", M, N, K)
    w, wv = _small_rows(N, K, N + K)
    xm, xv = _small_rows(M, K, M)
    assert np.array_equal(_np(gf.mx_product(xm, w)), xv @ wv.T)
    rng = np.random.default_rng(M * N)
    for dtype in TYPES.values():
        x = rng.integers(-8, 9, (M, K)).astype(np.float64)
        assert np.array_equal(_np(gf.mx_product(torch.from_numpy(x).to(dtype).cuda(), w, dtype=torch.float32)), x @ wv.T)
        y = rng.integers(-8, 9, (M, N)).astype(np.float64)
        assert np.array_equal(_np(gf.mx_product_grad(torch.from_numpy(y).to(dtype).cuda(), w, dtype=torch.float32)), y @ wv)


def test_fp32_values_enter_unrounded():
    """1 + 2^-23 times 1, minus 1: an input rounded to fewer bits gives 0."""
    _case("unrounded")
    for M in (1, 40, 300):
        K = 128
        x = torch.zeros(M, K, device="cuda")
        x[:, 0], x[:, 64] = 1 + 2.0 ** -23, -1.0
        wv = np.zeros((50, K))
        wv[:, 0] = wv[:, 64] = 1.0
        codes, scales = orc.quantise(wv)
        w = gf.MXRows(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), K)
        assert (gf.mx_product(x, w) == 2.0 ** -23).all()
        dy = torch.zeros(M, 50, device="cuda")
        dy[:, 0], dy[:, 49] = 1 + 2.0 ** -23, -1.0
        dx = gf.mx_product_grad(dy, w)
        assert (dx[:, 0] == 2.0 ** -23).all() and (dx[:, 1] == 0).all()


@pytest.mark.parametrize("M", [1, 7, 40, 300])
def test_infinities_and_nan_stay_in_their_rows(M):
    _case("non-finite", M)
    N, K = 150, 200
    w, wv = _mx(N, K, 5)
    scales = w.scales.clone()
    scales[3, 1] = 255                       # a NaN block in row 3
    wn = gf.MXRows(w.codes, scales, K)
    for dtype in TYPES.values():
        x = _rows(M, K, dtype, 6, spread=False)
        clean = gf.mx_product(x, wn, dtype=torch.float32)
        assert torch.isnan(clean[:, 3]).all() and torch.isfinite(clean[:, [0, 1, 2, 4, 149]]).all()
        x[M - 1, 199] = float("inf")
        out = gf.mx_product(x, w, dtype=torch.float32)
        assert torch.isfinite(out[:M - 1]).all()
        with np.errstate(invalid="ignore"):
            want = np.inf * np.sign(wv[:, 199])
        got = _np(out[M - 1])
        assert np.array_equal(got[wv[:, 199] != 0], want[wv[:, 199] != 0]) and np.isnan(got[wv[:, 199] == 0]).all()
        x[M - 1, 199] = float("nan")
        out = gf.mx_product(x, w, dtype=torch.float32)
        assert torch.isfinite(out[:M - 1]).all() and torch.isnan(out[M - 1]).all()
        dy = _rows(M, N, dtype, 8, spread=False)
        dy[M - 1, N - 1] = float("nan")
        dx = gf.mx_product_grad(dy, w, dtype=torch.float32)
        assert torch.isfinite(dx[:M - 1]).all() and torch.isnan(dx[M - 1]).all()
    xm = gf.mx_quantise(_rows(M, K, torch.float32, 6, spread=False))
    out = gf.mx_product(xm, wn)
    assert torch.isnan(out[:, 3]).all() and torch.isfinite(out[:, [0, 1, 2, 4, 149]]).all()


def test_largest_values():
    """The ends of fp32's range: no part of a split value overflows."""
    _case("largest")
    K = 64
    wv = np.zeros((20, K))
    wv[:, 0] = 0.5
    codes, scales = orc.quantise(wv)
    w = gf.MXRows(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), K)
    big = float(np.finfo(np.float32).max)
    for M in (1, 40, 200):
        x = torch.zeros(M, K, device="cuda")
        x[:, 0] = big
        assert (gf.mx_product(x, w) == big / 2).all()
        h = torch.zeros(M, K, device="cuda", dtype=torch.float16)
        h[:, 0] = 2.0 ** -24
        assert (gf.mx_product(h, w, dtype=torch.float32) == 2.0 ** -25).all()


def test_empty_and_slices():
    _case("empty")
    w, wv = _mx(40, 96, 1)
    x = _rows(6, 96, torch.float32, 2)
    assert gf.mx_product(x[:0], w).shape == (0, 40)
    assert gf.mx_product(x, w[:0]).shape == (6, 0)
    dx = gf.mx_product_grad(torch.empty(6, 0, device="cuda"), w[:0])
    assert dx.shape == (6, 96) and not dx.any()
    assert gf.mx_quantise(x[:0]).rows == 0 and gf.mx_dequantise(w[:0]).shape == (0, 96)
    _check_product(gf.mx_product(x, w[7:23]), _np(x), wv[7:23], "slice")
    r = gf.route(x[:0], 4)
    assert r.ids.shape == (0, 4) and not r.load.any()


def test_offsets_beyond_32_bits():
    """Input rows further than 2^32 bytes apart, and an output of more than
    2^32 elements."""
    _case("far rows")
    K, N = 96, 40
    w, wv = _mx(N, K, 3)
    far = 2 ** 31 + 64
    buf = torch.empty(2 * far + 128, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((3, K), (far, 1))
    ref = _rows(3, K, torch.bfloat16, 4)
    x.copy_(ref)
    _check_product(gf.mx_product(x, w, dtype=torch.float32), _np(ref), wv, "far x")
    assert torch.equal(gf.mx_quantise(x).codes, gf.mx_quantise(ref).codes)
    dy = buf.as_strided((3, N), (far, 1))
    dref = _rows(3, N, torch.bfloat16, 5)
    dy.copy_(dref)
    _check_product(gf.mx_product_grad(dy, w, dtype=torch.float32), _np(dref), np.ascontiguousarray(wv.T), "far dy")
    r = gf.route(dy, 4)
    assert torch.equal(r.ids, gf.route(dref, 4).ids)
    del buf, x, dy
    torch.cuda.empty_cache()
    _case("far outputs")
    M = N = 65600
    w = gf.mx_quantise(_rows(N, 32, torch.float32, 6, spread=False))
    xs = gf.mx_quantise(_rows(M, 32, torch.float32, 7, spread=False))
    out = gf.mx_product(xs, w, dtype=torch.bfloat16)
    some = torch.tensor([0, 1, 32768, 65535, 65536, 65599])
    xv, wvv = _np(gf.mx_dequantise(xs))[some], _np(gf.mx_dequantise(w))
    _check_product(out[some], xv, wvv, "far out")


# ---- routing --------------------------------------------------------------

ROUTES = [
    dict(T=1, E=1, k=1), dict(T=3, E=2, k=1), dict(T=70, E=8, k=2), dict(T=33, E=64, k=6), dict(T=50, E=60, k=60),
    dict(T=40, E=100, k=7, bias=True), dict(T=64, E=256, k=8, bias=True, groups=8, keep_groups=4, group_score="top2"),
    dict(T=64, E=256, k=8, groups=16, keep_groups=4), dict(T=20, E=1024, k=64), dict(T=21, E=1000, k=4, bias=True),
    dict(T=25, E=12, k=3, groups=4, keep_groups=1), dict(T=25, E=64, k=5, groups=64, keep_groups=9, group_score="top2"),
    dict(T=19, E=96, k=12, groups=3, keep_groups=2, group_score="top2", bias=True),
    dict(T=17, E=1024, k=16, groups=2, keep_groups=1, bias=True, group_score="top2"), dict(T=1, E=256, k=8, bias=True),
    dict(T=1000, E=160, k=6, groups=5, keep_groups=2), dict(T=32, E=200, k=9), dict(T=8, E=300, k=3), dict(T=9, E=300, k=4),
]


def _route_inputs(c, dtype, seed, masked):
    g = torch.Generator().manual_seed(seed)
    l = 2 * torch.randn(c["T"], c["E"], generator=g)
    if masked:
        l[torch.rand(l.shape, generator=g) < torch.rand(c["T"], 1, generator=g)] = float("-inf")
        l[::7] = float("-inf")
        l[3::9, ::5] = float("nan")
        l[5::11, 1::3] = float("inf")
        l[2::13] = torch.finfo(dtype).min
    bias = 0.01 * torch.randint(-10, 11, (c["E"],), generator=g).float() if c.get("bias") else None
    if bias is not None and masked:
        bias[c["E"] // 2] = float("-inf")
        bias[0] = float("nan")
    return l.to(dtype).cuda(), bias.cuda() if bias is not None else None


def _close(got, ref, bound, what):
    err = np.abs(_np(got) - ref)
    assert (err <= bound).all(), f"{what}: {err.max():.3g} against {np.max(bound):.3g}"


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("i", range(len(ROUTES)))
def test_route_and_gradient(i, dtype, masked, score):
    c = dict(ROUTES[i])
    _case("route", i, c, dtype, masked, score)
    l, bias = _route_inputs(c, TYPES[dtype], 31 * i + 1, masked)
    k = c["k"]
    how = {n: c[n] for n in ("groups", "keep_groups", "group_score") if n in c}
    b = None if bias is None else _np(bias)
    for renorm, scale, v in ((True, 1.0, l), (False, 2.5, _strided(l, 3, shift=1))):
        got = gf.route(v, k, bias=bias, score=score, renormalise=renorm, scale=scale, **how)
        ids, w, load = orc.route(_np(l), k, bias=b, score=score, renormalise=renorm, scale=scale, **how)
        assert np.array_equal(_np(got.ids), ids)
        assert np.array_equal(_np(got.load), load)
        _close(got.weights, w, orc.WEIGHT_RTOL * np.abs(w) + 2.0 ** -126, "weights")
        g = torch.randn(c["T"], k, generator=torch.Generator().manual_seed(i)).cuda()
        gn = g.clone()
        gn[torch.from_numpy(ids).cuda() < 0] = float("nan")     # weights that do not exist
        d = gf.route_grad(v, got.ids, gn, bias=bias, score=score, renormalise=renorm, scale=scale)
        ref = orc.route_grad(_np(l), ids, _np(g), bias=b, score=score, renormalise=renorm, scale=scale)
        assert d.dtype == l.dtype
        _close(d, ref, orc.grad_bound(ref, _np(g), scale, _name(d.dtype)), "dlogits")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_ties_and_near_ties(score):
    """Equal logits go to the lower index; sums of score and bias that differ
    only beyond 32 bits are told apart."""
    _case("ties", score)
    T, E, k = 200, 64, 8
    g = torch.Generator().manual_seed(9)
    l = torch.randint(-2, 3, (T, E), generator=g).float()
    for bias in (None, torch.zeros(E)):
        got = gf.route(l.cuda(), k, bias=None if bias is None else bias.cuda(), score=score)
        ids, _, _ = orc.route(l.numpy(), k, bias=None if bias is None else bias.numpy(), score=score)
        assert np.array_equal(_np(got.ids), ids)
    # logits one unit in the last place apart, in random order: scores that
    # agree in 32 bits for the most part
    base = torch.nextafter(torch.full((T, E), 1.0), torch.tensor(2.0))
    steps = torch.stack([torch.randperm(E, generator=g) for _ in range(T)])
    l = (base.view(torch.int32) + steps.int()).view(torch.float32)
    for groups, keep in ((1, 1), (8, 3)):
        got = gf.route(l.cuda(), k, bias=torch.full((E,), 0.25).cuda(), score=score, groups=groups, keep_groups=keep,
                       group_score="top2")
        ids, _, _ = orc.route(l.numpy(), k, bias=np.full(E, 0.25), score=score, groups=groups, keep_groups=keep,
                              group_score="top2")
        assert np.array_equal(_np(got.ids), ids)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,keep,k", [(12, 4, 2, 5), (120, 8, 8, 30), (256, 16, 4, 8), (300, 1, 1, 64), (320, 10, 4, 9),
                                             (512, 64, 20, 16), (1000, 8, 3, 12), (1024, 1, 1, 1), (16, 1, 1, 16),
                                             (16, 16, 9, 8), (60, 1, 1, 4), (64, 8, 3, 8), (250, 2, 1, 13), (400, 1, 1, 8),
                                             (700, 7, 7, 3), (1024, 16, 16, 16), (777, 1, 1, 17)])
def test_route_ties_of_rounded_logits(E, groups, keep, k, score):
    """Logits of few values: equal sums of score and bias, equal ranks of groups,
    in rows of every width; bias none, nothing, or of few values."""
    _case("rounded", E, groups, keep, k, score)
    g = torch.Generator().manual_seed(E + k)
    l = (2 * torch.randn(150, E, generator=g)).to(torch.bfloat16)
    l[1::2] = torch.round(l[1::2] * 2) / 2
    l[7::10, E // 3:] = float("-inf")
    for bias in (None, torch.zeros(E), torch.randint(-1, 2, (E,), generator=g) / 16):
        for rank in ("max", "top2"):
            got = gf.route(l.cuda(), k, bias=None if bias is None else bias.cuda(), score=score, groups=groups,
                           keep_groups=keep, group_score=rank)
            ids, w, load = orc.route(_np(l), k, bias=None if bias is None else bias.double().numpy(), score=score,
                                     groups=groups, keep_groups=keep, group_score=rank)
            assert np.array_equal(_np(got.ids), ids) and np.array_equal(_np(got.load), load)
            _close(got.weights, w, orc.WEIGHT_RTOL * np.abs(w) + 2.0 ** -126, "weights")


@pytest.mark.parametrize("keep", [2, 4])
def test_route_saturated_sigmoids(keep):
    """Sigmoids that are 1 in 64 bits tie where entries are ranked by score, not
    where they are by logit."""
    _case("saturated", keep)
    l = torch.arange(64, dtype=torch.float32).repeat(5, 1) + 40.0
    l[1:, ::3] = -60.0
    for rank in ("max", "top2"):
        for bias in (None, torch.zeros(64)):
            got = gf.route(l.cuda(), 6, bias=None if bias is None else bias.cuda(), score="sigmoid", groups=4,
                           keep_groups=keep, group_score=rank)
            ids, _, _ = orc.route(l.numpy(), 6, bias=None if bias is None else bias.numpy(), score="sigmoid", groups=4,
                                  keep_groups=keep, group_score=rank)
            assert np.array_equal(_np(got.ids), ids)


def test_route_grad_ignores_foreign_ids():
    _case("foreign ids")
    l = _rows(4, 16, torch.float32, 1, spread=False)
    ids = torch.tensor([[0, 1], [16, 2], [-5, 3], [2 ** 31 - 1, -1]], dtype=torch.int32).cuda()
    g = torch.ones(4, 2).cuda()
    d = gf.route_grad(l, ids, g, score="sigmoid", renormalise=False)
    kept = ids.cpu().numpy().copy()
    kept[(kept < 0) | (kept >= 16)] = -1
    ref = orc.route_grad(_np(l), kept, _np(g), score="sigmoid", renormalise=False)
    _close(d, ref, orc.grad_bound(ref, _np(g), 1.0, "float32"), "dlogits")


def test_results_do_not_change_from_run_to_run():
    """No sum's order depends on what else runs."""
    _case("repeat")
    w, _ = _mx(3000, 768, 1)
    x, dy = _rows(5, 768, torch.float32, 2), _rows(5, 3000, torch.float32, 3)
    first = gf.mx_product(x, w), gf.mx_product_grad(dy, w), gf.route(dy[:, :1024], 8).weights
    for _ in range(5):
        again = gf.mx_product(x, w), gf.mx_product_grad(dy, w), gf.route(dy[:, :1024], 8).weights
        assert all(torch.equal(a, b) for a, b in zip(first, again))


# ---- streams, graphs, autograd --------------------------------------------

def test_other_stream_and_graph():
    """Work goes to the current stream; a captured graph replays to the eager
    result after its inputs change."""
    _case("graph")
    w, _ = _mx(500, 256, 1)
    x, dy = _rows(9, 256, torch.float32, 2), _rows(9, 500, torch.float32, 3)
    bias = torch.zeros(500, device="cuda")

    def step():
        s = gf.mx_product(x, w)
        r = gf.route(s, 6, bias=bias)
        dl = gf.route_grad(s, r.ids, r.weights, bias=bias)
        return [s, r.ids, r.weights, r.load, gf.mx_product_grad(dl, w), gf.mx_product(gf.mx_quantise(x), w),
                gf.mx_product_grad(dy, w)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    eager = [t.clone() for t in step()]
    with torch.cuda.stream(side):
        other = [t.clone() for t in step()]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        x.copy_(_rows(9, 256, torch.float32, 10 + i))
        dy.copy_(_rows(9, 500, torch.float32, 20 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_autograd():
    """The nodes give what the gradient calls give, from any layout of dy."""
    _case("autograd")
    w, wv = _mx(60, 100, 1)
    x = _rows(7, 100, torch.float32, 2, spread=False).requires_grad_()
    s = gf.mx_product(x, w)
    r = gf.route(s, 5, score="softmax", groups=6, keep_groups=3)
    g = _rows(7, 5, torch.float32, 3, spread=False)
    (r.weights * g).sum().backward()
    ids = _np(r.ids)
    sv = _np(x) @ wv.T
    ds = orc.route_grad(sv, ids, _np(g))
    # the scores that route saw carry their own fp32 rounding
    bound = orc.grad_bound(ds, _np(g), 1.0, "float32") + 4 * orc.product_bound(_np(x), wv, "float32").max() * np.abs(_np(g)).max()
    _close(x.grad, ds @ wv, bound @ np.abs(wv) + orc.product_bound(ds, np.ascontiguousarray(wv.T), "float32"), "x.grad")
    assert not r.ids.requires_grad and not r.load.requires_grad
    x.grad = None
    gf.mx_product(x, w).sum().backward()     # an expanded dy
    _close(x.grad, np.ones((7, 60)) @ wv, orc.product_bound(np.ones((7, 60)), np.ascontiguousarray(wv.T), "float32"), "sum")
    x.grad = None
    gf.mx_product(x, w).t().matmul(torch.ones(7, 3, device="cuda")).sum().backward()   # a transposed dy
    _close(x.grad, 3 * np.ones((7, 60)) @ wv, orc.product_bound(3 * np.ones((7, 60)), np.ascontiguousarray(wv.T), "float32"), "dy^T")


def test_gradients_of_gradients_are_refused():
    _case("second derivatives")
    w, _ = _mx(20, 64, 1)
    x = _rows(3, 64, torch.float32, 2, spread=False).requires_grad_()
    for y in (gf.mx_product(x, w).square().sum(), gf.route(x, 4).weights.square().sum()):
        (d,) = torch.autograd.grad(y, x, create_graph=True)
        with pytest.raises(RuntimeError):
            d.sum().backward()
