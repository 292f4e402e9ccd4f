"""Operators of learned retrieval on torch tensors of the GPU (the device-memory
calls of include/garfield.h).

- ``mx_quantise`` / ``mx_dequantise``: rows to microscaled 4-bit floating point
  (``MXRows``) and back.
- ``mx_product``: scores of queries, real or quantised, against such rows;
  ``mx_product_grad`` its gradient with respect to the queries.
- ``route``: each query's k cells (experts) from its logits; ``route_grad`` the
  gradient with respect to the logits.

``mx_product`` and ``route`` take part in autograd.  Work goes to the current
stream of the tensors' device and nothing waits for it.  Matrices may have any
row distance; their last dimension must be contiguous.  Every call raises if
the library is missing; there is no other code path.
"""
import ctypes as C
import functools

from . import _lib

_SCORES = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORES = {"max": 0, "top2": 1}
MAX_CHOICES = 64    # of a row of route (GF_ROUTE_MAX_K)
_MAX_SIZE = 0x7FFFFF00     # rows or columns: the library counts them in 32 bits
torch = None        # imported by the first call: the rest of the package does without
_types = {}


def _need_torch():
    global torch
    if torch is None:
        import torch as t
        _types.update({t.float32: 0, t.float16: 1, t.bfloat16: 2})
        torch = t
    return torch


def _type(dtype, what):
    _need_torch()
    code = _types.get(dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {dtype}")
    return code


def _matrix(x, what):
    """x as the library reads it: (type, rows, columns, row distance)."""
    if not isinstance(x, _need_torch().Tensor) or x.ndim != 2:
        raise ValueError(f"{what} must be a matrix (a 2-d tensor)")
    n, d = x.shape
    if d > _MAX_SIZE:
        raise ValueError(f"{what} must have at most {_MAX_SIZE} columns")
    if not x.is_cuda:
        raise ValueError(f"{what} must be on the GPU")
    ld, one = x.stride()
    if one != 1 and d > 1:
        raise ValueError(f"{what}'s last dimension must be contiguous")
    if n < 2:
        ld = d
    elif ld < d:
        raise ValueError(f"{what}'s rows overlap")
    return _type(x.dtype, what), n, d, ld


def _count(x, what):
    """A whole number that the library's 32 bits hold."""
    try:
        n = int(x)
    except (TypeError, ValueError, OverflowError):
        n = -1
    if n != x or not 0 <= n <= _MAX_SIZE:
        raise ValueError(f"{what} must be a whole number from 0 to {_MAX_SIZE}, got {x!r}")
    return n


def _vector(x, shape, dtype, device, what):
    if x is None:
        return None
    if (not isinstance(x, torch.Tensor) or x.shape != shape or x.dtype != dtype or x.device != device
            or not x.is_contiguous()):
        raise ValueError(f"{what} must be a contiguous {tuple(shape)} {dtype} tensor on {device}")
    return x.data_ptr()


def _call(device, fn, *args):
    """fn on the current stream of the tensors' device."""
    i = device.index
    if torch._C._cuda_getDevice() == i:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if status:
        _lib._check(status)


class MXRows:
    """Rows at four bits: codes (rows, 64 S) and scales (rows, 4 S), uint8,
    S = ceil(K / 128); the layout is gf_mx_rows'.  Scale bytes of 253 and 254,
    which mx_quantise never writes, hold values beyond fp32 and bfloat16: only
    the product with both sides at four bits takes them."""

    def __init__(self, codes, scales, K):
        _need_torch()
        K = _count(K, "K")
        S = -(-K // 128)
        if K < 1:
            raise ValueError("K must be at least 1")
        for t, width, align, what in ((codes, 64 * S, 16, "codes"), (scales, 4 * S, 4, "scales")):
            if (not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or t.ndim != 2 or t.shape[1] != width
                    or t.shape[0] != codes.shape[0] or not t.is_contiguous() or not t.is_cuda
                    or t.device != codes.device):
                raise ValueError(f"{what} must be a contiguous (rows, {width}) uint8 tensor on the GPU")
            if t.data_ptr() % align:
                raise ValueError(f"{what} must be aligned to {align} bytes")
        self._parts = codes, scales
        self.K, self.rows, self.device = K, codes.shape[0], codes.device
        self._struct = _lib.MXRowsStruct(codes.data_ptr(), scales.data_ptr(), self.rows, self.K)

    @classmethod
    def _allocate(cls, rows, K, device):
        """Rows to be written: codes and scales one after the other in one
        allocation, split when somebody asks for them."""
        self = cls.__new__(cls)
        S = -(-K // 128)
        self._parts = torch.empty(rows * (68 * S), dtype=torch.uint8, device=device)
        self.K, self.rows, self.device = K, rows, device
        at = self._parts.data_ptr()
        self._struct = _lib.MXRowsStruct(at, at + rows * (64 * S), rows, K)
        return self

    def _versions(self):
        """What grows when the codes or scales are written to, but for tensors
        of inference mode, which keep no count."""
        codes, scales = self._split()
        return tuple(0 if t.is_inference() else t._version for t in (codes, scales))

    def _split(self):
        if not isinstance(self._parts, tuple):
            S = -(-self.K // 128)
            codes, scales = self._parts.split((self.rows * 64 * S, self.rows * 4 * S))
            self._parts = codes.view(self.rows, 64 * S), scales.view(self.rows, 4 * S)
        return self._parts

    @property
    def codes(self):
        return self._split()[0]

    @property
    def scales(self):
        return self._split()[1]

    def __getitem__(self, rows):
        """A run of whole rows (a slice of step 1), such as one cell's, without a copy."""
        if not isinstance(rows, slice) or rows.step not in (None, 1):
            raise TypeError("MXRows takes slices of consecutive rows")
        return MXRows(self.codes[rows], self.scales[rows], self.K)


def mx_quantise(x):
    """The rows of x (n, K) at four bits (gf_mx_quantise)."""
    t, n, K, ld = _matrix(x, "x")
    if K < 1:
        raise ValueError("x must have at least one column")
    w = MXRows._allocate(n, K, x.device)
    _call(w.device, _lib.load().gf_mx_quantise, x.data_ptr(), t, n, K, ld, w._struct.codes, w._struct.scales)
    return w


def mx_dequantise(w, dtype=None):
    """The values that w's rows stand for, (rows, K), float32 by default."""
    _need_torch()
    if not isinstance(w, MXRows):
        raise ValueError("w must be MXRows")
    dtype = dtype or torch.float32
    t = _type(dtype, "dtype")
    out = torch.empty((w.rows, w.K), dtype=dtype, device=w.device)
    _call(w.device, _lib.load().gf_mx_dequantise, C.byref(w._struct), t, out.data_ptr(), w.K)
    return out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(kind, off, t, M, ld, rows, K):
    """off: the address modulo 16, all that the size needs of it."""
    n = C.c_size_t()
    _lib._check(_lib.load().gf_mx_product_workspace_at(kind, off, t, M, ld, rows, K, C.byref(n)))
    return n.value


def _workspace(kind, x, t, M, ld, w):
    n = _workspace_bytes(kind, x.data_ptr() % 16, t, M, ld, w.rows, w.K)
    return (torch.empty(n, dtype=torch.uint8, device=w.device), n) if n else (None, 0)


def _product(x, w, dtype):
    if not isinstance(w, MXRows):
        raise ValueError("w must be MXRows")
    lib = _lib.load()
    if isinstance(x, MXRows):
        if x.K != w.K or x.device != w.device:
            raise ValueError(f"x holds {x.K} values a row on {x.device}, w {w.K} on {w.device}")
        dtype = dtype or torch.float32
        to = _type(dtype, "dtype")
        out = torch.empty((x.rows, w.rows), dtype=dtype, device=w.device)
        # this product takes no workspace
        _call(w.device, lib.gf_mx_product_mx, C.byref(x._struct), C.byref(w._struct), to, out.data_ptr(), w.rows,
              None, 0)
        return out
    t, M, K, ld = _matrix(x, "x")
    if K != w.K or x.device != w.device:
        raise ValueError(f"x holds {K} values a row on {x.device}, w {w.K} on {w.device}")
    dtype = dtype or x.dtype
    to = _type(dtype, "dtype")
    out = torch.empty((M, w.rows), dtype=dtype, device=w.device)
    ws, nws = _workspace(0, x, t, M, ld, w)
    _call(w.device, lib.gf_mx_product, x.data_ptr(), t, M, ld, C.byref(w._struct), to, out.data_ptr(), w.rows,
          ws.data_ptr() if nws else None, nws)
    return out


def mx_product_grad(dy, w, dtype=None):
    """The gradient of mx_product(x, w) with respect to x, (M, K), from dy
    (M, rows); dy's type by default (gf_mx_product_grad)."""
    if not isinstance(w, MXRows):
        raise ValueError("w must be MXRows")
    t, M, N, ld = _matrix(dy, "dy")
    if N != w.rows or dy.device != w.device:
        raise ValueError(f"dy holds {N} values a row on {dy.device}, w has {w.rows} rows on {w.device}")
    dtype = dtype or dy.dtype
    to = _type(dtype, "dtype")
    dx = torch.empty((M, w.K), dtype=dtype, device=w.device)
    ws, nws = _workspace(2, dy, t, M, ld, w)
    _call(w.device, _lib.load().gf_mx_product_grad, dy.data_ptr(), t, M, ld, C.byref(w._struct), to,
          dx.data_ptr(), w.K, ws.data_ptr() if nws else None, nws)
    return dx


_functions = None


def _autograd():
    """The autograd nodes, made at the first call that needs one."""
    global _functions
    if _functions is None:
        class Product(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, w, dtype):
                out = _product(x, w, dtype)
                ctx.w, ctx.dtype = w, x.dtype
                ctx.rows_as_they_were = w._versions()
                return out

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, dy):
                # not by save_for_backward, which takes no tensors of inference mode
                if ctx.rows_as_they_were != ctx.w._versions():
                    raise RuntimeError("mx_product: the rows have been modified by an inplace operation since the "
                                       "forward pass")
                if dy.ndim == 2 and dy.shape[1] > 1 and dy.stride(1) != 1 or dy.stride(0) < dy.shape[1]:
                    dy = dy.contiguous()
                return mx_product_grad(dy, ctx.w, ctx.dtype), None, None

        class Route(torch.autograd.Function):
            @staticmethod
            def forward(ctx, logits, k, bias, groups, keep_groups, group_score, score, renormalise, scale):
                ids, weights, load = _route(logits, k, bias, groups, keep_groups, group_score, score, renormalise,
                                            scale)
                ctx.save_for_backward(logits, ids, bias)
                ctx.how = dict(score=score, renormalise=renormalise, scale=scale)
                ctx.mark_non_differentiable(ids, load)
                return ids, weights, load

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, _ids, dweights, _load):
                logits, ids, bias = ctx.saved_tensors
                d = route_grad(logits, ids, dweights.contiguous(), bias=bias, **ctx.how)
                return (d,) + (None,) * 8

        _functions = Product, Route
    return _functions


def mx_product(x, w, dtype=None):
    """Scores (M, rows) of x against w's rows: x a matrix (M, K), whose values
    enter unrounded, or MXRows.  dtype: the result's type (by default x's, or
    float32 for MXRows).  Differentiable with respect to a matrix x."""
    if isinstance(x, _need_torch().Tensor) and x.requires_grad and torch.is_grad_enabled():
        return _autograd()[0].apply(x, w, dtype)
    return _product(x, w, dtype)


class Routes:
    """What route returns: ids (T, k) int32, best first and -1 where a row has
    fewer live entries; weights (T, k) float32; load (E,) int32, how many rows
    chose each entry."""

    __slots__ = ("ids", "weights", "load")

    def __init__(self, ids, weights, load):
        self.ids, self.weights, self.load = ids, weights, load

    def __iter__(self):
        return iter((self.ids, self.weights, self.load))


def _choice(table, key, what):
    code = table.get(key)
    if code is None:
        raise ValueError(f"{what} must be one of {', '.join(table)}, got {key!r}")
    return code


def _route(logits, k, bias, groups, keep_groups, group_score, score, renormalise, scale):
    t, T, E, ld = _matrix(logits, "logits")
    k = _count(k, "k")
    opts = _lib.RouteOpts(k, _choice(_SCORES, score, "score"), _count(groups, "groups"), _count(keep_groups, "keep_groups"),
                          _choice(_GROUP_SCORES, group_score, "group_score"), int(bool(renormalise)), float(scale))
    b = _vector(bias, (E,), torch.float32, logits.device, "bias")
    dev = logits.device
    # of a k that is refused, nothing is allocated
    ids = torch.empty((T, k if k <= MAX_CHOICES else 0), dtype=torch.int32, device=dev)
    weights = torch.empty((T, k if k <= MAX_CHOICES else 0), dtype=torch.float32, device=dev)
    load = torch.empty((E,), dtype=torch.int32, device=dev)
    _call(dev, _lib.load().gf_route, C.byref(opts), logits.data_ptr(), t, T, E, ld, b, ids.data_ptr(),
          weights.data_ptr(), load.data_ptr())
    return ids, weights, load


def route(logits, k, bias=None, groups=1, keep_groups=None, group_score="max", score="softmax", renormalise=True,
          scale=1.0):
    """The k cells (experts) of each row of logits (T, E), by softmax or
    sigmoid score plus bias (E,), among the keep_groups best of the groups of
    consecutive entries; entries at -inf (or NaN) are masked (gf_route).
    Returns Routes; the weights are differentiable with respect to the logits."""
    keep_groups = groups if keep_groups is None else keep_groups
    args = (logits, k, bias, groups, keep_groups, group_score, score, renormalise, scale)
    if isinstance(logits, _need_torch().Tensor) and logits.requires_grad and torch.is_grad_enabled():
        return Routes(*_autograd()[1].apply(*args))
    return Routes(*_route(*args))


def route_grad(logits, ids, dweights, bias=None, score="softmax", renormalise=True, scale=1.0):
    """The gradient of route's weights with respect to the logits, (T, E) in
    the logits' type, from dweights (T, k) float32 and route's ids; bias, score,
    renormalise and scale as in the call of route (gf_route_grad)."""
    t, T, E, ld = _matrix(logits, "logits")
    if not isinstance(ids, torch.Tensor) or ids.ndim != 2:
        raise ValueError("ids must be a (T, k) tensor")
    k = _count(ids.shape[1], "k")
    dev = logits.device
    i = _vector(ids, (T, k), torch.int32, dev, "ids")
    g = _vector(dweights, (T, k), torch.float32, dev, "dweights")
    b = _vector(bias, (E,), torch.float32, dev, "bias")
    opts = _lib.RouteOpts(k, _choice(_SCORES, score, "score"), 1, 1, 0, int(bool(renormalise)), float(scale))
    out = torch.empty((T, E), dtype=logits.dtype, device=dev)
    _call(dev, _lib.load().gf_route_grad, C.byref(opts), logits.data_ptr(), t, T, E, ld, b, i, g, out.data_ptr(),
          E)
    return out
