"""Products grouped by expert on data that is hard on their arithmetic: values far below the largest of their row or column,
alone where the other operand is not zero; zeros; infinities and NaN under an activation.  Tolerances: test_gpu_experts."""
import numpy as np
import pytest

from cortex_b200 import tensor as ct
from oracle import plain_operators as plain
from test_gpu_experts import _offsets, _product_tol, _within, stream  # noqa: F401

pytestmark = pytest.mark.gpu

# by size and always through scaled halves; the first sizes take them by themselves, the others are no multiple of anything
SHAPES = [(0, [700, 600, 0, 748], 2048, 1024), (2, [300, 0, 1, 130, 3, 31], 258, 129), (2, [90, 200], 130, 514)]


def _data(seed, sizes, n, k, tail=3):
    rng = np.random.default_rng(seed)
    rows = sum(sizes) + tail
    X, dY, W = (rng.standard_normal(s).astype(np.float32) for s in ((rows, k), (rows, n), (len(sizes), n, k)))
    return rng, X, dY, W


def _forward(X, W, sizes, act=None, bias=None):
    Y = ct.new_tensor([len(X), W.shape[1]], "float")
    ct.expert_gemm(Y, True, 1.0, ct.to_tensor(X, "float"), ct.to_tensor(W, "float"), 0.0, ct.to_tensor(_offsets(sizes), "int"), act=act)
    return ct.to_array(Y).reshape(len(X), W.shape[1])


def _input(dY, W, sizes):
    dX = ct.new_tensor([len(dY), W.shape[2]], "float")
    ct.expert_gemm(dX, False, 1.0, ct.to_tensor(dY, "float"), ct.to_tensor(W, "float"), 0.0, ct.to_tensor(_offsets(sizes), "int"))
    return ct.to_array(dX).reshape(len(dY), W.shape[2])


def _weights(dY, X, sizes):
    e, n, k = len(sizes), dY.shape[1], X.shape[1]
    dW, db = ct.new_tensor([e, n, k], "float"), ct.new_tensor([e, n], "float")
    ct.expert_gemm_weights(dW, 1.0, ct.to_tensor(dY, "float"), ct.to_tensor(X, "float"), 0.0, ct.to_tensor(_offsets(sizes), "int"),
                           bias_gradient=db)
    return ct.to_array(dW).reshape(e, n, k)


def _hold(way, sizes, X, dY, W):
    """The product against 64 bits, every element within the bound of its own terms."""
    zeros = np.zeros
    if way == "forward":
        want, size = plain.expert_gemm(zeros((len(X), W.shape[1])), True, 1.0, X, W, 0.0, _offsets(sizes))
        _within(_forward(X, W, sizes), want, size, _product_tol("float", W.shape[2]), way)
    elif way == "input":
        want, size = plain.expert_gemm(zeros((len(dY), W.shape[2])), False, 1.0, dY, W, 0.0, _offsets(sizes))
        _within(_input(dY, W, sizes), want, size, _product_tol("float", W.shape[1]), way)
    else:
        want, size = plain.expert_gemm_weights(zeros(W.shape), 1.0, dY, X, 0.0, _offsets(sizes))[:2]
        _within(_weights(dY, X, sizes), want, size, _product_tol("float", max(sizes)), way)


@pytest.mark.parametrize("route,sizes,n,k", SHAPES)
@pytest.mark.parametrize("small", [-22, -28, -34, -45])
@pytest.mark.parametrize("side", ["rows", "matrices"])
def test_small_values_that_alone_meet_others_forward(stream, route, sizes, n, k, small, side):  # noqa: F811
    """Up to 1 in 64 values of a row far below its largest, and a row of the other operand that is zero everywhere else."""
    stream.set_option("gemm-auto-presplit", route)
    rng, X, dY, W = _data(7, sizes, n, k)
    at = rng.choice(k, max(1, k // 64), replace=False)
    one, other = (X[:1], W[0, 3:4]) if side == "rows" else (W[0, 3:4], X[:1])
    one[:, at] *= np.float32(2.0 ** small)
    other[:, np.setdiff1d(np.arange(k), at)] = 0.0
    _hold("forward", sizes, X, dY, W)


@pytest.mark.parametrize("route,sizes,n,k", SHAPES)
@pytest.mark.parametrize("small", [-22, -28, -34, -45])
@pytest.mark.parametrize("columns", [1, 2, 20])
def test_one_large_value_that_meets_zeros_weights(stream, route, sizes, n, k, small, columns):  # noqa: F811
    """Columns of one operand with a single large value, and rows of the other that are zero there."""
    stream.set_option("gemm-auto-presplit", route)
    for swap in (False, True):
        rng, X, dY, W = _data(11, sizes, n, k)
        one, other = (X, dY) if swap else (dY, X)
        at = rng.choice(one.shape[1], columns, replace=False)
        at[-1] = one.shape[1] - 1                               # (the last of a width that is no multiple of 128)
        one[:, at] *= np.float32(2.0 ** small)
        for lo, hi in zip(_offsets(sizes)[:-1], _offsets(sizes)[1:]):
            if hi > lo:
                r = int(rng.integers(lo, hi))
                one[r, at] = 1.0
                other[r] = 0.0
        _hold("weights", sizes, X, dY, W)


@pytest.mark.parametrize("small", [-28, -45])
def test_sparse_columns_with_few_values_weights(stream, small):  # noqa: F811
    """The same where a column has few values at all: one large and some small ones among zeros."""
    stream.set_option("gemm-auto-presplit", 2)
    sizes, n, k = [512, 3, 200], 129, 70
    rng, X, dY, W = _data(13, sizes, n, k)
    for lo, hi in ((0, 512), (512, 515), (515, 715)):
        rows = rng.choice(np.arange(lo, hi), 3, replace=False)
        column = np.zeros(hi - lo, np.float32)
        column[rows - lo] = [1.0, 2.0 ** small, -1.5 * 2.0 ** small]
        dY[lo:hi, 5] = column
        X[rows[0]] = 0.0
    _hold("weights", sizes, X, dY, W)


@pytest.mark.parametrize("route,sizes,n,k", SHAPES)
@pytest.mark.parametrize("scale", [1e-6, 1e-8, 1e-10, 1e-13])
@pytest.mark.parametrize("columns", [1, 10])
def test_small_columns_of_the_matrices_input(stream, route, sizes, n, k, scale, columns):  # noqa: F811
    """Columns of a matrix that are small in every row: all terms of a result are small."""
    stream.set_option("gemm-auto-presplit", route)
    rng, X, dY, W = _data(17, sizes, n, k)
    W[:, :, rng.choice(k, columns, replace=False)] *= np.float32(scale)
    _hold("input", sizes, X, dY, W)


@pytest.mark.parametrize("route,sizes,n,k", SHAPES)
@pytest.mark.parametrize("small", [-24, -34])
@pytest.mark.parametrize("side", ["rows", "matrices"])
def test_small_values_that_alone_meet_others_input(stream, route, sizes, n, k, small, side):  # noqa: F811
    stream.set_option("gemm-auto-presplit", route)
    rng, X, dY, W = _data(19, sizes, n, k)
    at = rng.choice(n, max(1, n // 64), replace=False)
    rest = np.setdiff1d(np.arange(n), at)
    if side == "rows":
        dY[0, at] *= np.float32(2.0 ** small)
        W[0, rest, 5] = 0.0
    else:
        W[0, at, 5] *= np.float32(2.0 ** small)
        dY[0, rest] = 0.0
    _hold("input", sizes, X, dY, W)


@pytest.mark.parametrize("way", ["forward", "input", "weights"])
@pytest.mark.parametrize("act", [None, "relu", "tanh"])
def test_remainders_of_small_values(stream, way, act):  # noqa: F811
    """Some values far below the largest of their rows and columns, in both operands and at the same places, met by zeros but for
    them; results, signs and an accumulation into what is there; the same bits every time."""
    stream.set_option("gemm-auto-presplit", 2)
    sizes, n, k = [300, 1, 257, 0, 3], 260, 392
    rng, X, dY, W = _data(61, sizes, n, k)
    rows, e = len(X), len(sizes)
    for _ in range(40):
        lo, hi = [(0, 300), (301, 558)][rng.integers(2)]
        g = 0 if lo == 0 else 2
        r, i, j, small = rng.integers(lo, hi), rng.integers(n), rng.integers(k), np.float32(2.0 ** -rng.integers(22, 60))
        X[r, j] *= small
        dY[r, i] *= small
        W[g, i, j] *= small
        if way == "forward" and rng.random() < 0.5:
            keep = X[r, j]
            X[r] = 0.0                                  # the row meets the matrix there only
            X[r, j], X[r, (j + 7) % k] = keep, 0.0
            W[g, i, (j + 1) % k] = 0.0
    if way == "forward":
        for r, i, j in ((5, 9, 100), (400, 250, 391)):     # small times small, and nothing else
            g = 0 if r < 300 else 2
            W[g, i], W[g, i, j], W[g, i, (j + 5) % k] = 0.0, 2.0 ** -30, 1.0
            X[r, j], X[r, (j + 5) % k] = 2.0 ** -28, 0.0
    elif way == "input":
        for r, i, j in ((5, 9, 100), (400, 250, 391)):
            g = 0 if r < 300 else 2
            W[g, :, j], W[g, i, j], W[g, (i + 5) % n, j] = 0.0, 2.0 ** -30, 1.0
            dY[r, i], dY[r, (i + 5) % n] = 2.0 ** -28, 0.0
    else:
        for r, i, j in ((5, 9, 100), (400, 250, 391)):
            lo, hi = (0, 300) if r < 300 else (301, 558)
            X[lo:hi, j], X[r, j], X[r + 1, j] = 0.0, 2.0 ** -30, 1.0
            dY[r, i], dY[r + 1, i] = 2.0 ** -28, 0.0
    off, bias = ct.to_tensor(_offsets(sizes), "int"), rng.standard_normal((e, n)).astype(np.float32) * np.float32(1e-3)
    Xt, dYt, Wt = (ct.to_tensor(a, "float") for a in (X, dY, W))
    for alpha, beta in ((1.0, 0.0), (-2.0, 0.5)):
        if way == "weights":
            C0 = rng.standard_normal(W.shape).astype(np.float32) * np.float32(1e-6)
            run = lambda C: ct.expert_gemm_weights(C, alpha, dYt, Xt, beta, off)
            want, size = plain.expert_gemm_weights(C0, alpha, dY, X, beta, _offsets(sizes))[:2]
            length = max(sizes)
        else:
            C0 = rng.standard_normal((rows, n if way == "forward" else k)).astype(np.float32) * np.float32(1e-6)
            if way == "forward":
                run = lambda C: ct.expert_gemm(C, True, alpha, Xt, Wt, beta, off, bias=ct.to_tensor(bias, "float") if act else None, act=act)
                want, size = plain.expert_gemm(C0, True, alpha, X, W, beta, _offsets(sizes), bias if act else None, act)
            else:
                run = lambda C: ct.expert_gemm(C, False, alpha, dYt, Wt, beta, off, act=act)
                want, size = plain.expert_gemm(C0, False, alpha, dY, W, beta, _offsets(sizes), None, act)
            length = k if way == "forward" else n
        bits = []
        for _ in range(3):
            C = ct.to_tensor(C0, "float")
            run(C)
            bits.append(ct.to_array(C))
        assert all(np.array_equal(bits[0], b) for b in bits[1:])
        _within(bits[0], want, size + (np.abs(want) * 8 * 2.0 ** -24 / _product_tol("float", length) if act == "tanh" else 0.0),
                _product_tol("float", length), (way, alpha))


def _any_data(rng, shape):
    """Normal values, spread in every way over up to 60 powers of two, with outliers, with zeros in every way."""
    x = rng.standard_normal(shape)
    kind, a = rng.integers(8), rng.choice([0, 2, 5, 9, 14, 22, 30])
    rows, columns = shape[:-1] + (1,), (1,) * (len(shape) - 1) + shape[-1:]
    if kind in (1, 2, 3):
        where = (shape, rows, columns)[kind - 1]
        x = x * np.exp2(rng.uniform(-a, a, where))
    if kind == 4:
        x = _relu(x)
    if kind == 5:
        x = x * np.where(rng.random(shape) < rng.choice([1e-4, 1e-3, 1e-2]), np.exp2(-rng.uniform(18, 45, shape)), 1.0)
    if kind == 6:
        x = x * np.where(rng.random(shape) < 1e-4, np.exp2(rng.uniform(10, 40, shape)), 1.0)
    if rng.random() < 0.5:
        x = x * (rng.random(shape) < rng.choice([0.5, 0.1, 0.01]))
    for where in (rows, columns):
        if rng.random() < 0.3:
            x = x * (rng.random(where) < 0.9)
    return x.astype(np.float32)


@pytest.mark.parametrize("route", [1, 2])
@pytest.mark.parametrize("first", [900, 1000, 1250, 0, 100, 200, 300, 400])
def test_any_data_within_the_bound_of_its_own_terms(stream, route, first):  # noqa: F811
    """Every element of every direction, whatever it is made of."""
    stream.set_option("gemm-auto-presplit", route)
    for seed in range(first, first + 60):
        rng = np.random.default_rng(seed)
        sizes = [int(v) for v in rng.choice([0, 1, 2, 3, 7, 31, 64, 100, 256, 257, 300], rng.integers(1, 7))]
        n, k = int(rng.choice([1, 3, 8, 33, 64, 129, 200, 256, 300])), int(rng.choice([1, 2, 5, 16, 40, 64, 100, 130, 257, 520]))
        rows, e, o = sum(sizes) + 1, len(sizes), _offsets(sizes)
        X, W, dY = _any_data(rng, (rows, k)), _any_data(rng, (e, n, k)), _any_data(rng, (rows, n))
        off, Xt, Wt, dYt = ct.to_tensor(o, "int"), ct.to_tensor(X, "float"), ct.to_tensor(W, "float"), ct.to_tensor(dY, "float")
        alpha, beta = [(1.0, 0.0), (-0.5, 1.0)][rng.integers(2)]
        Y0, act = (rng.standard_normal((rows, n)) * 1e-3).astype(np.float32), [None, "relu"][rng.integers(2)]
        Y, dX, dW = ct.to_tensor(Y0, "float"), ct.new_tensor([rows, k], "float"), ct.new_tensor([e, n, k], "float")
        ct.expert_gemm(Y, True, alpha, Xt, Wt, beta, off, act=act)
        ct.expert_gemm(dX, False, 1.0, dYt, Wt, 0.0, off)
        ct.expert_gemm_weights(dW, 1.0, dYt, Xt, 0.0, off)
        least = 2.0 ** -120                                      # below the normal range nothing is promised
        for name, got, (want, size), length in (
                ("forward", Y, plain.expert_gemm(Y0, True, alpha, X, W, beta, o, None, act), k),
                ("input", dX, plain.expert_gemm(np.zeros((rows, k)), False, 1.0, dY, W, 0.0, o), n),
                ("weights", dW, plain.expert_gemm_weights(np.zeros((e, n, k)), 1.0, dY, X, 0.0, o)[:2], max(sizes + [1]))):
            _within(ct.to_array(got), want, size + least / _product_tol("float", length), _product_tol("float", length), (seed, name))


# ---- which way a call went: the fallback leaves the bits of a call that is certain to fall back ---------------------------

def _fell_back(way, sizes, X, dY, W):
    """Appends a group with a row outside the halves' range, which sends the whole call to the other kernels; were the other
    groups' results the same bits without it?"""
    more = sizes + [1]
    at = sum(sizes)
    big = lambda a: np.concatenate([a[:at], np.full((1, a.shape[1]), 1e25, np.float32), a[at:]])
    W2 = np.concatenate([W, W[:1]])
    run = {"forward": lambda s, x, d, w: _forward(x, w, s)[:at], "input": lambda s, x, d, w: _input(d, w, s)[:at],
           "weights": lambda s, x, d, w: _weights(d, x, s)[:len(sizes)]}[way]
    return np.array_equal(run(sizes, X, dY, W), run(more, big(X), big(dY), W2))


def _relu(x):
    return np.maximum(x, 0.0)


@pytest.mark.parametrize("way", ["forward", "input", "weights"])
def test_ordinary_data_stays_on_halves(stream, way):  # noqa: F811
    stream.set_option("gemm-auto-presplit", 2)
    sizes, n, k = [300, 1, 256, 90, 0, 31], 260, 520
    rng, X, dY, W = _data(23, sizes, n, k)
    assert not _fell_back(way, sizes, X, dY, W)
    if way == "forward":
        assert not _fell_back(way, sizes, _relu(X), dY, W)
    elif way == "input":
        assert not _fell_back(way, sizes, X, dY * (rng.random(dY.shape) < 0.5), W)
    else:
        assert not _fell_back(way, sizes, _relu(X), dY, W)
        assert not _fell_back(way, sizes, X, dY * (rng.random(dY.shape) < 0.5), W)
        rare = _relu(X)
        rare[:, ::10] *= rng.random(rare[:, ::10].shape) < 0.02            # features that hardly any row has
        assert not _fell_back(way, sizes, rare, dY * (rng.random(dY.shape) < 0.5), W)
    assert not _fell_back(way, sizes, X, dY, W * (rng.random(W.shape) < 0.1))      # most weights pruned
    spread = lambda a: a * np.exp2(rng.uniform(-30, 30, a.shape)).astype(np.float32)
    assert _fell_back(way, sizes, spread(X), spread(dY), spread(W))                 # far too many small values
    large = np.float32(1e25)
    assert _fell_back(way, sizes, X * (large if way == "forward" else 1), dY * (large if way != "forward" else 1), W)


def test_a_row_of_zeros_stays_on_halves_input(stream):  # noqa: F811
    """An output feature without weights (pruned, or padding) in one matrix, and a NaN that meets it."""
    stream.set_option("gemm-auto-presplit", 2)
    sizes, n, k = [300, 1, 256], 260, 520
    rng, X, dY, W = _data(29, sizes, n, k)
    W[0, 17] = 0.0
    W[2, :5] = 0.0
    assert not _fell_back("input", sizes, X, dY, W)
    _hold("input", sizes, X, dY, W)
    W[:, :, 33] = 0.0                                           # and an input feature without any
    assert not _fell_back("input", sizes, X, dY, W)
    _hold("input", sizes, X, dY, W)
    W[2] = 0.0
    assert not _fell_back("input", sizes, X, dY, W)
    _hold("input", sizes, X, dY, W)
    for bad in (np.nan, np.inf):                                # 0 * NaN and 0 * infinity are NaN
        dY2 = dY.copy()
        dY2[4, 17] = bad
        got = _input(dY2, W, sizes)
        assert np.isnan(got[4]).all() and np.isfinite(np.delete(got[:sum(sizes)], 4, 0)).all()


# ---- activations of what is no number ------------------------------------------------------------------------------------

@pytest.mark.parametrize("datatype", ["float", "double"])
@pytest.mark.parametrize("act", ["relu", "tanh", "logistic"])
# few rows, tiles that TMA cannot address, short reductions, long ones in a cluster's slices, halves and their fallback
@pytest.mark.parametrize("route,sizes,n,k", [(0, [1, 2], 40, 64), (0, [1, 2], 39, 63), (1, [100, 33], 129, 63), (1, [100, 33], 128, 64),
                                             (1, [30, 20], 128, 2048), (2, [100, 33], 128, 64), (2, [100, 33], 129, 63)])
def test_a_nan_stays_a_nan_under_an_activation(stream, datatype, act, route, sizes, n, k):  # noqa: F811
    stream.set_option("gemm-auto-presplit", route)
    rng = np.random.default_rng(31)
    X, W = rng.standard_normal((sum(sizes), k)), rng.standard_normal((2, n, k))
    X[0, 3] = np.nan
    W[1, 7, 2] = np.nan
    np_type = np.float32 if datatype == "float" else np.float64
    X, W = X.astype(np_type), W.astype(np_type)
    Y = ct.new_tensor([len(X), n], datatype)
    ct.expert_gemm(Y, True, 1.0, ct.to_tensor(X, datatype), ct.to_tensor(W, datatype), 0.0, ct.to_tensor(_offsets(sizes), "int"), act=act)
    got = ct.to_array(Y).reshape(len(X), n)
    want = np.zeros(got.shape, bool)
    want[0] = True
    want[sizes[0]:, 7] = True
    assert np.array_equal(np.isnan(got), want)


@pytest.mark.parametrize("route,sizes,n,k", [(0, [1, 2], 40, 64), (1, [100, 33], 128, 64), (1, [30, 20], 128, 2048), (2, [100, 33], 128, 64)])
def test_an_infinity_under_relu_is_no_finite_number_above_zero(stream, route, sizes, n, k):  # noqa: F811
    """Where 64 bits give +infinity the result is that or NaN (an infinity times a tail of zero), not a number."""
    stream.set_option("gemm-auto-presplit", route)
    rng = np.random.default_rng(37)
    X, W = rng.standard_normal((sum(sizes), k)).astype(np.float32), rng.standard_normal((2, n, k)).astype(np.float32)
    X[1, 3], W[0, :, 3] = np.inf, np.where(np.arange(n) % 2, 0.5, -0.5)      # exactly representable: no tail
    if sizes[0] < 2:
        X[0, 3] = np.inf
    row = 0 if sizes[0] < 2 else 1
    got = _forward(X, W, sizes, act="relu")
    up = np.arange(n) % 2 == 1
    assert not np.isfinite(got[row, up]).any()
    assert not (np.isfinite(got[row, ~up]) & (got[row, ~up] != 0)).any()     # exactly: 0
