"""Products grouped by expert, residual normalisation and gradient clipping on the B200 against plain 64-bit statements.

Tolerances are bounds, not fits.  With u = eps / 2 of the type:
  * a product's error is relative to S = |alpha| sum |a||b| + |beta c| + |bias| (the `magnitude` the plain statement
    returns).  fp32: operands are split into a head of 11 bits and a tail truncated to 11 bits and the product of the tails
    is dropped: below 3 * 2^-21 S; the tensor core adds with truncation, one addition per 8 values of k and per
    accumulator, 2^-23 S each at most; a few roundings at the end.  (k / 8 + 24) * 2^-23 + 2^-19 covers both and the
    plain-FMA kernels (k * 2^-24 at worst) up to k = 4096; longer reductions have k * 2^-24 on top.  fp64: (k + 8) * 2^-53.
  * tanh and logistic shrink an error and add a few units of their own: 8 u.
  * normalisations: a row sum of n terms as a tree of at most 8 + n / 128 levels, two of them in a row for a variance, and
    about 20 elementary operations: (64 + n / 32) u relative to the plain statement's magnitude; column sums over r rows
    (r + 64) u more.
"""
import numpy as np
import pytest

from cortex_b200 import _lib, nn, optimize
from cortex_b200 import tensor as ct
from oracle import plain_operators as plain
from test_experts import expert_block_step

pytestmark = pytest.mark.gpu
NP = {"float": np.float32, "double": np.float64}
U = {"float": 2.0 ** -24, "double": 2.0 ** -53}


@pytest.fixture
def stream(b200_driver):
    s = b200_driver.default_device().create_stream()
    with ct.with_stream(s):
        yield s
    s.sync()


def _product_tol(datatype, k):
    return ((k / 8 + 24) * 2.0 ** -23 + 2.0 ** -19 + k * 2.0 ** -24) if datatype == "float" else (k + 8) * 2.0 ** -53


def _within(got, value, magnitude, tol, what):
    got = np.asarray(got, np.float64).reshape(value.shape)
    assert np.array_equal(np.isfinite(got), np.isfinite(value)), what
    bad = np.abs(got - value) > tol * magnitude + 1e-300
    assert not bad.any(), (what, int(bad.sum()), float((np.abs(got - value) / np.maximum(magnitude, 1e-300)).max()), tol)


def _window(data, datatype, pad, shift=0):
    """The array as a window of a wider buffer: row pitch cols + pad, first element `shift` elements into the allocation."""
    rows, cols = data.shape
    wide = np.full((rows, cols + pad), 777.0, NP[datatype])
    wide[:, :cols] = data
    flat = np.concatenate([np.full(shift, 777.0, NP[datatype]), wide.reshape(-1)])
    t = ct.to_tensor(flat, datatype)
    buf = t.buffer.sub_buffer(shift, rows * (cols + pad))
    return ct.Tensor(t.device, {"shape": [rows, cols], "strides": [cols + pad, 1]}, buf), t


def _read(window, whole, pad, shift=0):
    rows, cols = window.shape()
    flat = ct.to_array(whole)
    assert np.all(flat[:shift] == 777.0)
    wide = flat[shift:].reshape(rows, cols + pad)
    assert np.all(wide[:, cols:] == 777.0), "the padding of the rows was written"
    return wide[:, :cols]


# rows, group sizes, n, k
PRODUCTS = [
    (1, [1], 1, 1), (2, [0, 1, 0, 1], 64, 32), (5, [5], 16, 16), (7, [0, 0, 0], 24, 40), (130, [1, 0, 128, 1], 128, 64),
    (129, [129], 130, 18), (300, [127, 129, 3, 0, 30], 260, 100), (64, [2] * 32, 96, 72), (257, [200, 0, 57], 33, 17),
    (40, [9, 8, 7, 6, 5, 4], 500, 784), (600, [64, 65, 63, 128, 192, 1, 87], 68, 1028), (1000, [700, 200], 132, 516),
    (3, [1, 1, 1], 1001, 333), (512, [511, 1], 257, 129), (96, [3] * 32, 40, 2052), (33, [16, 17], 4, 8),
    (70, [1] * 70, 20, 12),
    # few rows with long reductions (K slices), a group that outgrows the estimate its kernel was chosen by, short reductions in
    # many tiles, few tiles with long reductions
    (8, [1] * 8, 260, 1028), (14, [8, 0, 3, 1], 129, 2051), (4, [2, 2], 40, 4096), (99, [60, 1, 0, 35], 300, 520), (180, [90, 90], 1000, 68),
    (9, [0, 0, 7], 64, 64), (16, [0, 0, 16, 0], 257, 130), (515, [500, 0, 0, 0, 0, 12], 132, 260), (2103, [0, 2100, 3], 72, 100),
    (1320, [1300] + [1] * 14, 200, 136), (1200, [40] * 30, 516, 250), (450, [64, 65, 63, 1, 128, 129], 260, 256), (932, [400, 532], 20, 3332),
    (3000, [1000, 2000], 32, 36), (1040, [1024, 5, 11], 200, 1400),
]


def _offsets(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)


@pytest.mark.parametrize("datatype", ["float", "double"])
@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("case", range(len(PRODUCTS)))
def test_expert_gemm(stream, datatype, trans_b, case):
    rows, sizes, n, k = PRODUCTS[case]
    rng = np.random.default_rng(100 + case)
    A = rng.standard_normal((rows, k)).astype(NP[datatype])
    B = rng.standard_normal((len(sizes),) + ((n, k) if trans_b else (k, n))).astype(NP[datatype])
    C0 = rng.standard_normal((rows, n)).astype(NP[datatype])
    bias = rng.standard_normal((len(sizes), n)).astype(NP[datatype])
    off = ct.to_tensor(_offsets(sizes), "int")
    At, Bt, biast = ct.to_tensor(A, datatype), ct.to_tensor(B, datatype), ct.to_tensor(bias, datatype)
    for alpha, beta, with_bias, act in [(1.0, 0.0, True, "relu"), (-0.75, 0.5, False, None), (0.1, 0.0, True, "tanh")]:
        Ct = ct.to_tensor(C0, datatype)
        ct.expert_gemm(Ct, trans_b, alpha, At, Bt, beta, off, bias=biast if with_bias else None, act=act)
        got = ct.to_array(Ct).reshape(C0.shape)
        want, size = plain.expert_gemm(C0, trans_b, alpha, A, B, beta, _offsets(sizes), bias if with_bias else None, act)
        _within(got, want, size + (1.0 if act == "tanh" else 0.0) * 8 * U[datatype] / _product_tol(datatype, k),
                _product_tol(datatype, k), (PRODUCTS[case], alpha, act))
        used = sum(sizes)
        assert np.array_equal(got[used:], C0[used:])              # rows behind the last group are left as they were


@pytest.mark.parametrize("datatype", ["float", "double"])
@pytest.mark.parametrize("case", range(len(PRODUCTS)))
def test_expert_gemm_weights(stream, datatype, case):
    rows, sizes, n, k = PRODUCTS[case]
    rng = np.random.default_rng(200 + case)
    A, B = rng.standard_normal((rows, n)).astype(NP[datatype]), rng.standard_normal((rows, k)).astype(NP[datatype])
    used = sum(sizes)
    A[used:], B[used:] = np.nan, np.inf                            # rows outside every group do not enter
    C0 = rng.standard_normal((len(sizes), n, k)).astype(NP[datatype])
    bias0 = rng.standard_normal((len(sizes), n)).astype(NP[datatype])
    off = ct.to_tensor(_offsets(sizes), "int")
    At, Bt = ct.to_tensor(A, datatype), ct.to_tensor(B, datatype)
    for alpha, beta, with_bias in [(1.0, 0.0, True), (-0.5, 1.0, True), (0.3, 0.25, False)]:
        start = np.full_like(C0, np.nan) if beta == 0 else C0      # beta = 0 never reads C
        Ct, bt = ct.to_tensor(start, datatype), ct.to_tensor(np.full_like(bias0, np.nan) if beta == 0 else bias0, datatype)
        ct.expert_gemm_weights(Ct, alpha, At, Bt, beta, off, bias_gradient=bt if with_bias else None)
        want, size, bias, bias_size = plain.expert_gemm_weights(C0, alpha, A, B, beta, _offsets(sizes), bias0)
        tol = _product_tol(datatype, max(sizes))
        _within(ct.to_array(Ct), want, size, tol, (PRODUCTS[case], alpha, "weights"))
        if with_bias:
            _within(ct.to_array(bt), bias, bias_size, (max(sizes) + 8) * U[datatype], (PRODUCTS[case], alpha, "bias"))


@pytest.mark.parametrize("datatype", ["float", "double"])
@pytest.mark.parametrize("pad,shift", [(4, 0), (1, 0), (3, 1), (4, 4), (0, 1)])
def test_expert_gemm_pitches_and_alignments(stream, datatype, pad, shift):
    rows, sizes, n, k = 150, [40, 0, 100], 72, 56
    rng = np.random.default_rng(17)
    A, C0 = rng.standard_normal((rows, k)).astype(NP[datatype]), rng.standard_normal((rows, n)).astype(NP[datatype])
    W = rng.standard_normal((3, n, k)).astype(NP[datatype])
    off = ct.to_tensor(_offsets(sizes), "int")
    Aw, _ = _window(A, datatype, pad, shift)
    flat, whole = _window(W.reshape(3 * n, k), datatype, pad, shift)
    Ww = ct.Tensor(flat.device, {"shape": [3, n, k], "strides": [n * (k + pad), k + pad, 1]}, flat.buffer)
    Cw, Cwhole = _window(C0, datatype, pad, shift)
    ct.expert_gemm(Cw, True, 1.0, Aw, Ww, 0.5, off)
    want, size = plain.expert_gemm(C0, True, 1.0, A, W, 0.5, _offsets(sizes))
    _within(_read(Cw, Cwhole, pad, shift), want, size, _product_tol(datatype, k), "forward")
    Dw, Dwhole = _window(A, datatype, pad, shift)
    dY, _ = _window(C0, datatype, pad, shift)
    ct.expert_gemm(Dw, False, 1.0, dY, Ww, 0.0, off)
    want, size = plain.expert_gemm(A, False, 1.0, C0, W, 0.0, _offsets(sizes))
    _within(_read(Dw, Dwhole, pad, shift), want, size, _product_tol(datatype, n), "input gradient")
    ct.expert_gemm_weights(Ww, 2.0, dY, Aw, 1.0, off)
    want, size, _, _ = plain.expert_gemm_weights(W, 2.0, C0, A, 1.0, _offsets(sizes))
    _within(_read(flat, whole, pad, shift), want.reshape(3 * n, k), size.reshape(3 * n, k), _product_tol(datatype, 100), "weights")


@pytest.mark.parametrize("datatype", ["float", "double"])
def test_expert_gemm_keeps_other_experts_out(stream, datatype):
    """Infinities and NaN in the rows or weights of one expert reach no other one, in every direction."""
    sizes, n, k = [5, 3, 8, 130], 36, 20                           # no multiple of any tile: neighbours share tiles
    rng = np.random.default_rng(23)
    rows = sum(sizes) + 3
    off = ct.to_tensor(_offsets(sizes), "int")
    X, dY = rng.standard_normal((rows, k)).astype(NP[datatype]), rng.standard_normal((rows, n)).astype(NP[datatype])
    W = rng.standard_normal((4, n, k)).astype(NP[datatype])
    clean_y = plain.expert_gemm(np.zeros((rows, n)), True, 1.0, X, W, 0.0, _offsets(sizes))
    clean_x = plain.expert_gemm(np.zeros((rows, k)), False, 1.0, dY, W, 0.0, _offsets(sizes))
    clean_w = plain.expert_gemm_weights(np.zeros((4, n, k)), 1.0, dY, X, 0.0, _offsets(sizes))
    for bad in (0, 1, 2):
        lo, hi = _offsets(sizes)[bad:bad + 2]
        X2, dY2, W2 = X.copy(), dY.copy(), W.copy()
        X2[lo:hi], dY2[lo:hi], W2[bad] = np.nan, np.inf, np.nan
        X2[sum(sizes):] = np.inf
        others = np.array([r for r in range(sum(sizes)) if not lo <= r < hi])
        other_e = [e for e in range(4) if e != bad]
        Xt, dYt, Wt = ct.to_tensor(X2, datatype), ct.to_tensor(dY2, datatype), ct.to_tensor(W2, datatype)
        y, x, w = ct.new_tensor([rows, n], datatype), ct.new_tensor([rows, k], datatype), ct.new_tensor([4, n, k], datatype)
        ct.expert_gemm(y, True, 1.0, Xt, Wt, 0.0, off)
        ct.expert_gemm(x, False, 1.0, dYt, Wt, 0.0, off)
        ct.expert_gemm_weights(w, 1.0, dYt, Xt, 0.0, off)
        _within(ct.to_array(y).reshape(rows, n)[others], clean_y[0][others], clean_y[1][others], _product_tol(datatype, k), "y")
        _within(ct.to_array(x).reshape(rows, k)[others], clean_x[0][others], clean_x[1][others], _product_tol(datatype, n), "x")
        _within(ct.to_array(w).reshape(4, n, k)[other_e], clean_w[0][other_e], clean_w[1][other_e], _product_tol(datatype, 130), "w")


def test_expert_gemm_repeats_its_bits_and_replays(stream):
    """Two calls give the same bits, and so does a captured call replayed on new data in the same buffers."""
    sizes, n, k = [100, 3, 0, 200], 260, 512
    rows = sum(sizes)
    rng = np.random.default_rng(31)
    off = ct.to_tensor(_offsets(sizes), "int")
    X, dY = ct.to_tensor(rng.standard_normal((rows, k)), "float"), ct.to_tensor(rng.standard_normal((rows, n)), "float")
    W = ct.to_tensor(rng.standard_normal((4, n, k)), "float")
    y, x, w = ct.new_tensor([rows, n], "float"), ct.new_tensor([rows, k], "float"), ct.new_tensor([4, n, k], "float")
    wb = ct.new_tensor([4, n], "float")

    def run():
        ct.expert_gemm(y, True, 1.0, X, W, 0.0, off, act="relu")
        ct.expert_gemm(x, False, 1.0, dY, W, 0.0, off)
        ct.expert_gemm_weights(w, 1.0, dY, X, 0.0, off, bias_gradient=wb)

    run()
    first = [ct.to_array(t) for t in (y, x, w, wb)]
    run()
    assert all(np.array_equal(a, ct.to_array(t)) for a, t in zip(first, (y, x, w, wb)))
    stream.begin_capture()
    run()
    graph = stream.end_capture()
    sizes2 = [1, 150, 100, 20]                                      # other groups, other values, same buffers
    ct.assign(off, ct.to_tensor(_offsets(sizes2), "int"))
    X2 = rng.standard_normal((rows, k)).astype(np.float32)
    ct.assign(X, ct.to_tensor(X2, "float"))
    graph.launch(stream)
    replayed = [ct.to_array(t) for t in (y, x, w, wb)]
    run()
    eager = [ct.to_array(t) for t in (y, x, w, wb)]
    for i, (a, b) in enumerate(zip(replayed, eager)):
        assert np.array_equal(a, b), i
    graph.release()


@pytest.mark.parametrize("datatype", ["float", "double"])
@pytest.mark.parametrize("offsets", [[0, 50, 30, 64], [-5, 10, 20, 64], [0, 10, 20, 900], [0, 10, 2147483647, -2147483648]])
def test_expert_gemm_reports_bad_offsets(b200_driver, datatype, offsets):
    """Offsets that decrease or leave the rows: clamped, nothing outside is written, and the sync raises."""
    s = b200_driver.default_device().create_stream()
    rows, n, k = 64, 40, 24
    rng = np.random.default_rng(3)
    X, W = rng.standard_normal((rows, k)).astype(NP[datatype]), rng.standard_normal((3, n, k)).astype(NP[datatype])
    with ct.with_stream(s):
        off = ct.to_tensor(np.array(offsets, np.int32), "int")
        Xt, Wt, Y = ct.to_tensor(X, datatype), ct.to_tensor(W, datatype), ct.new_tensor([rows, n], datatype)
        dW = ct.new_tensor([3, n, k], datatype)
        ct.expert_gemm(Y, True, 1.0, Xt, Wt, 0.0, off)
        with pytest.raises(_lib.B200Error):
            s.sync()
        want, size = plain.expert_gemm(np.zeros((rows, n)), True, 1.0, X, W, 0.0, offsets)
        _within(ct.to_array(Y), want, size, _product_tol(datatype, k), "clamped")
        ct.expert_gemm_weights(dW, 1.0, Y, Xt, 0.0, off)
        with pytest.raises(_lib.B200Error):
            s.sync()
    s.sync()


def test_expert_gemm_many_experts_and_no_rows(stream):
    sizes = [0, 1, 2] * 700
    rows, n, k = sum(sizes), 12, 8
    rng = np.random.default_rng(4)
    X, W = rng.standard_normal((rows, k)).astype(np.float32), rng.standard_normal((len(sizes), n, k)).astype(np.float32)
    off = ct.to_tensor(_offsets(sizes), "int")
    Xt, Wt, Y = ct.to_tensor(X, "float"), ct.to_tensor(W, "float"), ct.new_tensor([rows, n], "float")
    ct.expert_gemm(Y, True, 1.0, Xt, Wt, 0.0, off)
    want, size = plain.expert_gemm(np.zeros((rows, n)), True, 1.0, X, W, 0.0, _offsets(sizes))
    _within(ct.to_array(Y), want, size, _product_tol("float", k), "many")
    dW = ct.new_tensor([len(sizes), n, k], "float")
    ct.expert_gemm_weights(dW, 1.0, Y, Xt, 0.0, off)
    want, size, _, _ = plain.expert_gemm_weights(np.zeros((len(sizes), n, k)), 1.0, ct.to_array(Y).reshape(rows, n), X, 0.0, _offsets(sizes))
    _within(ct.to_array(dW), want, size, _product_tol("float", 2), "many weights")


# ---- residual normalisation -------------------------------------------------------------------------------------

# rows, cols, gate rows (0 = none)
BLOCKS = [(1, 1, 0), (1, 5, 1), (3, 8, 3), (4, 100, 2), (7, 129, 7), (16, 1024, 4), (12, 2500, 3), (5, 4096, 1), (300, 64, 1),
          (257, 36, 257), (1000, 40, 125), (90, 513, 9), (2, 9000, 1), (3, 20001, 3), (6, 8192, 2), (640, 260, 5), (2000, 16, 2),
          (700, 4100, 7), (5, 4101, 5), (4, 6001, 1), (301, 2101, 1), (9, 4097, 0)]


def _block_inputs(rows, d, gate_rows, with_after, with_bias, datatype, seed):
    rng = np.random.default_rng(seed)
    f = lambda *s, scale=1.0, shift=0.0: (rng.standard_normal(s) * scale + shift).astype(NP[datatype])
    after = (f(d, scale=0.3, shift=1.0), f(d) if with_bias else None) if with_after else None
    before = (f(d, scale=0.3, shift=1.0), f(d) if with_bias else None)
    return dict(block=f(rows, d, scale=2.0, shift=0.3), residual=f(rows, d), gate=f(gate_rows, d) if gate_rows else None, after=after,
                before=before, dy=f(rows, d), dt=f(rows, d))


def _up(x, datatype):
    if isinstance(x, tuple):
        return tuple(_up(v, datatype) for v in x)
    return None if x is None else ct.to_tensor(x, datatype)


def _norm_tol(datatype, d, rows=0):
    return (64 + d / 32 + (rows + 64 if rows else 0)) * U[datatype]


@pytest.mark.parametrize("datatype", ["float", "double"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("case", range(len(BLOCKS)))
def test_block_normalize(stream, datatype, kind, case):
    rows, d, gate_rows = BLOCKS[case]
    for variant, (with_after, with_bias) in enumerate([(True, True), (False, False), (True, False)]):
        i = _block_inputs(rows, d, gate_rows, with_after, with_bias, datatype, 300 + case * 8 + variant)
        t = {k: _up(v, datatype) for k, v in i.items()}
        total, out = ct.new_tensor([rows, d], datatype), ct.new_tensor([rows, d], datatype)
        args = (t["gate"], 0.7, t["after"], t["before"], 1e-4, kind)
        ct.block_normalize(out, total, t["block"], t["residual"], *args)
        w_total, s_total, w_out, s_out = plain.block_normalize(i["block"], i["residual"], i["gate"], 0.7, i["after"], i["before"], 1e-4, kind)
        g_total, g_out = ct.to_array(total), ct.to_array(out)
        _within(g_total, w_total, s_total, _norm_tol(datatype, d), "total")
        _within(g_out, w_out, s_out, 2 * _norm_tol(datatype, d), "output")
        # in place on the residual stream, and the output over the block: the same bits
        ct.block_normalize(t["block"], t["residual"], t["block"], t["residual"], *args)
        assert np.array_equal(ct.to_array(t["residual"]), g_total) and np.array_equal(ct.to_array(t["block"]), g_out)
        # without a block: the residual is normalised, and may be copied
        r = ct.to_tensor(i["residual"], datatype)
        ct.block_normalize(out, total if variant else None, None, r, None, 0.7, None, t["before"], 1e-4, kind)
        _, _, w_out, s_out = plain.block_normalize(None, i["residual"], None, 0.7, None, i["before"], 1e-4, kind)
        _within(ct.to_array(out), w_out, s_out, _norm_tol(datatype, d), "output alone")
        if variant:
            assert np.array_equal(ct.to_array(total), i["residual"].reshape(-1))
    # no normalisation before the next block: only the sum
    t = {k: _up(v, datatype) for k, v in i.items()}
    ct.block_normalize(None, total, t["block"], t["residual"], t["gate"], 0.7, t["after"], None, 1e-4, kind)
    assert np.array_equal(ct.to_array(total), g_total)


@pytest.mark.parametrize("datatype", ["float", "double"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("case", range(len(BLOCKS)))
def test_block_normalize_gradients(stream, datatype, kind, case):
    rows, d, gate_rows = BLOCKS[case]
    new = lambda *s: ct.new_tensor(list(s), datatype)
    for variant, (with_after, with_bias, with_dt) in enumerate([(True, True, True), (False, False, True), (True, False, False)]):
        i = _block_inputs(rows, d, gate_rows, with_after, with_bias, datatype, 500 + case * 8 + variant)
        total = plain.block_normalize(i["block"], i["residual"], i["gate"], 0.7, i["after"], i["before"], 1e-4, kind)[0].astype(NP[datatype])
        t = {k: _up(v, datatype) for k, v in i.items()}
        tt = ct.to_tensor(total, datatype)
        g = {"block": new(rows, d), "residual": new(rows, d), "before": new(d), "before_b": new(d)}
        if with_after:
            g.update(after=new(d), after_b=new(d))
        if gate_rows:
            g["gate"] = new(gate_rows, d)
        call = lambda dt, rg: ct.block_normalize_gradients(
            g["block"], rg, g.get("gate"), (g["after"], g["after_b"]) if with_after else None, (g["before"], g["before_b"]), t["dy"], dt, tt,
            t["block"], t["gate"], 0.7, t["after"], t["before"], 1e-4, kind)
        call(t["dt"] if with_dt else None, g["residual"])
        want = plain.block_normalize_gradients(i["dy"], i["dt"] if with_dt else None, total, i["block"], i["gate"], 0.7, i["after"],
                                               i["before"], 1e-4, kind)
        first = {}
        for name, (value, size) in want.items():
            first[name] = ct.to_array(g[name])
            per = {"block": 0, "residual": 0, "gate": rows // max(gate_rows, 1)}.get(name, rows)
            _within(first[name], value, size, 4 * _norm_tol(datatype, d, per), (BLOCKS[case], variant, name))
        if with_dt:                                                  # over the gradient that reached the sum: the same bits
            call(t["dt"], t["dt"])
            first["residual"], g["residual"] = first["residual"], t["dt"]
            for name in want:
                assert np.array_equal(ct.to_array(g[name]), first[name]), name


@pytest.mark.parametrize("datatype", ["float", "double"])
@pytest.mark.parametrize("pad,shift", [(4, 0), (1, 0), (3, 1), (0, 1)])
def test_block_normalize_pitches_and_alignments(stream, datatype, pad, shift):
    rows, d = 9, 132
    i = _block_inputs(rows, d, 3, True, True, datatype, 77)
    win = {k: _window(i[k], datatype, pad, shift) for k in ("block", "residual", "dy", "dt")}
    out, total = _window(i["dy"], datatype, pad, shift), _window(i["dy"], datatype, pad, shift)
    gate, after, before = _up(i["gate"], datatype), _up(i["after"], datatype), _up(i["before"], datatype)
    ct.block_normalize(out[0], total[0], win["block"][0], win["residual"][0], gate, 0.7, after, before, 1e-4, "layer")
    w_total, s_total, w_out, s_out = plain.block_normalize(i["block"], i["residual"], i["gate"], 0.7, i["after"], i["before"], 1e-4, "layer")
    g_total = _read(*total, pad, shift)
    _within(g_total, w_total, s_total, _norm_tol(datatype, d), "total")
    _within(_read(*out, pad, shift), w_out, s_out, 2 * _norm_tol(datatype, d), "output")
    bg, rg = _window(i["dy"], datatype, pad, shift), _window(i["dy"], datatype, pad, shift)
    ct.block_normalize_gradients(bg[0], rg[0], None, None, None, win["dy"][0], win["dt"][0], total[0], win["block"][0], gate, 0.7, after,
                                 before, 1e-4, "layer")
    want = plain.block_normalize_gradients(i["dy"], i["dt"], g_total, i["block"], i["gate"], 0.7, i["after"], i["before"], 1e-4, "layer")
    _within(_read(*rg, pad, shift), *want["residual"], 4 * _norm_tol(datatype, d, 1), "residual gradient")
    _within(_read(*bg, pad, shift), *want["block"], 4 * _norm_tol(datatype, d, 1), "block gradient")


def test_block_normalize_without_parts(stream):
    """No block: only the normalised sum has gradients.  No normalisation before the next block: only the sum."""
    i = _block_inputs(6, 40, 0, True, True, "double", 9)
    t = {k: _up(v, "double") for k, v in i.items()}
    rg, bg, s, b = (ct.new_tensor(x, "double") for x in ([6, 40], [6, 40], [40], [40]))
    ct.block_normalize_gradients(None, rg, None, None, (s, b), t["dy"], None, t["residual"], None, None, 1.0, None, t["before"], 1e-4)
    want = plain.block_normalize_gradients(i["dy"], None, i["residual"], None, None, 1.0, None, i["before"], 1e-4, "rms")
    for got, name in ((rg, "residual"), (s, "before"), (b, "before_b")):
        _within(ct.to_array(got), *want[name], 4 * _norm_tol("double", 40, 6), name)
    ct.block_normalize_gradients(bg, rg, None, (s, b), None, None, t["dt"], None, t["block"], None, 0.5, t["after"], None, 1e-4)
    want = plain.block_normalize_gradients(None, i["dt"], None, i["block"], None, 0.5, i["after"], None, 1e-4, "rms")
    for got, name in ((rg, "residual"), (bg, "block"), (s, "after"), (b, "after_b")):
        _within(ct.to_array(got), *want[name], 4 * _norm_tol("double", 40, 6), name)


def test_block_normalize_rows_that_stand_out(stream):
    """A row of zeros, of one value, of the type's largest values, with an infinity or a NaN: its neighbours do not notice."""
    rows, d = 8, 260
    rng = np.random.default_rng(12)
    x = rng.standard_normal((rows, d)).astype(np.float32)
    x[1], x[2], x[3, 5], x[4, 0] = 0.0, 3.0, np.inf, np.nan
    w = np.ones(d, np.float32)
    out = ct.new_tensor([rows, d], "float")
    for kind in ("rms", "layer"):
        ct.block_normalize(out, None, None, ct.to_tensor(x, "float"), None, 1.0, None, (ct.to_tensor(w, "float"), None), 1e-5, kind)
        got = ct.to_array(out).reshape(rows, d)
        fine = [0, 1, 2, 5, 6, 7]
        _, _, want, size = plain.block_normalize(None, x[fine], None, 1.0, None, (w, None), 1e-5, kind)
        _within(got[fine], want, size, _norm_tol("float", d), kind)
        assert np.isnan(got[4]).all() and not np.isfinite(got[3, 5])
        assert np.array_equal(got[1], np.zeros(d))


# ---- the global gradient norm -----------------------------------------------------------------------------------

SHAPES = [[1], [7], [[3, 5]], [4096, 1, 33], [100003, 0, 17, [64, 48]], [8192, 8191, 8193, 24577], [5] * 700, [1 << 20, 3, 999999]]


@pytest.mark.parametrize("datatype", ["float", "double"])
@pytest.mark.parametrize("shapes", SHAPES, ids=lambda s: "%dx%s" % (len(s), s[0]))
def test_clip_gradients(stream, datatype, shapes):
    rng = np.random.default_rng(41)
    data = [(rng.standard_normal(s) * rng.uniform(0.1, 3.0)).astype(NP[datatype]) for s in shapes]
    norm = plain.global_norm(data)
    n = sum(g.size for g in data)
    tensors = [ct.to_tensor(g, datatype) for g in data]
    got = ct.to_array(optimize.global_norm(tensors))
    # squares and sums in double: n roundings at the very worst, one of the result to the type
    assert abs(got[0] - norm) <= norm * (n * 2.0 ** -53 + 2 * U[datatype])
    for bound in (norm * 0.37, norm * 4.0):
        scale = plain.clip_scale(norm, bound)
        apart = [ct.new_tensor(list(g.shape), datatype) for g in data]
        before = ct.to_array(optimize.clip_gradients(tensors, bound, clipped=apart))
        assert np.array_equal(before, got)
        for t, c, g in zip(tensors, apart, data):
            assert np.array_equal(ct.to_array(t).reshape(g.shape), g)
            _within(ct.to_array(c), g.astype(np.float64) * scale, np.abs(g) * scale, n * 2.0 ** -53 + 4 * U[datatype], bound)
    assert all(np.array_equal(ct.to_array(c).reshape(g.shape), g) for c, g in zip(apart, data))      # within the bound: copied
    want = [ct.to_array(c) for c in apart]
    bound = norm * 0.37
    apart = [ct.new_tensor(list(g.shape), datatype) for g in data]
    optimize.clip_gradients(tensors, bound, clipped=apart)
    optimize.clip_gradients(tensors, bound)                          # in place: the same bits as apart
    assert all(np.array_equal(ct.to_array(t), ct.to_array(c)) for t, c in zip(tensors, apart))
    assert len(want) == len(data)


@pytest.mark.parametrize("datatype", ["float", "double"])
def test_clip_gradients_unaligned_pieces(stream, datatype):
    """Pieces of flat buffers at odd offsets; source and destination may be aligned differently."""
    rng = np.random.default_rng(43)
    flat = rng.standard_normal(50000).astype(NP[datatype])
    src, dst = ct.to_tensor(flat, datatype), ct.to_tensor(np.full(50010, 777.0), datatype)
    cuts = [0, 1, 4, 9, 8201, 8202, 30001, 49999]
    for shift in (0, 1, 3):
        g = [ct.Tensor(src.device, {"shape": [b - a], "strides": [1]}, src.buffer.sub_buffer(a, b - a)) for a, b in zip(cuts[:-1], cuts[1:])]
        c = [ct.Tensor(dst.device, {"shape": [b - a], "strides": [1]}, dst.buffer.sub_buffer(a + shift, b - a)) for a, b in zip(cuts[:-1], cuts[1:])]
        norm = float(ct.to_array(optimize.clip_gradients(g, 1.0, clipped=c))[0])
        want = np.linalg.norm(flat[:49999].astype(np.float64))
        assert abs(norm - want) <= want * 4 * U["float" if datatype == "float" else "double"] * (1 if datatype == "float" else 50000)
        got = ct.to_array(dst)
        np.testing.assert_allclose(got[shift:49999 + shift], flat[:49999] / want, rtol=8 * U[datatype] + 50000 * 2.0 ** -53)
        assert np.all(got[49999 + 3:] == 777.0)


def test_clip_gradients_extremes(stream):
    """Squares that no float holds; infinities and NaN leave the gradients alone; zeros."""
    big = np.array([3e38, -2e38, 1e-40], np.float32)
    t, c = ct.to_tensor(big, "float"), ct.new_tensor([3], "float")
    norm = ct.to_array(optimize.clip_gradients([t], 1.0, clipped=[c]))[0]
    assert np.isinf(norm)                       # 3.6e38 is no float: the norm says so, the scaling used the double
    np.testing.assert_allclose(ct.to_array(c)[:2], big[:2] / np.linalg.norm(big.astype(np.float64)), rtol=2.0 ** -22)
    for bad in (np.inf, np.nan):
        data = np.array([1.0, bad, 2.0], np.float32)
        norm = ct.to_array(optimize.clip_gradients([ct.to_tensor(data, "float")], 1.0, clipped=[c]))[0]
        assert not np.isfinite(norm) and np.array_equal(ct.to_array(c), data, equal_nan=True)
    zero = ct.new_tensor([100], "float")
    assert ct.to_array(optimize.clip_gradients([zero], 1.0))[0] == 0.0 and not ct.to_array(zero).any()


def test_clip_gradients_repeats_its_bits_and_replays(stream):
    rng = np.random.default_rng(47)
    tensors = [ct.to_tensor(rng.standard_normal(n), "float") for n in (300001, 5, 77777)]
    out = [ct.new_tensor([t.ecount()], "float") for t in tensors]
    norm = ct.new_tensor([1], "float")
    run = lambda: optimize.clip_gradients(tensors, 2.0, clipped=out, norm=norm)
    run()
    first = [ct.to_array(t) for t in out + [norm]]
    for _ in range(3):
        run()
        assert all(np.array_equal(a, ct.to_array(t)) for a, t in zip(first, out + [norm]))
    stream.begin_capture()
    run()
    graph = stream.end_capture()
    for t in tensors:
        ct.unary_op(t, 3.0, t, "noop")
    graph.launch(stream)
    replayed = [ct.to_array(t) for t in out + [norm]]
    run()
    assert all(np.array_equal(a, ct.to_array(t)) for a, t in zip(replayed, out + [norm]))
    assert not np.array_equal(replayed[-1], first[-1])
    graph.release()


# ---- together ------------------------------------------------------------------------------------------------------

def test_expert_block_step_matches_the_oracle(b200_driver, oracle_driver):
    """A training step of a residual block of experts (forward, every gradient, clipping, Adam), twice."""
    got = {}
    for name, driver in (("gpu", b200_driver), ("cpu", oracle_driver)):
        s = driver.default_device().create_stream()
        with ct.with_stream(s), ct.with_datatype("double"):
            got[name] = expert_block_step(3, "double", rows=150, routed=140, d=36, hidden=52, experts=5)
        s.sync()
    for key, want in got["cpu"].items():
        # everything in 64 bits on both sides; Adam's step divides by the root of a square: 1e-9 leaves room for that
        np.testing.assert_allclose(got["gpu"][key], want, rtol=1e-9, atol=1e-9 * np.abs(want).max(), err_msg=key)


def test_expert_layers_backward_accumulates(stream):
    rng = np.random.default_rng(51)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    w, b, x, dy, off = f(3, 20, 12), f(3, 20), f(30, 12), f(30, 20), _offsets([10, 0, 18])
    layer = nn.ExpertLinear(ct.to_tensor(w, "float"), ct.to_tensor(b, "float"))
    o = ct.to_tensor(off, "int")
    wg, bg = ct.new_tensor([3, 20, 12], "float"), ct.new_tensor([3, 20], "float")
    for times in (1, 2):
        layer.backward(ct.to_tensor(x, "float"), None, ct.to_tensor(dy, "float"), wg, bg, o)
        want, size, bias, bias_size = plain.expert_gemm_weights(np.zeros_like(w), times, dy, x, 0.0, off, np.zeros_like(b))
        _within(ct.to_array(wg), want, size, _product_tol("float", 18) + 2 * U["float"], "weights")
        _within(ct.to_array(bg), bias, bias_size, 32 * U["float"], "bias")


@pytest.mark.parametrize("tile_n", [64, 128, 256])
@pytest.mark.parametrize("slices", [1, 2, 8])
def test_expert_gemm_tile_widths_slices_and_long_reductions(stream, tile_n, slices):
    """Every tile width and slice count (chosen by size otherwise), reductions that are cut into several roundings."""
    rng = np.random.default_rng(61)
    stream.set_option("gemm-tile-n", tile_n)
    stream.set_option("gemm-k-slices", slices)
    sizes, n, k = [127, 129, 3, 0, 30], 264, 4500
    rows = sum(sizes) + 2
    off = ct.to_tensor(_offsets(sizes), "int")
    X, W, b = (rng.standard_normal(s).astype(np.float32) for s in ((rows, k), (5, n, k), (5, n)))
    Xt, Wt, Y = ct.to_tensor(X, "float"), ct.to_tensor(W, "float"), ct.new_tensor([rows, n], "float")
    ct.expert_gemm(Y, True, 0.5, Xt, Wt, 0.0, off, bias=ct.to_tensor(b, "float"), act="logistic")
    want, size = plain.expert_gemm(np.zeros((rows, n)), True, 0.5, X, W, 0.0, _offsets(sizes), b, "logistic")
    _within(ct.to_array(Y), want, size + 8 * U["float"] / _product_tol("float", k), _product_tol("float", k), "forward")
    sizes, n, k = [4700, 0, 300, 17], 136, 265
    rows = sum(sizes) + 5
    off = ct.to_tensor(_offsets(sizes), "int")
    dY, X, C0 = (rng.standard_normal(s).astype(np.float32) for s in ((rows, n), (rows, k), (4, n, k)))
    Ct = ct.to_tensor(C0, "float")
    ct.expert_gemm_weights(Ct, 1.0, ct.to_tensor(dY, "float"), ct.to_tensor(X, "float"), 1.0, off)
    want, size, _, _ = plain.expert_gemm_weights(C0, 1.0, dY, X, 1.0, _offsets(sizes))
    _within(ct.to_array(Ct), want, size, _product_tol("float", 4700), "weights")


def test_bias_of_a_layer_may_start_anywhere(stream):
    """A bias that is a view at an odd offset of its buffer, in a layer with an even row pitch."""
    rng = np.random.default_rng(67)
    X, W, flat = (rng.standard_normal(s).astype(np.float32) for s in ((40, 64), (36, 64), 64))
    layer_bias = ct.to_tensor(flat, "float")
    for at in (1, 2, 3):
        bias = ct.Tensor(layer_bias.device, {"shape": [36], "strides": [1]}, layer_bias.buffer.sub_buffer(at, 36))
        Y = ct.new_tensor([40, 36], "float")
        nn.Linear(ct.to_tensor(W, "float"), bias).forward_fused(ct.to_tensor(X, "float"), Y, "relu")
        want, size = plain.expert_gemm(np.zeros((40, 36)), True, 1.0, X, W[None], 0.0, [0, 40], flat[None, at:at + 36], "relu")
        _within(ct.to_array(Y), want, size, _product_tol("float", 64), at)


@pytest.mark.parametrize("route", [0, 1, 2])
@pytest.mark.parametrize("n,k", [(256, 64), (260, 2600), (500, 129), (33, 40)])
def test_expert_gemm_scaled_halves(stream, route, n, k):
    """The three ways an fp32 product can go (by size, never / always through scaled halves), all directions, on data that
    fits them, that spans too wide a range, that is too large, and with an infinity in one group."""
    rng = np.random.default_rng(71)
    stream.set_option("gemm-auto-presplit", route)
    sizes = [300, 0, 1, 256, 90, 31]
    rows, e = sum(sizes) + 7, len(sizes)
    off = ct.to_tensor(_offsets(sizes), "int")
    for data in ("plain", "scaled", "wide", "large", "inf"):
        X, dY, W = (rng.standard_normal(s).astype(np.float32) for s in ((rows, k), (rows, n), (e, n, k)))
        if data == "scaled":                                   # every row and column at a scale of its own
            X *= np.exp2(rng.integers(-18, 18, (rows, 1))).astype(np.float32)
            W *= np.exp2(rng.integers(-12, 12, (e, n, 1))).astype(np.float32)
            dY *= np.exp2(rng.integers(-12, 12, (1, n))).astype(np.float32)
        elif data == "wide":                                   # one value that dwarfs its row, and meets a zero
            X[:, 0], W[:, :, 0], dY[0] = -3e38, 0.0, 0.0
            X[0] = 0.0
        elif data == "large":
            X *= np.float32(1e25)
        elif data == "inf":
            X[305, 3] = np.inf                                  # group 3: rows 301 .. 557
        Y0, W0 = rng.standard_normal((rows, n)).astype(np.float32), rng.standard_normal((e, n, k)).astype(np.float32)
        Y, dX, dW = ct.to_tensor(Y0, "float"), ct.new_tensor([rows, k], "float"), ct.to_tensor(W0, "float")
        Xt, dYt, Wt = ct.to_tensor(X, "float"), ct.to_tensor(dY, "float"), ct.to_tensor(W, "float")
        ct.expert_gemm(Y, True, 0.5, Xt, Wt, 0.5, off)
        ct.expert_gemm(dX, False, 1.0, dYt, Wt, 0.0, off)
        ct.expert_gemm_weights(dW, 1.0, dYt, Xt, 1.0, off)
        stream.sync()
        keep = np.ones(rows, bool)
        keep_e = np.ones(e, bool)
        if data == "inf":
            keep[305], keep_e[3] = False, False
        with np.errstate(all="ignore"):
            want, size = plain.expert_gemm(Y0, True, 0.5, X, W, 0.5, _offsets(sizes))
            want_x, size_x = plain.expert_gemm(np.zeros((rows, k)), False, 1.0, dY, W, 0.0, _offsets(sizes))
            want_w, size_w, _, _ = plain.expert_gemm_weights(W0, 1.0, dY, X, 1.0, _offsets(sizes))
        if data == "wide":
            size_w[:, :, 0] = np.inf                            # sums of the giant values themselves: anything near them goes
        _within(ct.to_array(Y).reshape(rows, n)[keep], want[keep], size[keep], _product_tol("float", k), (data, "forward"))
        _within(ct.to_array(dX), want_x, size_x, _product_tol("float", n), (data, "input"))
        got_w = ct.to_array(dW).reshape(e, n, k)
        if data != "wide":
            _within(got_w[keep_e], want_w[keep_e], size_w[keep_e], _product_tol("float", 300), (data, "weights"))
        else:
            _within(got_w[:, :, 1:], want_w[:, :, 1:], size_w[:, :, 1:], _product_tol("float", 300), (data, "weights"))


@pytest.mark.parametrize("way", ["forward", "input", "weights"])
@pytest.mark.parametrize("route,sizes,n,k", [(1, [200, 0, 56], 264, 512), (1, [20, 4, 8], 264, 512), (2, [200, 0, 56], 264, 512)])
def test_expert_gemm_waits_that_run_out(b200_driver, way, route, sizes, n, k):
    _waits_that_run_out(b200_driver, way, route, sizes, n, k, 128 if route == 1 else 0)  # (tensor cores also where there are few rows)


# tiles that follow one another, 128 and 64 wide; slices that meet in L2, of a product and of a weight gradient
@pytest.mark.parametrize("way,sizes,n,k", [("forward", [200, 0, 56], 264, 512), ("input", [20, 9, 8], 264, 512), ("weights", [100, 0, 56], 264, 512),
                                           ("forward", [200, 0, 56], 264, 16000), ("weights", [400, 0, 112], 264, 512)])
def test_expert_gemm_waits_that_run_out_by_sizes(b200_driver, way, sizes, n, k):
    _waits_that_run_out(b200_driver, way, 1, sizes, n, k, 0)


def _waits_that_run_out(b200_driver, way, route, sizes, n, k, tile_n):
    """Producers that deliver nothing (a setting, not a fault): every role gives up in time, the sync raises, and the next call
    on the stream is right."""
    s = b200_driver.default_device().create_stream()
    s.set_option("gemm-auto-presplit", route)
    s.set_option("gemm-tile-n", tile_n)
    rng = np.random.default_rng(5)
    rows, off = sum(sizes), _offsets(sizes)
    X, dY, W = (rng.standard_normal(sh).astype(np.float32) for sh in ((rows, k), (rows, n), (3, n, k)))
    with ct.with_stream(s):
        o, Xt, dYt, Wt = ct.to_tensor(off, "int"), ct.to_tensor(X, "float"), ct.to_tensor(dY, "float"), ct.to_tensor(W, "float")
        out = {"forward": ct.new_tensor([rows, n], "float"), "input": ct.new_tensor([rows, k], "float"),
               "weights": ct.new_tensor([3, n, k], "float")}[way]

        def run():
            if way == "forward":
                ct.expert_gemm(out, True, 1.0, Xt, Wt, 0.0, o)
            elif way == "input":
                ct.expert_gemm(out, False, 1.0, dYt, Wt, 0.0, o)
            else:
                ct.expert_gemm_weights(out, 1.0, dYt, Xt, 0.0, o)

        run()
        s.sync()
        s.set_option("wait-limit-cycles", 1 << 20)
        s.set_option("inject-fault", 1)
        run()
        with pytest.raises(_lib.B200Error) as err:
            s.sync()
        assert err.value.code == 4
        s.set_option("inject-fault", 0)
        s.set_option("wait-limit-cycles", 0)
        run()
        s.sync()
        want = {"forward": lambda: plain.expert_gemm(np.zeros((rows, n)), True, 1.0, X, W, 0.0, off),
                "input": lambda: plain.expert_gemm(np.zeros((rows, k)), False, 1.0, dY, W, 0.0, off),
                "weights": lambda: plain.expert_gemm_weights(np.zeros((3, n, k)), 1.0, dY, X, 0.0, off)[:2]}[way]()
        _within(ct.to_array(out), *want, _product_tol("float", max(k, n)), way)


@pytest.mark.parametrize("offsets", [[0, 500, 300, 640], [-5, 100, 200, 640], [0, 10, 20, 900], [0, 10, 2147483647, -2147483648]])
def test_expert_gemm_scaled_halves_reports_bad_offsets(b200_driver, offsets):
    s = b200_driver.default_device().create_stream()
    s.set_option("gemm-auto-presplit", 2)
    rows, n, k = 640, 72, 104
    rng = np.random.default_rng(3)
    X, dY, W = (rng.standard_normal(sh).astype(np.float32) for sh in ((rows, k), (rows, n), (3, n, k)))
    with ct.with_stream(s):
        off = ct.to_tensor(np.array(offsets, np.int32), "int")
        Xt, dYt, Wt = ct.to_tensor(X, "float"), ct.to_tensor(dY, "float"), ct.to_tensor(W, "float")
        Y, dX, dW, db = ct.new_tensor([rows, n], "float"), ct.new_tensor([rows, k], "float"), ct.new_tensor([3, n, k], "float"), ct.new_tensor([3, n], "float")
        ct.expert_gemm(Y, True, 1.0, Xt, Wt, 0.0, off)
        with pytest.raises(_lib.B200Error):
            s.sync()
        ct.expert_gemm(dX, False, 1.0, dYt, Wt, 0.0, off)
        with pytest.raises(_lib.B200Error):
            s.sync()
        ct.expert_gemm_weights(dW, 1.0, dYt, Xt, 0.0, off, bias_gradient=db)
        with pytest.raises(_lib.B200Error):
            s.sync()
        _within(ct.to_array(Y), *plain.expert_gemm(np.zeros((rows, n)), True, 1.0, X, W, 0.0, offsets), _product_tol("float", k), "y")
        _within(ct.to_array(dX), *plain.expert_gemm(np.zeros((rows, k)), False, 1.0, dY, W, 0.0, offsets), _product_tol("float", n), "x")
        w, ws, b, bs = plain.expert_gemm_weights(np.zeros((3, n, k)), 1.0, dY, X, 0.0, offsets, np.zeros((3, n)))
        _within(ct.to_array(dW), w, ws, _product_tol("float", rows), "w")
        _within(ct.to_array(db), b, bs, (rows + 8) * U["float"], "b")
    s.sync()


def test_no_rows(stream):
    """A batch without rows: nothing to compute, gradients of zero."""
    off = ct.to_tensor(np.zeros(4, np.int32), "int")
    W = ct.new_tensor([3, 8, 4], "float")
    X, Y, D = (ct.new_tensor([0, c], "float") for c in (4, 8, 4))
    ct.expert_gemm(Y, True, 1.0, X, W, 0.0, off)
    ct.expert_gemm(D, False, 1.0, Y, W, 0.0, off)
    dW, db = ct.to_tensor(np.ones((3, 8, 4)), "float"), ct.to_tensor(np.ones((3, 8)), "float")
    ct.expert_gemm_weights(dW, 1.0, Y, X, 0.5, off, bias_gradient=db)
    assert np.all(ct.to_array(dW) == 0.5) and np.all(ct.to_array(db) == 0.5)
    ct.expert_gemm_weights(dW, 1.0, Y, X, 0.0, off, bias_gradient=db)
    assert not ct.to_array(dW).any() and not ct.to_array(db).any()
    w, e = ct.to_tensor(np.ones(4), "float"), [ct.new_tensor([0, 4], "float") for _ in range(7)]
    ct.block_normalize(e[0], e[1], e[2], e[3], None, 1.0, (w, None), (w, None), 1e-5)
    ga, gb = ct.to_tensor(np.ones(4), "float"), ct.to_tensor(np.ones(4), "float")
    ct.block_normalize_gradients(e[4], e[5], None, (ga, None), (gb, None), e[0], e[1], e[2], e[3], None, 1.0, (w, None), (w, None), 1e-5)
    assert not ct.to_array(ga).any() and not ct.to_array(gb).any()


def test_offsets_beyond_32_bits(stream):
    """Matrices of more than 2^31 elements: the last rows are found and right."""
    rows, d = (1 << 19) + 5, 4100
    rng = np.random.default_rng(81)
    last, w = rng.standard_normal((3, d)).astype(np.float32), rng.standard_normal(d).astype(np.float32)
    x, y = ct.new_tensor([rows, d], "float", init_value=None), ct.new_tensor([rows, d], "float", init_value=None)

    def fill(value):                                 # (memset takes fewer than 2^31 elements at a time)
        for first in (0, rows // 2):
            n = (rows // 2 if first == 0 else rows - rows // 2) * d
            ct.assign(ct.Tensor(x.device, {"shape": [n], "strides": [1]}, x.buffer.sub_buffer(first * d, n)), value)

    fill(1.0)
    tail = lambda t: ct.Tensor(t.device, {"shape": [3, d], "strides": [d, 1]}, t.buffer.sub_buffer((rows - 3) * d, 3 * d))
    ct.assign(tail(x), ct.to_tensor(last, "float"))
    wt, gate = ct.to_tensor(w, "float"), ct.to_tensor(w[None], "float")
    ct.block_normalize(y, x, x, x, gate, 0.5, (wt, None), (wt, None), 1e-5, "layer")
    total, t_size, out, o_size = plain.block_normalize(last, last, w[None], 0.5, (w, None), (w, None), 1e-5, "layer")
    _within(ct.to_array(tail(x)), total, t_size, _norm_tol("float", d), "total")
    _within(ct.to_array(tail(y)), out, o_size, 2 * _norm_tol("float", d), "output")
    # the product: all rows are one expert's but the last three
    A, W = ct.new_tensor([rows, 8], "float"), rng.standard_normal((2, d, 8)).astype(np.float32)
    a_last = rng.standard_normal((3, 8)).astype(np.float32)
    at = ct.Tensor(A.device, {"shape": [3, 8], "strides": [8, 1]}, A.buffer.sub_buffer((rows - 3) * 8, 24))
    ct.assign(at, ct.to_tensor(a_last, "float"))
    ct.expert_gemm(y, True, 1.0, A, ct.to_tensor(W, "float"), 0.0, ct.to_tensor(np.array([0, rows - 3, rows], np.int32), "int"))
    want, size = plain.expert_gemm(np.zeros((3, d)), True, 1.0, a_last, W, 0.0, [0, 0, 3])
    _within(ct.to_array(tail(y)), want, size, _product_tol("float", 8), "product")
    # the norm, and a piece behind 2^31 elements
    fill(0.5)
    flat = ct.as_vector(x)
    norm = ct.to_array(optimize.clip_gradients([flat], 1.0))[0]
    n = rows * d
    assert abs(norm - 0.5 * np.sqrt(n)) <= norm * 2.0 ** -23
    np.testing.assert_allclose(ct.to_array(tail(x)), 1.0 / np.sqrt(n), rtol=2.0 ** -22)
