"""Calls of the expert products that their documentation allows: bad offsets anywhere, no rows under every option, captured and
replayed calls and calls of two streams at once on scaled halves, narrow tiles in slices."""
import numpy as np
import pytest

from cortex_b200 import _lib
from cortex_b200 import tensor as ct
from oracle import plain_operators as plain
from test_gpu_experts import NP, _offsets, _product_tol, _within, stream  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("datatype", ["float", "double"])
@pytest.mark.parametrize("tile_n", [0, 64, 128])
@pytest.mark.parametrize("rows,experts,at,value", [(1, 64, 33, 0), (1, 64, 64, 2), (8, 100, 70, 9), (8, 100, 99, -1), (3, 4096, 4095, 0),
                                                   (60, 64, 64, 61), (100, 128, 127, 3), (40, 33, 33, 41)])
def test_bad_offsets_of_groups_behind_the_last_row(b200_driver, datatype, tile_n, rows, experts, at, value):
    """The rows lie in the first groups, and only offsets far behind them are bad: clamped, and reported."""
    s = b200_driver.default_device().create_stream()
    s.set_option("gemm-tile-n", tile_n)
    n, k = 24, 40
    rng = np.random.default_rng(41)
    X, W = rng.standard_normal((rows, k)).astype(NP[datatype]), rng.standard_normal((experts, n, k)).astype(NP[datatype])
    good = np.minimum(np.arange(experts + 1), rows).astype(np.int32)
    bad = good.copy()
    bad[at] = value
    with ct.with_stream(s):
        Xt, Wt, Y = ct.to_tensor(X, datatype), ct.to_tensor(W, datatype), ct.new_tensor([rows, n], datatype)
        for trans_b, M, out in ((True, Wt, Y), (False, ct.to_tensor(W.reshape(experts, k, n), datatype), Y)):
            ct.expert_gemm(out, trans_b, 1.0, Xt, M, 0.0, ct.to_tensor(good, "int"))
            s.sync()
            ct.expert_gemm(out, trans_b, 1.0, Xt, M, 0.0, ct.to_tensor(bad, "int"))
            with pytest.raises(_lib.B200Error):
                s.sync()
            want, size = plain.expert_gemm(np.zeros((rows, n)), trans_b, 1.0, X, W if trans_b else W.reshape(experts, k, n), 0.0, bad)
            _within(ct.to_array(out), want, size, _product_tol(datatype, k), trans_b)
    s.sync()


@pytest.mark.parametrize("options", [{"gemm-tile-n": 64}, {"gemm-tile-n": 128, "gemm-k-slices": 4}, {"gemm-auto-presplit": 2}, {"gemm-auto-presplit": 1}])
def test_no_rows_under_options(stream, options):  # noqa: F811
    for name, value in options.items():
        stream.set_option(name, value)
    off = ct.to_tensor(np.zeros(4, np.int32), "int")
    X, Y, D = (ct.new_tensor([0, c], "float") for c in (40, 80, 40))
    W = ct.new_tensor([3, 80, 40], "float")
    ct.expert_gemm(Y, True, 1.0, X, W, 0.0, off)
    ct.expert_gemm(D, False, 1.0, Y, W, 0.0, off)
    for beta in (0.5, 0.0):
        dW, db = ct.to_tensor(np.ones((3, 80, 40)), "float"), ct.to_tensor(np.ones((3, 80)), "float")
        ct.expert_gemm_weights(dW, 1.0, Y, X, beta, off, bias_gradient=db)
        assert np.all(ct.to_array(dW) == beta) and np.all(ct.to_array(db) == beta)


# sizes that take scaled halves by themselves, in every direction
LARGE = ([700, 600, 0, 748], 2048, 1024)


def _large(seed):
    sizes, n, k = LARGE
    rng = np.random.default_rng(seed)
    rows = sum(sizes) + 3
    return rng, [rng.standard_normal(s).astype(np.float32) for s in ((rows, k), (rows, n), (len(sizes), n, k))]


def _all_ways(X, dY, W, off, out):
    y, dx, dw, db = out
    ct.expert_gemm(y, True, 1.0, X, W, 0.0, off, act="relu")
    ct.expert_gemm(dx, False, 1.0, dY, W, 0.0, off)
    ct.expert_gemm_weights(dw, 1.0, dY, X, 1.0, off, bias_gradient=db)


def _outputs(rows):
    sizes, n, k = LARGE
    return [ct.new_tensor(list(s), "float") for s in ((rows, n), (rows, k), (len(sizes), n, k), (len(sizes), n))]


def test_scaled_halves_repeat_their_bits_and_replay(stream):  # noqa: F811
    """A captured pass serves other routings and other data: such that fit halves, and such that fall back inside the replay."""
    sizes, n, k = LARGE
    rng, (X, dY, W) = _large(43)
    rows = len(X)
    off = ct.to_tensor(_offsets(sizes), "int")
    Xt, dYt, Wt = (ct.to_tensor(a, "float") for a in (X, dY, W))
    out, zero = _outputs(rows), lambda ts: [ct.assign(t, 0.0) for t in ts]
    _all_ways(Xt, dYt, Wt, off, out)
    first = [ct.to_array(t) for t in out]
    zero(out)
    _all_ways(Xt, dYt, Wt, off, out)
    assert all(np.array_equal(a, ct.to_array(t)) for a, t in zip(first, out))
    stream.begin_capture()
    _all_ways(Xt, dYt, Wt, off, out)
    graph = stream.end_capture()
    wide = X.copy()
    wide[5] *= np.exp2(-rng.integers(0, 60, k)).astype(np.float32)
    wide[1000, 7] = 1e30
    for sizes2, data in (([1, 0, 2000, 50], X), (sizes, wide), ([500, 500, 500, 551], X)):
        ct.assign(off, ct.to_tensor(_offsets(sizes2), "int"))
        ct.assign(Xt, ct.to_tensor(data, "float"))
        zero(out)
        graph.launch(stream)
        replayed = [ct.to_array(t) for t in out]
        zero(out)
        _all_ways(Xt, dYt, Wt, off, out)
        assert all(np.array_equal(a, ct.to_array(t)) for a, t in zip(replayed, out)), sizes2
        want, size = plain.expert_gemm(np.zeros((rows, n)), True, 1.0, data, W, 0.0, _offsets(sizes2), act="relu")
        _within(replayed[0], want, size, _product_tol("float", k), sizes2)
    graph.release()


def test_two_streams_at_once_on_scaled_halves(b200_driver):
    device = b200_driver.default_device()
    made = []
    for seed in (47, 53):
        s = device.create_stream()
        with ct.with_stream(s):
            _, arrays = _large(seed)
            tensors = [ct.to_tensor(a, "float") for a in arrays] + [ct.to_tensor(_offsets(LARGE[0]), "int")]
            alone = _outputs(len(arrays[0]))
            _all_ways(*tensors, alone)
            made.append((s, tensors, [ct.to_array(t) for t in alone], [_outputs(len(arrays[0])) for _ in range(4)]))
    for s, _, _, _ in made:
        s.sync()
    for i in range(4):
        for s, tensors, _, outs in made:
            with ct.with_stream(s):
                _all_ways(*tensors, outs[i])
    for s, _, alone, outs in made:
        with ct.with_stream(s):
            assert all(np.array_equal(a, ct.to_array(t)) for out in outs for a, t in zip(alone, out))
        s.sync()


# even rows per expert up to 32, more than the kernels of few rows take: one slice, a cluster's slices, slices that meet in L2
@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("sizes,n,k", [([30, 20], 2048, 260), ([30, 20], 128, 2048), ([40, 0, 9], 300, 1100), ([30, 20], 128, 16000), ([33, 31], 64, 9000),
                                       ([17], 100, 20000)])
def test_narrow_tiles_in_slices(stream, trans_b, sizes, n, k):  # noqa: F811
    rng = np.random.default_rng(59)
    rows = sum(sizes) + 1
    X, W, b = (rng.standard_normal(s).astype(np.float32) for s in ((rows, k), (len(sizes),) + ((n, k) if trans_b else (k, n)), (len(sizes), n)))
    C0 = rng.standard_normal((rows, n)).astype(np.float32)
    for beta, act in ((0.0, None), (0.5, "relu")):
        Y = ct.to_tensor(C0, "float")
        ct.expert_gemm(Y, trans_b, 0.5, ct.to_tensor(X, "float"), ct.to_tensor(W, "float"), beta, ct.to_tensor(_offsets(sizes), "int"),
                       bias=ct.to_tensor(b, "float"), act=act)
        want, size = plain.expert_gemm(C0, trans_b, 0.5, X, W, beta, _offsets(sizes), b, act)
        _within(ct.to_array(Y), want, size, _product_tol("float", k), (sizes, beta))
        assert np.array_equal(ct.to_array(Y).reshape(rows, n)[-1], C0[-1])


@pytest.mark.parametrize("route", [1, 2])
@pytest.mark.parametrize("sizes,n,k", [([1], 1, 1), ([3, 0, 2], 2, 1), ([1, 1], 1, 9), ([5, 300], 7, 8), ([65, 64, 63], 31, 65), ([0, 1, 2] * 300, 24, 16),
                                       ([256, 257, 255], 257, 127), ([4], 8200, 3), ([2, 1], 3, 8200)])
def test_smallest_and_oddest_sizes_on_either_route(stream, route, sizes, n, k):  # noqa: F811
    stream.set_option("gemm-auto-presplit", route)
    rng = np.random.default_rng(67)
    rows, e = sum(sizes) + 1, len(sizes)
    X, dY, W = (rng.standard_normal(s).astype(np.float32) for s in ((rows, k), (rows, n), (e, n, k)))
    off = ct.to_tensor(_offsets(sizes), "int")
    Xt, dYt, Wt = (ct.to_tensor(a, "float") for a in (X, dY, W))
    Y, dX, dW, db = (ct.new_tensor(list(s), "float") for s in ((rows, n), (rows, k), (e, n, k), (e, n)))
    ct.expert_gemm(Y, True, 1.0, Xt, Wt, 0.0, off)
    ct.expert_gemm(dX, False, 1.0, dYt, Wt, 0.0, off)
    ct.expert_gemm_weights(dW, 1.0, dYt, Xt, 0.0, off, bias_gradient=db)
    o = _offsets(sizes)
    _within(ct.to_array(Y), *plain.expert_gemm(np.zeros((rows, n)), True, 1.0, X, W, 0.0, o), _product_tol("float", k), "forward")
    _within(ct.to_array(dX), *plain.expert_gemm(np.zeros((rows, k)), False, 1.0, dY, W, 0.0, o), _product_tol("float", n), "input")
    w, ws, b, bs = plain.expert_gemm_weights(np.zeros((e, n, k)), 1.0, dY, X, 0.0, o, np.zeros((e, n)))
    _within(ct.to_array(dW), w, ws, _product_tol("float", max(sizes)), "weights")
    _within(ct.to_array(db), b, bs, (max(sizes) + 8) * 2.0 ** -24, "bias")


def test_no_memory_left_for_the_halves(b200_driver):
    """The halves' workspace does not fit beside what a program holds: the call runs without them."""
    device = b200_driver.default_device()
    s = device.create_stream()
    s.set_option("gemm-auto-presplit", 2)
    sizes, n, k = [130, 0, 126, 256], 4096, 4096                 # halves of 268 MB
    rows = sum(sizes)
    rng = np.random.default_rng(73)
    X, W, dY = rng.standard_normal((rows, k)).astype(np.float32), rng.standard_normal((4, n, k)).astype(np.float32), None
    dY = rng.standard_normal((rows, n)).astype(np.float32)
    with ct.with_stream(s):
        off, Xt, Wt, dYt = ct.to_tensor(_offsets(sizes), "int"), ct.to_tensor(X, "float"), ct.to_tensor(W, "float"), ct.to_tensor(dY, "float")
        Y, dX = ct.new_tensor([rows, n], "float"), ct.new_tensor([rows, k], "float")
        s.sync()
        held, room = [], device.memory_info()["free"] - (96 << 20)
        while room > (8 << 20):
            size = min(room, 8 << 30)
            held.append(device.allocate_device_buffer(size // 8, "double"))
            room = min(room - size, device.memory_info()["free"] - (96 << 20))
        ct.expert_gemm(Y, True, 1.0, Xt, Wt, 0.0, off)
        ct.expert_gemm(dX, False, 1.0, dYt, Wt, 0.0, off)
        s.sync()
        for b in held:
            b.release()
        lo, hi = 120, 140                                        # rows of two experts
        w, ws = plain.expert_gemm(np.zeros((20, n)), True, 1.0, X[lo:hi], W[[0, 2]], 0.0, [0, 10, 20])
        _within(ct.to_array(Y).reshape(rows, n)[lo:hi], w, ws, _product_tol("float", k), "forward")
        w, ws = plain.expert_gemm(np.zeros((20, k)), False, 1.0, dY[lo:hi], W[[0, 2]], 0.0, [0, 10, 20])
        _within(ct.to_array(dX).reshape(rows, k)[lo:hi], w, ws, _product_tol("float", n), "input")
