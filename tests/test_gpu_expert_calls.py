"""Calls of the expert products that their documentation allows: bad offsets anywhere, no rows under every option."""
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
