"""Residual normalisation of rows whose squares leave the type's range."""
import numpy as np
import pytest

from cortex_b200 import tensor as ct
from oracle import plain_operators as plain
from test_gpu_experts import NP, _norm_tol, _within, stream  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("datatype,large", [("float", 3e38), ("float", 1e25), ("double", 1.5e308), ("double", 1e200)])
@pytest.mark.parametrize("cols", [8, 33, 260, 5000, 20000])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_rows_of_the_types_largest_values(stream, datatype, large, cols, kind):  # noqa: F811
    """Such a row comes out as the bias, or as NaN where even its values have no sum; its neighbours do not notice."""
    rng = np.random.default_rng(71)
    x = rng.standard_normal((5, cols)).astype(NP[datatype])
    x[1] = np.where(np.arange(cols) % 3 == 0, -large, large)
    w, b = (rng.standard_normal(cols).astype(NP[datatype]) for _ in range(2))
    out = ct.new_tensor([5, cols], datatype)
    ct.block_normalize(out, None, None, ct.to_tensor(x, datatype), None, 1.0, None, (ct.to_tensor(w, datatype), ct.to_tensor(b, datatype)), 1e-5, kind)
    got = ct.to_array(out).reshape(5, cols)
    fine = [0, 2, 3, 4]
    _, _, want, size = plain.block_normalize(None, x[fine], None, 1.0, None, (w, b), 1e-5, kind)
    _within(got[fine], want, size, _norm_tol(datatype, cols), kind)
    assert np.array_equal(got[1], b) or (kind == "layer" and np.isnan(got[1]).all())
