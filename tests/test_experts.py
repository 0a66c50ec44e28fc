"""Expert layers, residual normalisation and gradient clipping without a GPU: the plain statements against differences,
the refusals of the tensor API and of the C ABI, and a training step of the layers on the CPU oracle."""
import ctypes as C

import numpy as np
import pytest

from cortex_b200 import _lib, nn, optimize
from cortex_b200 import tensor as ct
from oracle import plain_operators as plain


@pytest.fixture
def bound(oracle_driver):
    with ct.with_stream(oracle_driver.default_device().create_stream()), ct.with_datatype("double"):
        yield


def _numeric(f, x, h=1e-6):
    g = np.zeros(x.shape)
    for i in np.ndindex(*x.shape):
        keep = x[i]
        x[i] = keep + h
        hi = f()
        x[i] = keep - h
        lo = f()
        x[i] = keep
        g[i] = (hi - lo) / (2 * h)
    return g


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate_rows", [0, 1, 2, 6])
@pytest.mark.parametrize("with_after", [True, False])
def test_plain_block_gradients_against_differences(kind, gate_rows, with_after):
    rng = np.random.default_rng(5 + gate_rows)
    rows, d, eps = 6, 5, 1e-3
    block, residual = rng.standard_normal((rows, d)), rng.standard_normal((rows, d))
    gate = rng.standard_normal((gate_rows, d)) if gate_rows else None
    aw, ab, bw, bb = (rng.standard_normal(d) for _ in range(4))
    after, before = ((aw, ab) if with_after else None), (bw, bb)
    c_total, c_out = rng.standard_normal((rows, d)), rng.standard_normal((rows, d))

    def loss():
        total, _, out, _ = plain.block_normalize(block, residual, gate, 0.7, after, before, eps, kind)
        return float((total * c_total).sum() + (out * c_out).sum())

    total = plain.block_normalize(block, residual, gate, 0.7, after, before, eps, kind)[0]
    got = plain.block_normalize_gradients(c_out, c_total, total, block, gate, 0.7, after, before, eps, kind)
    wanted = {"block": block, "residual": residual, "before": bw, "before_b": bb}
    if with_after:
        wanted.update(after=aw, after_b=ab)
    if gate_rows:
        wanted["gate"] = gate
    assert set(wanted) == set(got)
    for name, x in wanted.items():
        # central differences of step 1e-6: truncation ~1e-12 * f''', rounding ~1e-16 * |loss| / 1e-6, |loss| < 1e3
        np.testing.assert_allclose(got[name][0], _numeric(loss, x), atol=1e-6, rtol=1e-6, err_msg=name)


def test_plain_expert_gradients_against_differences():
    rng = np.random.default_rng(8)
    offsets = [0, 3, 3, 5]
    x, w, b = rng.standard_normal((7, 4)), rng.standard_normal((3, 2, 4)), rng.standard_normal((3, 2))
    c = rng.standard_normal((7, 2))
    c[5:] = 0.0                                       # rows outside every group

    def loss():
        return float((plain.expert_gemm(np.zeros((7, 2)), True, 1.0, x, w, 0.0, offsets, b, "tanh")[0] * c).sum())

    y = plain.expert_gemm(np.zeros((7, 2)), True, 1.0, x, w, 0.0, offsets, b, "tanh")[0]
    dy = c * (1 - y * y)
    dx = plain.expert_gemm(np.zeros((7, 4)), False, 1.0, dy, w, 0.0, offsets)[0]
    dw, _, db, _ = plain.expert_gemm_weights(np.zeros((3, 2, 4)), 1.0, dy, x, 0.0, offsets, np.zeros((3, 2)))
    for got, arg in ((dx, x), (dw, w), (db, b)):
        np.testing.assert_allclose(got, _numeric(loss, arg), atol=1e-7)


def _t(shape, dt=None):
    return ct.new_tensor(list(shape), datatype=dt)


def test_expert_gemm_refusals(bound):
    A, B, Cm, off = _t([6, 4]), _t([3, 5, 4]), _t([6, 5]), _t([4], "int")
    ct.expert_gemm(Cm, True, 1.0, A, B, 0.0, off)
    bad = [
        dict(A=_t([6, 3])), dict(B=_t([3, 4, 5])), dict(C=_t([5, 5])), dict(C=_t([6, 4])), dict(offsets=_t([3], "int")),
        dict(offsets=_t([4], "float")), dict(A=_t([6, 4], "float")), dict(B=_t([5, 4])), dict(bias=_t([3, 4])),
        dict(bias=_t([15])), dict(act="softmax"), dict(act="gelu"), dict(C=ct.transpose(_t([5, 6]), [1, 0])),
        dict(A=ct.transpose(_t([4, 6]), [1, 0])), dict(A=_t([6, 4], "int"), B=_t([3, 5, 4], "int"), C=_t([6, 5], "int")),
    ]
    for change in bad:
        args = {"C": Cm, "A": A, "B": B, "offsets": off, "bias": None, "act": None, **change}
        with pytest.raises(ct.TensorError):
            ct.expert_gemm(args["C"], True, 1.0, args["A"], args["B"], 0.0, args["offsets"], bias=args["bias"], act=args["act"])
    square = _t([8, 4])
    with pytest.raises(ct.TensorError, match="overlaps"):      # the product over its own input
        ct.expert_gemm(square, True, 1.0, square, _t([3, 4, 4]), 0.0, off)
    # windows of one buffer that share no memory are fine
    both = _t([12, 4])
    ct.expert_gemm(ct.submatrix(both, 6, 6, 0, 4), True, 1.0, ct.submatrix(both, 0, 6, 0, 4), _t([3, 4, 4]), 0.0, off)


def test_expert_gemm_weights_refusals(bound):
    A, B, Cm, off = _t([6, 5]), _t([6, 4]), _t([3, 5, 4]), _t([4], "int")
    ct.expert_gemm_weights(Cm, 1.0, A, B, 0.0, off, bias_gradient=_t([3, 5]))
    for change in [dict(A=_t([5, 5])), dict(B=_t([6, 5])), dict(C=_t([3, 4, 5])), dict(off=_t([5], "int")), dict(bg=_t([3, 4])),
                   dict(bg=_t([3, 5], "float")), dict(C=_t([15, 4]))]:
        a = {"A": A, "B": B, "C": Cm, "off": off, "bg": None, **change}
        with pytest.raises(ct.TensorError):
            ct.expert_gemm_weights(a["C"], 1.0, a["A"], a["B"], 0.0, a["off"], bias_gradient=a["bg"])


def test_block_normalize_refusals(bound):
    x, r, out, tot, w, gate = _t([6, 4]), _t([6, 4]), _t([6, 4]), _t([6, 4]), _t([4]), _t([3, 4])
    ok = dict(output=out, total=tot, block=x, residual=r, gate=gate, residual_scale=1.0, after=(w, None), before=(w, w), epsilon=1e-5)
    ct.block_normalize(**ok)
    ct.block_normalize(**{**ok, "total": r})                            # in place on the residual stream
    ct.block_normalize(out, None, None, r, None, 1.0, None, (w, None), 1e-5, kind="layer")
    for change in [dict(residual=None), dict(output=None), dict(before=None), dict(total=None), dict(epsilon=0.0), dict(kind="group"),
                   dict(gate=_t([4, 4])), dict(gate=_t([3, 5])), dict(gate=_t([0, 4])), dict(block=_t([5, 4])), dict(after=(_t([5]), None)),
                   dict(before=(_t([4], "float"), None)), dict(block=None), dict(output=_t([4, 6])),
                   dict(output=ct.transpose(_t([4, 6]), [1, 0]))]:
        with pytest.raises(ct.TensorError):
            ct.block_normalize(**{**ok, **change})
    ok = dict(block_gradient=_t([6, 4]), residual_gradient=_t([6, 4]), gate_gradient=_t([3, 4]), after_gradients=(_t([4]), None),
              before_gradients=(_t([4]), _t([4])), output_gradient=out, total_gradient=tot, total=r, block=x, gate=gate,
              residual_scale=1.0, after=(w, None), before=(w, w), epsilon=1e-5)
    ct.block_normalize_gradients(**ok)
    for change in [dict(residual_gradient=None), dict(block_gradient=None), dict(block=None), dict(output_gradient=None), dict(total=None),
                   dict(gate=None), dict(gate_gradient=_t([1, 4])), dict(after=None), dict(after_gradients=(w, None)),
                   dict(before_gradients=(_t([5]), None)), dict(total_gradient=_t([6, 5]))]:
        with pytest.raises(ct.TensorError):
            ct.block_normalize_gradients(**{**ok, **change})


def test_clip_refusals(bound):
    a, b = _t([6]), _t([2, 3])
    optimize.clip_gradients([a, b], 1.0)
    with pytest.raises(ct.TensorError):
        optimize.clip_gradients([], 1.0)
    for bound_ in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ct.TensorError):
            optimize.clip_gradients([a], bound_)
    with pytest.raises(ct.TensorError):
        optimize.clip_gradients([a, _t([3], "float")], 1.0)
    with pytest.raises(ct.TensorError):
        optimize.clip_gradients([ct.transpose(_t([2, 3]), [1, 0])], 1.0)
    with pytest.raises(ct.TensorError):
        optimize.clip_gradients([a], 1.0, clipped=[_t([5])])
    with pytest.raises(ct.TensorError):
        optimize.global_norm([a], norm=_t([2]))
    with pytest.raises(ct.TensorError):
        optimize.global_norm([_t([3], "int")])


def test_streams_of_another_device_are_refused(oracle_driver):
    """A stream's kernels cannot reach the memory of another device: the call is refused before it is launched."""
    from oracle.cpu_backend import OracleDriver
    other = OracleDriver().default_device().create_stream()
    with ct.with_stream(oracle_driver.default_device().create_stream()), ct.with_datatype("double"):
        x, w, y, off, v = _t([6, 4]), _t([3, 5, 4]), _t([6, 5]), _t([4], "int"), _t([4])
        a, b, c, d, norm = _t([6, 4]), _t([6, 4]), _t([6, 4]), _t([6, 4]), _t([1])
    calls = [lambda: ct.expert_gemm(y, True, 1.0, x, w, 0.0, off), lambda: ct.expert_gemm_weights(w, 1.0, y, x, 0.0, off),
             lambda: ct.block_normalize(a, b, c, x, None, 1.0, None, (v, None), 1e-5),
             lambda: ct.block_normalize_gradients(a, b, None, None, None, c, None, x, d, None, 1.0, None, (v, None), 1e-5),
             lambda: optimize.global_norm([x], norm=norm), lambda: optimize.clip_gradients([x], 1.0, norm=norm)]
    with ct.with_stream(oracle_driver.default_device().create_stream()), ct.with_datatype("double"):
        for call in calls:
            call()
    with ct.with_stream(other), ct.with_datatype("double"):
        for call in calls:
            with pytest.raises(ct.TensorError, match="another device"):
                call()


# ---- the C ABI refuses before it touches a device: a block of zeros stands in for the stream, and made-up addresses that
# ---- nothing reads for the buffers

P = 0x7000_0000_0000


def _refused(name, *args, match):
    lib = _lib.load()
    stream = C.create_string_buffer(4096)
    rc = getattr(lib, name)(C.addressof(stream), *args)
    assert rc == 1 and match in _lib.last_error(), (rc, _lib.last_error())


def test_c_abi_expert_refusals():
    def call(dtype=4, C_=P, ldc=8, A=P + 4096, rows=4, k=8, lda=8, B=P + 8192, e=2, n=8, bs=64, ldb=8, off=P + 16384, act=0):
        return ("cb200_expert_gemm", dtype, C_, ldc, 1, 1.0, A, rows, k, lda, B, e, n, bs, ldb, 0.0, off, None, act)

    for kw, text in [(dict(C_=None), "null"), (dict(off=None), "null"), (dict(dtype=2), "float and double"), (dict(e=0), "experts"),
                     (dict(e=5000), "experts"), (dict(rows=-1), "row count"), (dict(k=0), "extents"), (dict(ldc=7), "pitch"),
                     (dict(lda=7), "pitch"), (dict(ldb=7), "pitch"), (dict(bs=63), "overlap"), (dict(act=4), "activation"),
                     (dict(act=-1), "activation"), (dict(A=P + 4098), "aligned"), (dict(off=P + 2), "aligned"),
                     (dict(dtype=5, A=P + 4100), "aligned")]:
        c = call(**kw)
        _refused(c[0], *c[1:], match=text)

    def weights(c_stride=64, ldc=8, lda=8, ldb=8, m=8, n=8, e=2):
        return ("cb200_expert_gemm_weights", 4, P, c_stride, ldc, 1.0, P + 4096, 4, m, lda, P + 8192, n, ldb, e, 0.0, P + 16384, None)

    for kw, text in [(dict(c_stride=63), "overlap"), (dict(ldc=7), "pitch"), (dict(lda=7), "pitch"), (dict(ldb=7), "pitch"),
                     (dict(m=0), "extents"), (dict(e=0), "experts")]:
        c = weights(**kw)
        _refused(c[0], *c[1:], match=text)


@pytest.mark.parametrize("extent", [2 ** 31 - 65535, 2 ** 31 - 1, 2 ** 31])
def test_c_abi_expert_extents_leave_room_for_the_kernels_indexes(extent):
    """Kernels step 32-bit indexes past the last row and column by a tile at most."""
    big = 2 ** 33
    _refused("cb200_expert_gemm", 4, P, big, 1, 1.0, P + 4096, 4, extent, big, P + 8192, 1, 8, 64, big, 0.0, P + 16384, None, 0, match="extents")
    _refused("cb200_expert_gemm", 4, P, big, 1, 1.0, P + 4096, 4, 8, big, P + 8192, 1, extent, 64, big, 0.0, P + 16384, None, 0, match="extents")
    _refused("cb200_expert_gemm", 4, P, big, 1, 1.0, P + 4096, extent, 8, big, P + 8192, 1, 8, 64, big, 0.0, P + 16384, None, 0, match="row count")
    for m, n in ((extent, 8), (8, extent)):
        _refused("cb200_expert_gemm_weights", 4, P, 64, big, 1.0, P + 4096, 4, m, big, P + 8192, n, big, 1, 0.0, P + 16384, None, match="extents")


def test_c_abi_block_refusals():
    M = [P + i * 65536 for i in range(12)]

    def desc(kind=0, eps=1e-5, rows=4, cols=8, gate_rows=2):
        return C.byref(_lib.BlockDesc(kind, eps, 1.0, rows, cols, gate_rows))

    def call(d=None, out=M[0], total=M[1], block=M[2], res=M[3], gate=M[4], aw=M[5], bw=M[6], ab=None, ld=8):
        return ("cb200_block_normalize", 4, out, ld, total, ld, block, ld, res, ld, gate, aw, ab, bw, None, d or desc())

    for kw, text in [(dict(d=desc(kind=2)), "unknown"), (dict(d=desc(eps=0.0)), "epsilon"), (dict(d=desc(eps=float("nan"))), "epsilon"),
                     (dict(d=desc(rows=-1)), "extents"), (dict(d=desc(cols=0)), "extents"), (dict(d=desc(gate_rows=3)), "gate rows"),
                     (dict(d=desc(gate_rows=0)), "gate rows"), (dict(res=None), "residual"), (dict(total=None), "total"),
                     (dict(block=None), "belong"), (dict(bw=None), "together"), (dict(aw=None, ab=M[7]), "bias without"), (dict(ld=7), "pitch"),
                     (dict(out=M[1]), "output and total"), (dict(total=M[3] + 32), "total and residual"),
                     (dict(out=M[2] + 4), "output and block"), (dict(out=M[4]), "gate"), (dict(res=M[3] + 2), "aligned")]:
        c = call(**kw)
        _refused(c[0], *c[1:], match=text)

    def grads(d=None, bg=M[0], rg=M[1], gg=M[2], dy=M[3], dt=M[4], total=M[5], block=M[6], gate=M[7], aw=M[8], bw=M[9], ab_g=None):
        return ("cb200_block_normalize_gradients", 4, bg, 8, rg, 8, gg, None, ab_g, None, None, dy, 8, dt, 8, total, 8, block, 8, gate,
                aw, None, bw, d or desc())

    for kw, text in [(dict(rg=None), "residual_gradient"), (dict(dy=None, dt=None, bw=None), "arrives"), (dict(dy=None), "together"),
                     (dict(total=None), "total"), (dict(block=None), "together"), (dict(gate=None), "not there"),
                     (dict(aw=None, ab_g=M[10]), "not there"), (dict(bg=M[6]), "operand"), (dict(rg=M[5]), "operand"),
                     (dict(bg=M[4]), "operand"), (dict(rg=M[4] + 32), "operand"), (dict(bg=M[1]), "residual_gradient"),
                     (dict(gg=M[7]), "gate"), (dict(gg=M[3]), "gate_gradient"), (dict(gg=M[0] + 32), "gate_gradient")]:
        c = grads(**kw)
        _refused(c[0], *c[1:], match=text)


M12 = [P + i * 65536 for i in range(14)]


def _block_call(out=M12[0], total=M12[1], block=M12[2], res=M12[3], gate=M12[4], aw=M12[5], ab=M12[6], bw=M12[7], bb=M12[8], ld=8, eps=1e-5,
                dtype=4):
    return ("cb200_block_normalize", dtype, out, ld, total, ld, block, ld, res, ld, gate, aw, ab, bw, bb,
            C.byref(_lib.BlockDesc(0, eps, 1.0, 4, 8, 2)))


def _block_gradient_call(bg=M12[0], rg=M12[1], gg=M12[2], gaw=M12[3], gab=M12[4], gbw=M12[5], gbb=M12[6], dy=M12[7], dt=M12[8], total=M12[9],
                         block=M12[10], gate=M12[11], aw=M12[12], ab=M12[13], bw=M12[13] + 4096, ld=8, eps=1e-5, dtype=4):
    return ("cb200_block_normalize_gradients", dtype, bg, ld, rg, ld, gg, gaw, gab, gbw, gbb, dy, ld, dt, ld, total, ld, block, ld, gate,
            aw, ab, bw, C.byref(_lib.BlockDesc(0, eps, 1.0, 4, 8, 2)))


def test_c_abi_block_results_over_scales_and_biases():
    """No result is written over a scale, a bias or (of the gradients' vectors) anything else."""
    for name in ("aw", "ab", "bw", "bb"):
        for result, text in ((M12[0], "output overlaps"), (M12[1], "total overlaps")):
            for at in (result, result + 3 * 32 + 28, result - 28, result + 40):
                c = _block_call(**{name: at})
                _refused(c[0], *c[1:], match=text)
    for name in ("aw", "ab", "bw"):
        for result, text in ((M12[0], "block_gradient overlaps"), (M12[1], "residual_gradient overlaps"), (M12[2], "gate_gradient overlaps")):
            c = _block_gradient_call(**{name: result + 36})
            _refused(c[0], *c[1:], match=text)
    everything = [M12[0], M12[1], M12[2], M12[7], M12[8], M12[9], M12[10], M12[11], M12[12], M12[13], M12[13] + 4096]
    for i, name in enumerate(("gaw", "gab", "gbw", "gbb")):
        for other in everything + [M12[3 + j] for j in range(4) if j != i]:
            c = _block_gradient_call(**{name: other + 20})
            _refused(c[0], *c[1:], match="overlaps")
    # a vector in the gap between a matrix's rows shares nothing with it: the next check refuses (a misfit of another kind)
    c = _block_call(aw=M12[0] + 32, ld=16, out=M12[0], total=M12[0] + 4)
    _refused(c[0], *c[1:], match="output and total")
    c = _block_call(aw=M12[0] + 32, ab=M12[0] + 96, bw=M12[0] + 160, bb=M12[1] + 24, ld=16)
    _refused(c[0], *c[1:], match="total overlaps a bias")


@pytest.mark.parametrize("call", [_block_call, _block_gradient_call])
def test_c_abi_block_epsilon_of_the_element_type(call):
    """An epsilon that is 0 or infinite as a float: a row of zeros would become NaN."""
    for eps, dtype in [(1e-46, 4), (1e39, 4), (float("inf"), 5), (0.0, 5)]:
        c = call(eps=eps, dtype=dtype, ld=7)
        _refused(c[0], *c[1:], match="epsilon")
    for eps, dtype in [(1e-44, 4), (1e-300, 5)]:                       # these are fine: the next check refuses
        c = call(eps=eps, dtype=dtype, ld=7)
        _refused(c[0], *c[1:], match="pitch")


def test_c_abi_vectors_off_their_element_type():
    """Gates, scales, biases and their gradients are loaded as elements: an address between two would fault on the device."""
    for name in ("gate", "aw", "ab", "bw", "bb"):
        for dtype, by in ((4, 2), (5, 4)):
            c = _block_call(**{name: M12[4] + 1024 + by}, dtype=dtype)
            _refused(c[0], *c[1:], match="aligned")
    for name in ("gg", "gaw", "gab", "gbw", "gbb", "gate", "aw", "ab", "bw"):
        for dtype, by in ((4, 2), (5, 4)):
            c = _block_gradient_call(**{name: M12[2] + 1024 + by}, dtype=dtype)
            _refused(c[0], *c[1:], match="aligned")
    for dtype, by in ((4, 2), (5, 4)):
        _refused("cb200_expert_gemm", dtype, P, 8, 1, 1.0, P + 4096, 4, 8, 8, P + 8192, 2, 8, 64, 8, 0.0, P + 16384, P + 32768 + by, 0, match="aligned")
        _refused("cb200_expert_gemm_weights", dtype, P, 64, 8, 1.0, P + 4096, 4, 8, 8, P + 8192, 8, 8, 2, 0.0, P + 16384, P + 32768 + by, match="aligned")


def test_c_abi_clip_refusals():
    def lists(g, n, out):
        return (C.c_void_p * len(g))(*g), (C.c_int64 * len(n))(*n), (C.c_void_p * len(out))(*out)

    def clip(g, n, out, bound=1.0, norm=None, dtype=4, count=None):
        a, b, c = lists(g, n, out)
        return ("cb200_clip_gradients", dtype, len(g) if count is None else count, a, b, c, bound, norm)

    A, B = P, P + 4096
    for args, text in [(clip([A], [8], [A], bound=0.0), "bound"), (clip([A], [8], [A], bound=float("inf")), "bound"),
                       (clip([A], [8], [A], dtype=3), "float and double"), (clip([A], [-1], [A]), "negative"),
                       (clip([0], [8], [A]), "null"), (clip([A], [8], [0]), "null"), (clip([A + 2], [8], [A]), "aligned"),
                       (clip([A], [8], [A + 2]), "aligned"), (clip([A], [8], [A], count=-1), "outside"),
                       (clip([A, A], [8, 8], [A, A]), "overlap"),                       # one gradient twice, in place
                       (clip([A, B], [8, 8], [B, A]), "another gradient"), (clip([A], [8], [A + 4]), "another gradient"),
                       (clip([A, B], [8, 8], [A, A + 16]), "overlap"), (clip([A], [8], [B], norm=B + 4), "norm"),
                       (clip([A], [8], [B], norm=A + 4), "norm"), (clip([A], [8], [B], norm=P + 8194), "aligned")]:
        _refused(args[0], *args[1:], match=text)


# ---- the layers together -------------------------------------------------------------------------------------------

def expert_block_step(rng_seed, datatype, rows=14, routed=12, d=6, hidden=10, experts=3, steps=2, max_norm=0.05):
    """A residual block of experts, trained: normalise, two expert layers, normalise + gate + add + normalise, a linear
    loss on both outputs; gradients of everything, clipped together, Adam.  Returns named arrays of the last step."""
    rng = np.random.default_rng(rng_seed)
    np_type = {"float": np.float32, "double": np.float64}[datatype]
    draw = lambda *s, scale=1.0: ct.to_tensor((rng.standard_normal(s) * scale).astype(np_type), datatype)
    new = lambda *s: ct.new_tensor(list(s), datatype=datatype)
    sizes = rng.multinomial(routed, np.ones(experts) / experts)
    offsets = ct.to_tensor(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32), "int")
    x, c_total, c_out = draw(rows, d), draw(rows, d, scale=0.1), draw(rows, d, scale=0.1)
    up = nn.ExpertLinear(draw(experts, hidden, d, scale=0.5), draw(experts, hidden, scale=0.1))
    down = nn.ExpertLinear(draw(experts, d, hidden, scale=0.5), draw(experts, d, scale=0.1))
    first = nn.ResidualNormalization(before=(draw(d), draw(d)), kind="layer")
    step = nn.ResidualNormalization(after=(draw(d), None), before=(draw(d), draw(d)), gate=draw(1, d), residual_scale=0.5)
    parameters = [up.weights, up.bias, down.weights, down.bias, *first.before, step.after[0], *step.before, step.gate]
    adam = optimize.Adam(alpha=0.01)
    total_n = sum(p.ecount() for p in parameters)
    state = {"m": new(total_n), "v": new(total_n)}
    out = {}
    for _ in range(steps):
        gradients = [new(*p.shape()) for p in parameters]
        gu, gub, gd, gdb, g1, g1b, ga, g2, g2b, gg = gradients
        n1, h, y, total, n2 = new(rows, d), new(rows, hidden), new(rows, d), new(rows, d), new(rows, d)
        first.forward(None, x, None, n1)
        up.forward(n1, h, offsets, act="relu")
        down.forward(h, y, offsets)
        step.forward(y, x, total, n2)
        dy, dx, dh, dh_act, dn1, dx1 = new(rows, d), new(rows, d), new(rows, hidden), new(rows, hidden), new(rows, d), new(rows, d)
        step.backward(y, total, c_out, c_total, dy, dx, gg, (ga, None), (g2, g2b))
        down.backward(h, dh, dy, gd, gdb, offsets)
        ct.activation_gradient(dh_act, dh, h, "relu")
        up.backward(n1, dn1, dh_act, gu, gub, offsets)
        first.backward(None, x, dn1, dx, None, dx1, before_gradients=(g1, g1b))
        out = {"total": ct.to_array(total), "out": ct.to_array(n2), "dx": ct.to_array(dx1)}
        out.update({"g%d" % i: ct.to_array(g) for i, g in enumerate(gradients)})
        out["norm"] = ct.to_array(optimize.clip_gradients(gradients, max_norm))
        out.update({"c%d" % i: ct.to_array(g) for i, g in enumerate(gradients)})
        adam = adam.batch_update()
        at = 0
        for p, g in zip(parameters, gradients):
            adam.compute_parameters(state, 1.0, at, g, p)
            at += p.ecount()
        out.update({"p%d" % i: ct.to_array(p) for i, p in enumerate(parameters)})
    return out


def test_expert_block_step_on_the_oracle(oracle_driver):
    with ct.with_stream(oracle_driver.default_device().create_stream()), ct.with_datatype("double"):
        got = expert_block_step(3, "double")
    flat = np.concatenate([got["g%d" % i] for i in range(10)])
    assert np.isclose(got["norm"][0], np.linalg.norm(flat))
    clipped = np.concatenate([got["c%d" % i] for i in range(10)])
    assert np.isclose(np.linalg.norm(clipped), 0.05) and np.allclose(clipped * np.linalg.norm(flat), flat * 0.05)
