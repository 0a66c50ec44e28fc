"""Plain numpy statements, in 64 bits, of the operators that have no counterpart in the reference: the products grouped by
expert, the normalisations around a residual block, the global gradient norm.  TEST INFRASTRUCTURE, like the rest of this
package.

Every function returns values and, where it says so, magnitudes: the same formula with every term replaced by its absolute
value, which is what rounding errors are relative to."""
import numpy as np


def activation(v, act):
    if act in (None, "none"):
        return v
    if act == "relu":
        return np.maximum(v, 0.0)
    if act == "tanh":
        return np.tanh(v)
    return 1.0 / (1.0 + np.exp(-v))


def groups(offsets, rows):
    """(first, end) of every group, clamped as the device does."""
    out, last = [], 0
    offs = [min(max(int(o), 0), rows) for o in offsets]
    for lo, hi in zip(offs[:-1], offs[1:]):
        lo = max(lo, last)
        hi = max(hi, lo)
        last = hi
        out.append((lo, hi))
    return out


def expert_gemm(C, trans_b, alpha, A, B, beta, offsets, bias=None, act=None):
    """New C and the magnitude before the activation (rows outside every group: C, 0)."""
    A, B = A.astype(np.float64), B.astype(np.float64)
    out, size = C.astype(np.float64).copy(), np.zeros(C.shape)
    for e, (lo, hi) in enumerate(groups(offsets, len(A))):
        if lo == hi:
            continue
        m = B[e].T if trans_b else B[e]
        v, a = alpha * (A[lo:hi] @ m), abs(alpha) * (np.abs(A[lo:hi]) @ np.abs(m))
        if beta != 0:
            v, a = v + beta * out[lo:hi], a + np.abs(beta * out[lo:hi])
        if bias is not None:
            v, a = v + bias[e].astype(np.float64), a + np.abs(bias[e].astype(np.float64))
        out[lo:hi], size[lo:hi] = activation(v, act), a
    return out, size


def expert_gemm_weights(C, alpha, A, B, beta, offsets, bias_gradient=None):
    """New C, its magnitude, new bias_gradient, its magnitude."""
    A, B = A.astype(np.float64), B.astype(np.float64)
    out = C.astype(np.float64) * beta if beta != 0 else np.zeros(C.shape)
    size = np.abs(out)
    bias = np.zeros(C.shape[:2]) if bias_gradient is None or beta == 0 else beta * bias_gradient.astype(np.float64)
    bias_size = np.abs(bias)
    for e, (lo, hi) in enumerate(groups(offsets, len(A))):
        out[e] += alpha * (A[lo:hi].T @ B[lo:hi])
        size[e] += abs(alpha) * (np.abs(A[lo:hi]).T @ np.abs(B[lo:hi]))
        bias[e] += alpha * A[lo:hi].sum(0)
        bias_size[e] += abs(alpha) * np.abs(A[lo:hi]).sum(0)
    return out, size, bias, bias_size


def normalized(x, kind, epsilon):
    """N(x), 1 / std, and what an error of N(x) is relative to (the row's mean enters every element)."""
    x = x.astype(np.float64)
    mean = x.mean(-1, keepdims=True) if kind == "layer" else 0.0
    rstd = 1.0 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + epsilon)
    size = np.abs(x) * rstd
    if kind == "layer":
        # the centred values carry an error relative to |x| and the mean's own terms, and so does their variance
        size = size + np.abs(x).mean(-1, keepdims=True) * rstd
        size = size * (1.0 + (x ** 2).mean(-1, keepdims=True) * rstd ** 2)
    return (x - mean) * rstd, rstd, size


def _gate(gate, rows):
    return 1.0 if gate is None else np.repeat(gate.astype(np.float64).reshape(-1, gate.shape[-1]), rows // (gate.size // gate.shape[-1]), 0)


def block_normalize(block, residual, gate, residual_scale, after, before, epsilon, kind):
    """total, its magnitude, output (None without before), its magnitude."""
    r = residual.astype(np.float64)
    total, size = r, np.abs(r)
    if block is not None:
        u, _, us = normalized(block, kind, epsilon) if after is not None else (block.astype(np.float64), None, np.abs(block.astype(np.float64)))
        if after is not None:
            w, b = after[0].astype(np.float64), 0.0 if after[1] is None else after[1].astype(np.float64)
            u, us = u * w + b, us * np.abs(w) + np.abs(b)
        g = _gate(gate, len(r))
        total, size = r + residual_scale * g * u, np.abs(r) + abs(residual_scale) * np.abs(g) * us
    if before is None:
        return total, size, None, None
    hat, rstd, hs = normalized(total, kind, epsilon)
    w, b = before[0].astype(np.float64), 0.0 if before[1] is None else before[1].astype(np.float64)
    # an error of the sum moves the row's statistics and the element itself
    hs = hs + size * rstd + np.abs(hat) * (size * np.abs(total)).mean(-1, keepdims=True) * rstd ** 2
    return total, size, hat * w + b, hs * np.abs(w) + np.abs(b)


def _vjp(x, d, ds, kind, epsilon):
    """N'(x, d) and its magnitude; ds is the magnitude of d."""
    hat, rstd, hs = normalized(x, kind, epsilon)
    dot = (d * hat).mean(-1, keepdims=True)
    dots = (ds * hs).mean(-1, keepdims=True)
    v, s = d - hat * dot, ds + hs * dots
    if kind == "layer":
        v, s = v - d.mean(-1, keepdims=True), s + ds.mean(-1, keepdims=True)
        s = s * (1.0 + (x.astype(np.float64) ** 2).mean(-1, keepdims=True) * rstd ** 2)
    return v * rstd, s * rstd, hat, hs


def block_normalize_gradients(output_gradient, total_gradient, total, block, gate, residual_scale, after, before, epsilon, kind):
    """{name: (value, magnitude)} of residual, block, gate, after, after_b, before, before_b (those that exist)."""
    out = {}
    some = output_gradient if output_gradient is not None else total_gradient
    rows = len(some)
    d = np.zeros(some.shape) if total_gradient is None else total_gradient.astype(np.float64)
    ds = np.abs(d)
    if before is not None:
        dy, w = output_gradient.astype(np.float64), before[0].astype(np.float64)
        v, s, hat, hs = _vjp(total, dy * w, np.abs(dy * w), kind, epsilon)
        d, ds = d + v, ds + s
        out["before"] = ((dy * hat).sum(0), (np.abs(dy) * hs).sum(0))
        out["before_b"] = (dy.sum(0), np.abs(dy).sum(0))
    out["residual"] = (d, ds)
    if block is None:
        return out
    x = block.astype(np.float64)
    u, us = x, np.abs(x)
    if after is not None:
        hat, _, hs = normalized(block, kind, epsilon)
        w, b = after[0].astype(np.float64), 0.0 if after[1] is None else after[1].astype(np.float64)
        u, us = hat * w + b, hs * np.abs(w) + np.abs(b)
    g = _gate(gate, rows)
    du, dus = residual_scale * d, abs(residual_scale) * ds
    if gate is not None:
        per = rows // (gate.size // gate.shape[-1])
        shape = (rows // per, per, x.shape[1])
        out["gate"] = ((du * u).reshape(shape).sum(1).reshape(gate.shape), (dus * us).reshape(shape).sum(1).reshape(gate.shape))
    du, dus = du * g, dus * np.abs(g)
    if after is not None:
        out["after"] = ((du * hat).sum(0), (dus * hs).sum(0))
        out["after_b"] = (du.sum(0), dus.sum(0))
        du, dus, _, _ = _vjp(block, du * w, dus * np.abs(w), kind, epsilon)
    out["block"] = (du, dus)
    return out


def global_norm(gradients):
    return float(np.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in gradients)))


def clip_scale(norm, max_norm):
    return max_norm / norm if np.isfinite(norm) and norm > max_norm else 1.0
