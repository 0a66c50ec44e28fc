"""The operators that carry the training and serving of expert layers, measured against their plain forms.

Three families, used next to one another in one residual block (normalise, run the experts, normalise, gate, add; then
the gradients, their norm and the optimiser's step):

  experts   a product per expert over ragged groups of rows: forward (bias and activation joined), gradient of the
            input, gradients of weights and bias
  block     normalisation after a block, its gate, the residual scale and add, and the normalisation before the next
            block, in one call; and the gradients of all of it
  clip      the global norm over many gradient tensors and the clipped gradients

``own`` selects what run() computes with: the plain form in elementary torch operations, or the framework's calls.
"""
import math

import numpy as np
import torch

own = False


# ---- cases -----------------------------------------------------------------------------------------------------

def listed():
    return [
        # serving one token: its row goes to two of the experts, and the call is as long as reading their weights
        {"name": "experts forward, one token", "op": "experts", "way": "forward", "dtype": "float", "experts": 8,
         "rows": 2, "routed": 2, "n_out": 4096, "n_in": 1024, "act": "relu"},
        # a layer of the size of an MNIST classifier's, four experts: launch latency and ragged tiles
        {"name": "experts forward, small", "op": "experts", "way": "forward", "dtype": "float", "experts": 4,
         "rows": 128, "routed": 121, "n_out": 500, "n_in": 784, "act": "relu"},
        # rows that no 16-byte load can address: 333 inputs, 1001 outputs, in double
        {"name": "experts forward, odd double", "op": "experts", "way": "forward", "dtype": "double", "experts": 7,
         "rows": 1000, "routed": 1000, "n_out": 1001, "n_in": 333, "act": "tanh"},
        # a training batch over many experts of ordinary width, padded at its end
        {"name": "experts forward, batch", "op": "experts", "way": "forward", "dtype": "float", "experts": 32,
         "rows": 8192, "routed": 8000, "n_out": 2048, "n_in": 1024, "act": "relu"},
        # the widest layer: the cost is the product itself
        {"name": "experts forward, wide", "op": "experts", "way": "forward", "dtype": "float", "experts": 8,
         "rows": 16384, "routed": 16384, "n_out": 4096, "n_in": 4096, "act": "none"},
        # the two gradients of the training batch
        {"name": "experts input gradient", "op": "experts", "way": "input", "dtype": "float", "experts": 32,
         "rows": 8192, "routed": 8000, "n_out": 2048, "n_in": 1024, "act": "none"},
        {"name": "experts weight gradient", "op": "experts", "way": "weights", "dtype": "float", "experts": 32,
         "rows": 8192, "routed": 8000, "n_out": 2048, "n_in": 1024, "act": "none"},
        # the block around a single token: nothing but latency
        {"name": "block forward, one token", "op": "block", "way": "forward", "dtype": "float", "kind": "rms", "rows": 1,
         "width": 4096, "gate": "channel", "after": True, "bias": False},
        # the block over a whole training batch
        {"name": "block forward, batch", "op": "block", "way": "forward", "dtype": "float", "kind": "rms", "rows": 16384,
         "width": 4096, "gate": "channel", "after": True, "bias": False},
        # its gradients, with biases, a gate row for each of several samples, and a width that is not a power of two
        {"name": "block gradients", "op": "block", "way": "gradients", "dtype": "float", "kind": "layer", "rows": 8192,
         "width": 2500, "gate": "sample", "after": True, "bias": True},
        # the parameters of a small classifier: latency
        {"name": "clip, small network", "op": "clip", "dtype": "float", "tensors": 4, "total": 397510, "seed": 1,
         "bound": 0.5},
        # the parameters of a large network, in buffers of very different lengths
        {"name": "clip, large network", "op": "clip", "dtype": "float", "tensors": 160, "total": 1 << 28, "seed": 2,
         "bound": 0.25},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["experts", "experts", "block", "clip"])
    dtype = rng.choice(["float", "float", "float", "double"])
    if op == "experts":
        way = rng.choice(["forward", "input", "weights"])
        experts = _log(rng, 1, 64)
        n_out, n_in = _log(rng, 16, 4096), _log(rng, 16, 4096)
        if rng.random() < 0.6:      # most layers have widths that are multiples of 4
            n_out, n_in = (n_out + 3) // 4 * 4, (n_in + 3) // 4 * 4
        while experts * n_out * n_in > 1 << 27:
            experts = max(1, experts // 2)
        rows = _log(rng, 1, 16384)
        top = 5.4e11 if dtype == "float" else 1e11
        while 2.0 * rows * n_out * n_in > top:
            rows //= 2
        routed = max(1, rows - rng.choice([0, 0, rows // 16, rows // 3]))
        return {"op": op, "way": way, "dtype": dtype, "experts": experts, "rows": rows, "routed": routed, "n_out": n_out,
                "n_in": n_in, "act": rng.choice(["none", "relu", "tanh", "logistic"]) if way == "forward" else "none"}
    if op == "block":
        width = _log(rng, 32, 8192)
        if rng.random() < 0.6:
            width = (width + 3) // 4 * 4
        rows = _log(rng, 1, 16384)
        while rows * width > (1 << 26 if dtype == "float" else 1 << 25):
            rows //= 2
        rows = max(1, rows)
        gate = rng.choice(["none", "channel", "sample", "row"])
        return {"op": op, "way": rng.choice(["forward", "gradients"]), "dtype": dtype, "kind": rng.choice(["rms", "layer"]),
                "rows": rows, "width": width, "gate": gate, "after": rng.random() < 0.7, "bias": rng.random() < 0.5}
    total = _log(rng, 1000, 1 << (28 if dtype == "float" else 27))
    return {"op": op, "dtype": dtype, "tensors": min(_log(rng, 1, 400), total // 8), "total": total,
            "seed": rng.randrange(1 << 20), "bound": rng.choice([1e-3, 0.1, 0.25, 0.9, 2.0])}


# ---- inputs ----------------------------------------------------------------------------------------------------

_TYPE = {"float": torch.float32, "double": torch.float64}
EPSILON = 1e-5
RESIDUAL_SCALE = 0.7


def _group_sizes(experts, routed, seed):
    """Uneven groups as a router makes them, some of them empty."""
    rng = np.random.default_rng(seed + 77)
    share = rng.exponential(size=experts)
    if experts > 4:
        share[rng.random(experts) < 0.1] = 0.0
    share = share + 1e-9
    return rng.multinomial(routed, share / share.sum()).tolist()


def _piece_lengths(case):
    """Buffers of very different lengths that add up to the total; fixed by the case, as a network's are."""
    rng = np.random.default_rng(case["seed"])
    n, total = case["tensors"], case["total"]
    share = np.exp(rng.uniform(0.0, 7.0, size=n))
    lengths = np.maximum(1, (share / share.sum() * (total - n)).astype(np.int64))
    lengths[int(np.argmax(lengths))] += total - int(lengths.sum())
    return lengths.tolist()


def _gate_rows(case):
    """Rows of the gate tensor; each serves rows / gate rows consecutive rows of the batch."""
    if case["gate"] == "none":
        return 0
    if case["gate"] == "channel":
        return 1
    if case["gate"] == "row":
        return case["rows"]
    return max(g for g in (16, 8, 7, 5, 4, 3, 2, 1) if case["rows"] % g == 0)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    t = _TYPE[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=t).mul_(scale)

    s = {"case": case}
    if case["op"] == "experts":
        e, rows, n, k = case["experts"], case["rows"], case["n_out"], case["n_in"]
        s["sizes"] = _group_sizes(e, case["routed"], int(seed))
        s["offsets"] = torch.tensor(np.concatenate([[0], np.cumsum(s["sizes"])]), dtype=torch.int32, device="cuda")
        if case["way"] != "input":
            s["x"] = normal(rows, k)
        if case["way"] != "forward":
            s["dy"] = normal(rows, n, scale=0.02)
        if case["way"] != "weights":
            s["w"] = normal(e, n, k, scale=math.sqrt(2.0 / k))
        if case["way"] == "forward":
            s["b"] = normal(e, n, scale=0.1)
            s["out"] = torch.full((rows, n), 0.25, device="cuda", dtype=t)
        elif case["way"] == "input":
            s["out"] = torch.full((rows, k), 0.25, device="cuda", dtype=t)
        else:
            s["out"] = torch.empty(e, n, k, device="cuda", dtype=t)
            s["out_b"] = torch.empty(e, n, device="cuda", dtype=t)
    elif case["op"] == "block":
        rows, d = case["rows"], case["width"]
        s["block"], s["gate"] = normal(rows, d, scale=2.0).add_(0.3), None
        s["residual"] = normal(rows, d)
        if case["gate"] != "none":
            s["gate"] = normal(_gate_rows(case), d, scale=0.5)
        for name in ("after", "before"):
            on = name == "before" or case["after"]
            s[name] = normal(d, scale=0.2).add_(1.0) if on else None
            s[name + "_b"] = normal(d, scale=0.2) if on and case["bias"] else None
        s["total"], s["out"] = torch.empty(rows, d, device="cuda", dtype=t), torch.empty(rows, d, device="cuda", dtype=t)
        if case["way"] == "gradients":
            s["total"] = normal(rows, d, scale=1.5).add_(0.1)      # the forward call's sum, kept for this pass
            s["d_out"], s["d_total"] = normal(rows, d, scale=0.02), normal(rows, d, scale=0.02)
            s["residual_grad"] = torch.empty(rows, d, device="cuda", dtype=t)
            for name in ("gate", "after", "after_b", "before", "before_b"):
                s[name + "_grad"] = torch.empty_like(s[name]) if s[name] is not None else None
    else:
        lengths = _piece_lengths(case)
        flat = normal(case["total"], scale=1.0)
        scales = torch.tensor(np.random.default_rng(int(seed)).uniform(0.1, 2.0, len(lengths)), device="cuda", dtype=t)
        s["flat"] = flat.mul_(torch.repeat_interleave(scales, torch.tensor(lengths, device="cuda"), output_size=case["total"]))
        s["gradients"] = list(torch.split(s["flat"], lengths))
        s["clipped_flat"] = torch.empty_like(flat)
        s["clipped"] = list(torch.split(s["clipped_flat"], lengths))
        s["norm"] = torch.empty(1, device="cuda", dtype=t)
        s["max_norm"] = case["bound"] * math.sqrt(case["total"])
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------

_ACT = {"none": lambda v: v, "relu": lambda v: v.clamp_min(0), "tanh": torch.tanh, "logistic": torch.sigmoid}


def _experts_plain(s):
    case, sizes = s["case"], s["sizes"]
    rest = case["rows"] - case["routed"]
    if case["way"] == "forward":
        act = _ACT[case["act"]]
        parts = [act(x @ w.T + b) for x, w, b in zip(s["x"].split(sizes + [rest]), s["w"], s["b"])]
        return torch.cat(parts + [s["out"][case["routed"]:]])
    if case["way"] == "input":
        parts = [dy @ w for dy, w in zip(s["dy"].split(sizes + [rest]), s["w"])]
        return torch.cat(parts + [s["out"][case["routed"]:]])
    pairs = list(zip(s["dy"].split(sizes + [rest]), s["x"].split(sizes + [rest])))[:-1]
    return torch.stack([dy.T @ x for dy, x in pairs]), torch.stack([dy.sum(0) for dy, _ in pairs])


def _normed(x, kind):
    c = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    r = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + EPSILON)
    return c * r, r


def _affine(x, w, b):
    y = x * w
    return y if b is None else y + b


def _normed_gradient(d, w, hat, r, kind):
    d = d * w
    g = d - hat * (d * hat).mean(-1, keepdim=True)
    if kind == "layer":
        g = g - d.mean(-1, keepdim=True)
    return g * r


def _rows_of(gate, rows):
    return gate.repeat_interleave(rows // gate.shape[0], 0) if gate.shape[0] > 1 else gate


def _block_plain(s):
    case, kind = s["case"], s["case"]["kind"]
    hat_a, r_a = _normed(s["block"], kind) if case["after"] else (s["block"], None)
    u = _affine(hat_a, s["after"], s["after_b"]) if case["after"] else s["block"]
    gate = _rows_of(s["gate"], case["rows"]) if s["gate"] is not None else None
    if case["way"] == "forward":
        total = s["residual"] + RESIDUAL_SCALE * (u if gate is None else gate * u)
        hat, _ = _normed(total, kind)
        return total, _affine(hat, s["before"], s["before_b"])
    hat, r = _normed(s["total"], kind)
    out = {"before": (s["d_out"] * hat).sum(0)}
    if case["bias"]:
        out["before_b"] = s["d_out"].sum(0)
    d_total = s["d_total"] + _normed_gradient(s["d_out"], s["before"], hat, r, kind)
    out["residual"] = d_total
    du = RESIDUAL_SCALE * d_total
    if gate is not None:
        out["gate"] = (du * u).reshape(s["gate"].shape[0], -1, case["width"]).sum(1)
        du = du * gate
    if case["after"]:
        out["after"] = (du * hat_a).sum(0)
        if case["bias"]:
            out["after_b"] = du.sum(0)
        du = _normed_gradient(du, s["after"], hat_a, r_a, kind)
    out["block"] = du
    return out


def _clip_plain(s):
    # the sum over all elements is a long one: 64 bits
    norm = torch.sqrt(torch.stack([(g.double() * g.double()).sum() for g in s["gradients"]]).sum())
    scale = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm)).to(s["flat"].dtype)
    return torch.cat([g * scale for g in s["gradients"]]), norm.to(s["flat"].dtype).reshape(1)


# ---- the framework's calls -------------------------------------------------------------------------------------

_framework = {}


def _stream():
    if "stream" not in _framework:
        from cortex_b200.driver import driver
        device = driver().default_device()
        _framework.update(device=device, stream=device.create_stream())
    return _framework["stream"]


def _tensor(x):
    """A framework tensor on the memory of a torch tensor."""
    from cortex_b200 import dimensions, tensor
    from cortex_b200.driver import Buffer
    if x is None:
        return None
    names = {torch.float32: "float", torch.float64: "double", torch.int32: "int"}
    buffer = Buffer(x.data_ptr(), names[x.dtype], x.numel(), _framework["device"], owner=x)
    return tensor.Tensor(_framework["device"], dimensions.dimensions(list(x.shape)), buffer)


def _handles(s):
    """The framework's descriptors of the state's buffers: what a program that uses it holds anyway."""
    if "handles" not in s:
        s["handles"] = {k: _tensor(v) if isinstance(v, torch.Tensor) else [_tensor(x) for x in v]
                        for k, v in s.items() if isinstance(v, torch.Tensor) or k in ("gradients", "clipped")}
    return s["handles"]


def _own(s):
    from cortex_b200 import optimize
    from cortex_b200 import tensor as ct
    case = s["case"]
    with ct.with_stream(_stream()):
        h = _handles(s)
        get = h.get
        if case["op"] == "experts":
            if case["way"] == "forward":
                ct.expert_gemm(h["out"], True, 1.0, h["x"], h["w"], 0.0, h["offsets"], bias=h["b"], act=case["act"])
                return s["out"]
            if case["way"] == "input":
                ct.expert_gemm(h["out"], False, 1.0, h["dy"], h["w"], 0.0, h["offsets"])
                return s["out"]
            ct.expert_gemm_weights(h["out"], 1.0, h["dy"], h["x"], 0.0, h["offsets"], bias_gradient=h["out_b"])
            return s["out"], s["out_b"]
        if case["op"] == "block":
            after = (h["after"], get("after_b")) if case["after"] else None
            before = (h["before"], get("before_b"))
            if case["way"] == "forward":
                ct.block_normalize(h["out"], h["total"], h["block"], h["residual"], get("gate"), RESIDUAL_SCALE, after,
                                   before, EPSILON, kind=case["kind"])
                return s["total"], s["out"]
            ct.block_normalize_gradients(
                h["out"], h["residual_grad"], get("gate_grad"),
                (h["after_grad"], get("after_b_grad")) if case["after"] else None, (h["before_grad"], get("before_b_grad")),
                h["d_out"], h["d_total"], h["total"], h["block"], get("gate"), RESIDUAL_SCALE, after, before, EPSILON,
                kind=case["kind"])
            out = {"block": s["out"], "residual": s["residual_grad"], "gate": s["gate_grad"], "after": s["after_grad"],
                   "after_b": s["after_b_grad"], "before": s["before_grad"], "before_b": s["before_b_grad"]} \
                if "gate_grad" in s else {}
            return {k: v for k, v in out.items() if v is not None}
        optimize.clip_gradients(h["gradients"], s["max_norm"], clipped=h["clipped"], norm=h["norm"])
        return s["clipped_flat"], s["norm"]


def run(state):
    if own:
        return _own(state)
    return {"experts": _experts_plain, "block": _block_plain, "clip": _clip_plain}[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "float" else 8
    if case["op"] == "experts":
        e, rows, n, k = case["experts"], case["routed"], case["n_out"], case["n_in"]
        used = min(e, rows)        # experts without rows are not read; their gradients are still written
        weights = e * n * k if case["way"] == "weights" else used * n * k
        return {"bytes": size * (rows * (n + k) + weights + (used * n if case["way"] == "forward" else 0)),
                "flops": 2 * rows * n * k}
    if case["op"] == "block":
        cells = case["rows"] * case["width"]
        gate = _gate_rows(case) * case["width"]
        if case["way"] == "forward":
            return {"bytes": size * (4 * cells + gate), "flops": 12 * cells}
        return {"bytes": size * (6 * cells + 2 * gate), "flops": 30 * cells}
    return {"bytes": 2 * size * case["total"], "flops": 3 * case["total"]}


# ---- the definitions, in 64 bits -------------------------------------------------------------------------------

def _exact_norm(x, kind):
    m = x.sum(-1, keepdim=True) / x.shape[-1] if kind == "layer" else 0.0
    v = ((x - m) ** 2).sum(-1, keepdim=True) / x.shape[-1]
    return (x - m) / (v + EPSILON) ** 0.5, (v + EPSILON) ** -0.5


def _exact_norm_vjp(hat, inv, d, kind):
    """Product of d with the Jacobian of the normalisation: (I - hat hat^T / D [- 1 1^T / D]) / std."""
    width = hat.shape[-1]
    out = d - hat * torch.einsum("rc,rc->r", hat, d)[:, None] / width
    if kind == "layer":
        out = out - torch.einsum("rc->r", d)[:, None] / width
    return out * inv


def exact(case, seed):
    s = prepare(case, seed)
    f = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "experts":
        bounds = np.concatenate([[0], np.cumsum(s["sizes"])]).tolist()
        if case["way"] == "weights":
            dw, db = torch.zeros_like(f["out"]), torch.zeros_like(f["out_b"])
            for e, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
                dw[e] = torch.einsum("rn,rk->nk", f["dy"][lo:hi], f["x"][lo:hi])
                db[e] = torch.einsum("rn->n", f["dy"][lo:hi])
            return dw, db
        y = f["out"].clone()
        for e, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
            if case["way"] == "input":
                y[lo:hi] = torch.einsum("rn,nk->rk", f["dy"][lo:hi], f["w"][e])
                continue
            v = torch.einsum("rk,nk->rn", f["x"][lo:hi], f["w"][e]) + f["b"][e]
            if case["act"] == "relu":
                v = torch.where(v > 0, v, torch.zeros_like(v))
            elif case["act"] == "tanh":
                v = 1.0 - 2.0 / (torch.exp(2.0 * v) + 1.0)
            elif case["act"] == "logistic":
                v = 1.0 / (1.0 + torch.exp(-v))
            y[lo:hi] = v
        return y
    if case["op"] == "block":
        rows, d, kind = case["rows"], case["width"], case["kind"]
        zero, one = torch.zeros(d, device="cuda", dtype=torch.float64), torch.ones(d, device="cuda", dtype=torch.float64)
        if case["gate"] == "none":
            gate = one.expand(rows, d)
        else:
            per = rows // f["gate"].shape[0]
            gate = f["gate"][torch.arange(rows, device="cuda") // per]
        u, hat_a, inv_a = f["block"], None, None
        if case["after"]:
            hat_a, inv_a = _exact_norm(f["block"], kind)
            u = hat_a * f["after"] + f.get("after_b", zero)
        if case["way"] == "forward":
            total = f["residual"] + RESIDUAL_SCALE * gate * u
            return total, _exact_norm(total, kind)[0] * f["before"] + f.get("before_b", zero)
        hat, inv = _exact_norm(f["total"], kind)
        d_total = f["d_total"] + _exact_norm_vjp(hat, inv, f["d_out"] * f["before"], kind)
        du = RESIDUAL_SCALE * gate * d_total
        out = {"block": du, "residual": d_total, "before": torch.einsum("rc,rc->c", f["d_out"], hat)}
        if case["after"]:
            out["block"] = _exact_norm_vjp(hat_a, inv_a, du * f["after"], kind)
            out["after"] = torch.einsum("rc,rc->c", du, hat_a)
        if case["gate"] != "none":
            out["gate"] = torch.zeros_like(f["gate"]).index_add_(0, torch.arange(rows, device="cuda") // per,
                                                                 RESIDUAL_SCALE * d_total * u)
        if case["bias"]:
            out["before_b"] = torch.einsum("rc->c", f["d_out"])
            if case["after"]:
                out["after_b"] = torch.einsum("rc->c", du)
        return out
    flat = f["flat"]
    norm = torch.dot(flat, flat) ** 0.5
    return flat * min(1.0, s["max_norm"] / float(norm)), norm.reshape(1)
