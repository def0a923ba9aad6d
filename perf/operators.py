"""Workloads of the feature-head operators: root-mean-square norm, linear layer with a fused epilogue, gated linear layer.

A head of this kind turns rows of any width (descriptors, network taps) into the rows that the fused kNN match takes.  Every case is
one call of one operator, forward only ("train" false) or forward and backward.  With `own` false `run` computes the operators from
elementary torch operations in 32 bits; with `own` true it calls the framework.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6


def listed():
    return [
        # --- rms_norm
        # one row on its way through a served head: latency
        {"name": "norm, one row", "op": "norm", "rows": 1, "d": 4096, "dtype": "bf16", "residual": True, "train": False, "fp8": False},
        # the style set of the style loop (65 536 rows of 256 features), one training step
        {"name": "norm, style rows, train", "op": "norm", "rows": 65536, "d": 256, "dtype": "bf16", "residual": True, "train": True, "fp8": False},
        # the content rows of the style loop (1M Gaussians of 256 features), on their way into the fp8 match
        {"name": "norm, scene rows, fp8", "op": "norm", "rows": 1000000, "d": 256, "dtype": "bf16", "residual": True, "train": False, "fp8": True},
        # --- linear
        # one row against a wide layer: the weights are read once, nothing else counts
        {"name": "linear, one row", "op": "linear", "rows": 1, "k": 4096, "n": 4096, "dtype": "bf16", "act": "silu", "bias": True, "residual": False, "train": False, "fp8": False},
        # the 512-wide taps of the feature network, in its own 32 bits
        {"name": "linear, 512-wide taps, f32, train", "op": "linear", "rows": 784, "k": 512, "n": 512, "dtype": "f32", "act": "relu", "bias": True, "residual": True, "train": True, "fp8": False},
        # the wide layer of a head in training
        {"name": "linear, wide, train", "op": "linear", "rows": 16384, "k": 1024, "n": 4096, "dtype": "bf16", "act": "gelu", "bias": True, "residual": False, "train": True, "fp8": False},
        # neighbour descriptors of an odd length, an odd number of points, onto an odd width
        {"name": "linear, odd sizes, f16, train", "op": "linear", "rows": 4999, "k": 999, "n": 515, "dtype": "f16", "act": "relu", "bias": True, "residual": True, "train": True, "fp8": False},
        # the second product of a block on 8-bit rows, added to the stream
        {"name": "linear, fp8 rows", "op": "linear", "rows": 16384, "k": 2048, "n": 2048, "dtype": "bf16", "act": "none", "bias": True, "residual": True, "train": False, "fp8": True},
        # --- gated_linear
        # a few rows of a served head
        {"name": "gated, four rows", "op": "gated", "rows": 4, "k": 1024, "n": 4096, "dtype": "bf16", "act": "silu", "bias": False, "train": False, "fp8": False},
        # the style set through a gated layer four times as wide
        {"name": "gated, style rows", "op": "gated", "rows": 65536, "k": 256, "n": 1024, "dtype": "f16", "act": "gelu", "bias": True, "train": False, "fp8": False},
        # one training step of a wide gated layer
        {"name": "gated, wide, train", "op": "gated", "rows": 16384, "k": 1024, "n": 2816, "dtype": "bf16", "act": "silu", "bias": False, "train": True, "fp8": False},
        # the largest: a long batch of 8-bit rows through a very wide layer
        {"name": "gated, fp8 rows", "op": "gated", "rows": 8192, "k": 4096, "n": 8192, "dtype": "bf16", "act": "silu", "bias": False, "train": False, "fp8": True},
    ]


def _spread(rng, lo, hi, step=1):
    """A whole number of [lo, hi], even over its logarithm; a multiple of `step` where that is over one."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, v // step * step or step))


def draw(rng):
    op = rng.choice(["norm", "linear", "gated"])
    fp8 = rng.random() < 0.25
    train = not fp8 and rng.random() < 0.5
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"]) if not fp8 else rng.choice(["bf16", "f16"])
    if op == "norm":
        d = _spread(rng, 8, 8192, 4 if fp8 else rng.choice([1, 8, 64]))
        rows = _spread(rng, 1, min(1000000, (1 << 27) // d))
        return {"op": "norm", "rows": rows, "d": d, "dtype": dtype, "residual": rng.random() < 0.5, "train": train, "fp8": fp8}
    step = rng.choice([1, 16, 64])
    k, n = _spread(rng, 16, 4096, step), _spread(rng, 16, 4096, step)
    most = (1 << 36) // (k * n) if dtype != "f32" else (1 << 34) // (k * n)
    rows = _spread(rng, 1, max(16, min(65536, most)), rng.choice([1, 1, 64]))
    case = {"op": op, "rows": rows, "k": k, "n": n, "dtype": dtype, "act": rng.choice(["relu", "gelu", "silu", "sigmoid", "none"]), "bias": rng.random() < 0.5}
    if op == "linear":
        case["residual"] = rng.random() < 0.5
    return {**case, "train": train, "fp8": fp8}


# ------------------------------------------------------------------------------------------------ inputs
def _to_fp8(v):
    """Rows as a user of the fp8 match holds them: e4m3 bytes and one E8M0 exponent a row, the smallest that keeps the row within 448."""
    top = v.abs().amax(1).double()
    e = torch.where(top > 0, torch.ceil(torch.log2(top.clamp_min(1e-300) / 448.0)), torch.zeros_like(top)).clamp(-126, 127)
    q = (v.double() * torch.exp2(-e)[:, None]).clamp(-448, 448).float().to(torch.float8_e4m3fn)
    return q.view(torch.uint8), (e + 127).to(torch.int32)


def _rows(shape, g, dtype):
    """Feature rows: normal values, the rows of different lengths."""
    v = torch.randn(shape, generator=g, device="cuda")
    return (v * torch.exp(0.5 * torch.randn(shape[0], 1, generator=g, device="cuda"))).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, R = DTYPES[case["dtype"]], case["rows"]
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    st = {"case": case}
    if case["op"] == "norm":
        d = case["d"]
        st["x"] = _rows((R, d), g, dt)
        st["w"] = (1.0 + 0.1 * normal(d)).to(dt)
        st["res"] = _rows((R, d), g, dt) if case["residual"] else None
        if case["train"]:
            st["dy"] = normal(R, d).to(dt)
            st["ds"] = normal(R, d).to(dt) if case["residual"] else None
        leaves = ("x", "w", "res")
    else:
        K, N = case["k"], case["n"]
        x = _rows((R, K), g, dt)
        names = ["w"] if case["op"] == "linear" else ["w", "v"]
        if case["fp8"]:
            st["x"], st["xs"] = _to_fp8(x)
            for i in names:
                st[i], st[i + "s"] = _to_fp8(normal(N, K) / math.sqrt(K))
        else:
            st["x"] = x
            for i in names:
                st[i] = (normal(N, K) / math.sqrt(K)).to(dt)
        for i in names:
            st["b" + i] = normal(N).to(dt) if case["bias"] else None
        st["res"] = _rows((R, N), g, dt) if case.get("residual") else None
        if case["train"]:
            st["dy"] = normal(R, N).to(dt)
        leaves = ("x", "w", "v", "bw", "bv", "res")
    if case["train"]:
        st["leaves"] = [i for i in leaves if st.get(i) is not None]
        for i in st["leaves"]:
            st[i].requires_grad_(True)
    return st


# ------------------------------------------------------------------------------------------------ the plain forms
def _act(z, name):
    """act(z) and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    sig = 1.0 / (1.0 + torch.exp(-z))
    if name == "silu":
        return z * sig, sig * (1.0 + z * (1.0 - sig))
    return sig, sig * (1.0 - sig)


def _values(st, name):
    """A matrix in 32 bits, whatever it is held in."""
    if name + "s" in st:
        return st[name].view(torch.float8_e4m3fn).float() * torch.exp2(st[name + "s"].float() - 127.0)[:, None]
    return st[name].detach().float()


def _plain_norm(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    s = st["x"].detach().float()
    if case["residual"]:
        s = s + st["res"].detach().float()
    w = st["w"].detach().float()
    r = 1.0 / torch.sqrt((s * s).sum(1, keepdim=True) / case["d"] + EPS)
    unit = s * r
    y = unit * w
    if case["fp8"]:
        top = y.abs().amax(1, keepdim=True)
        m, e = torch.frexp(top)
        e = torch.where(top > 0, e - 8 - (m <= 0.875).to(e.dtype), torch.zeros_like(e))
        q = torch.clamp(y * torch.exp2(-e.float()), -448, 448).to(torch.float8_e4m3fn).float() * torch.exp2(e.float())
        out = {"rows": q.to(torch.bfloat16)}
    else:
        out = {"y": y.to(dt)}
    if case["residual"]:
        out["s"] = s.to(dt)
    if case["train"]:
        dy = st["dy"].float()
        g = dy * w
        dx = r * (g - unit * ((g * unit).sum(1, keepdim=True) / case["d"]))
        if case["residual"]:
            dx = dx + st["ds"].float()
            out["dres"] = dx.to(dt)
        out["dx"], out["dw"] = dx.to(dt), (dy * unit).sum(0).to(dt)
    return out


def _plain_linear(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    x, w = _values(st, "x"), _values(st, "w")
    z = x @ w.t()
    if case["bias"]:
        z = z + st["bw"].detach().float()
    a, da = _act(z, case["act"])
    y = a + st["res"].detach().float() if case["residual"] else a
    out = {"y": y.to(dt)}
    if case["train"]:
        dz = st["dy"].float() * da
        out["dx"], out["dw"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
        if case["bias"]:
            out["db"] = dz.sum(0).to(dt)
        if case["residual"]:
            out["dres"] = st["dy"].clone()
    return out


def _plain_gated(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    x, w, v = _values(st, "x"), _values(st, "w"), _values(st, "v")
    g, u = x @ w.t(), x @ v.t()
    if case["bias"]:
        g, u = g + st["bw"].detach().float(), u + st["bv"].detach().float()
    a, da = _act(g, case["act"])
    out = {"y": (a * u).to(dt)}
    if case["train"]:
        dy = st["dy"].float()
        du, dg = dy * a, dy * u * da
        out["dx"] = (dg @ w + du @ v).to(dt)
        out["dw"], out["dv"] = (dg.t() @ x).to(dt), (du.t() @ x).to(dt)
        if case["bias"]:
            out["db"], out["dc"] = dg.sum(0).to(dt), du.sum(0).to(dt)
    return out


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(st):
    from wast3d_amd import ops

    case = st["case"]
    if case["op"] == "norm":
        if case["fp8"]:
            q, e, *s = ops.rms_norm_fp8(st["x"], st["w"], residual=st["res"], eps=EPS)
            out = {"rows": (q.view(torch.float8_e4m3fn).float() * torch.exp2(e.float() - 127.0)[:, None]).to(torch.bfloat16)}
            return {**out, "s": s[0]} if s else out
        got = ops.rms_norm(st["x"], st["w"], residual=st["res"], eps=EPS)
        out = {"y": got[0], "s": got[1]} if case["residual"] else {"y": got}
    elif case["op"] == "linear":
        act = None if case["act"] == "none" else case["act"]
        if case["fp8"]:
            return {"y": ops.linear_fp8(st["x"], st["xs"], st["w"], st["ws"], st["bw"], activation=act, residual=st["res"], out_dtype=DTYPES[case["dtype"]])}
        out = {"y": ops.linear(st["x"], st["w"], st["bw"], activation=act, residual=st["res"])}
    else:
        act = None if case["act"] == "none" else case["act"]
        if case["fp8"]:
            return {"y": ops.gated_linear_fp8(st["x"], st["xs"], st["w"], st["ws"], st["v"], st["vs"], st["bw"], st["bv"], activation=act, out_dtype=DTYPES[case["dtype"]])}
        out = {"y": ops.gated_linear(st["x"], st["w"], st["v"], st["bw"], st["bv"], activation=act)}
    if case["train"]:
        given = [st["dy"]] + ([st["ds"]] if st.get("ds") is not None else [])
        grads = torch.autograd.grad(list(out.values()), [st[i] for i in st["leaves"]], given)
        out = {i: v.detach() for i, v in out.items()}
        out.update(zip([{"bw": "db", "bv": "dc"}.get(i, "d" + i) for i in st["leaves"]], grads))
    return out


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "linear": _plain_linear, "gated": _plain_gated}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    R, b = case["rows"], SIZE[case["dtype"]]
    if case["op"] == "norm":
        d = case["d"]
        total = R * d * b * (2 if case["residual"] else 1) + d * b                      # x, residual, weight
        total += R * (d + 4) if case["fp8"] else R * d * b                              # y
        total += R * d * b if case["residual"] else 0                                   # s
        if case["train"]:
            total += R * d * b * (4 if case["residual"] else 2) + d * b                 # dy, ds; dx, dres; dw
        return {"bytes": total, "flops": R * d * (10 if case["train"] else 4)}
    K, N, m = case["k"], case["n"], 1 if case["op"] == "linear" else 2
    read = R * (K + 4) + m * N * (K + 4) if case["fp8"] else (R * K + m * N * K) * b
    bias, res = (m * N * b if case["bias"] else 0), (R * N * b if case.get("residual") else 0)
    total = read + bias + res + R * N * b
    if case["train"]:
        total += R * N * b + R * K * b + m * N * K * b + bias + res                     # dy; dx, the weights', the biases' and the residual's gradients
    return {"bytes": total, "flops": 2 * m * R * N * K * (3 if case["train"] else 1)}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)

    def leaf(name):
        if st.get(name) is None:
            return None
        if name + "s" in st:                                                            # 8-bit rows
            return torch.ldexp(st[name].view(torch.float8_e4m3fn).double(), (st[name + "s"] - 127)[:, None].double())
        return st[name].detach().double().requires_grad_(case["train"])

    x, w, v, bw, bv, res = (leaf(i) for i in ("x", "w", "v", "bw", "bv", "res"))
    squash = {"none": lambda t: t, "relu": lambda t: t.clamp_min(0), "gelu": lambda t: t * torch.special.ndtr(t), "silu": lambda t: t * torch.sigmoid(t), "sigmoid": torch.sigmoid}
    out, given = {}, [st["dy"].double()] if case["train"] else []
    if case["op"] == "norm":
        s = x if res is None else x + res
        y = w * s * torch.rsqrt(s.square().mean(1, keepdim=True) + EPS)
        if case["fp8"]:
            scale = torch.exp2(torch.ceil(torch.log2(y.abs().amax(1, keepdim=True) / 448.0)).clamp_min(-126))
            out["rows"] = (y / scale).float().to(torch.float8_e4m3fn).double() * scale
        else:
            out["y"] = y
        if res is not None:
            out["s"] = s
            if case["train"]:
                given.append(st["ds"].double())
    elif case["op"] == "linear":
        y = squash[case["act"]](torch.matmul(x, w.t()) + (0.0 if bw is None else bw))
        out["y"] = y if res is None else y + res
    else:
        gate = torch.matmul(x, w.t()) + (0.0 if bw is None else bw)
        out["y"] = squash[case["act"]](gate) * (torch.matmul(x, v.t()) + (0.0 if bv is None else bv))
    if case["train"]:
        by = {"dx": x, "dw": w, "dv": v, "db": bw, "dc": bv, "dres": res}
        by = {n: t for n, t in by.items() if t is not None}
        grads = torch.autograd.grad(list(out.values()), list(by.values()), given)
        out = {n: t.detach() for n, t in out.items()}
        out.update(zip(by, grads))
    return out
