"""Cases of the 16-bit feed-forward operators: layer norm, a linear layer with
its bias, activation and residual, and the gated (GEGLU / SwiGLU) projection,
each forward alone or with its backward pass.

Kinds of case:

* ``norm``    ``layer_norm`` over the last dim of ``[rows, dim]``;
* ``linear``  ``linear_act``: ``act(x W^T + b) + residual``, ``[rows, k] -> [rows, n]``;
* ``gated``   ``gated_linear``: ``(x Wv^T + bv) * act(x Wg^T + bg)``,
  ``[rows, k] -> [rows, n]``, the two weights stacked (``fused``) or apart.

``train`` cases return the output and the gradient of every input. Activations
are N(0, 1) with 0.5% of the channels 8 times larger for layer norm (and an
offset, as a residual stream has), N(0, 1) for the products (a norm's output);
weights N(0, 1 / k), biases N(0, 0.1), residuals N(0, 1), output gradients
N(0, 1 / 32) (a scaled loss).
"""

import math

import torch

own = False   # False: the plain form in elementary torch operations; True: the framework's operators

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # the smallest: a text encoder's layer norm over a 77-token prompt pair; latency
        {"name": "norm_text", "kind": "norm", "rows": 154, "dim": 768, "x": "fp16", "w": "fp16", "train": False},
        # a fine-tuning step's layer norm at SDXL's 640-channel level, 16 images, float32 master weights
        {"name": "norm_train", "kind": "norm", "rows": 65536, "dim": 640, "x": "bf16", "w": "fp32", "train": True},
        # wide rows of an odd width: a single-precision stream
        {"name": "norm_train_odd", "kind": "norm", "rows": 4099, "dim": 2731, "x": "fp32", "w": "fp32",
         "train": True},
        # a UNet's time embedding, the CFG pair: two rows, latency
        {"name": "linear_time_embed", "kind": "linear", "rows": 2, "k": 320, "n": 1280, "dtype": "fp16",
         "act": "silu", "bias": True, "res": False, "train": False, "pad": 0},
        # one token through a square projection with its residual: the weights' bytes
        {"name": "linear_token", "kind": "linear", "rows": 1, "k": 4096, "n": 4096, "dtype": "bf16",
         "act": "none", "bias": False, "res": True, "train": False, "pad": 0},
        # the SDXL feed-forward's output layer with its bias and residual
        {"name": "linear_ff_out", "kind": "linear", "rows": 8192, "k": 2560, "n": 640, "dtype": "fp16",
         "act": "none", "bias": True, "res": True, "train": False, "pad": 0},
        # the first layer of a DiT's MLP in a fine-tuning step: the largest
        {"name": "linear_train_mlp", "kind": "linear", "rows": 4608, "k": 2048, "n": 8192, "dtype": "bf16",
         "act": "gelu_tanh", "bias": True, "res": False, "train": True, "pad": 0},
        # odd sizes in every direction
        {"name": "linear_train_odd", "kind": "linear", "rows": 1001, "k": 1155, "n": 577, "dtype": "fp16",
         "act": "silu", "bias": True, "res": True, "train": True, "pad": 0},
        # one token through a language model's gated projection, weights apart
        {"name": "gated_token", "kind": "gated", "rows": 1, "k": 2048, "n": 8192, "dtype": "bf16", "act": "silu",
         "bias": False, "fused": False, "train": False, "pad": 0},
        # SDXL's GEGLU at the 640-channel level, 1024^2, the CFG pair
        {"name": "gated_unet", "kind": "gated", "rows": 8192, "k": 640, "n": 2560, "dtype": "fp16", "act": "gelu",
         "bias": True, "fused": True, "train": False, "pad": 0},
        # the same at the 1280-channel level in a fine-tuning step of 4 images
        {"name": "gated_train", "kind": "gated", "rows": 4096, "k": 1280, "n": 5120, "dtype": "bf16", "act": "gelu",
         "bias": True, "fused": True, "train": True, "pad": 0},
        # ragged sizes, weights apart, rows strided as a slice of a wider buffer has them
        {"name": "gated_train_ragged", "kind": "gated", "rows": 777, "k": 1000, "n": 2731, "dtype": "bf16",
         "act": "silu", "bias": True, "fused": False, "train": True, "pad": 24},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size over the logarithm of its range: two in three a multiple of 16, as layer widths are."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 1 / 3 else max(16, (v + 8) // 16 * 16)


def draw(rng):
    kind = rng.choice(["norm", "linear", "linear", "gated", "gated"])
    train = rng.random() < 0.5
    if kind == "norm":
        while True:
            rows, dim = _log(rng, 1, 65536), _size(rng, 8, 16384)
            if rows * dim <= 65536 * 640:
                break
        x = rng.choice(["fp16", "bf16", "fp32"])
        return {"kind": kind, "rows": rows, "dim": dim, "x": x, "w": rng.choice([x, "fp32"]), "train": train}
    most = 6.0 * 4608 * 2048 * 8192
    while True:
        rows, k, n = _log(rng, 1, 16384), _size(rng, 16, 8192), _size(rng, 16, 8192)
        if (6.0 if train else 2.0) * (2 if kind == "gated" else 1) * rows * k * n <= most:
            break
    case = {"kind": kind, "rows": rows, "k": k, "n": n, "dtype": rng.choice(["fp16", "bf16"]),
            "bias": rng.random() < 0.7, "train": train, "pad": rng.choice([0, 0, 64, 5])}
    if kind == "linear":
        case["act"] = rng.choice(["none", "gelu", "gelu_tanh", "silu", "quick_gelu"])
        case["res"] = rng.random() < 0.5
    else:
        case["act"] = rng.choice(["gelu", "gelu_tanh", "silu", "quick_gelu"])
        case["fused"] = rng.random() < 0.5
    return case


def _inputs(case, seed):
    """Every input of a case by name, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    rows = case["rows"]
    if case["kind"] == "norm":
        dim, xt, wt = case["dim"], DTYPES[case["x"]], DTYPES[case["w"]]
        loud = torch.where(torch.rand(dim, generator=g, device="cuda") < 0.005, 8.0, 1.0)
        x = (randn(rows, dim) * loud + randn(rows, 1, std=0.5)).to(xt)
        t = {"x": x, "w": (1.0 + randn(dim, std=0.2)).to(wt), "b": randn(dim, std=0.1, dtype=wt)}
        if case["train"]:
            t["dy"] = randn(rows, dim, std=1 / 32, dtype=xt)
        return t
    k, n, dt = case["k"], case["n"], DTYPES[case["dtype"]]
    t = {"x": randn(rows, k + case["pad"], dtype=dt)[:, :k]}
    if case["kind"] == "linear":
        t["w"] = randn(n, k, std=k ** -0.5, dtype=dt)
        if case["bias"]:
            t["b"] = randn(n, std=0.1, dtype=dt)
        if case["res"]:
            t["res"] = randn(rows, n, dtype=dt)
    elif case["fused"]:
        t["w"] = randn(2 * n, k, std=k ** -0.5, dtype=dt)
        if case["bias"]:
            t["b"] = randn(2 * n, std=0.1, dtype=dt)
    else:
        t["w"], t["wg"] = randn(n, k, std=k ** -0.5, dtype=dt), randn(n, k, std=k ** -0.5, dtype=dt)
        if case["bias"]:
            t["b"], t["bg"] = randn(n, std=0.1, dtype=dt), randn(n, std=0.1, dtype=dt)
    if case["train"]:
        t["dy"] = randn(rows, n, std=1 / 32, dtype=dt)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    if case["train"]:
        for name, v in t.items():
            if name != "dy":
                v.requires_grad_(True)
    return {"case": case, "t": t}


def run(state):
    return _own(state["case"], state["t"]) if own else _plain(state["case"], state["t"])


def _own(case, t):
    import diffucore_amd as dc
    if case["kind"] == "norm":
        y = dc.layer_norm(t["x"], t["w"], t["b"], EPS)
    elif case["kind"] == "linear":
        y = dc.linear_act(t["x"], t["w"], t.get("b"), act=case["act"], residual=t.get("res"))
    elif case["fused"]:
        y = dc.gated_linear(t["x"], t["w"], t.get("b"), act=case["act"])
    else:
        y = dc.gated_linear(t["x"], t["w"], t.get("b"), gate_weight=t["wg"], gate_bias=t.get("bg"), act=case["act"])
    out = {"y": y.detach()}
    if case["train"]:
        names = [name for name in t if name != "dy"]
        for name, grad in zip(names, torch.autograd.grad(y, [t[name] for name in names], t["dy"])):
            out["d" + name] = grad
    return out


# ---------------------------------------------------------------- the plain form, in float32

def _act(z, act):
    """The activation of z and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "gelu":
        c = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * c, c + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        r = math.sqrt(2.0 / math.pi)
        th = torch.tanh(r * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * r * (1.0 + 0.134145 * z * z)
    a = 1.0 if act == "silu" else 1.702
    s = 1.0 / (1.0 + torch.exp(-a * z))
    return z * s, s + a * z * s * (1.0 - s)


@torch.no_grad()
def _plain(case, t):
    f = {name: v.float() for name, v in t.items()}
    out = {}
    if case["kind"] == "norm":
        mean = f["x"].mean(-1, keepdim=True)
        d = f["x"] - mean
        r = torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS)
        xh = d * r
        out["y"] = xh * f["w"] + f["b"]
        if case["train"]:
            g = f["dy"] * f["w"]
            out["dx"] = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
            out["dw"] = (f["dy"] * xh).sum(0)
            out["db"] = f["dy"].sum(0)
    elif case["kind"] == "linear":
        z = f["x"] @ f["w"].t()
        if "b" in f:
            z = z + f["b"]
        y, slope = _act(z, case["act"])
        out["y"] = y + f["res"] if "res" in f else y
        if case["train"]:
            dz = f["dy"] * slope
            out["dx"], out["dw"] = dz @ f["w"], dz.t() @ f["x"]
            if "b" in f:
                out["db"] = dz.sum(0)
            if "res" in f:
                out["dres"] = f["dy"]
    else:
        wv, wg = f["w"].chunk(2) if case["fused"] else (f["w"], f["wg"])
        a, g = f["x"] @ wv.t(), f["x"] @ wg.t()
        if case["bias"]:
            bv, bg = f["b"].chunk(2) if case["fused"] else (f["b"], f["bg"])
            a, g = a + bv, g + bg
        y, slope = _act(g, case["act"])
        out["y"] = a * y
        if case["train"]:
            da, dg = f["dy"] * y, f["dy"] * a * slope
            out["dx"] = da @ wv + dg @ wg
            dw = [da.t() @ f["x"], dg.t() @ f["x"]]
            db = [da.sum(0), dg.sum(0)]
            if case["fused"]:
                out["dw"] = torch.cat(dw)
                if case["bias"]:
                    out["db"] = torch.cat(db)
            else:
                out["dw"], out["dwg"] = dw
                if case["bias"]:
                    out["db"], out["dbg"] = db
    like = lambda name: t["x" if name == "y" else name[1:]].dtype   # noqa: E731
    return {name: v.to(like(name)) for name, v in out.items()}


# ---------------------------------------------------------------- the definition, in float64

@torch.no_grad()
def exact(case, seed):
    """The outputs from the operators' definitions in 64 bits; gradients of the
    products by the chain rule through each operand, one weight at a time."""
    i = {name: v.double() for name, v in _inputs(case, seed).items()}
    x = i["x"]
    res = {}
    if case["kind"] == "norm":
        n = x.shape[1]
        mu = x.sum(1, keepdim=True) / n
        var = ((x - mu) ** 2).sum(1, keepdim=True) / n
        sd = (var + EPS).sqrt()
        res["y"] = (x - mu) / sd * i["w"] + i["b"]
        if case["train"]:
            up = i["dy"] * i["w"]
            # d y_j / d x_k = w_j (delta_jk - 1/n - (x_j - mu)(x_k - mu) / (n sd^2)) / sd
            proj = (up * (x - mu)).sum(1, keepdim=True) / (n * sd * sd)
            res["dx"] = (up - up.sum(1, keepdim=True) / n - (x - mu) * proj) / sd
            res["dw"] = (i["dy"] * ((x - mu) / sd)).sum(0)
            res["db"] = i["dy"].sum(0)
        return res

    def value_and_slope(u, act):
        if act == "none":
            return u, torch.ones_like(u)
        if act == "gelu":
            cdf = 0.5 * torch.erfc(-u / math.sqrt(2.0))
            return u * cdf, cdf + u * torch.exp(-u * u / 2.0) / math.sqrt(2.0 * math.pi)
        if act == "gelu_tanh":   # 0.5 (1 + tanh v) = sigmoid(2 v)
            q = 2.0 * math.sqrt(2.0 / math.pi)
            s = torch.sigmoid(q * (u + 0.044715 * u ** 3))
            return u * s, s + u * s * (1.0 - s) * q * (1.0 + 3.0 * 0.044715 * u ** 2)
        q = {"silu": 1.0, "quick_gelu": 1.702}[act]
        s = torch.sigmoid(q * u)
        return u * s, s * (1.0 + q * u * (1.0 - s))

    n = case["n"]
    if case["kind"] == "linear":
        u = torch.matmul(x, i["w"].T) + (i["b"] if "b" in i else 0.0)
        v, slope = value_and_slope(u, case["act"])
        res["y"] = v + (i["res"] if "res" in i else 0.0)
        if case["train"]:
            du = i["dy"] * slope
            res["dx"] = torch.matmul(du, i["w"])
            res["dw"] = torch.matmul(du.T, x)
            if "b" in i:
                res["db"] = du.sum(0)
            if "res" in i:
                res["dres"] = i["dy"]
        return res
    w = i["w"] if case["fused"] else torch.cat([i["w"], i["wg"]])
    u = torch.matmul(x, w.T)
    if case["bias"]:
        u = u + (i["b"] if case["fused"] else torch.cat([i["b"], i["bg"]]))
    v, slope = value_and_slope(u[:, n:], case["act"])
    res["y"] = u[:, :n] * v
    if case["train"]:
        du = torch.cat([i["dy"] * v, i["dy"] * u[:, :n] * slope], 1)
        res["dx"] = torch.matmul(du, w)
        dw, db = torch.matmul(du.T, x), du.sum(0)
        if case["fused"]:
            res["dw"] = dw
            if case["bias"]:
                res["db"] = db
        else:
            res["dw"], res["dwg"] = dw[:n], dw[n:]
            if case["bias"]:
                res["db"], res["dbg"] = db[:n], db[n:]
    return res


def work(case):
    """Each input read once, each output written once (a residual's gradient is
    the output's own and costs nothing); the products' operations."""
    rows, train = case["rows"], case["train"]
    if case["kind"] == "norm":
        dim, xb, wb = case["dim"], DTYPES[case["x"]].itemsize, DTYPES[case["w"]].itemsize
        return {"bytes": (4 if train else 2) * rows * dim * xb + (4 if train else 2) * dim * wb,
                "flops": (20 if train else 8) * rows * dim}
    k, n = case["k"], case["n"]
    wide = 2 * n if case["kind"] == "gated" else n
    elems = rows * k + wide * k + rows * n + (wide if case["bias"] else 0)
    if case.get("res"):
        elems += rows * n
    if train:
        elems += rows * n + rows * k + wide * k + (wide if case["bias"] else 0)
    return {"bytes": 2 * elems, "flops": (6 if train else 2) * rows * k * wide}
