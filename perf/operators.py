"""What is measured of the transformer-layer operators: the linear layer with its epilogue and its
gradient, and the root-mean-square norm with the residual's addition and its gradient.

Each case names one operator (`op`), its sizes, types and options.  `run` computes it either in plain
torch operations in 32 bits (`own` false) or through this package's entry points (`own` true);
`exact` is the definition in 64 bits.
"""

import math

import torch

own = False

EPS = 1e-5
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
E4M3_MAX = 448.0
TINY = 2.0 ** -126  # the smallest scale of a row held in 8 bits
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def linear(name, m, k, n, dtype, act, bias=True, residual="", out="bf16", pre=False, trans_b=True):
    """m tokens of k features to n; `residual` is the residual's type or empty; `trans_b`: weights n x k."""
    c = {"op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias, "residual": residual,
         "out": out, "pre": pre, "trans_b": trans_b}
    return {"name": name, **c} if name else c


def linear_backward(name, m, k, n, act, bias=True, trans_b=True):
    c = {"op": "linear_backward", "m": m, "k": k, "n": n, "act": act, "bias": bias, "trans_b": trans_b}
    return {"name": name, **c} if name else c


def rms_norm(name, m, n, dtype, out, residual=True):
    c = {"op": "rms_norm", "m": m, "n": n, "dtype": dtype, "out": out, "residual": residual}
    return {"name": name, **c} if name else c


def rms_norm_backward(name, m, n, dtype, residual=True):
    c = {"op": "rms_norm_backward", "m": m, "n": n, "dtype": dtype, "residual": residual}
    return {"name": name, **c} if name else c


def listed():
    return [
        # One token's down projection back onto the residual stream while decoding.
        linear("linear bf16 1", 1, 4096, 4096, "bf16", "none", bias=False, residual="bf16"),
        # A decoding batch through an 8-bit up projection.
        linear("linear e4m3 16", 16, 4096, 16384, "e4m3", "silu"),
        # A training batch's up projection; the value before the activation is kept for the gradient.
        linear("linear bf16 4096", 4096, 4096, 16384, "bf16", "gelu_tanh", pre=True, trans_b=False),
        # A prefill's 8-bit down projection onto the residual stream.
        linear("linear e4m3 8192", 8192, 16384, 4096, "e4m3", "none", residual="bf16"),
        # Ragged sizes (no row a multiple of 16 bytes), f32 out and residual.
        linear("linear bf16 777", 777, 333, 1111, "bf16", "gelu", residual="f32", out="f32", trans_b=False),
        # The gradient of the training batch's up projection.
        linear_backward("linear_backward 8192", 8192, 4096, 16384, "gelu_tanh", trans_b=False),
        # A small ragged layer's gradient.
        linear_backward("linear_backward 500", 500, 1000, 1000, "silu"),
        # The norm before a layer while decoding, its output in 8 bits for an 8-bit product.
        rms_norm("rms_norm e4m3 16", 16, 4096, "bf16", "e4m3"),
        # The same for a long prefill.
        rms_norm("rms_norm e4m3 16384", 16384, 8192, "bf16", "e4m3"),
        # An f32 model with an odd width and no residual.
        rms_norm("rms_norm f32 4097", 4097, 1111, "f32", "f32", residual=False),
        # The norm's gradient for a training batch, joined with the residual stream's.
        rms_norm_backward("rms_norm_backward 16384", 16384, 4096, "bf16"),
        # The norm's gradient of a small f32 model with an odd width.
        rms_norm_backward("rms_norm_backward 300", 300, 1111, "f32", residual=False),
    ]


def spread(rng, lo, hi):
    """A size between lo and hi, even over its logarithm; half of them multiples of 64 where there is room."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(64, v // 64 * 64) if hi >= 1024 and v >= 64 and rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_backward", "rms_norm", "rms_norm_backward"])
    if op == "linear":
        dtype = rng.choice(["bf16", "e4m3"])
        while True:
            m, k, n = spread(rng, 1, 16384), spread(rng, 32, 16384), spread(rng, 32, 16384)
            if m * k * n <= 4096 * 4096 * 16384:
                break
        return linear("", m, k, n, dtype, rng.choice(ACTIVATIONS), rng.random() < 0.7, rng.choice(["", "bf16", "f32"]),
                      rng.choice(["bf16", "bf16", "f32"]), rng.random() < 0.3, dtype == "e4m3" or rng.random() < 0.5)
    if op == "linear_backward":
        while True:
            m, k, n = spread(rng, 8, 16384), spread(rng, 32, 16384), spread(rng, 32, 16384)
            if m * k * n <= 4096 * 4096 * 16384:
                break
        return linear_backward("", m, k, n, rng.choice(ACTIVATIONS), rng.random() < 0.7, rng.random() < 0.5)
    while True:
        m, n = spread(rng, 1, 65536), spread(rng, 32, 16384)
        if m * n <= 16384 * 8192:
            break
    dtype = rng.choice(["bf16", "f32"])
    if op == "rms_norm":
        return rms_norm("", m, n, dtype, rng.choice(["e4m3", dtype]), rng.random() < 0.7)
    return rms_norm_backward("", m, n, dtype, rng.random() < 0.7)


# ---- inputs -----------------------------------------------------------------------------------


def rows_e4m3(x):
    """Rows of x in 8 bits and a scale a row, as an 8-bit model's weights and activations are held."""
    scale = (x.abs().amax(1) / E4M3_MAX).clamp_min(TINY)
    return (x / scale[:, None]).to(torch.float8_e4m3fn), scale


def activations(m, n, g, dtype=torch.float32):
    """Normal values with a few large channels, as the residual stream of a trained model has."""
    x = torch.randn(m, n, generator=g, device="cuda")
    x[:, :: max(1, n // 7)] *= 8.0
    return x.to(dtype)


def weights(c, g):
    shape = (c["n"], c["k"]) if c["trans_b"] else (c["k"], c["n"])
    return torch.randn(*shape, generator=g, device="cuda") * (1.0 / math.sqrt(c["k"]))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = dict(case)
    s = {"case": c}
    m, n = c["m"], c["n"]
    if c["op"] in ("linear", "linear_backward"):
        k = c["k"]
        a, b = activations(m, k, g), weights(c, g)
        if c["bias"]:
            s["bias"] = 0.1 * torch.randn(n, generator=g, device="cuda")
        if c["op"] == "linear":
            if c["dtype"] == "e4m3":
                s["a"], s["a_scale"] = rows_e4m3(a)
                s["b"], s["b_scale"] = rows_e4m3(b)
            else:
                s["a"], s["b"] = a.bfloat16(), b.bfloat16()
            if c["residual"]:
                s["residual"] = activations(m, n, g, DTYPES[c["residual"]])
        else:
            s["a"], s["b"] = a.bfloat16(), b.bfloat16()
            s["dout"] = (torch.randn(m, n, generator=g, device="cuda") * 0.01).bfloat16()
            if c["act"] != "none":
                s["pre"] = (1.5 * torch.randn(m, n, generator=g, device="cuda")).bfloat16()
        return s
    dtype = DTYPES[c["dtype"]]
    x = activations(m, n, g, dtype)
    if m > 2:
        x[m // 2] = 0  # a padded token
    s["weight"] = 1.0 + 0.2 * torch.randn(n, generator=g, device="cuda")
    if c["op"] == "rms_norm":
        s["x"] = x
        if c["residual"]:
            r = activations(m, n, g, dtype)
            if m > 2:
                r[m // 2] = 0
            s["residual"] = r
        return s
    s["s"] = x
    s["rstd"] = (x.double().square().mean(1) + EPS).rsqrt().float()
    s["dy"] = (torch.randn(m, n, generator=g, device="cuda") * 0.01).to(dtype)
    if c["residual"]:
        s["ds"] = (torch.randn(m, n, generator=g, device="cuda") * 0.01).to(dtype)
    return s


# ---- the plain form -----------------------------------------------------------------------------


def activation(z, name):
    if name == "relu":
        return torch.clamp_min(z, 0.0)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def slope(z, name):
    """The activation's derivative."""
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == "gelu_tanh":
        t = torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * z * z)
    if name == "silu":
        e = 1.0 / (1.0 + torch.exp(-z))
        return e * (1.0 + z * (1.0 - e))
    return torch.ones_like(z)


def plain_linear(s, c):
    a, b = s["a"].float(), s["b"].float()
    z = a @ (b.t() if c["trans_b"] else b)
    if c["dtype"] == "e4m3":
        z = z * s["a_scale"][:, None] * s["b_scale"]
    if c["bias"]:
        z = z + s["bias"]
    y = activation(z, c["act"])
    if c["residual"]:
        y = y + s["residual"].float()
    to = DTYPES[c["out"]]
    return {"out": y.to(to), "pre": z.to(to)} if c["pre"] else {"out": y.to(to)}


def plain_linear_backward(s, c):
    a, b, dz = s["a"].float(), s["b"].float(), s["dout"].float()
    if c["act"] != "none":
        dz = dz * slope(s["pre"].float(), c["act"])
    da = dz @ (b if c["trans_b"] else b.t())
    db = dz.t() @ a if c["trans_b"] else a.t() @ dz
    out = {"da": da.bfloat16(), "db": db.bfloat16()}
    if c["bias"]:
        out["dbias"] = dz.sum(0)
    return out


def plain_rms_norm(s, c):
    x = s["x"].float()
    if c["residual"]:
        x = x + s["residual"].float()
    rstd = torch.rsqrt((x * x).mean(1) + EPS)
    y = x * rstd[:, None] * s["weight"]
    out = {"rstd": rstd}
    if c["residual"]:
        out["sum"] = x.to(DTYPES[c["dtype"]])
    if c["out"] == "e4m3":
        out["out"], out["scale"] = rows_e4m3(y)
    else:
        out["out"] = y.to(DTYPES[c["out"]])
    return out


def plain_rms_norm_backward(s, c):
    hat = s["s"].float() * s["rstd"][:, None]
    dy = s["dy"].float()
    g = dy * s["weight"]
    dx = (g - hat * (g * hat).mean(1, keepdim=True)) * s["rstd"][:, None]
    if c["residual"]:
        dx = dx + s["ds"].float()
    return {"dx": dx.to(DTYPES[c["dtype"]]), "dweight": (dy * hat).sum(0)}


# ---- the framework's calls ------------------------------------------------------------------------


def own_run(s, c):
    from tensorforge_b200 import _lib

    code = {"f32": _lib.F32, "bf16": _lib.BF16, "e4m3": _lib.E4M3}
    stream = torch.cuda.current_stream().cuda_stream
    m, n = c["m"], c["n"]

    def ptr(name):
        return s[name].data_ptr() if name in s else None

    def new(*shape, dtype=torch.float32):
        return torch.empty(shape, device="cuda", dtype=dtype)

    if c["op"] == "linear":
        to = DTYPES[c["out"]]
        out = {"out": new(m, n, dtype=to)}
        if c["pre"]:
            out["pre"] = new(m, n, dtype=to)
        _lib.linear(ptr("a"), ptr("b"), out["out"].data_ptr(), m, n, c["k"], activation=c["act"], bias=ptr("bias"),
                    residual=ptr("residual"), pre=out["pre"].data_ptr() if c["pre"] else None, a_scale=ptr("a_scale"),
                    b_scale=ptr("b_scale"), a_dtype=code[c["dtype"]], b_dtype=code[c["dtype"]], out_dtype=code[c["out"]],
                    residual_dtype=code[c["residual"] or "bf16"], trans_b=c["trans_b"], stream=stream)
        return out
    if c["op"] == "linear_backward":
        out = {"da": torch.empty_like(s["a"]), "db": torch.empty_like(s["b"])}
        if c["bias"]:
            out["dbias"] = new(n)
        _lib.linear_backward(ptr("dout"), ptr("a"), ptr("b"), m, n, c["k"], activation=c["act"], pre=ptr("pre"),
                             dA=out["da"].data_ptr(), dB=out["db"].data_ptr(),
                             dbias=out["dbias"].data_ptr() if c["bias"] else None, dtype=_lib.BF16, grad_dtype=_lib.BF16,
                             trans_b=c["trans_b"], stream=stream)
        return out
    dtype = DTYPES[c["dtype"]]
    if c["op"] == "rms_norm":
        out = {"rstd": new(m), "out": new(m, n, dtype=DTYPES[c["out"]])}
        if c["residual"]:
            out["sum"] = new(m, n, dtype=dtype)
        if c["out"] == "e4m3":
            out["scale"] = new(m)
        _lib.rms_norm(ptr("x"), out["out"].data_ptr(), m, n, EPS, weight=ptr("weight"), residual=ptr("residual"),
                      sum_out=out["sum"].data_ptr() if c["residual"] else None, rstd=out["rstd"].data_ptr(),
                      scale=out["scale"].data_ptr() if c["out"] == "e4m3" else None, dtype=code[c["dtype"]],
                      out_dtype=code[c["out"]], stream=stream)
        return out
    out = {"dx": new(m, n, dtype=dtype), "dweight": new(n)}
    _lib.rms_norm_backward(ptr("dy"), ptr("s"), ptr("rstd"), out["dx"].data_ptr(), m, n, weight=ptr("weight"), ds=ptr("ds"),
                           dweight=out["dweight"].data_ptr(), dtype=code[c["dtype"]], stream=stream)
    return out


def run(state):
    c = state["case"]
    if own:
        return own_run(state, c)
    return {"linear": plain_linear, "linear_backward": plain_linear_backward, "rms_norm": plain_rms_norm,
            "rms_norm_backward": plain_rms_norm_backward}[c["op"]](state, c)


def work(case):
    c = case
    m, n = c["m"], c["n"]
    size = {"f32": 4, "bf16": 2, "e4m3": 1, "": 0}
    if c["op"] == "linear":
        k, e, o = c["k"], size[c["dtype"]], size[c["out"]]
        b = e * (m * k + k * n) + m * n * (o * (2 if c["pre"] else 1) + size[c["residual"]]) + (4 * n if c["bias"] else 0)
        return {"bytes": b + (4 * (m + n) if c["dtype"] == "e4m3" else 0), "flops": 2.0 * m * n * k}
    if c["op"] == "linear_backward":
        k = c["k"]
        b = 2 * (2 * m * k + 2 * k * n + m * n * (1 if c["act"] == "none" else 2)) + (4 * n if c["bias"] else 0)
        return {"bytes": b, "flops": 4.0 * m * n * k}
    e = size[c["dtype"]]
    if c["op"] == "rms_norm":
        return {"bytes": m * n * (e * (3 if c["residual"] else 1) + size[c["out"]]) + 4 * n + 4 * m * (2 if c["out"] == "e4m3" else 1),
                "flops": 6.0 * m * n}
    return {"bytes": m * n * e * (4 if c["residual"] else 3) + 8 * n + 4 * m, "flops": 10.0 * m * n}


# ---- the definition in 64 bits --------------------------------------------------------------------


def phi(z):
    """The normal distribution's cumulative function."""
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))


def exact_activation(z, name):
    """The activation's value and derivative."""
    if name == "relu":
        return z.relu(), torch.where(z > 0, 1.0, 0.0)
    if name == "gelu":
        return z * phi(z), phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        # 0.5 (1 + tanh u) is the logistic function of 2 u.
        u2 = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        du2 = 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2)
        p = torch.sigmoid(u2)
        return z * p, p + z * p * (1 - p) * du2
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    return z, torch.ones_like(z)


def exact(case, seed):
    s, c = prepare(case, seed), case
    d = {k: v.double() for k, v in s.items() if k != "case"}
    if c["op"] in ("linear", "linear_backward"):
        w = d["b"].T if c["trans_b"] else d["b"]  # k x n
        if c["op"] == "linear":
            if "a_scale" in d:
                d["a"] = d["a"] * d["a_scale"].unsqueeze(1)
                w = w * d["b_scale"].unsqueeze(0)
            z = torch.matmul(d["a"], w)
            if "bias" in d:
                z += d["bias"]
            y = exact_activation(z, c["act"])[0]
            y = y + d["residual"] if "residual" in d else y
            return {"out": y, "pre": z} if c["pre"] else {"out": y}
        dz = d["dout"]
        if "pre" in d:
            dz = dz * exact_activation(d["pre"], c["act"])[1]
        dw = torch.matmul(d["a"].T, dz)
        out = {"da": torch.matmul(dz, w.T), "db": dw.T if c["trans_b"] else dw}
        if "bias" in d:
            out["dbias"] = dz.sum(dim=0)
        return out
    if c["op"] == "rms_norm":
        x = d["x"] + d["residual"] if "residual" in d else d["x"]
        rms = (x.pow(2).sum(1) / c["n"] + EPS).sqrt()
        y = x / rms.unsqueeze(1) * d["weight"]
        out = {"rstd": 1 / rms, "out": y}
        if "residual" in d:
            out["sum"] = x
        if c["out"] == "e4m3":
            out["scale"] = (y.abs().max(dim=1).values / E4M3_MAX).clamp(min=TINY)
            out["out"] = y / out["scale"].unsqueeze(1)  # the number that the 8 bits stand for, unrounded
        return out
    # y = w s rstd(s): dL/ds_i = rstd (w_i dy_i - s_i rstd^2 / n sum_j w_j dy_j s_j), and the stream's own.
    s_, r, wdy = d["s"], d["rstd"].unsqueeze(1), d["dy"] * d["weight"]
    dx = r * wdy - s_ * r ** 3 * (wdy * s_).sum(1, keepdim=True) / c["n"]
    if "ds" in d:
        dx = dx + d["ds"]
    return {"dx": dx, "dweight": (d["dy"] * s_ * r).sum(dim=0)}
