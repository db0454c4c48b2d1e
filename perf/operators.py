"""The layer operators of ``smrt_amd.autoencode.layers`` as cases to measure: what they compute, in elementary torch
operations, and the calls a user makes of them.

Five kinds of case:

``dense``    one dense layer, ``act(x W + b) + residual``: its forward pass, or a training step of it
``norm``     layer norm's forward and backward pass, with the gradients of its weight and bias
``pack``     a batch of activations held in 8 bits (32 columns share a power of two) and read back
``ckpt``     a training step of a dense layer, or of a layer norm, whose saved activations are held in those 8 bits
``grouped``  the dense layers of several classes on one batch whose rows are sorted by class: forward, or a training step
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 32                       # columns that share a scale
EPS = 1e-5


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one row through a hidden layer of the wide net 256-[1024]x4-64: a request answered row by row
        {"name": "dense row", "op": "dense", "step": False, "dtype": "bf16", "rows": 1, "k": 1024, "n": 1024,
         "act": "sigmoid", "residual": False},
        # the same net over its large batch: encode, decode and generate of many rows
        {"name": "dense forward wide", "op": "dense", "step": False, "dtype": "bf16", "rows": 65536, "k": 1024, "n": 1024,
         "act": "relu", "residual": True},
        # first layer of 784-450-10 at the data-parallel batch of a rank: widths that no tile divides
        {"name": "dense step odd", "op": "dense", "step": True, "dtype": "f32", "rows": 8192, "k": 784, "n": 450,
         "act": "sigmoid", "residual": False},
        # a residual hidden layer of the wide net at the large batch, in the framework's own type: the largest
        {"name": "dense step wide", "op": "dense", "step": True, "dtype": "f32", "rows": 65536, "k": 1024, "n": 1024,
         "act": "tanh", "residual": True},
        # a default mini-batch of 64 features: latency
        {"name": "norm batch", "op": "norm", "dtype": "f32", "rows": 128, "n": 64},
        # odd rows and an odd width
        {"name": "norm odd", "op": "norm", "dtype": "f16", "rows": 8191, "n": 450},
        # the wide net's hidden width at the large batch: bandwidth
        {"name": "norm wide", "op": "norm", "dtype": "bf16", "rows": 65536, "n": 1024},
        # a layer norm over 784 pixels whose input is kept in 8 bits between the passes
        {"name": "norm checkpointed", "op": "ckpt", "layer": "norm", "dtype": "bf16", "rows": 16384, "n": 784},
        # a hidden layer of the wide net that keeps its input and its activation in 8 bits
        {"name": "dense checkpointed", "op": "ckpt", "layer": "dense", "dtype": "bf16", "rows": 32768, "k": 1024, "n": 1024,
         "act": "elu", "residual": False},
        # a class of 19 608 rows of 450 activations, put away in 8 bits and read back: the last block of a row is ragged
        {"name": "pack odd", "op": "pack", "dtype": "f32", "rows": 19608, "n": 450},
        # three synthetic rows each of eight classes, one decoder layer per class: latency
        {"name": "grouped rows", "op": "grouped", "step": False, "dtype": "f32", "rows": 24, "k": 450, "n": 784, "groups": 8,
         "act": "sigmoid"},
        # eight classes of about 5 000 rows of 784 pixels: every class's first layer, forward and backward
        {"name": "grouped step", "op": "grouped", "step": True, "dtype": "bf16", "rows": 40000, "k": 784, "n": 450, "groups": 8,
         "act": "relu"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["dense", "dense", "norm", "pack", "ckpt", "ckpt", "grouped", "grouped"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    rows = _log(rng, 1, 65536)
    if op in ("norm", "pack"):
        c = {"op": op, "dtype": dtype, "rows": rows, "n": _log(rng, 8, 4000)}
        c["rows"] = max(1, min(rows, 65536 * 1024 // c["n"]))
        return c
    k, n = _log(rng, 16, 2000), _log(rng, 16, 2000)
    if rng.random() < 0.4:                                  # widths of whole tiles as often as a user picks them
        k, n = -(-k // 64) * 64, -(-n // 64) * 64
    if op == "ckpt":
        # the activation that a layer computes and packs is held in a 16-bit type: in 32 bits a last-bit difference of two
        # orders of summation moves a value over a border between two 8-bit steps
        if rng.random() < 0.4:
            return {"op": "ckpt", "layer": "norm", "dtype": dtype, "rows": max(1, min(rows, 65536 * 1024 // n)), "n": n}
        return {"op": "ckpt", "layer": "dense", "dtype": rng.choice(["bf16", "f16"]), "rows": max(1, min(rows, 32768 * 1024 * 1024 // (k * n))),
                "k": k, "n": n, "act": rng.choice(["identity", "sigmoid", "tanh", "elu"]), "residual": False}
    step = rng.random() < 0.5
    # relu's gradient jumps at zero, so in 32 bits a training step of it is not compared closely
    act = rng.choice(["identity", "sigmoid", "tanh", "elu"] + (["relu"] if not step or dtype != "f32" else []))
    if op == "dense":
        return {"op": "dense", "step": step, "dtype": dtype, "rows": max(1, min(rows, 65536 * 1024 * 1024 // (k * n))), "k": k, "n": n,
                "act": act, "residual": rng.random() < 0.4}
    groups = _log(rng, 2, 64)
    k, n = min(k, 1100), min(n, 1100)
    return {"op": "grouped", "step": step, "dtype": dtype, "rows": max(1, min(rows, 20000 * 1024 * 1024 // (k * n))), "k": k, "n": n,
            "groups": groups, "act": act}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    m, n, op = case["rows"], case["n"], case["op"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def rows_of(width):
        # activations of a trained layer: every column has its own centre and spread
        return (normal(m, width) * torch.exp(0.5 * normal(width)) + 0.5 * normal(width)).to(dtype)

    s = {"case": dict(case)}
    if op == "pack":
        s["x"] = rows_of(n)
        return s
    if op == "norm" or case.get("layer") == "norm":
        s["x"], s["grad"] = rows_of(n), normal(m, n).to(dtype)
        s["weight"], s["bias"] = (1 + 0.2 * normal(n)).to(dtype), (0.2 * normal(n)).to(dtype)
        return s
    k = case["k"]
    s["x"] = rows_of(k)
    lead = (case["groups"],) if op == "grouped" else ()
    # the Xavier bound of the framework's initial weights, at the inputs' spread
    s["weight"] = ((2 * torch.rand(lead + (k, n), generator=gen, device="cuda") - 1) * math.sqrt(6.0 / (k + n)) * 0.7).to(dtype)
    s["bias"] = (0.2 * normal(*lead, n)).to(dtype)
    s["residual"] = normal(m, n).to(dtype) if case.get("residual") else None
    if case.get("step", op == "ckpt"):
        s["grad"] = normal(m, n).to(dtype)
    if op == "grouped":
        # class sizes that differ by a factor of a few, every eighth class without rows: their running sums, as the caller
        # who sorted the rows by class has them, and the largest of them
        share = torch.exp(0.5 * normal(case["groups"])).double()
        share[5::8] = 0.0
        ends = torch.round(torch.cumsum(share, 0) / share.sum() * m).to(torch.int64)
        ends[-1] = m
        s["ends"] = ends
        s["most"] = int(torch.diff(ends, prepend=ends.new_zeros(1)).max())
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _act(z, name):
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    if name == "tanh":
        return torch.tanh(z)
    if name == "relu":
        return torch.clamp(z, min=0.0)
    if name == "elu":
        return torch.where(z > 0, z, torch.expm1(z))
    return z


def _act_grad(a, name):
    """The activation's derivative, from its value."""
    if name == "sigmoid":
        return a * (1.0 - a)
    if name == "tanh":
        return 1.0 - a * a
    if name == "relu":
        return (a > 0).to(a.dtype)
    if name == "elu":
        return torch.where(a < 0, a + 1.0, torch.ones_like(a))
    return torch.ones_like(a)


def _packed(x, dtype):
    """The values that the 8-bit form of ``x`` (values of ``dtype``, in 32 bits) stands for: whole numbers up to 127 times the
    smallest power of two with which the largest of 32 columns fits, halves to even."""
    m, n = x.shape
    short = -n % BLOCK
    b = torch.cat([x, x.new_zeros(m, short)], 1).reshape(m, -1, BLOCK)
    top = b.abs().amax(2, keepdim=True)
    low = -24 if dtype == torch.float16 else -126
    e = torch.frexp(top)[1] - 7                                             # top < 128 * 2^e
    e = torch.where(top > torch.ldexp(torch.full_like(top, 127.0), e), e + 1, e)
    e = torch.where(top > 0, e, torch.full_like(e, low)).clamp(min=low)
    up, down = ((127 + sign * e.to(torch.int32) << 23).view(torch.float32) for sign in (1, -1))     # 2^e, 2^-e to the bit
    return (torch.round(b * down) * up).reshape(m, -1)[:, :n]


def _dense_plain(s, packed=False):
    c, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    act = c["act"]
    a = _act(x @ w + b, act)
    y = (a if s["residual"] is None else a + s["residual"].float()).to(dtype)
    if "grad" not in s:
        return {"y": y}
    a = a.to(dtype).float()
    g = s["grad"].float()
    if packed:
        x, a = _packed(x, dtype), _packed(a, dtype)
    dz = g * _act_grad(a, act)
    return {"y": y, "dx": (dz @ w.t()).to(dtype), "dw": (x.t() @ dz).to(dtype), "db": dz.sum(0).to(dtype)}


def _norm_plain(s, packed=False):
    dtype = s["x"].dtype
    x, w, b, g = s["x"].float(), s["weight"].float(), s["bias"].float(), s["grad"].float()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + EPS)
    y = (x - mean) * rstd * w + b
    if packed:
        x = _packed(x, dtype)
    xhat = (x - mean) * rstd
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))
    return {"y": y.to(dtype), "mean": mean[:, 0], "rstd": rstd[:, 0], "dx": dx.to(dtype), "dw": (g * xhat).sum(0).to(dtype), "db": g.sum(0).to(dtype)}


def _spread(s):
    """Each row's class, and its place in a batch of ``most`` rows a class."""
    m = s["x"].shape[0]
    row = torch.arange(m, device="cuda")
    group = torch.searchsorted(s["ends"], row, right=True)
    begin = torch.cat([s["ends"].new_zeros(1), s["ends"][:-1]])
    return group, row - begin[group]


def _grouped_plain(s):
    c, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    act, k, n = c["act"], c["k"], c["n"]
    group, at = _spread(s)
    w = s["weight"].float()
    xs = torch.zeros(c["groups"], s["most"], k, device="cuda")
    xs[group, at] = s["x"].float()
    a = _act(torch.bmm(xs, w) + s["bias"].float()[:, None], act)
    y = a[group, at].to(dtype)
    if "grad" not in s:
        return {"y": y}
    dz = s["grad"].float() * _act_grad(y.float(), act)
    dzs = torch.zeros(c["groups"], s["most"], n, device="cuda")
    dzs[group, at] = dz
    dx = torch.bmm(dzs, w.transpose(1, 2).contiguous())[group, at]
    dw = torch.bmm(xs.transpose(1, 2).contiguous(), dzs)
    return {"y": y, "dx": dx.to(dtype), "dw": dw.to(dtype), "db": dzs.sum(1).to(dtype)}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _dense_own(s, packed=False):
    from smrt_amd.autoencode import dense, dense_backward, pack_rows
    x, w, b, act = s["x"], s["weight"], s["bias"], s["case"]["act"]
    if "grad" not in s:
        return {"y": dense(x, w, b, activation=act, residual=s["residual"])}
    kept = pack_rows(x) if packed else x
    y, saved = dense(x, w, b, activation=act, residual=s["residual"], save="packed" if packed else "activation")
    dx, dw, db = dense_backward(s["grad"], kept, w, saved, activation=act)
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _norm_own(s, packed=False):
    from smrt_amd.autoencode import layer_norm, layer_norm_backward, pack_rows
    kept = pack_rows(s["x"]) if packed else s["x"]
    y, mean, rstd = layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
    dx, dw, db = layer_norm_backward(s["grad"], kept, mean, rstd, s["weight"])
    return {"y": y, "mean": mean, "rstd": rstd, "dx": dx, "dw": dw, "db": db}


def _grouped_own(s):
    from smrt_amd.autoencode import dense_grouped, dense_grouped_backward
    x, ends, w, b, act = s["x"], s["ends"], s["weight"], s["bias"], s["case"]["act"]
    if "grad" not in s:
        return {"y": dense_grouped(x, ends, w, b, activation=act)}
    y, saved = dense_grouped(x, ends, w, b, activation=act, save="activation")
    dx, dw, db = dense_grouped_backward(s["grad"], x, ends, w, saved, activation=act)
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def run(state):
    op = state["case"]["op"]
    layer = state["case"].get("layer", op)
    if own:
        if op == "pack":
            from smrt_amd.autoencode import pack_rows, unpack_rows
            return {"x": unpack_rows(pack_rows(state["x"]))}
        if op == "grouped":
            return _grouped_own(state)
        return (_norm_own if layer == "norm" else _dense_own)(state, op == "ckpt")
    if op == "pack":
        return {"x": _packed(state["x"].float(), state["x"].dtype).to(state["x"].dtype)}
    if op == "grouped":
        return _grouped_plain(state)
    return (_norm_plain if layer == "norm" else _dense_plain)(state, op == "ckpt")


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    m, n, op = case["rows"], case["n"], case["op"]
    eight = m * n + m * -(-n // BLOCK)                                          # the 8-bit form of [m, n]
    if op == "pack":
        return {"bytes": 2 * m * n * size + 2 * eight, "flops": 4 * m * n}
    if op == "norm" or case.get("layer") == "norm":
        # forward reads x and writes y; backward reads the gradient and what was kept of x, and writes dx; the statistics both ways
        kept = 2 * eight if op == "ckpt" else m * n * size
        return {"bytes": 4 * m * n * size + kept + 16 * m + 5 * n * size, "flops": 18 * m * n}
    k, groups = case["k"], case.get("groups", 1)
    some = groups - len(range(5, groups, 8)) if op == "grouped" else 1           # classes with rows
    some = min(some, m)
    weights = (k * n + n) * size
    b = m * k * size + some * weights + m * n * size * (2 if case.get("residual") else 1)
    f = 2 * m * k * n
    if case.get("step", op == "ckpt"):
        act = case.get("act") != "identity"
        if op == "ckpt":
            kept_x = m * k + m * -(-k // BLOCK)
            b += 2 * kept_x + 2 * eight * act
        else:
            b += m * k * size + m * n * size * act * (2 if case.get("residual") else 1)
        b += m * n * size + some * k * n * size + m * k * size + groups * weights     # grad and weights in, gradients out
        f *= 3
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def _exact_packed(v, dtype):
    """8-bit values of ``v`` (64 bits), written with logarithms of the block maxima instead of their exponents."""
    m, n = v.shape
    wide = torch.zeros(m, -(-n // BLOCK) * BLOCK, dtype=torch.float64, device=v.device)
    wide[:, :n] = v
    blocks = wide.view(m, -1, BLOCK)
    top = blocks.abs().max(dim=2).values
    e = torch.ceil(torch.log2(top / 127.0))
    e = torch.maximum(e, torch.full_like(e, -24.0 if dtype == torch.float16 else -126.0))
    scale = ((e.long() + 1023) << 52).view(torch.float64)[:, :, None]
    return (torch.round(blocks / scale) * scale).reshape(m, -1)[:, :n]


def _exact_dense(x, w, b, r, g, act, dtype, packed):
    z = torch.addmm(b, x, w)
    a = {"sigmoid": torch.sigmoid, "tanh": torch.tanh, "relu": torch.relu, "elu": torch.nn.functional.elu, "identity": torch.clone}[act](z)
    y = a if r is None else a + r
    if g is None:
        return {"y": y}
    a = a.to(dtype).double()                                   # what the layer hands to its backward pass
    if packed:
        a, x = _exact_packed(a, dtype), _exact_packed(x, dtype)
    slope = {"sigmoid": lambda: a - a * a, "tanh": lambda: (1 - a) * (1 + a), "relu": lambda: (a > 0).double(),
             "elu": lambda: torch.clamp(a, max=0.0) + 1.0, "identity": lambda: 1.0}[act]()
    dz = g * slope
    return {"y": y, "dx": torch.mm(dz, w.t()), "dw": torch.mm(x.t(), dz), "db": dz.sum(dim=0)}


def exact(case, seed):
    s = prepare(case, seed)
    dtype = DTYPES[case["dtype"]]
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    op = case["op"]
    if op == "pack":
        return {"x": _exact_packed(d["x"], dtype)}
    if op == "norm" or case.get("layer") == "norm":
        n = case["n"]
        x, g = d["x"], d["grad"]
        mu = x.sum(1) / n
        r = ((x * x).sum(1) / n - mu * mu + EPS) ** -0.5
        y = (x - mu[:, None]) * r[:, None] * d["weight"] + d["bias"]
        if op == "ckpt":
            x = _exact_packed(x, dtype)
        h = (x - mu[:, None]) * r[:, None]
        gw = g * d["weight"]
        dx = (n * gw - gw.sum(1, keepdim=True) - h * (gw * h).sum(1, keepdim=True)) * (r / n)[:, None]
        return {"y": y, "mean": mu, "rstd": r, "dx": dx, "dw": (g * h).sum(0), "db": g.sum(0)}
    if op != "grouped":
        return _exact_dense(d["x"], d["weight"], d["bias"], d.get("residual"), d.get("grad"), case["act"], dtype, op == "ckpt")
    ends = [0] + s["ends"].tolist()
    parts = [_exact_dense(d["x"][lo:hi], d["weight"][i], d["bias"][i], None, d["grad"][lo:hi] if "grad" in d else None, case["act"], dtype, False)
             for i, (lo, hi) in enumerate(zip(ends[:-1], ends[1:]))]
    return {k: torch.cat([p[k] for p in parts]) if k in ("y", "dx") else torch.stack([p[k] for p in parts]) for k in parts[0]}
