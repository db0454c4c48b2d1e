"""Layer operators on the GPU against their formulas in 64 bits on the CPU.

Tolerances are bounds of the arithmetic, element by element.  u = 2^-24 (fp32), half = eps / 2 of the result's type.  A sum of K products in fp32, in any
order, is off by at most 2 (K + 10) u times the sum of the magnitudes (the factor 2: the matrix cores' inner additions are not
specified to round to nearest).  An activation has slope <= 1 and its own error is a few u of 1 + |z|.  Storing rounds by half, twice
where a rounded value goes into a product (dz)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]
ACTS = ["identity", "sigmoid", "tanh", "relu", "elu"]
U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps      # the step below the normal numbers


def make(rng, dtype, *shape, scale=1.0):
    """Values of dtype as a CPU tensor."""
    return torch.from_numpy(rng.standard_normal(shape) * scale).to(dtype)


def odd_rows(t, lead=3, offset=1):
    """The same matrix on the GPU with rows that start at odd places."""
    big = torch.full(t.shape[:-1] + (t.shape[-1] + lead + offset,), float("nan"), dtype=t.dtype, device="cuda")
    view = big[..., offset:offset + t.shape[-1]]
    view.copy_(t)
    return view


def act64(z, name):
    return {"identity": lambda: z, "sigmoid": lambda: 1 / (1 + torch.exp(-z)), "tanh": lambda: torch.tanh(z), "relu": lambda: torch.where(z < 0, 0.0, z),
            "elu": lambda: torch.where(z > 0, z, torch.expm1(z))}[name]()


def slope64(a, name):
    return {"identity": lambda: torch.ones_like(a), "sigmoid": lambda: a * (1 - a), "tanh": lambda: 1 - a * a, "relu": lambda: (a > 0).double(),
            "elu": lambda: torch.where(a < 0, a + 1, 1.0)}[name]()


def close(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol) & ~((got == want) | (got.isnan() & want.isnan()))
    assert not bad.any(), "%s: %d of %d off, first at %s: got %r, want %r, tol %r" % (
        what, int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item(),
        tol[bad][0].item() if isinstance(tol, torch.Tensor) and tol.shape == bad.shape else tol)


def product_tol(a, b, k):
    return 2 * (k + 10) * U * (a.abs() @ b.abs())


def check_dense(x, w, b, r, act, y, saved=None, dtype=F32):
    """Forward result (and saved activation, None to skip) of CPU inputs; returns nothing."""
    X, W = x.double(), w.double()
    z = X @ W + (0 if b is None else b.double())
    zt = product_tol(X, W, X.shape[1]) + 4 * U * z.abs()
    a = act64(z, act)
    at = zt + 8 * U * (1 + a.abs())
    out = a + (0 if r is None else r.double())
    close(y, out, at + 2 * U * out.abs() + half(dtype) * (out.abs() + at) + tiny(dtype), "y")
    if saved is not None:
        close(saved, a, at + half(dtype) * (a.abs() + at) + tiny(dtype), "saved")


def check_dense_backward(g, x, w, a, act, dx, dw, db, dtype=F32):
    """Gradients at CPU values g, x, w and the activation's value a (None: identity)."""
    G, X, W = g.double(), x.double(), w.double()
    s = slope64(a.double(), act) if a is not None else torch.ones_like(G)
    dz = G * s
    dzt = 4 * U * G.abs()                                       # the slope's few roundings, in fp32
    rt = dzt + half(dtype) * dz.abs() + tiny(dtype) if act != "identity" else torch.zeros_like(dz)
    m, n = G.shape
    if dx is not None:
        want, D = dz @ W.T, dz.abs() + rt
        tol = product_tol(D, W.T, n) + rt @ W.abs().T
        close(dx, want, tol + half(dtype) * (want.abs() + tol) + tiny(dtype), "dx")
    if dw is not None:
        want = X.T @ dz
        tol = product_tol(X.T, dz.abs() + rt, m) + X.abs().T @ rt
        close(dw, want, tol + half(dtype) * (want.abs() + tol) + tiny(dtype), "dw")
    if db is not None:
        want = dz.sum(0)
        tol = 2 * (m + 10) * U * dz.abs().sum(0) + dzt.sum(0)
        close(db, want, tol + half(dtype) * (want.abs() + tol) + tiny(dtype), "db")


SIZES = [(1, 1, 1), (1, 64, 64), (2, 3, 5), (3, 129, 1), (5, 1, 130), (7, 45, 33), (16, 64, 128), (31, 33, 31), (33, 96, 100), (64, 128, 64), (65, 65, 65),
         (127, 130, 129), (128, 256, 128), (129, 31, 257), (300, 100, 60), (600, 450, 10), (1100, 20, 450), (257, 784, 450)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("i", range(len(SIZES)), ids=[str(s) for s in SIZES])
def test_dense_forward_and_backward(i, dtype):
    from smrt_amd.autoencode import dense, dense_backward
    m, k, n = SIZES[i]
    rng = np.random.default_rng(1000 + i)
    act, with_b, with_r, odd = ACTS[(i + DTYPES.index(dtype)) % 5], i % 3 != 0, i % 2 == 1, i % 4 in (1, 2)
    x, w, b = make(rng, dtype, m, k), make(rng, dtype, k, n, scale=k ** -0.5), make(rng, dtype, n) if with_b else None
    r, g = make(rng, dtype, m, n) if with_r else None, make(rng, dtype, m, n)
    put = odd_rows if odd else (lambda v: v.cuda())
    dev = lambda v: None if v is None else put(v)
    y, saved = dense(dev(x), dev(w), None if b is None else b.cuda(), residual=dev(r), activation=act, save="activation")
    assert y.dtype == dtype and (saved is None) == (act == "identity") and (saved is y) == (act != "identity" and r is None)
    check_dense(x, w, b, r, act, y, saved, dtype)
    a = None if saved is None else saved.cpu()
    dx, dw, db = dense_backward(dev(g), dev(x), dev(w), None if saved is None else put(a), activation=act)
    check_dense_backward(g, x, w, a, act, dx, dw, db, dtype)
    only = dense_backward(dev(g), dev(x), dev(w), saved, activation=act, need_x=False, need_weight=False)
    assert only[0] is None and only[1] is None and torch.equal(only[2], db)
    only = dense_backward(dev(g), dev(x), dev(w), saved, activation=act, need_weight=False, need_bias=False)
    assert torch.equal(only[0], dx) and only[1] is None and only[2] is None


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("act", ACTS)
def test_dense_every_activation(act, dtype):
    from smrt_amd.autoencode import dense, dense_backward
    rng = np.random.default_rng(7)
    m, k, n = 70, 96, 72
    x, w, b, g = make(rng, dtype, m, k, scale=3.0), make(rng, dtype, k, n, scale=0.3), make(rng, dtype, n), make(rng, dtype, m, n)
    y, saved = dense(x.cuda(), w.cuda(), b.cuda(), activation=act, save="activation")
    check_dense(x, w, b, None, act, y, saved, dtype)
    assert torch.equal(dense(x.cuda(), w.cuda(), b.cuda(), activation=act), y)
    a = None if saved is None else saved.cpu()
    check_dense_backward(g, x, w, a, act, *dense_backward(g.cuda(), x.cuda(), w.cuda(), saved, activation=act), dtype)


def test_dense_long_sum_of_rows_and_fp32_accuracy():
    """dW and db over many rows (slices that are joined), and fp32 products as exact as fp32 products are: an fp32 product rounds
    every addition, here 2e-6 of the norm is far below what two bf16 parts instead of three would give (1e-5)."""
    from smrt_amd.autoencode import dense, dense_backward
    rng = np.random.default_rng(3)
    m, k, n = 20000, 160, 130
    x, w, g = make(rng, F32, m, k), make(rng, F32, k, n, scale=0.1), make(rng, F32, m, n)
    dx, dw, db = dense_backward(g.cuda(), x.cuda(), w.cuda())
    check_dense_backward(g, x, w, None, "identity", dx, dw, db, F32)
    for got, want in ((dx, g.double() @ w.double().T), (dw, x.double().T @ g.double()), (db, g.double().sum(0)),
                      (dense(x.cuda(), w.cuda()), x.double() @ w.double())):
        assert (got.cpu().double() - want).norm() <= 2e-6 * want.norm()
    again = dense_backward(g.cuda(), x.cuda(), w.cuda())
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


@pytest.mark.parametrize("m,k,n", [(0, 3, 4), (3, 0, 4), (3, 4, 0), (0, 0, 0)])
def test_dense_empty(m, k, n):
    from smrt_amd.autoencode import dense, dense_backward
    x, w, b, g = (torch.randn(s, device="cuda") for s in ((m, k), (k, n), (n,), (m, n)))
    y, saved = dense(x, w, b, activation="sigmoid", save="activation")
    assert y.shape == (m, n)
    if k == 0:
        close(y, torch.sigmoid(b.cpu().double()).expand(m, n), 8 * U, "y")
    dx, dw, db = dense_backward(g, x, w, saved, activation="sigmoid")
    assert dx.shape == (m, k) and dw.shape == (k, n) and db.shape == (n,)
    if m == 0:
        assert not dw.any() and not db.any()
    if n == 0:
        assert not dx.any()


def test_dense_not_finite():
    """Infinities and NaN go where the formula takes them, in fp32 too, whose numbers are multiplied in parts."""
    from smrt_amd.autoencode import dense, dense_backward
    rng = np.random.default_rng(5)
    for dtype in DTYPES:
        x, w = make(rng, dtype, 40, 70), make(rng, dtype, 70, 50)
        x[3, 5], x[7, 69], x[11, 0], x[12, 1] = float("inf"), float("-inf"), float("nan"), torch.finfo(dtype).max
        w[2, 9], w[4, 11] = float("inf"), 0.0
        z = x.double() @ w.double()
        big = z.abs() > torch.finfo(dtype).max * 0.9                # may or may not overflow: not compared
        y = dense(x.cuda(), w.cuda()).cpu().double()
        for f in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(f(y)[~big], f(z)[~big]) or dtype != F32 and torch.equal(f(y)[~big & z.isfinite()], f(z)[~big & z.isfinite()])
        assert torch.equal(y.isnan(), z.isnan())
        # a NaN that reaches the activation leaves it as NaN
        for act in ACTS:
            a = dense(x.cuda(), w.cuda(), activation=act).cpu()
            assert torch.equal(a.isnan(), z.isnan()), act
        g = torch.ones(40, 50, dtype=dtype)
        dx, dw, db = dense_backward(g.cuda(), x.cuda(), w.cuda())
        assert torch.equal(dw.cpu().isnan(), (x.double().T @ g.double()).isnan())
        assert db.isfinite().all()


def test_dense_small_and_large_numbers():
    """fp32 numbers whose lower parts are below the normal range, f16 numbers below it, and numbers near the largest."""
    from smrt_amd.autoencode import dense
    rng = np.random.default_rng(6)
    x, w = make(rng, F32, 33, 64), make(rng, F32, 64, 40)
    z = x.double() @ w.double()
    for s in (2.0 ** -100, 2.0 ** 120):
        y = dense((x * s).cuda(), w.cuda()).cpu().double() / s
        assert (y - z).norm() <= 2e-6 * z.norm()
    x = (torch.arange(64).reshape(4, 16).float() * 2.0 ** -24).to(F16)          # every one is below 2^-14
    w = torch.eye(16, dtype=F16)
    assert torch.equal(dense(x.cuda(), w.cuda()).cpu(), x)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_dense_out_and_residual_in_place(dtype):
    from smrt_amd import _hip
    from smrt_amd.autoencode import dense
    rng = np.random.default_rng(8)
    x, w, r = make(rng, dtype, 130, 50), make(rng, dtype, 50, 70, scale=0.2), make(rng, dtype, 130, 70)
    want = dense(x.cuda(), w.cuda(), residual=r.cuda(), activation="tanh")
    buf = odd_rows(r)
    got = dense(x.cuda(), w.cuda(), residual=buf, activation="tanh", out=buf)
    assert got is buf and torch.equal(buf, want)
    big = torch.full((134, 81), 7.0, dtype=dtype, device="cuda")
    dense(x.cuda(), w.cuda(), residual=r.cuda(), activation="tanh", out=big[2:132, 5:75])
    assert torch.equal(big[2:132, 5:75], want)
    big[2:132, 5:75] = 7.0
    assert (big == 7.0).all()                                    # nothing around it was written
    sq = make(rng, dtype, 70, 70).cuda()
    with pytest.raises(_hip.HipLibraryError):
        dense(sq, make(rng, dtype, 70, 70).cuda(), out=sq)
    with pytest.raises(_hip.HipLibraryError):
        dense(x.cuda(), w.cuda(), residual=big[1:131, 5:75], out=big[2:132, 5:75])


# ------------------------------------------------------------------------------------------------ 8 bits
def packed_reference(x, dtype):
    """q and scale bytes of a CPU matrix, by integer arithmetic on exact fractions of its values in 64 bits."""
    v = x.double().numpy()
    m, n = v.shape
    blocks = -(-n // 32)
    wide = np.zeros((m, blocks * 32))
    wide[:, :n] = v
    wide = wide.reshape(m, blocks, 32)
    q, scale = np.zeros((m, blocks, 32), np.int8), np.zeros((m, blocks), np.uint8)
    low, high = (-24, 10) if dtype == F16 else (-126, 122)
    for i in range(m):
        for j in range(blocks):
            b = wide[i, j]
            if not np.isfinite(b).all():
                scale[i, j] = 255
                continue
            top, e = np.abs(b).max(), low
            while top > 127 * 2.0 ** e:
                e += 1
            scale[i, j] = e + 127
            q[i, j] = np.clip(np.rint(b / 2.0 ** e), -63 if e == high else -127, 63 if e == high else 127)
    return torch.from_numpy(q.reshape(m, blocks * 32)), torch.from_numpy(scale)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,n", [(1, 1), (2, 31), (3, 32), (5, 33), (70, 100), (129, 450), (0, 5), (3, 0)])
def test_pack(m, n, dtype):
    from smrt_amd.autoencode import pack_rows, unpack_rows
    rng = np.random.default_rng(9)
    x = torch.from_numpy(rng.standard_normal((m, n)) * np.exp2(rng.integers(-12, 9, (m, 1)))).to(dtype)
    if m > 2 and n > 2:
        x[0], x[1, :2] = 0.0, torch.finfo(dtype).max
        x[2, 0], x[2, 1] = float("nan") if n > 40 else 1.0, -0.0
        x[2, -1] = float("-inf") if n == 450 else 2.0 ** -24
    for put in (lambda v: v.cuda(), odd_rows):
        p = pack_rows(put(x))
        q, scale = packed_reference(x, dtype)
        assert torch.equal(p.scale.cpu(), scale) and torch.equal(p.q.cpu(), q)
        assert p.shape == (m, n) and p.dtype == dtype
        v = unpack_rows(p).cpu()
        bits = np.ldexp(1.0, scale.numpy().astype(int) - 127)
        bits[scale.numpy() == 255] = np.nan
        want = (q.double().numpy().reshape(m, -(-n // 32), 32) * bits[:, :, None]).reshape(m, -(-n // 32) * 32)[:, :n]
        assert v.dtype == dtype
        close(v, torch.from_numpy(want), 0.0, "values")           # exact in every type
        again = pack_rows(v.cuda())                                # a packed matrix packs to itself, where the scale is the smallest
        close(unpack_rows(again).cpu(), v.double(), 0.0, "again")


def test_pack_borders():
    """The largest of a block just at, below and above 127 steps, halves to even, the lowest and the highest scales."""
    from smrt_amd.autoencode import pack_rows
    rows = [[127.0, 0.5, 1.5, 2.5, -0.5], [127.00001, 1.0, 3.0, 5.0], [126.5, 1.0], [254.0, 1.0, 3.0], [2.0 ** -126, 2.0 ** -127], [2.0 ** -140],
            [3.0e38, 1.0e38], [3.4028235e38, 2.0 ** 121], [2.0 ** -149]]
    x = torch.zeros(len(rows), 32)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r)
    p = pack_rows(x.cuda())
    q, scale = packed_reference(x, F32)
    assert torch.equal(p.scale.cpu(), scale) and torch.equal(p.q.cpu(), q)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,k,n,act", [(5, 3, 31, "tanh"), (130, 100, 70, "elu"), (257, 64, 450, "sigmoid"), (700, 33, 32, "relu"), (40, 200, 64, "identity")])
def test_checkpointed_dense(m, k, n, act, dtype):
    """The activation packed by the forward launch is the packed activation, and the backward pass is the one at the values that 8 bits stand for."""
    from smrt_amd.autoencode import dense, dense_backward, pack_rows, unpack_rows
    rng = np.random.default_rng(10)
    x, w, b, g = make(rng, dtype, m, k), make(rng, dtype, k, n, scale=k ** -0.5), make(rng, dtype, n), make(rng, dtype, m, n)
    r = make(rng, dtype, m, n).cuda()
    dev = [v.cuda() for v in (x, w, b)]
    y, a = dense(*dev, residual=r, activation=act, save="activation")
    y8, p = dense(*dev, residual=r, activation=act, save="packed")
    assert torch.equal(y, y8)
    if act == "identity":
        assert p is None and a is None
    else:
        want = pack_rows(a)
        assert torch.equal(p.q, want.q) and torch.equal(p.scale, want.scale)
    px = pack_rows(dev[0])
    got = dense_backward(g.cuda(), px, dev[1], p, activation=act)
    check_dense_backward(g, unpack_rows(px).cpu(), w, None if p is None else unpack_rows(p).cpu(), act, *got, dtype)


def test_checkpoint_of_not_finite_activations_gives_nan_gradients():
    from smrt_amd.autoencode import dense_backward, pack_rows
    x = torch.ones(40, 64)
    x[3, 40] = float("inf")
    g, w = torch.ones(40, 16), torch.ones(64, 16)
    for dtype in DTYPES:
        dx, dw, db = dense_backward(g.to(dtype).cuda(), pack_rows(x.to(dtype).cuda()), w.to(dtype).cuda())
        assert dw[32:].isnan().all() and dw[:32].isfinite().all() and dx.isfinite().all()


# ------------------------------------------------------------------------------------------------ groups
def sound_ends(ends, rows):
    out, last = [], 0
    for e in ends:
        last = max(last, min(max(e, 0), rows))
        out.append(last)
    return out


GROUPS = [(10, [10]), (10, [4]), (300, [0, 129, 129, 300]), (257, [1, 2, 3, 257]), (64, [64, 10, 64, -5]), (50, [1 << 40, 3]), (130, [-(1 << 62), 60, 50, 130]),
          (500, [128, 256, 384]), (0, [0, 0]), (200, sorted(np.random.default_rng(1).integers(0, 200, 70).tolist())),
          (900, sorted(np.random.default_rng(2).integers(0, 900, 150).tolist())), (1300, [1200, 1300]), (66, [0] * 64 + [66])]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("i", range(len(GROUPS)))
def test_grouped(i, dtype):
    from smrt_amd.autoencode import dense_grouped, dense_grouped_backward, pack_rows, unpack_rows
    m, ends = GROUPS[i]
    rng = np.random.default_rng(50 + i)
    k, n = ((40, 70), (64, 64), (33, 130))[i % 3]
    G, act, with_r = len(ends), ACTS[(i + DTYPES.index(dtype)) % 5], i % 2 == 0
    x, w, b, g = make(rng, dtype, m, k), make(rng, dtype, G, k, n, scale=k ** -0.5), make(rng, dtype, G, n), make(rng, dtype, m, n)
    r = make(rng, dtype, m, n) if with_r else None
    e_dev = torch.tensor(ends, dtype=torch.int64, device="cuda")
    wd = odd_rows(w) if i % 2 else w.cuda()
    xd, gd, bd = odd_rows(x), g.cuda(), b.cuda()
    y, saved = dense_grouped(xd, e_dev, wd, bd, residual=None if r is None else r.cuda(), activation=act, save="activation")
    dx, dw, db = dense_grouped_backward(gd, xd, e_dev, wd, saved, activation=act)
    px = pack_rows(xd)
    p_dx, p_dw, p_db = dense_grouped_backward(gd, px, e_dev, wd, saved, activation=act)
    assert torch.equal(p_dx, dx) and torch.equal(p_db, db)
    lo, x8 = 0, unpack_rows(px).cpu()
    for j, hi in enumerate(sound_ends(ends, m)):
        s = slice(lo, hi)
        a = None if saved is None else saved[s].cpu()
        check_dense(x[s], w[j], b[j], None if r is None else r[s], act, y[s], None if saved is None else saved[s], dtype)
        check_dense_backward(g[s], x[s], w[j], a, act, dx[s], dw[j], db[j], dtype)
        check_dense_backward(g[s], x8[s], w[j], a, act, None, p_dw[j], None, dtype)
        lo = hi
    assert not y[lo:].any() and not dx[lo:].any()                # rows of no class
    out = torch.full_like(y, 5.0)
    dense_grouped(xd, e_dev, wd, bd, residual=None if r is None else r.cuda(), activation=act, out=out)
    assert torch.equal(out[:lo], y[:lo]) and (out[lo:] == 5.0).all()


def test_grouped_is_dense_for_one_group():
    from smrt_amd.autoencode import dense, dense_grouped
    x, w = torch.randn(300, 90, device="cuda"), torch.randn(90, 64, device="cuda")
    assert torch.equal(dense_grouped(x, torch.tensor([300], device="cuda"), w[None]), dense(x, w))


# ------------------------------------------------------------------------------------------------ layer norm
NORMS = [(1, 1), (3, 2), (33, 7), (5, 8), (200, 63), (31, 64), (128, 65), (17, 128), (40, 200), (9, 256), (70, 450), (8, 512), (6, 513), (700, 784), (3, 1024),
         (5, 1500), (2, 2048), (3, 4000), (2, 9000), (2, 20000), (1, 32768), (0, 64), (3000, 40)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("i", range(len(NORMS)), ids=[str(s) for s in NORMS])
def test_layer_norm(i, dtype):
    from smrt_amd.autoencode import layer_norm, layer_norm_backward, pack_rows, unpack_rows
    m, n = NORMS[i]
    rng = np.random.default_rng(200 + i)
    wt = F32 if i % 3 == 0 else dtype
    x, g = make(rng, dtype, m, n), make(rng, dtype, m, n)
    if m > 2:
        x[1] = 3.0                                               # a row without variance
        x[2] = (x[2].double() * 0.01 + 50).to(dtype)             # a mean far above the spread
    w = None if i % 5 == 4 else make(rng, wt, n)
    b = None if w is None or i % 4 == 3 else make(rng, wt, n)
    put = odd_rows if i % 2 else (lambda v: v.cuda())
    wd, bd = (None if v is None else v.cuda() for v in (w, b))
    y, mean, rstd = layer_norm(put(x), wd, bd, eps=1e-5)
    X, G = x.double(), g.double()
    W = torch.ones(n, dtype=torch.float64) if w is None else w.double()
    mu = X.mean(1, keepdim=True)
    d = X - mu
    var = (d * d).mean(1, keepdim=True)
    rs = (var + 1e-5) ** -0.5
    # the mean is off by (n + 2) u of the mean magnitude, a difference by that much too; the variance is second order in it
    mt = 2 * (n + 4) * U * X.abs().mean(1, keepdim=True)
    dt = mt + U * X.abs()
    vt = 2 * (n + 8) * U * var + 2 * (d.abs() * dt).mean(1, keepdim=True) + (dt * dt).mean(1, keepdim=True)
    rt = rs * (0.5 * vt / (var + 1e-5) * 1.5 + 8 * U)
    close(mean, mu[:, 0], mt[:, 0], "mean")
    close(rstd, rs[:, 0], rt[:, 0], "rstd")
    want = d * rs * W + (0 if b is None else b.double())
    tol = (dt * rs + d.abs() * rt + dt * rt) * W.abs() + 8 * U * ((d * rs * W).abs() + want.abs())
    close(y, want, tol + half(dtype) * (want.abs() + tol) + tiny(dtype), "y")
    # the backward pass from the statistics that the forward pass gave
    for packed in (False, True):
        kept = pack_rows(put(x)) if packed else put(x)
        K = unpack_rows(kept).cpu().double() if packed else X
        dx, dw, db = layer_norm_backward(put(g), kept, mean, rstd, wd)
        M, R = mean.cpu().double()[:, None], rstd.cpu().double()[:, None]
        h, gw = (K - M) * R, G * W
        s1, s2 = gw.mean(1, keepdim=True), (gw * h).mean(1, keepdim=True)
        want = R * (gw - s1 - h * s2)
        ht = 3 * U * h.abs()
        c = 2 * (n + 8) * U
        s1t, s2t = c * gw.abs().mean(1, keepdim=True), c * (gw * h).abs().mean(1, keepdim=True) + (gw.abs() * ht).mean(1, keepdim=True)
        tol = R * (s1t + h.abs() * s2t + ht * s2.abs() + 8 * U * (gw.abs() + s1.abs() + (h * s2).abs()))
        close(dx, want, tol + half(dtype) * (want.abs() + tol) + tiny(dtype), "dx")
        if w is None:
            assert dw is None and db is None
            continue
        c = 2 * (m + 10) * U
        tol = c * (G * h).abs().sum(0) + (G.abs() * ht).sum(0)
        close(dw, (G * h).sum(0), tol + half(wt) * ((G * h).sum(0).abs() + tol) + tiny(wt), "dw")
        tol = c * G.abs().sum(0)
        close(db, G.sum(0), tol + half(wt) * (G.sum(0).abs() + tol) + tiny(wt), "db")


def test_layer_norm_many_rows_and_not_finite():
    from smrt_amd.autoencode import layer_norm, layer_norm_backward
    torch.manual_seed(0)
    x, g, w = torch.randn(30001, 72, device="cuda"), torch.randn(30001, 72, device="cuda"), torch.randn(72, device="cuda")
    x[5, 3], x[9, 0] = float("nan"), float("inf")
    y, mean, rstd = layer_norm(x, w)
    bad = torch.zeros(30001, dtype=torch.bool, device="cuda")
    bad[5] = bad[9] = True
    assert torch.equal(y.isnan().all(1), bad) and torch.equal(y.isnan().any(1), bad)
    g[5], g[9] = 0, 0
    dx, dw, db = layer_norm_backward(g, x, mean, rstd, w)
    assert torch.equal(dx.isnan().any(1), bad)
    first = layer_norm_backward(g[10:], x[10:], mean[10:], rstd[10:], w)
    h = (x[10:].double() - mean[10:, None].double()) * rstd[10:, None].double()
    assert ((first[1].double() - (g[10:].double() * h).sum(0)).norm() <= 1e-6 * (g[10:].double() * h).sum(0).norm())
    assert all(torch.equal(p, q) for p, q in zip(first, layer_norm_backward(g[10:], x[10:], mean[10:], rstd[10:], w)))
    only = layer_norm_backward(g[10:], x[10:], mean[10:], rstd[10:], w, need_x=False, need_weight=False)
    assert only[0] is None and only[1] is None and torch.equal(only[2], first[2])
    z = x[10:40].clone()
    want = layer_norm(z, w)[0]
    assert layer_norm(z, w, out=z)[0] is z and torch.equal(z, want)          # in place


# ------------------------------------------------------------------------------------------------ together, differences, streams, graphs
def block(x, p, ends, eight):
    """A pre-norm residual block whose layers keep their inputs (in 8 bits), forward."""
    from smrt_amd.autoencode import dense, dense_grouped, layer_norm, pack_rows
    h, mean, rstd = layer_norm(x, p["gamma"], p["beta"])
    u, su = dense(h, p["w1"], p["b1"], activation="tanh", save="packed" if eight else "activation")
    y, _ = dense_grouped(u, ends, p["w2"], p["b2"], residual=x, save="activation")
    keep = pack_rows if eight else (lambda v: v)
    return y, (keep(x), mean, rstd, keep(h), su if eight else u, su)


def block_backward(gy, p, ends, kept):
    from smrt_amd.autoencode import dense_backward, dense_grouped_backward, layer_norm_backward
    x, mean, rstd, h, u, su = kept
    du, dw2, db2 = dense_grouped_backward(gy, u, ends, p["w2"])
    dh, dw1, db1 = dense_backward(du, h, p["w1"], su, activation="tanh")
    dx, dg, dbeta = layer_norm_backward(dh, x, mean, rstd, p["gamma"])
    return {"x": dx + gy, "w1": dw1, "b1": db1, "w2": dw2, "b2": db2, "gamma": dg, "beta": dbeta}


def block_inputs(dtype, m=200, d=96, hid=130, groups=3, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s, scale=1.0: (torch.randn(s, generator=gen) * scale).to(dtype).cuda()
    p = {"gamma": 1 + r(d, scale=0.2), "beta": r(d, scale=0.2), "w1": r(d, hid, scale=d ** -0.5), "b1": r(hid, scale=0.1),
         "w2": r(groups, hid, d, scale=hid ** -0.5), "b2": r(groups, d, scale=0.1)}
    return r(m, d), p, torch.tensor([m // 4, m // 4, m], device="cuda"), r(m, d)


def test_block_against_autograd_in_64_bits():
    x, p, ends, gy = block_inputs(F32)
    y, kept = block(x, p, ends, False)
    got = block_backward(gy, p, ends, kept)
    leaves = {k: v.cpu().double().requires_grad_() for k, v in dict(p, x=x).items()}
    L = leaves
    h = torch.nn.functional.layer_norm(L["x"], (96,), L["gamma"], L["beta"], 1e-5)
    u = torch.tanh(h @ L["w1"] + L["b1"])
    e = [0] + ends.tolist()
    out = torch.cat([u[e[g]:e[g + 1]] @ L["w2"][g] + L["b2"][g] for g in range(3)]) + L["x"]
    out.backward(gy.cpu().double())
    assert (y.cpu().double() - out).norm() <= 2e-6 * out.norm()
    for k, v in leaves.items():
        assert (got[k].cpu().double() - v.grad).norm() <= 5e-6 * max(v.grad.norm(), 1e-30), k


def test_checkpointed_block_is_near_the_exact_one():
    """8 bits hold a block of 32 to half a step, 1/254 to 1/127 of its largest value: for normal values, largest 2 to 2.6 spreads, that is 0.3 to
    0.6 percent of a value's spread (uniform error: half a step over sqrt 3).  A gradient passes through three such layers, and tanh's
    slope 1 - a^2 doubles a's error: 3 percent holds them with room."""
    x, p, ends, gy = block_inputs(F32)
    exact, near = (block_backward(gy, p, ends, block(x, p, ends, e)[1]) for e in (False, True))
    for k in exact:
        assert (near[k] - exact[k]).norm() <= 0.03 * exact[k].norm(), k


@pytest.mark.parametrize("name", ["x", "w1", "b1", "w2", "b2", "gamma", "beta"])
def test_block_gradient_is_the_difference_quotient(name):
    """Along a direction v: (L(t + h v) - L(t - h v)) / 2 h, L summed in 64 bits from fp32 outputs.  Truncation is h^2 times a third derivative, the
    outputs' errors (2e-6 of their norm) come in over 2 h: with h = 0.01 both stay below 1 percent of |grad| |v| / sqrt(size)."""
    x, p, ends, gy = block_inputs(F32, m=150)
    got = block_backward(gy, p, ends, block(x, p, ends, False)[1])[name]
    gen = torch.Generator().manual_seed(3)
    v = torch.randn(got.shape, generator=gen).cuda() + got / got.norm() * got.numel() ** 0.5
    v = v / v.norm() * got.numel() ** 0.5 * (0.1 if name.startswith("w") else 1.0)
    loss = lambda q, z: (block(z, q, ends, False)[0].double() * gy.double()).sum()
    step = lambda s: loss(p, x + s * v) if name == "x" else loss(dict(p, **{name: p[name] + s * v}), x)
    slope = (step(0.01) - step(-0.01)) / 0.02
    assert abs(float(slope - (got.double() * v.double()).sum())) <= 0.01 * float(got.norm() * v.norm())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_block_on_another_stream_and_in_two_graphs(dtype):
    x, p, ends, gy = block_inputs(dtype)
    y, kept = block(x, p, ends, True)
    want = block_backward(gy, p, ends, kept)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2, kept2 = block(x, p, ends, True)
        got = block_backward(gy, p, ends, kept2)
    side.synchronize()
    assert torch.equal(y2, y) and all(torch.equal(got[k], want[k]) for k in want)
    # two graphs of different inputs, replayed in turn with eager work between them
    sets, graphs = [(x.clone(), gy.clone()), tuple(v.clone() for v in block_inputs(dtype, seed=1)[0::3])], []
    eager = []
    for z, g in sets:
        ye, ke = block(z, p, ends, True)
        eager.append((ye, block_backward(g, p, ends, ke)))
    torch.cuda.synchronize()
    for z, g in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            yg, kg = block(z, p, ends, True)
            out = block_backward(g, p, ends, kg)
        graphs.append((graph, yg, out))
    for turn in range(4):
        for graph, yg, out in graphs:
            yg.zero_()
            for v in out.values():
                v.zero_()
        for i in ((0, 1), (1, 0))[turn % 2]:
            graphs[i][0].replay()
            block(x, p, ends, True)
        torch.cuda.synchronize()
        for (graph, yg, out), (ye, oe) in zip(graphs, eager):
            assert torch.equal(yg, ye) and all(torch.equal(out[k], oe[k]) for k in oe)


def test_rows_past_32_bits():
    """Offsets in bytes and in elements past 2^32: the last rows of a matrix of 2.2e9 elements."""
    from smrt_amd.autoencode import dense, dense_backward, layer_norm, pack_rows, unpack_rows
    rows, ld = 530000, 4160
    big = torch.zeros(rows, ld, dtype=BF16, device="cuda")
    x = big[:, 4096:]
    tail = torch.randn(64, 64).to(BF16)
    x[-64:] = tail.cuda()
    w = torch.randn(64, 32).to(BF16)
    y = dense(x, w.cuda())
    check_dense(tail, w, None, None, "identity", y[-64:], None, BF16)
    assert not y[:-64].any()
    g = torch.randn(64, 32).to(BF16)
    full = torch.zeros(rows, 32, dtype=BF16, device="cuda")
    full[-64:] = g.cuda()
    dx, dw, db = dense_backward(full, x, w.cuda())
    check_dense_backward(g, tail, w, None, "identity", dx[-64:], dw, db, BF16)
    assert torch.equal(layer_norm(x)[0][-64:], layer_norm(tail.cuda())[0])
    assert torch.equal(unpack_rows(pack_rows(x))[-64:], unpack_rows(pack_rows(tail.cuda())))


TILES = [(16500, 100, 700), (70000, 40, 260), (5000, 300, 1030), (4200, 1032, 520), (3001, 515, 2050), (33000, 257, 263)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("i", range(len(TILES)), ids=[str(s) for s in TILES])
def test_dense_larger_tiles(i, dtype):
    """Sizes that get the larger product tiles, with edges in every direction; rows at odd places for every other one."""
    from smrt_amd.autoencode import dense, dense_backward, pack_rows, unpack_rows
    m, k, n = TILES[i]
    rng = np.random.default_rng(300 + i)
    x, w, g = make(rng, dtype, m, k), make(rng, dtype, k, n, scale=k ** -0.5), make(rng, dtype, m, n)
    put = odd_rows if i % 2 else (lambda v: v.cuda())
    y = dense(put(x), put(w))
    check_dense(x, w, None, None, "identity", y, None, dtype)
    dx, dw, db = dense_backward(put(g), put(x), put(w))
    check_dense_backward(g, x, w, None, "identity", dx, dw, db, dtype)
    px = pack_rows(put(x))
    _, dw, _ = dense_backward(put(g), px, put(w), need_x=False, need_bias=False)
    check_dense_backward(g, unpack_rows(px).cpu(), w, None, "identity", None, dw, None, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_grouped_larger_tiles(dtype):
    from smrt_amd.autoencode import dense_grouped, dense_grouped_backward
    rng = np.random.default_rng(400)
    ends, m, k, n = [9000, 9000, 21001, 40000], 40100, 130, 270
    x, w, b, g = make(rng, dtype, m, k), make(rng, dtype, 4, k, n, scale=k ** -0.5), make(rng, dtype, 4, n), make(rng, dtype, m, n)
    e = torch.tensor(ends, device="cuda")
    y, saved = dense_grouped(x.cuda(), e, w.cuda(), b.cuda(), activation="sigmoid", save="activation")
    dx, dw, db = dense_grouped_backward(g.cuda(), x.cuda(), e, w.cuda(), saved, activation="sigmoid")
    lo = 0
    for j, hi in enumerate(ends):
        s, a = slice(lo, hi), saved[lo:hi].cpu()
        check_dense(x[s], w[j], b[j], None, "sigmoid", y[s], saved[s], dtype)
        check_dense_backward(g[s], x[s], w[j], a, "sigmoid", dx[s], dw[j], db[j], dtype)
        lo = hi
    assert not y[lo:].any() and not dx[lo:].any()


# ------------------------------------------------------------------------------------------------ the classes' decoders
@pytest.fixture(scope="module")
def fitted():
    from smrt_amd.autoencode import VariationalAutoEncoder
    rs = np.random.RandomState(0)
    return [VariationalAutoEncoder([40, 24], 5, activation_function="elu", n_epochs=2, batch_size=32, learning_rate=0.01, random_state=i).fit(
        rs.uniform(size=(70 + 30 * i, 50))) for i in range(3)]


def test_class_decoders_match_the_estimators(fitted):
    """fp32: the same products and activations in another order of summation; 1e-4 is the agreement that all paths of the decoder are held to."""
    from smrt_amd.autoencode import ClassDecoders
    d = ClassDecoders(fitted)
    rs = np.random.RandomState(1)
    z, ends = rs.normal(size=(90, 5)).astype(np.float32), [20, 20, 85]
    got = d.decode(torch.from_numpy(z).cuda(), torch.tensor(ends, device="cuda")).cpu().numpy()
    assert got.shape == (90, 50)
    np.testing.assert_allclose(got[:20], fitted[0].feed_forward(z[:20]), rtol=1e-4, atol=1e-6)
    np.testing.assert_allclose(got[20:85], fitted[2].feed_forward(z[20:85]), rtol=1e-4, atol=1e-6)


def test_class_decoders_generate_is_the_estimators_generate(fitted):
    from smrt_amd.autoencode import ClassDecoders
    counts = [7, 0, 30]
    got = ClassDecoders(fitted).generate(counts, np.random.RandomState(5), loc=0.1, scale=0.5).cpu().numpy()
    rs, want = np.random.RandomState(5), []
    for e, n in zip(fitted, counts):
        want.append(e.feed_forward(rs.normal(0.1, 0.5, size=(n, 5))) if n else np.zeros((0, 50), np.float32))
    np.testing.assert_allclose(got, np.concatenate(want), rtol=1e-4, atol=1e-6)
    with pytest.raises(ValueError):
        ClassDecoders(fitted).generate([1, 2], np.random.RandomState(0))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
def test_class_decoders_in_16_bits(fitted, dtype):
    """Against the chain in 64 bits on the rounded weights, with each layer's rounding carried on by the next layer's weights."""
    from smrt_amd.autoencode import ClassDecoders
    d = ClassDecoders(fitted, dtype)
    z = make(np.random.default_rng(2), dtype, 64, 5)
    ends = [30, 50, 64]
    got = d.decode(z.cuda(), torch.tensor(ends, device="cuda"))
    lo = 0
    for c, hi in enumerate(ends):
        a, e = z[lo:hi].double(), torch.zeros(hi - lo, 5, dtype=torch.float64)
        for w, b, act in d.layers:
            W = w[c].cpu().double()
            e = e @ W.abs() + product_tol(a.abs() + e, W, W.shape[0]) + 8 * U
            a = act64(a @ W + b[c].cpu().double(), act)
            e = e + 8 * U * (1 + a.abs())
            e = e + half(dtype) * (a.abs() + e) + tiny(dtype)
        close(got[lo:hi], a, e, "class %d" % c)
        lo = hi


def test_class_decoders_refuse_other_shapes(fitted):
    from smrt_amd.autoencode import ClassDecoders, VariationalAutoEncoder
    other = VariationalAutoEncoder(24, 5, n_epochs=1, batch_size=32, random_state=0).fit(np.random.RandomState(0).uniform(size=(40, 50)))
    with pytest.raises(ValueError):
        ClassDecoders([fitted[0], other])


ROWS = [(1, 64, 64), (1, 1100, 70), (2, 5, 1030), (7, 700, 9), (20, 513, 300), (32, 130, 1000), (33, 40, 64), (64, 65, 520), (3, 8, 8), (5, 1, 1)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("i", range(len(ROWS)), ids=[str(s) for s in ROWS])
def test_dense_few_rows(i, dtype):
    """The kernels for a few rows, at their limits and over several steps of each sum, from tensors and from 8-bit forms."""
    from smrt_amd.autoencode import dense, dense_backward, pack_rows, unpack_rows
    m, k, n = ROWS[i]
    rng = np.random.default_rng(500 + i)
    act = ACTS[(i + DTYPES.index(dtype)) % 5]
    x, w, b, r, g = make(rng, dtype, m, k), make(rng, dtype, k, n, scale=k ** -0.5), make(rng, dtype, n), make(rng, dtype, m, n), make(rng, dtype, m, n)
    put = odd_rows if i % 2 else (lambda v: v.cuda())
    y, saved = dense(put(x), put(w), b.cuda(), residual=put(r), activation=act, save="activation")
    check_dense(x, w, b, r, act, y, saved, dtype)
    y8, p = dense(put(x), put(w), b.cuda(), residual=put(r), activation=act, save="packed")
    assert torch.equal(y, y8)
    if p is not None:
        want = pack_rows(saved)
        assert torch.equal(p.q, want.q) and torch.equal(p.scale, want.scale)
    got = dense_backward(put(g), put(x), put(w), saved, activation=act)
    check_dense_backward(g, x, w, None if saved is None else saved.cpu(), act, *got, dtype)
    assert all(torch.equal(u, v) for u, v in zip(got, dense_backward(put(g), put(x), put(w), saved, activation=act)))
    px = pack_rows(put(x))
    got = dense_backward(put(g), px, put(w), p, activation=act)
    check_dense_backward(g, unpack_rows(px).cpu(), w, None if p is None else unpack_rows(p).cpu(), act, *got, dtype)
    only = dense_backward(put(g), px, put(w), p, activation=act, need_x=False, need_weight=False)
    assert only[0] is None and only[1] is None and torch.equal(only[2], got[2])
    only = dense_backward(put(g), px, put(w), p, activation=act, need_weight=False, need_bias=False)
    assert torch.equal(only[0], got[0])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,ends", [(24, [3, 6, 6, 20, 24]), (10, [4, 2, 7]), (1, [0, 1]), (30, [0] * 70 + [30]), (60, list(range(1, 61))), (12, [-3, 1 << 50])])
def test_grouped_few_rows(m, ends, dtype):
    from smrt_amd.autoencode import dense_grouped, dense_grouped_backward
    rng = np.random.default_rng(600)
    k, n, G = 90, 70, len(ends)
    x, w, b, g = make(rng, dtype, m, k), make(rng, dtype, G, k, n, scale=k ** -0.5), make(rng, dtype, G, n), make(rng, dtype, m, n)
    e = torch.tensor(ends, dtype=torch.int64, device="cuda")
    out = torch.full((m, n), 5.0, dtype=dtype, device="cuda")
    dense_grouped(x.cuda(), e, w.cuda(), b.cuda(), activation="elu", out=out)
    y, saved = dense_grouped(x.cuda(), e, w.cuda(), b.cuda(), activation="elu", save="activation")
    dx, dw, db = dense_grouped_backward(g.cuda(), x.cuda(), e, w.cuda(), saved, activation="elu")
    lo = 0
    for j, hi in enumerate(sound_ends(ends, m)):
        s = slice(lo, hi)
        check_dense(x[s], w[j], b[j], None, "elu", y[s], None, dtype)
        check_dense_backward(g[s], x[s], w[j], saved[s].cpu(), "elu", dx[s], dw[j], db[j], dtype)
        lo = hi
    assert not y[lo:].any() and not dx[lo:].any()
    assert torch.equal(out[:lo], y[:lo]) and (out[lo:] == 5.0).all()


# ------------------------------------------------------------------------------------------------ the ends of what the calls allow
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_columns_of_one_buffer(dtype):
    """Input and output as different columns of one matrix, with rows that interleave in memory; columns that meet are refused."""
    from smrt_amd import _hip
    from smrt_amd.autoencode import dense, layer_norm
    rng = np.random.default_rng(70)
    x, w, r = make(rng, dtype, 90, 50), make(rng, dtype, 50, 70, scale=0.2), make(rng, dtype, 90, 70)
    buf = torch.full((90, 200), 3.0, dtype=dtype, device="cuda")
    buf[:, :50], buf[:, 120:190] = x.cuda(), r.cuda()
    dense(buf[:, :50], w.cuda(), residual=buf[:, 120:190], activation="elu", out=buf[:, 50:120])
    check_dense(x, w, None, r, "elu", buf[:, 50:120], None, dtype)
    assert torch.equal(buf[:, :50].cpu(), x) and torch.equal(buf[:, 120:190].cpu(), r) and (buf[:, 190:] == 3.0).all()
    want = layer_norm(x.cuda())[0]
    layer_norm(buf[:, :50], out=buf[:, 150:])
    assert torch.equal(buf[:, 150:], want) and torch.equal(buf[:, :50].cpu(), x)
    for out in (buf[:, 49:119], buf[1:, 49:119]):
        with pytest.raises(_hip.HipLibraryError):
            dense(buf[:out.shape[0], :50], w.cuda(), out=out)
    with pytest.raises(_hip.HipLibraryError):
        layer_norm(buf[:89, :50], out=buf[1:, :50])


WIDTHS = [1, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 71, 72, 73, 127, 128, 129, 135]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("k", WIDTHS)
def test_every_way_a_piece_is_cut(k, dtype):
    """Widths around the pieces and tiles in both directions, rows between NaN, in forward and backward products."""
    from smrt_amd.autoencode import dense, dense_backward
    rng = np.random.default_rng(7000 + k)
    m = 150
    x = make(rng, dtype, m, k)
    for n in WIDTHS:
        w, g = make(rng, dtype, k, n, scale=k ** -0.5), make(rng, dtype, m, n)
        y = dense(odd_rows(x), odd_rows(w))
        check_dense(x, w, None, None, "identity", y, None, dtype)
        dx, dw, db = dense_backward(odd_rows(g), odd_rows(x), odd_rows(w))
        check_dense_backward(g, x, w, None, "identity", dx, dw, db, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_widest_strides(dtype):
    """Rows 2^21 elements apart, the most that the products take: the same bits as from rows next to each other."""
    from smrt_amd import _hip
    from smrt_amd.autoencode import dense, dense_backward, layer_norm, pack_rows
    big = torch.empty((300, 1 << 21), dtype=dtype, device="cuda")
    gen = torch.Generator().manual_seed(5)
    put = lambda col, r, c: big[:r, col:col + c].copy_(torch.randn((r, c), generator=gen).to(dtype))
    x, w, g = put(1, 300, 270), put(400, 270, 261), put((1 << 21) - 261, 300, 261)
    X, W, G = x.contiguous(), w.contiguous(), g.contiguous()
    out = big[:, 1000:1261]
    dense(x, w, activation="tanh", out=out)
    want = dense(X, W, activation="tanh")
    assert torch.equal(out, want)
    for p, q in zip(dense_backward(g, x, w, out, activation="tanh"), dense_backward(G, X, W, want, activation="tanh")):
        assert torch.equal(p, q)
    assert torch.equal(layer_norm(x)[0], layer_norm(X)[0])
    assert torch.equal(pack_rows(x).q, pack_rows(X).q)
    del big, x, w, g, out
    wide = torch.zeros((2, (1 << 21) + 8), dtype=dtype, device="cuda")
    with pytest.raises(_hip.HipLibraryError):
        dense(wide[:, :8], W[:8])


def test_most_groups():
    """65 535 groups, most of one row, some empty, some of several."""
    from smrt_amd.autoencode import dense_grouped, dense_grouped_backward
    G, k, n = 65535, 9, 7
    gen = torch.Generator().manual_seed(6)
    sizes = torch.randint(0, 3, (G,), generator=gen)
    sizes[1000], sizes[G - 1] = 700, 5
    ends = sizes.cumsum(0)
    m = int(ends[-1])
    which = torch.repeat_interleave(torch.arange(G), sizes)
    x, w, g = torch.randn((m, k), generator=gen), torch.randn((G, k, n), generator=gen), torch.randn((m, n), generator=gen)
    y = dense_grouped(x.cuda(), ends.cuda(), w.cuda())
    dx, dw, db = dense_grouped_backward(g.cuda(), x.cuda(), ends.cuda(), w.cuda())
    X, W, D = x.double(), w.double(), g.double()
    own = W[which]
    tol = lambda terms, count: 2 * (count + 10) * U * terms + half(F32) * 2 * terms + tiny(F32)
    close(y, (X[:, :, None] * own).sum(1), tol((X[:, :, None] * own).abs().sum(1), k), "y")
    close(dx, (own * D[:, None]).sum(2), tol((own * D[:, None]).abs().sum(2), n), "dx")
    outer = X[:, :, None] * D[:, None]
    zero = torch.zeros((G, k, n), dtype=torch.float64)
    close(dw, zero.index_add(0, which, outer), tol(zero.index_add(0, which, outer.abs()), 700), "dw")
    zero = torch.zeros((G, n), dtype=torch.float64)
    close(db, zero.index_add(0, which, D), tol(zero.index_add(0, which, D.abs()), 700), "db")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,ends", [(50, [10, 20, 41]), (900, [200, 500, 801])])
def test_nan_stays_in_its_class(m, ends, dtype):
    """A class of NaN rows, a class with a NaN weight, and NaN rows of no class leave the others' results as they are."""
    from smrt_amd.autoencode import dense_grouped, dense_grouped_backward
    rng = np.random.default_rng(80)
    k, n = 70, 45
    x, w, g = make(rng, dtype, m, k), make(rng, dtype, 3, k, n, scale=0.1), make(rng, dtype, m, n)
    e = torch.tensor(ends, device="cuda")

    def run(x, w, g):
        y, saved = dense_grouped(x.cuda(), e, w.cuda(), activation="sigmoid", save="activation")
        return (y, *dense_grouped_backward(g.cuda(), x.cuda(), e, w.cuda(), saved, activation="sigmoid"))
    want = run(x, w, g)
    x, w, g = x.clone(), w.clone(), g.clone()
    x[ends[0]:ends[1]] = float("nan")
    x[ends[2]:], g[ends[2]:] = float("nan"), float("nan")
    y, dx, dw, db = run(x, w, g)
    a, b, c = slice(0, ends[0]), slice(ends[0], ends[1]), slice(ends[1], ends[2])
    for s in (a, c):
        assert torch.equal(y[s], want[0][s]) and torch.equal(dx[s], want[1][s])
    assert y[b].isnan().all() and dx[b].isnan().all() and dw[1].isnan().all() and db[1].isnan().all()
    for j in (0, 2):
        assert torch.equal(dw[j], want[2][j]) and torch.equal(db[j], want[3][j])
    assert not y[ends[2]:].any() and not dx[ends[2]:].any()
    w[2, 5, 7] = float("nan")
    y = run(x, w, g)[0]
    assert torch.equal(y[a], want[0][a]) and y[c, 7].isnan().all() and torch.equal(y[c, :7], want[0][c, :7]) and torch.equal(y[c, 8:], want[0][c, 8:])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_many_groups_of_few_rows(dtype):
    """60 rows over 20 000 groups, most of them empty, with ends that fall back and leave the rows."""
    from smrt_amd.autoencode import dense_grouped, dense_grouped_backward
    G, m, k, n = 20000, 60, 33, 70
    rng = np.random.default_rng(90)
    ends = np.sort(rng.integers(0, m + 1, G))
    ends[::7] -= 25
    ends[-3:] = [m - 1, -5, 1 << 40]
    x, w, g = make(rng, dtype, m, k), torch.randn((G, k, n), generator=torch.Generator().manual_seed(2)).to(dtype), make(rng, dtype, m, n)
    e = torch.from_numpy(ends).cuda()
    y = dense_grouped(x.cuda(), e, w.cuda())
    dx, dw, db = dense_grouped_backward(g.cuda(), x.cuda(), e, w.cuda())
    used, lo = torch.zeros(G, dtype=torch.bool), 0
    for j, hi in enumerate(sound_ends(ends.tolist(), m)):
        if hi > lo:
            s = slice(lo, hi)
            used[j] = True
            check_dense(x[s], w[j], None, None, "identity", y[s], None, dtype)
            check_dense_backward(g[s], x[s], w[j], None, "identity", dx[s], dw[j], db[j], dtype)
        lo = hi
    assert lo == m and not dw[~used.cuda()].any() and not db[~used.cuda()].any()


@pytest.mark.parametrize("dtype", [F32, F16], ids=str)
def test_two_threads_with_a_stream_each(dtype):
    """The same calls from two host threads at once, each on its own stream: workspaces and results do not mix."""
    import threading
    sets = [block_inputs(dtype, m=m, seed=m) for m in (40, 700)]
    want = []
    for x, p, ends, gy in sets:
        y, kept = block(x, p, ends, True)
        want.append((y, block_backward(gy, p, ends, kept)))
    torch.cuda.synchronize()
    bad = []

    def work(i):
        x, p, ends, gy = sets[i]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                y, kept = block(x, p, ends, True)
                got = block_backward(gy, p, ends, kept)
                if not torch.equal(y, want[i][0]) or not all(torch.equal(got[k], want[i][1][k]) for k in got):
                    bad.append(i)
        stream.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_class_decoders_without_rows(fitted):
    from smrt_amd.autoencode import ClassDecoders
    d = ClassDecoders(fitted)
    assert d.generate([0, 0, 0], np.random.RandomState(1)).shape == (0, 50)
    some = d.generate([0, 4, 0], np.random.RandomState(1))
    assert torch.equal(some, ClassDecoders(fitted[1:2]).generate([4], np.random.RandomState(1)))


WIDE_NORMS = [(2051, 1437), (2050, 2000), (1031, 2500), (1029, 4000), (1025, 8000), (517, 12000)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("i", range(len(WIDE_NORMS)), ids=[str(s) for s in WIDE_NORMS])
def test_layer_norm_of_many_wide_rows(i, dtype, monkeypatch):
    """Every way to share a row among waves, with more rows than one turn of the workgroups and odd numbers of them."""
    import sys
    monkeypatch.setattr(sys.modules[__name__], "NORMS", WIDE_NORMS)
    test_layer_norm(i, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("k", [1, 7, 9, 33, 65, 72, 129, 135])
def test_every_way_a_piece_is_cut_with_many_rows(k, dtype):
    """The same widths forward with more rows than the kernels for a few rows take, bias, residual and the saved activation among them."""
    from smrt_amd.autoencode import dense, pack_rows
    rng = np.random.default_rng(7500 + k)
    m = 1301
    x = make(rng, dtype, m, k)
    for n in WIDTHS:
        w, b, r = make(rng, dtype, k, n, scale=k ** -0.5), make(rng, dtype, n), make(rng, dtype, m, n)
        y, saved = dense(odd_rows(x), odd_rows(w), b.cuda(), residual=odd_rows(r), activation="tanh", save="activation")
        check_dense(x, w, b, r, "tanh", y, saved, dtype)
        y8, kept = dense(odd_rows(x), odd_rows(w), b.cuda(), residual=odd_rows(r), activation="tanh", save="packed")
        want = pack_rows(saved)
        assert torch.equal(y8, y) and torch.equal(kept.q, want.q) and torch.equal(kept.scale, want.scale)


# ------------------------------------------------------------------------------------------------ what a C caller may ask for besides
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,k,n,ends,act", [(40, 90, 70, [7, 7, 31], "elu"), (12, 33, 130, [0, 5], "identity"), (300, 90, 70, [100, 90, 221], "sigmoid"),
                                            (700, 90, 70, [100, 301, 333], "tanh"), (9000, 300, 520, [4000, 8001], "identity"),
                                            (40, 90, 70, [0, 0], "relu"), (700, 90, 70, [0, 0], "relu")])
def test_backward_entry_keeps_rows_of_no_class(m, k, n, ends, act, dtype):
    """keep_rest of the C entry: dx of rows behind the last end stays as it was, from the kernels for a few rows and from the product tiles alike."""
    import ctypes as C
    from smrt_amd import _hip
    from smrt_amd.autoencode import dense_grouped, dense_grouped_backward
    rng = np.random.default_rng(900)
    G, ids = len(ends), {F32: 0, BF16: 1, F16: 2}
    x, w, g = make(rng, dtype, m, k).cuda(), make(rng, dtype, G, k, n, scale=k ** -0.5).cuda(), make(rng, dtype, m, n).cuda()
    e = torch.tensor(ends, device="cuda")
    saved = dense_grouped(x, e, w, activation=act, save="activation")[1]
    want = dense_grouped_backward(g, x, e, w, saved, activation=act)
    lib = _hip.load()
    for keep in (1, 0):
        dx, dw, db = torch.full((m, k), 5.0, dtype=dtype, device="cuda"), torch.empty_like(w), torch.empty((G, n), dtype=dtype, device="cuda")
        args = _hip.Dense(ids[dtype], _hip.ACTIVATION_IDS[act], m, k, n, G, keep, e.data_ptr(), x.data_ptr(), k, None, 0, w.data_ptr(), n, k * n, None, n,
                          None, 0, None, 0, None if saved is None else saved.data_ptr(), n, None, 0, g.data_ptr(), n, dx.data_ptr(), k, dw.data_ptr(), n, k * n,
                          db.data_ptr())
        size = lib.smrt_dense_backward_workspace(C.byref(args))
        assert (size > 0) == (m >= 300)
        work = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
        assert lib.smrt_dense_backward(C.byref(args), work.data_ptr(), size, torch.cuda.current_stream().cuda_stream) == 0
        last = max(ends)
        assert torch.equal(dx[:last], want[0][:last]) and torch.equal(dw, want[1]) and torch.equal(db, want[2])
        assert (dx[last:] == (5.0 if keep else 0.0)).all()


TILED = [(1408, 70, 50), (1500, 9, 450), (16500, 70, 700), (70000, 40, 260)]       # 64x64 tiles, the same, 128x128 and, in 16 bits, 256x256


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [(40, 70, 50)] + TILED)
def test_infinities_and_nan_from_rows_and_tiles(m, k, n, dtype):
    """Infinities keep their sign and NaN its place in all three products, whichever kernel takes them."""
    from smrt_amd.autoencode import dense, dense_backward
    rng = np.random.default_rng(920)
    inf, nan, top = float("inf"), float("nan"), torch.finfo(dtype).max
    x, w, g = make(rng, dtype, m, k), make(rng, dtype, k, n), make(rng, dtype, m, n)
    x[3, 5], x[7, k - 1], x[11, 0], x[12, 1], x[m - 1, k - 1] = inf, -inf, nan, top, inf
    w[2, 9], w[4, 11], w[k - 1, n - 1] = inf, 0.0, -inf
    g[20, 3], g[21, n - 1], g[m - 2, 0], g[23, 7] = inf, -inf, nan, top

    def doubtful(a, b):
        """What 32-bit sums may take elsewhere: results near the largest number of the type, and sums in which a term of the largest number and a factor
        above 1, an infinity in 32 bits (not in f16, whose products stay far below), meets an infinity or another such term."""
        want, has = a @ b, lambda f, d: f.any(d)
        big = want.isfinite() & (want.abs() > 0.9 * top)
        if dtype != F16:
            huge = lambda v: (v.abs() == top) | v.isinf()
            big |= has(a.abs() == top, 1)[:, None] & has(huge(b), 0) | has(huge(a), 1)[:, None] & has(b.abs() == top, 0)
        return big

    def check(got, a, b, what):
        got, want, big = got.cpu().double(), a @ b, doubtful(a, b)
        for f in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(f(got)[~big], f(want)[~big]), (what, f.__name__)
        assert want.isposinf().any() and want.isneginf().any() and want.isnan().any() and want.isfinite().any()
    X, W, D = x.double(), w.double(), g.double()
    check(dense(x.cuda(), w.cuda()), X, W, "y")
    dx, dw, db = dense_backward(g.cuda(), x.cuda(), w.cuda())
    check(dx, D, W.T, "dx")
    check(dw, X.T, D, "dw")
    check(db[None], torch.ones(1, m, dtype=torch.float64), D, "db")
    nans, sure = (X @ W).isnan(), ~doubtful(X, W)
    for act in ACTS:
        assert torch.equal(dense(x.cuda(), w.cuda(), activation=act).cpu().isnan()[sure], nans[sure]), act


@pytest.mark.parametrize("m,k,n", TILED)
def test_small_and_large_numbers_from_tiles(m, k, n):
    """fp32 in parts over the range in which all three parts are normal numbers (x from 2^-103, so that x's last bit is 2^-126), and near the largest."""
    from smrt_amd.autoencode import dense, dense_backward
    rng = np.random.default_rng(930)
    x, w, g = make(rng, F32, m, k).clamp(-3, 3), make(rng, F32, k, n, scale=k ** -0.5), make(rng, F32, m, n).clamp(-3, 3)
    X, W, D = x.double(), w.double(), g.double()
    for s in (2.0 ** -100, 2.0 ** 110):
        y = dense((x * s).cuda(), w.cuda()).cpu().double() / s
        assert (y - X @ W).norm() <= 2e-6 * (X @ W).norm()
        dx, dw, _ = dense_backward((g * s).cuda(), x.cuda(), w.cuda())
        assert (dx.cpu().double() / s - D @ W.T).norm() <= 2e-6 * (D @ W.T).norm()
        assert (dw.cpu().double() / s - X.T @ D).norm() <= 2e-6 * (X.T @ D).norm()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,ends,k,n", [(1500, [300, 701, 1400], 70, 45), (17000, [5000, 9001, 16800], 70, 700)])
def test_nan_stays_in_its_class_in_tiles(m, ends, k, n, dtype):
    """A class of NaN rows, NaN rows of no class and a NaN weight leave the other classes' results as they are."""
    from smrt_amd.autoencode import dense_grouped, dense_grouped_backward
    rng = np.random.default_rng(940)
    nan = float("nan")
    x, w, g = make(rng, dtype, m, k), make(rng, dtype, 3, k, n, scale=0.1), make(rng, dtype, m, n)
    e = torch.tensor(ends, device="cuda")

    def run(x, w, g):
        y, saved = dense_grouped(x.cuda(), e, w.cuda(), activation="sigmoid", save="activation")
        return (y, *dense_grouped_backward(g.cuda(), x.cuda(), e, w.cuda(), saved, activation="sigmoid"))
    want = run(x, w, g)
    x, w, g = x.clone(), w.clone(), g.clone()
    x[ends[0]:ends[1]] = nan
    x[ends[2]:], g[ends[2]:] = nan, nan
    y, dx, dw, db = run(x, w, g)
    a, b, c = slice(0, ends[0]), slice(ends[0], ends[1]), slice(ends[1], ends[2])
    for s in (a, c):
        assert torch.equal(y[s], want[0][s]) and torch.equal(dx[s], want[1][s])
    assert y[b].isnan().all() and dx[b].isnan().all() and dw[1].isnan().all() and db[1].isnan().all()
    for j in (0, 2):
        assert torch.equal(dw[j], want[2][j]) and torch.equal(db[j], want[3][j])
    assert not y[ends[2]:].any() and not dx[ends[2]:].any()
    w[2, 5, 7] = nan
    y = run(x, w, g)[0]
    assert torch.equal(y[a], want[0][a]) and y[c, 7].isnan().all() and torch.equal(y[c, :7], want[0][c, :7]) and torch.equal(y[c, 8:], want[0][c, 8:])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,k,n", TILED)
def test_grouped_tiles_are_dense_tiles_for_one_group(m, k, n, dtype):
    from smrt_amd.autoencode import dense, dense_grouped
    rng = np.random.default_rng(950)
    x, w = make(rng, dtype, m, k).cuda(), make(rng, dtype, k, n).cuda()
    assert torch.equal(dense_grouped(x, torch.tensor([m], device="cuda"), w[None]), dense(x, w))


def test_out_counts_as_written():
    """A tensor that autograd kept and a call writes over ends its backward pass with an error, as after any in-place operation."""
    from smrt_amd.autoencode import dense, layer_norm
    x, w = torch.randn(6, 8, device="cuda"), torch.randn(8, 8, device="cuda")
    for call in (lambda out: dense(x, w, out=out), lambda out: layer_norm(x, out=out), lambda out: dense(x, w, residual=out, out=out)):
        leaf = torch.randn(6, 8, device="cuda", requires_grad=True)
        h = torch.exp(leaf)                                  # keeps its result
        loss = h.sum()
        call(h.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        out = torch.empty(6, 8, device="cuda")
        assert dense(x, w, out=out) is out


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_one_row_of_a_wide_matrix(dtype):
    """A single row has no distance to another: the width of the matrix that it is cut from does not count."""
    from smrt_amd.autoencode import dense, dense_backward, dense_grouped
    rng = np.random.default_rng(960)
    x, w, g = make(rng, dtype, 1, 8), make(rng, dtype, 8, 16), make(rng, dtype, 1, 16)
    wide = torch.zeros((2, (1 << 21) + 64), dtype=dtype, device="cuda")
    wide[0, :8], wide[0, 8:24] = x[0].cuda(), g[0].cuda()
    X, D = wide[:1, :8], wide[:1, 8:24]
    y = dense(X, w.cuda())
    check_dense(x, w, None, None, "identity", y, None, dtype)
    check_dense_backward(g, x, w, None, "identity", *dense_backward(D, X, w.cuda()), dtype)
    assert torch.equal(dense_grouped(X, torch.tensor([1], device="cuda"), w.cuda()[None]), y)


# ------------------------------------------------------------------------------------------------ fp32 products in three bf16 parts
def worst_fp32(rng, count):
    """fp32 numbers of one binade whose upper parts end in ones or in halves, where cutting and rounding leave the most, among ordinary ones."""
    bits = rng.integers(0, 1 << 23, count).astype(np.uint32)
    special = np.array([0x00ffff, 0x7fffff, 0x00ff80, 0x00ff7f, 0x007fff, 0x008000, 0x00fe80, 0x40ffff, 0x01ffff, 0x00ff81, 0x00fe7f], np.uint32)
    some = rng.random(count) < 0.7
    bits[some] = special[rng.integers(0, len(special), int(some.sum()))]
    sign = rng.integers(0, 2, count).astype(np.uint32) << 31
    return torch.from_numpy((bits | np.uint32(0x3f800000) | sign).view(np.float32))


@pytest.mark.parametrize("m,n", [(1408, 64), (16512, 704)], ids=["64x64 tiles", "128x128 tiles"])
def test_fp32_products_of_single_terms(m, n):
    """Sums of one product each, from the tiles: parts are h (cut off, so m = x - h is at most 2^-7 of x's power of two) and m (cut off in one operand, away from zero in
    the other), which leaves l below 2^-15.  m l and l m, which are not multiplied, have different signs and stay below 2^-22 = 4 u of the product.  hh and the
    products of the other parts are exact in fp32; their sum, below 2^-6, is rounded on the way (a few u of 2^-6), and hh plus that sum once: 5.25 u altogether."""
    from smrt_amd.autoencode import dense, dense_backward
    rng = np.random.default_rng(910)
    k = 16
    one = lambda rows, cols: torch.zeros(rows, cols).scatter_(1, torch.from_numpy(rng.integers(0, cols, (rows, 1))), worst_fp32(rng, rows)[:, None])

    def check(got, a, b, what):
        want = a.double() @ b.double()                       # one term
        close(got, want, 5.25 * U * want.abs(), what)
    x, w, g = one(m, k), worst_fp32(rng, k * n).reshape(k, n), one(m, n)
    check(dense(x.cuda(), w.cuda()), x, w, "y")
    dx = dense_backward(g.cuda(), x.cuda(), w.cuda(), need_weight=False, need_bias=False)[0]
    check(dx, g, w.T, "dx")
    row = int(rng.integers(0, m))
    x, g = torch.zeros(m, k), worst_fp32(rng, m * n).reshape(m, n)
    x[row] = worst_fp32(rng, k)
    dw = dense_backward(g.cuda(), x.cuda(), w.cuda(), need_x=False, need_bias=False)[1]
    check(dw, x.T, g, "dw")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_pack_holds_its_bounds(dtype):
    """1/126 of a block's largest magnitude at every scale but the ends: half a step at the lowest (every f16 number there is a whole number of steps), 1/64 at the
    highest, whose 64 steps would be an infinity."""
    from smrt_amd.autoencode import pack_rows, unpack_rows
    rng = np.random.default_rng(970)
    low, high = (-24, 10) if dtype == F16 else (-126, 122)
    top = torch.finfo(dtype).max
    exps = rng.integers(-24 if dtype == F16 else -149, 16 if dtype == F16 else 128, 4000)
    x = torch.from_numpy((rng.uniform(-1, 1, (4000, 32)) * np.exp2(exps)[:, None]).clip(-top, top)).to(dtype)
    step = 2.0 ** high
    ends = [[top], [-top, top / 2, step, 0.5 * step], [63.5 * step], [63.49 * step], [127.0 * step / 2], [127.02 * step / 2], [2.0 ** low], [2.0 ** low / 2],
            [2.0 ** low / 2, 2.0 ** low * 1.5], [2.0 ** low / 4], [127 * 2.0 ** low, 2.0 ** low / 2], [63.5 * 2.0 ** low]]
    for i, e in enumerate(ends):
        x[i] = 0
        x[i, :len(e)] = torch.tensor(e, dtype=torch.float64).clamp(-top, top).to(dtype)
    p = pack_rows(x.cuda())
    v, X, byte = unpack_rows(p).cpu().double(), x.double(), p.scale.cpu().int()
    assert v.isfinite().all() and (p.q.cpu().int().abs()[byte[:, 0] == high + 127] <= 63).all()
    most = X.abs().amax(1, keepdim=True)
    bound = torch.where(byte == high + 127, most / 64, torch.where(byte == low + 127, 0.0 if dtype == F16 else 2.0 ** (low - 1), most / 126))
    assert ((v - X).abs() <= bound).all()
    for b in (low + 127, low + 128, 127, high + 126, high + 127):
        assert (byte == b).any(), b
