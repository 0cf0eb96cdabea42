"""The dense operators (quickrank_amd/dense.py) against plain implementations in 64 bits.

Tolerances count roundings: a result is rounded once (half a step of its type, U[type] relative), sums
and products are held in f32 (2^-24 a step, at most as many steps as there are terms, over the sum of the
terms' absolute values), and a value that passes through memory in the element type costs U[type] more."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U32 = 2.0 ** -24
# the smallest step of a type near zero (f16's subnormals; the others' are far below what is tested)
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"]


@pytest.fixture(scope="module")
def dense():
    from quickrank_amd import dense
    return dense


def rand(seed, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)


def padded(t, pad, fill=float("nan")):
    """The same matrix inside rows that are `pad` longer and hold NaN behind it."""
    buf = torch.full((t.shape[0], t.shape[1] + pad), fill, dtype=t.dtype, device=t.device)
    buf[:, :t.shape[1]] = t
    return buf[:, :t.shape[1]]


def shifted(t, by):
    """The same contiguous tensor `by` elements behind a 16-byte boundary, NaN on both sides."""
    buf = torch.full((t.numel() + 64,), float("nan"), dtype=t.dtype, device=t.device)
    v = buf[by:by + t.numel()].view(t.shape)
    v.copy_(t)
    return v


def close(got, want, tol, dtype, what):
    """|got - want| <= tol + half a step of the result, elementwise."""
    assert got.dtype == dtype and got.shape == want.shape, (what, got.dtype, got.shape, want.shape)
    err = (got.double() - want).abs()
    lim = tol + U[dtype] * (want.abs() + tol) + TINY[dtype]
    bad = ~(err <= lim)
    assert not bad.any(), (what, int(bad.sum()), float((err / lim).nan_to_num(1e30).max()))


# ---- layer norm ----------------------------------------------------------------------------------

def norm64(x, w, b, eps):
    x = x.double()
    mean = x.mean(1)
    var = (x - mean[:, None]).square().mean(1)
    rstd = 1 / (var + eps).sqrt()
    hat = (x - mean[:, None]) * rstd[:, None]
    y = hat * (w.double() if w is not None else 1.0) + (b.double() if b is not None else 0.0)
    return y, mean, rstd, hat


def steps(cols):
    """An upper bound of the roundings in a row's sum: eight lanes at least share it."""
    return cols / 8 + 32


def norm_tolerances(x, w, b, eps):
    y, mean, rstd, hat = norm64(x, w, b, eps)
    c, s = x.shape[1], steps(x.shape[1])
    tm = U32 * s * x.double().abs().mean(1) + U32 * mean.abs()
    # the squares' sum: its own roundings, and the error of every difference from the mean
    dist = (x.double() - mean[:, None]).abs()
    tv = U32 * (s + 4) * dist.square().mean(1) + 2 * (tm[:, None] + U32 * dist).mul(dist).mean(1) + tm * tm
    tr = rstd * (0.5 * tv * rstd * rstd * 1.5 + 8 * U32)
    th = (tm[:, None] + U32 * dist) * rstd[:, None] + dist * tr[:, None] + 2 * U32 * hat.abs()
    aw = w.double().abs() if w is not None else torch.ones(c, dtype=torch.float64, device=x.device)
    ty = th * aw + 2 * U32 * (hat.abs() * aw + (b.double().abs() if b is not None else 0.0))
    return (y, mean, rstd), (ty, tm, tr)


NORM_SHAPES = [(1, 1), (1, 2), (3, 7), (100, 136), (257, 64), (33, 200), (65, 513), (7, 1000), (5, 1001), (1000, 8), (9, 2048),
               (4, 4099), (2, 16384), (3, 33001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_norm_forward(dense, dtype, rows, cols):
    x = rand(rows + cols, rows, cols, dtype=dtype, scale=1.5, shift=0.5)
    for params in {dtype, torch.float32}:
        w, b = rand(1, cols, dtype=params, scale=0.2, shift=1), rand(2, cols, dtype=params)
        for v in (x, padded(x, 3), shifted(x, 1)):
            y, mean, rstd = dense.layer_norm(v, w, b, 1e-5)
            want, tol = norm_tolerances(x, w, b, 1e-5)
            for g, t, e, d, n in zip((y, mean, rstd), want, tol, (dtype, torch.float32, torch.float32), ("y", "mean", "rstd")):
                close(g, t, e, d, n)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_without_parameters_and_leading_dimensions(dense, dtype):
    x = rand(3, 4, 9, 136, dtype=dtype)
    y, mean, rstd = dense.layer_norm(x)
    want, tol = norm_tolerances(x.view(36, 136), None, None, 1e-5)
    assert y.shape == x.shape and mean.shape == (36,)
    close(y.view(36, 136), want[0], tol[0], dtype, "y")
    w = rand(4, 136)
    for weight, bias in ((w, None), (None, w)):
        want, tol = norm_tolerances(x.view(36, 136), weight, bias, 1e-5)
        close(dense.layer_norm(x, weight, bias)[0].view(36, 136), want[0], tol[0], dtype, "y")


def test_norm_of_far_values_equal_values_and_broken_rows(dense):
    """A mean far from zero keeps its digits (the squares are taken from the mean), a row of one value gives the
    bias, NaN and infinity stay in their row."""
    x = rand(5, 40, 136, shift=4096.0)
    x[7] = 3.25
    x[9, 100] = float("nan")
    x[11, 5] = float("inf")
    w, b = rand(6, 136), rand(7, 136)
    y, mean, rstd = dense.layer_norm(x, w, b)
    ok = [r for r in range(40) if r not in (9, 11)]
    want, tol = norm_tolerances(x[ok], w, b, 1e-5)
    close(y[ok], want[0], tol[0], torch.float32, "y")
    assert torch.equal(y[7], b) and torch.isnan(y[9]).all() and torch.isnan(y[11]).all()


NORM_GRAD_SHAPES = [(1, 1), (1, 64), (2, 7), (100, 136), (4097, 136), (257, 200), (65, 1000), (130, 1001), (1031, 33), (70, 2048),
                    (9, 4099), (3, 16384), (2, 33001), (20000, 8)]


def norm_grad_check(dense, dtype, params, rows, cols, seed=0):
    x = rand(seed + 1, rows, cols, dtype=dtype, scale=1.5, shift=0.5)
    w, dy = rand(seed + 2, cols, dtype=params, scale=0.2, shift=1), rand(seed + 3, rows, cols, dtype=dtype)
    _, mean, rstd, _ = norm64(x, w, None, 1e-5)
    mean, rstd = mean.float(), rstd.float()
    # from the given statistics: the formula in 64 bits
    hat = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    g = dy.double() * w.double()
    a, c = g.mean(1, keepdim=True), (g * hat).mean(1, keepdim=True)
    dx = rstd.double()[:, None] * (g - a - hat * c)
    s = steps(cols)
    ta, tc = U32 * (s + 2) * g.abs().mean(1, keepdim=True), U32 * (s + 6) * (g * hat).abs().mean(1, keepdim=True)
    tdx = rstd.double()[:, None].abs() * (4 * U32 * (g.abs() + a.abs() + (hat * c).abs()) + ta + hat.abs() * tc)
    dw, db = (dy.double() * hat).sum(0), dy.double().sum(0)
    tw = U32 * (rows + 8) * (dy.double() * hat).abs().sum(0)
    tb = U32 * (rows + 8) * dy.double().abs().sum(0)
    for v, d in ((x, dy), (padded(x, 5), padded(dy, 1)), (shifted(x, 3), shifted(dy, 1))):
        got = dense.layer_norm_backward(d, v, w, mean, rstd)
        close(got[0], dx, tdx, dtype, "dx")
        close(got[1], dw, tw, params, "dw")
        close(got[2], db, tb, params, "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", NORM_GRAD_SHAPES)
def test_norm_backward(dense, dtype, rows, cols):
    for params in {dtype, torch.float32}:
        norm_grad_check(dense, dtype, params, rows, cols)


def test_norm_backward_broadcast_gradient(dense):
    """One gradient row for all rows (a sum over documents): a stride of 0."""
    x, w = rand(1, 50, 136), rand(2, 136)
    dy = rand(3, 1, 136).expand(50, 136)
    _, mean, rstd = dense.layer_norm(x, w)
    a = dense.layer_norm_backward(dy, x, w, mean, rstd)
    b = dense.layer_norm_backward(dy.contiguous(), x, w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_no_rows(dense, dtype):
    x, w = torch.empty(0, 40, dtype=dtype, device="cuda"), rand(1, 40, dtype=dtype)
    y, mean, rstd = dense.layer_norm(x, w, w)
    assert y.shape == (0, 40) and mean.shape == (0,)
    dx, dw, db = dense.layer_norm_backward(x, x, w, mean, rstd)
    assert dx.shape == (0, 40) and not dw.any() and not db.any()


def test_norm_gradient_against_differences(dense):
    x, w, b = rand(1, 12, 136), rand(2, 136), rand(3, 136)
    c, v = rand(4, 12, 136).double(), rand(5, 12, 136)
    _, mean, rstd = dense.layer_norm(x, w, b)
    dx, dw, db = dense.layer_norm_backward(c.float(), x, w, mean, rstd)
    h = 2.0 ** -6
    vw = rand(6, 136)

    def diff(f, w_, vx, vw_):
        return ((c * f(x + h * vx, w_ + h * vw_)).sum() - (c * f(x - h * vx, w_ - h * vw_)).sum()) / (2 * h)
    for vx, vw_, grad in ((v, 0 * vw, (dx.double() * v).sum()), (0 * v, vw, (dw.double() * vw).sum())):
        own = diff(lambda p, q: dense.layer_norm(p, q, b)[0].double(), w, vx, vw_)
        far = diff(lambda p, q: norm64(p.double(), q, b, 1e-5)[0], w, vx, vw_)
        xd, wd = x.double().requires_grad_(True), w.double().requires_grad_(True)
        gx, gw = torch.autograd.grad((norm64(xd, wd, b, 1e-5)[0] * c).sum(), (xd, wd))
        true = (gx * vx).sum() + (gw * vw_).sum()
        y = dense.layer_norm(x, w, b)[0].double()
        # the forward pass's own roundings over the step, and what the difference quotient itself is off
        lim = 40 * U32 * (c.abs() * (y.abs() + 1)).sum() / h + (far - true).abs()
        assert (own - grad).abs() <= lim and lim < 0.05 * (c.abs() * (y.abs() + 1)).sum()
        assert (grad - true).abs() <= 200 * U32 * (c.abs().sum() * 10)


# ---- dropout -------------------------------------------------------------------------------------

MASK = (1 << 64) - 1


def words64(seed, offset, n):
    """The generator in Python's whole numbers."""
    def mix(z):
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & MASK
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & MASK
        return z ^ (z >> 31)
    key = mix(seed & MASK)
    out = []
    for w in range((n + 3) // 4):
        bits = mix((key + 0x9E3779B97F4A7C15 * (offset + w + 1)) & MASK)
        out += [(bits >> s) & 0xFFFF for s in (0, 16, 32, 48)]
    return torch.tensor(out[:n])


def drop64(x, p, seed, offset, residual=None):
    t = int(p * 65536 + 0.5)
    keep = (words64(seed, offset, x.numel()) >= t).view(x.shape).to(x.device)
    y = torch.where(keep, x.double() * (65536.0 / (65536 - t) if t < 65536 else 0.0), 0.0)
    return (y if residual is None else y + residual.double()), keep


DROP_SHAPES = [(1, 1), (1, 3), (3, 1), (2, 2), (5, 7), (100, 136), (33, 511), (17, 1001), (257, 24), (1, 4099), (64, 512)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", DROP_SHAPES)
def test_dropout(dense, dtype, rows, cols):
    x, res = rand(1, rows, cols, dtype=dtype), rand(2, rows, cols, dtype=dtype)
    for p, seed, offset in ((0.1, 12345, 0), (0.5, (1 << 64) - 3, (1 << 40) + 7), (0.0, 0, 5), (1.0, 1, 1), (0.9999999, 7, 3)):
        for r in (None, res, padded(res, 2)):
            want, keep = drop64(x, p, seed, offset, r)
            tol = 2 * U32 * want.abs() + U32 * (2 * x.double().abs() * 65536 if p > 0.99 else 4 * x.double().abs())
            for v in (x, padded(x, 3), shifted(x, 1), shifted(x, 4)):
                close(dense.dropout(v, p, seed, offset, residual=r), want, tol, dtype, (p, seed))
        back = dense.dropout_backward(x, p, seed, offset)
        assert torch.equal(back != 0, keep & (x != 0))


def test_dropout_is_a_function_of_the_element(dense):
    """The same bits whatever the stride, the split into calls or the type; NaN in dropped places is gone."""
    x = torch.ones(60, 128, device="cuda")
    whole = dense.dropout(x, 0.3, 99, 11)
    assert torch.equal(dense.dropout(padded(x, 8), 0.3, 99, 11), whole)
    assert torch.equal(dense.dropout(x.half(), 0.3, 99, 11) != 0, whole != 0)
    halves = [dense.dropout(x[:30], 0.3, 99, 11), dense.dropout(x[30:], 0.3, 99, 11 + dense.dropout_words(x[:30]))]
    assert torch.equal(torch.cat(halves), whole)
    assert torch.equal(dense.dropout(x, 0.3, 99, 5, counter=torch.tensor([6], device="cuda")), whole)
    y = dense.dropout(torch.full_like(x, float("nan")), 0.3, 99, 11)
    assert torch.equal(torch.isnan(y), whole != 0) and not y[whole == 0].any()
    assert not torch.equal(dense.dropout(x, 0.3, 100, 11), whole)


def test_dropout_share_and_mean(dense):
    """Of n elements about p n are dropped: within 6 standard deviations of a binomial count."""
    n, p = 1 << 22, 0.1
    y = dense.dropout(torch.ones(n // 1024, 1024, device="cuda"), p, 2024)
    dropped = int((y == 0).sum())
    t = int(p * 65536 + 0.5) / 65536
    assert abs(dropped - t * n) < 6 * (n * t * (1 - t)) ** 0.5


def test_dropout_no_elements(dense):
    for shape in ((0, 8), (5, 0), (0,)):
        assert dense.dropout(torch.empty(shape, device="cuda"), 0.5, 1).shape == shape


# ---- gated feed-forward --------------------------------------------------------------------------

def act64(name, g):
    f = {"relu": torch.relu, "sigmoid": torch.sigmoid, "silu": lambda v: v * torch.sigmoid(v),
         "gelu": lambda v: 0.5 * v * (1 + torch.erf(v / 2 ** 0.5)),
         "gelu_tanh": lambda v: 0.5 * v * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3)))}[name]
    g = g.detach().requires_grad_(True)
    a = f(g)
    d, = torch.autograd.grad(a.sum(), g)
    return a.detach(), d


# an activation and its derivative are off by at most this many f32 roundings of (1 + |g|)
ACT_STEPS = 24


def ffn_forward_check(dense, dtype, act, x, wg, wu, views=()):
    m, k = x.shape
    g, u = x.double() @ wg.double().T, x.double() @ wu.double().T
    # k products and k additions in f32
    tg = 2 * U32 * (k + 8) * (x.double().abs() @ wg.double().abs().T)
    tu = 2 * U32 * (k + 8) * (x.double().abs() @ wu.double().abs().T)
    a, _ = act64(act, g)
    ta = 1.2 * tg + ACT_STEPS * U32 * (1 + g.abs())
    th = ta * u.abs() + a.abs() * tu + ta * tu + 2 * U32 * (a * u).abs()
    for args in ((x, wg, wu),) + tuple(views):
        h, sg, su = dense.gated_ffn(*args, act=act, save=True)
        close(h, a * u, th, dtype, "h")
        close(sg, g, tg, dtype, "gate")
        close(su, u, tu, dtype, "up")
        assert torch.equal(dense.gated_ffn(*args, act=act), h)


def ffn_backward_check(dense, dtype, act, x, wg, wu, seed=9, views=False):
    m, k = x.shape
    n = wg.shape[0]
    g, u = ((x.float() @ w.float().T).to(dtype) for w in (wg, wu))
    dh = rand(seed, m, n, dtype=dtype)
    a, d = act64(act, g.double())
    dg, du = dh.double() * u.double() * d, dh.double() * a
    # each passes through memory in the element type
    te = ACT_STEPS * U32 * (1 + g.double().abs())
    tg = U[dtype] * dg.abs() * 1.01 + te * (dh.double() * u.double()).abs() + 4 * U32 * dg.abs() + TINY[dtype]
    tu = U[dtype] * du.abs() * 1.01 + te * dh.double().abs() + 4 * U32 * du.abs() + TINY[dtype]
    W = [w.double() for w in (wg, wu)]
    dx = dg @ W[0] + du @ W[1]
    tx = tg @ W[0].abs() + tu @ W[1].abs() + 2 * U32 * (2 * n + 8) * (dg.abs() @ W[0].abs() + du.abs() @ W[1].abs())
    X = x.double()
    dw = [dg.T @ X, du.T @ X]
    tw = [t.T @ X.abs() + 2 * U32 * (m + 8) * (v.abs().T @ X.abs()) for t, v in ((tg, dg), (tu, du))]
    sets = [(dh, x, wg, wu, g, u)]
    if views:
        sets += [(padded(dh, 3), padded(x, 5), padded(wg, 1), padded(wu, 1), g, u),
                 (shifted(dh, 1), shifted(x, 3), shifted(wg, 5), shifted(wu, 7), shifted(g, 1), shifted(u, 2)),
                 (padded(dh, 8), padded(x, 16), padded(wg, 8), padded(wu, 8), g, u)]
    for args in sets:
        got = dense.gated_ffn_backward(*args, act=act)
        close(got[0], dx, tx, dtype, "dx")
        close(got[1], dw[0], tw[0], dtype, "dw_gate")
        close(got[2], dw[1], tw[1], dtype, "dw_up")


FFN_SHAPES = [(1, 1, 1), (1, 7, 5), (1, 64, 64), (1, 1024, 512), (2, 136, 512), (3, 8, 16), (5, 1000, 33), (16, 200, 130),
              (17, 136, 129), (33, 264, 250), (64, 64, 64), (100, 136, 512), (128, 100, 255), (129, 65, 257), (257, 72, 96),
              (300, 520, 1030), (1000, 24, 40), (513, 256, 384), (70, 2048, 72)]


def ffn_inputs(seed, m, k, n, dtype):
    return rand(seed, m, k, dtype=dtype), rand(seed + 1, n, k, dtype=dtype, scale=k ** -0.5), rand(seed + 2, n, k, dtype=dtype,
                                                                                                    scale=k ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", FFN_SHAPES)
def test_ffn_forward(dense, dtype, m, k, n):
    x, wg, wu = ffn_inputs(m + k, m, k, n, dtype)
    views = [(padded(x, 3), padded(wg, 1), padded(wu, 1)), (shifted(x, 1), shifted(wg, 3), shifted(wu, 5)),
             (padded(x, 8), padded(wg, 16), padded(wu, 16))]
    ffn_forward_check(dense, dtype, ACTS[(m + k + n) % 5], x, wg, wu, views)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", FFN_SHAPES)
def test_ffn_backward(dense, dtype, m, k, n):
    ffn_backward_check(dense, dtype, ACTS[(m + k) % 5], *ffn_inputs(m + n, m, k, n, dtype), views=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_ffn_activations(dense, dtype, act):
    """Each activation over a wide range of arguments, far tails included."""
    x, wg, wu = ffn_inputs(3, 40, 16, 48, dtype)
    x = x * 6
    ffn_forward_check(dense, dtype, act, x, wg, wu)
    ffn_backward_check(dense, dtype, act, x, wg, wu)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(2100, 256, 1100), (4096, 192, 768), (2050, 1032, 516), (9000, 136, 256), (600, 1024, 2048)])
def test_ffn_many_tiles(dense, dtype, m, k, n):
    x, wg, wu = ffn_inputs(m, m, k, n, dtype)
    ffn_forward_check(dense, dtype, "silu", x, wg, wu)
    ffn_backward_check(dense, dtype, "silu", x, wg, wu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(4090, 2040, 2044), (2000, 2041, 4090), (8192, 512, 1024), (4001, 1000, 2009), (1030, 2016, 8190)])
def test_ffn_large_tiles(dense, dtype, m, k, n):
    """Sizes whose products, forward or backward, are made in tiles of 256 x 256: whole and partial tiles and stages."""
    x, wg, wu = ffn_inputs(14, m, k, n, dtype)
    ffn_forward_check(dense, dtype, "silu", x, wg, wu)
    ffn_backward_check(dense, dtype, "gelu", x, wg, wu)


def test_ffn_broken_values_stay_in_their_row_and_column(dense):
    x, wg, wu = ffn_inputs(1, 130, 72, 200, torch.bfloat16)
    ref = dense.gated_ffn(x, wg, wu)
    x2, wg2 = x.clone(), wg.clone()
    x2[77, 71] = float("nan")
    wg2[150, 3] = float("inf")
    h = dense.gated_ffn(x2, wg2, wu)
    keep = torch.ones_like(h, dtype=torch.bool)
    keep[77], keep[:, 150] = False, False
    assert torch.equal(h[keep], ref[keep]) and torch.isnan(h[77]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_ffn_no_rows_and_leading_dimensions(dense, dtype):
    x, wg, wu = ffn_inputs(1, 12, 40, 24, dtype)
    empty = x[:0]
    h, g, u = dense.gated_ffn(empty, wg, wu, save=True)
    dx, dwg, dwu = dense.gated_ffn_backward(h, empty, wg, wu, g, u)
    assert h.shape == (0, 24) and dx.shape == (0, 40) and not dwg.any() and not dwu.any()
    flat, cube = dense.gated_ffn(x, wg, wu, save=True), dense.gated_ffn(x.view(3, 4, 40), wg, wu, save=True)
    assert all(torch.equal(p, q.view(12, 24)) and q.shape == (3, 4, 24) for p, q in zip(flat, cube))
    dh = rand(2, 12, 24, dtype=dtype)
    one = dense.gated_ffn_backward(dh, x, wg, wu, *flat[1:])
    two = dense.gated_ffn_backward(dh.view(3, 4, 24), x.view(3, 4, 40), wg, wu, *cube[1:])
    assert two[0].shape == (3, 4, 40) and all(torch.equal(p, q.view(p.shape)) for p, q in zip(one, two))


def test_ffn_gradient_against_differences(dense):
    x, wg, wu = ffn_inputs(4, 20, 48, 40, torch.float32)
    c = rand(5, 20, 40)
    h0, g, u = dense.gated_ffn(x, wg, wu, "silu", save=True)
    grads = dense.gated_ffn_backward(c, x, wg, wu, g, u, "silu")
    step = 2.0 ** -6

    def f64(x_, a_, b_):
        ga = x_.double() @ a_.double().T
        return ga * torch.sigmoid(ga) * (x_.double() @ b_.double().T)
    ins = (x, wg, wu)
    for i in range(3):
        v = rand(6 + i, *ins[i].shape, scale=0.3)
        hi = [t + step * v if j == i else t for j, t in enumerate(ins)]
        lo = [t - step * v if j == i else t for j, t in enumerate(ins)]
        own = ((dense.gated_ffn(*hi).double() - dense.gated_ffn(*lo).double()) * c.double()).sum() / (2 * step)
        far = ((f64(*hi) - f64(*lo)) * c.double()).sum() / (2 * step)
        leaf = [t.double().requires_grad_(True) for t in ins]
        true = (torch.autograd.grad((f64(*leaf) * c.double()).sum(), leaf)[i] * v).sum()
        grad = (grads[i].double() * v).sum()
        size = (c.double().abs() * (h0.double().abs() + 1)).sum()
        # k = 48 terms a product, two products
        lim = 2 * 2 * 56 * U32 * size / step + (far - true).abs()
        assert (own - grad).abs() <= lim and lim < 0.05 * size
        assert (grad - true).abs() <= 4 * 56 * U32 * (grads[i].double().abs() * v.abs()).sum() * 10


# ---- how they are called -------------------------------------------------------------------------

def raw(dense):
    from quickrank_amd import _capi
    return _capi.lib()


@pytest.mark.parametrize("dtype", TYPES)
def test_outputs_of_longer_rows_leave_the_rest_alone(dense, dtype):
    """The C calls write rows of any stride and nothing behind them."""
    L, code, e = raw(dense), dense.TYPES[dtype], torch.finfo(dtype)
    m, k, n = 37, 45, 21
    x, wg, wu = ffn_inputs(1, m, k, n, dtype)
    s = torch.cuda.current_stream().cuda_stream

    def out(rows, cols, pad):
        buf = torch.full((rows + 1, cols + pad), 7.0, dtype=dtype, device="cuda")
        return buf, buf[:rows, :cols]

    def untouched(buf, rows, cols):
        b = buf.clone()
        b[:rows, :cols] = 7.0
        return bool((b == 7.0).all())
    by, y = out(m, k, 3)
    assert L.qr_layer_norm_async(0, s, code, code, m, k, x.data_ptr(), k, None, None, 1e-5, y.data_ptr(), k + 3, None, None) == 0
    ref, mean, rstd = dense.layer_norm(x)
    assert torch.equal(y, ref) and untouched(by, m, k)
    bd, d = out(m, k, 5)
    assert L.qr_dropout_async(0, s, code, m, k, x.data_ptr(), k, None, 0, d.data_ptr(), k + 5, 0.25, 3, 4, None) == 0
    assert torch.equal(d, dense.dropout(x, 0.25, 3, 4)) and untouched(bd, m, k)
    bh, h = out(m, n, 2)
    need = C.c_size_t()
    assert L.qr_gated_ffn_workspace(code, m, k, n, C.byref(need)) == 0
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    assert L.qr_gated_ffn_async(0, s, code, 0, m, k, n, x.data_ptr(), k, wg.data_ptr(), wu.data_ptr(), k, h.data_ptr(), n + 2,
                                None, None, ws.data_ptr(), need.value) == 0
    hr, g, u = dense.gated_ffn(x, wg, wu, save=True)
    assert torch.equal(h, hr) and untouched(bh, m, n)
    bx, dx = out(m, k, 7)
    assert L.qr_gated_ffn_backward_workspace(code, m, k, n, C.byref(need)) == 0
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    dw = torch.empty(2, n, k, dtype=dtype, device="cuda")
    assert L.qr_gated_ffn_backward_async(0, s, code, 0, m, k, n, hr.data_ptr(), n, x.data_ptr(), k, wg.data_ptr(), wu.data_ptr(), k,
                                         g.data_ptr(), u.data_ptr(), dx.data_ptr(), k + 7, dw.data_ptr(), dw[1].data_ptr(),
                                         ws.data_ptr(), need.value) == 0
    want = dense.gated_ffn_backward(hr, x, wg, wu, g, u)
    assert torch.equal(dx, want[0]) and torch.equal(dw[0], want[1]) and untouched(bx, m, k)
    assert L.qr_layer_norm_backward_workspace(m, k, C.byref(need)) == 0
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    bn, dn = out(m, k, 1)
    dp = torch.empty(2, k, dtype=dtype, device="cuda")
    assert L.qr_layer_norm_backward_async(0, s, code, code, m, k, y.data_ptr(), k + 3, x.data_ptr(), k, None, mean.data_ptr(),
                                          rstd.data_ptr(), dn.data_ptr(), k + 1, dp.data_ptr(), dp[1].data_ptr(), ws.data_ptr(),
                                          need.value) == 0
    want = dense.layer_norm_backward(ref, x, None, mean, rstd)
    assert torch.equal(dn, want[0]) and torch.equal(dp[0], want[1]) and torch.equal(dp[1], want[2]) and untouched(bn, m, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [45, 136, 4099])
def test_in_place(dense, dtype, cols):
    """y over x, dx over dy: what the C calls allow."""
    L, code, m = raw(dense), dense.TYPES[dtype], 37
    x, dy = rand(1, m, cols, dtype=dtype), rand(2, m, cols, dtype=dtype)
    s = torch.cuda.current_stream().cuda_stream
    y, mean, rstd = dense.layer_norm(x)
    want = dense.layer_norm_backward(dy, x, None, mean, rstd)
    v, d = x.clone(), dy.clone()
    need = C.c_size_t()
    assert L.qr_layer_norm_backward_workspace(m, cols, C.byref(need)) == 0
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    dp = torch.empty(2, cols, dtype=dtype, device="cuda")
    assert L.qr_layer_norm_backward_async(0, s, code, code, m, cols, d.data_ptr(), cols, x.data_ptr(), cols, None, mean.data_ptr(),
                                          rstd.data_ptr(), d.data_ptr(), cols, dp.data_ptr(), dp[1].data_ptr(), ws.data_ptr(),
                                          need.value) == 0
    assert torch.equal(d, want[0]) and torch.equal(dp[0], want[1]) and torch.equal(dp[1], want[2])
    assert L.qr_layer_norm_async(0, s, code, code, m, cols, v.data_ptr(), cols, None, None, 1e-5, v.data_ptr(), cols, None, None) == 0
    assert torch.equal(v, y)
    want = dense.dropout(x, 0.3, 5, residual=dy)
    r = dy.clone()
    assert L.qr_dropout_async(0, s, code, m, cols, x.data_ptr(), cols, r.data_ptr(), cols, r.data_ptr(), cols, 0.3, 5, 0, None) == 0
    assert torch.equal(r, want)


def block(dense, x, w, b, wg, wu, wd, p, seed, counter=None):
    """x + dropout(gated(norm(x)) wd^T), and the gradients for a gradient of ones."""
    y, mean, rstd = dense.layer_norm(x, w, b)
    h, g, u = dense.gated_ffn(y, wg, wu, save=True)
    out = dense.dropout(h @ wd.T, p, seed, residual=x, counter=counter)
    do = torch.ones_like(out)
    dz = dense.dropout_backward(do, p, seed, counter=counter)
    dy, dwg, dwu = dense.gated_ffn_backward(dz @ wd, y, wg, wu, g, u)
    dx, dw, db = dense.layer_norm_backward(dy, x, w, mean, rstd)
    return out, dx + do, dw, db, dwg, dwu


def block_inputs(dtype=torch.bfloat16, m=300, k=136, n=264):
    x, wg, wu = ffn_inputs(1, m, k, n, dtype)
    return x, rand(4, k, shift=1), rand(5, k), wg, wu, rand(6, k, n, dtype=dtype, scale=n ** -0.5)


def test_the_same_call_twice_gives_the_same_bits(dense):
    ins = block_inputs()
    a, b = block(dense, *ins, 0.2, 3), block(dense, *ins, 0.2, 3)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_on_another_stream(dense):
    ins = block_inputs()
    want = block(dense, *ins, 0.2, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block(dense, *ins, 0.2, 3)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_two_captured_graphs_replayed_side_by_side(dense):
    """Two graphs of the whole block, each with memory of its own, replayed on two streams at once and among eager work."""
    ins = block_inputs()
    counters = [torch.zeros(1, dtype=torch.int64, device="cuda") for _ in range(2)]
    block(dense, *ins, 0.2, 3, counters[0])  # the libraries' handles exist before a capture
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in counters:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(block(dense, *ins, 0.2, 3, c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step in range(4):
        for i, c in enumerate(counters):
            c.fill_(1000 * step + 17 * i)
        want = [block(dense, *ins, 0.2, 3, c) for c in counters]
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(got, ref)), step
    assert not torch.equal(outs[0][0], outs[1][0])


def test_threads_call_at_once(dense):
    import threading
    ins = block_inputs()
    want = block(dense, *ins, 0.2, 3)
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got = block(dense, *ins, 0.2, 3)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(p, q) for p, q in zip(got, want)):
                    bad.append(1)
    ts = [threading.Thread(target=work) for _ in range(3)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_refusals_on_the_gpu(dense):
    from quickrank_amd import QrError
    x, wg, wu = ffn_inputs(1, 4, 8, 6, torch.float32)
    w = rand(1, 8)
    _, mean, rstd = dense.layer_norm(x, w)
    h, g, u = dense.gated_ffn(x, wg, wu, save=True)
    for call in (lambda: dense.layer_norm(x.t()),                       # columns of a stride
                 lambda: dense.layer_norm(x, w[:7]),
                 lambda: dense.layer_norm(x, w.half()),
                 lambda: dense.layer_norm(x.bfloat16(), w, w.bfloat16()),
                 lambda: dense.layer_norm(x, w, eps=-1.0),
                 lambda: dense.layer_norm(x, w, eps=float("nan")),
                 lambda: dense.layer_norm(x.double()),
                 lambda: dense.layer_norm(x[:, :0]),
                 lambda: dense.layer_norm(x.clone().requires_grad_(True)),
                 lambda: dense.layer_norm_backward(x[:3], x, w, mean, rstd),
                 lambda: dense.layer_norm_backward(x.half(), x, w, mean, rstd),
                 lambda: dense.layer_norm_backward(x, x, w, mean[:3], rstd),
                 lambda: dense.layer_norm_backward(x, x, w, mean.half(), rstd),
                 lambda: dense.dropout(x, -0.1, 1),
                 lambda: dense.dropout(x, 1.1, 1),
                 lambda: dense.dropout(x, float("nan"), 1),
                 lambda: dense.dropout(x, 0.1, 1, residual=x[:2]),
                 lambda: dense.dropout(x, 0.1, 1, residual=x.half()),
                 lambda: dense.dropout(x, 0.1, 1, counter=torch.zeros(1)),
                 lambda: dense.dropout(x, 0.1, 1, counter=torch.zeros(2, dtype=torch.int64, device="cuda")),
                 lambda: dense.gated_ffn(x, wg, wu[:5]),
                 lambda: dense.gated_ffn(x, wg[:, :7], wu[:, :7]),
                 lambda: dense.gated_ffn(x, wg.half(), wu.half()),
                 lambda: dense.gated_ffn(x, wg, wu, "tanh"),
                 lambda: dense.gated_ffn(x, wg[:0], wu[:0]),
                 lambda: dense.gated_ffn(x, wg.cpu(), wu),
                 lambda: dense.gated_ffn_backward(h[:3], x, wg, wu, g, u),
                 lambda: dense.gated_ffn_backward(h, x, wg, wu, g.half(), u),
                 lambda: dense.gated_ffn_backward(h, x, wg, wu, padded(g, 1), u)):
        with pytest.raises(QrError):
            call()
    x.requires_grad_(True)
    with torch.no_grad():
        dense.layer_norm(x, w)


# ---- offsets beyond 32 bits ------------------------------------------------------------------------

def test_dropout_beyond_2_32_elements(dense):
    """The tail of 2^32 + 4099 elements equals a call of its own at its word's offset."""
    n = (1 << 32) + 4099
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = dense.dropout(x, 0.3, 17, 5)
    start = (1 << 32) - 8
    tail = dense.dropout(x[start:].contiguous(), 0.3, 17, 5 + start // 4)
    assert torch.equal(y[start:], tail) and torch.equal(y[:64], dense.dropout(x[:64], 0.3, 17, 5))
    wide = y.view(1, n)
    assert torch.equal(dense.dropout(x.view(1, n), 0.3, 17, 5)[0, start:], tail) and wide.shape == (1, n)


def test_norm_beyond_2_32_elements(dense):
    """Rows at the end of 2^32 + 2^20 elements, forward and backward."""
    cols = 2048
    rows = (1 << 21) + 512
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    x[-3:] = rand(1, 3, cols, dtype=torch.bfloat16)
    w, b = rand(2, cols), rand(3, cols)
    y, mean, rstd = dense.layer_norm(x, w, b)
    want = dense.layer_norm(x[-3:].clone(), w, b)
    assert torch.equal(y[-3:], want[0]) and torch.equal(mean[-3:], want[1]) and torch.equal(rstd[-3:], want[2])
    dy = y.zero_()
    dy[-3:] = rand(4, 3, cols, dtype=torch.bfloat16)
    got = dense.layer_norm_backward(dy, x, w, mean, rstd)
    ref = dense.layer_norm_backward(dy[-3:].clone(), x[-3:].clone(), w, mean[-3:].clone(), rstd[-3:].clone())
    assert torch.equal(got[0][-3:], ref[0])
    for p, q in zip(got[1:], ref[1:]):
        # (three addends a column, in another order: two additions and a product, each half a step of f32)
        size = dy[-3:].double().abs().max() * 8 * 3
        assert (p.double() - q.double()).abs().max() <= 8 * U32 * size


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_far_apart(dense, dtype):
    """Rows 2^24 elements apart: offsets beyond 2^31 elements, strides longer than the product kernel's tiles reach."""
    m, k, n, far = 200, 72, 136, 1 << 24
    x, wg, wu = ffn_inputs(1, m, k, n, dtype)
    buf = torch.full(((m - 1) * far + k,), float("nan"), dtype=dtype, device="cuda")
    v = buf.as_strided((m, k), (far, 1))
    v.copy_(x)
    w = rand(4, k)
    assert all(torch.equal(p, q) for p, q in zip(dense.layer_norm(v, w), dense.layer_norm(x, w)))
    assert torch.equal(dense.dropout(v, 0.4, 3), dense.dropout(x, 0.4, 3))
    h = dense.gated_ffn(x, wg, wu, save=True)
    assert all(torch.equal(p, q) for p, q in zip(dense.gated_ffn(v, wg, wu, save=True), h))
    want = dense.gated_ffn_backward(h[0], x, wg, wu, *h[1:])
    assert all(torch.equal(p, q) for p, q in zip(dense.gated_ffn_backward(h[0], v, wg, wu, *h[1:]), want))
    many = rand(5, 4000, k, dtype=dtype)  # (the tiled kernels)
    far_w = buf.as_strided((n, k), (far, 1))
    far_w.copy_(wg)
    far_u = torch.empty_like(buf).as_strided((n, k), (far, 1))
    far_u.copy_(wu)
    h = dense.gated_ffn(many, wg, wu, save=True)
    assert all(torch.equal(p, q) for p, q in zip(dense.gated_ffn(many, far_w, far_u, save=True), h))
    want = dense.gated_ffn_backward(h[0], many, wg, wu, *h[1:])
    assert all(torch.equal(p, q) for p, q in zip(dense.gated_ffn_backward(h[0], many, far_w, far_u, *h[1:]), want))


@pytest.mark.parametrize("dtype", TYPES)
def test_ffn_broadcast_inputs(dense, dtype):
    """One row for all rows of x, of dh, of the weights: strides of 0."""
    x, wg, wu = ffn_inputs(1, 1, 72, 130, dtype)
    many = x.expand(700, 72)
    a, b = dense.gated_ffn(many, wg, wu, save=True), dense.gated_ffn(many.contiguous(), wg, wu, save=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    dh = rand(2, 1, 130, dtype=dtype).expand(700, 130)
    a = dense.gated_ffn_backward(dh, many, wg, wu, *b[1:])
    b = dense.gated_ffn_backward(dh.contiguous(), many.contiguous(), wg, wu, *b[1:])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    one = wg[:1].expand(130, 72)
    assert torch.equal(dense.gated_ffn(many, one, one), dense.gated_ffn(many.contiguous(), one.contiguous(), one.contiguous()))


def test_f32_products_keep_24_bits(dense):
    """Numbers whose low mantissa bits decide: (1 + 2^-23) (1 - 2^-23) summed against -1, in units that f32 holds."""
    m, k, n = 130, 64, 130
    x, w = torch.zeros(m, k, device="cuda"), torch.zeros(n, k, device="cuda")
    x[:, 0], w[:, 0] = 1 + 2.0 ** -23, 1.0
    x[:, 1], w[:, 1] = -1.0, 1.0
    x[:, 2], w[:, 2] = 2.0 ** -40, 3.0
    _, g, u = dense.gated_ffn(x, w, w, "relu", save=True)
    want = torch.full_like(g, 2.0 ** -23 + 3 * 2.0 ** -40)
    # the first two cancel exactly; what the split leaves out is below 2^-21 of the largest product
    assert (g - want).abs().max() <= 2.0 ** -40 and torch.equal(g, u)


def test_dropout_seeds_of_numpy(dense):
    np = pytest.importorskip("numpy")
    x = rand(70, 9, 40)
    want = dense.dropout(x, 0.5, 7, offset=3)
    assert torch.equal(dense.dropout(x, 0.5, np.int64(7), offset=np.int32(3)), want)
    assert torch.equal(dense.dropout(x, 0.5, np.uint64(7), offset=np.int64(3)), want)
    assert torch.equal(dense.dropout(x, 0.5, np.int64(-1)), dense.dropout(x, 0.5, 2 ** 64 - 1))
    with pytest.raises(dense.QrError):
        dense.dropout(x, 0.5, 7.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(3000, 601, 64), (700, 65, 333), (2500, 129, 50), (300, 1023, 1000), (4100, 63, 4000), (9000, 8, 127),
                                   (65, 5, 9000)])
def test_ffn_rows_off_boundaries(dense, dtype, m, k, n):
    """Odd rows, rows of whole pieces at odd strides and bases: read as they lie or copied, by the sizes."""
    x, wg, wu = ffn_inputs(31, m, k, n, dtype)
    ffn_forward_check(dense, dtype, "gelu_tanh", x, wg, wu,
                      [(padded(x, 3), padded(wg, 5), padded(wu, 5)), (shifted(x, 1), shifted(wg, 3), shifted(wu, 2)),
                       (x, padded(wg, 1), padded(wu, 1)), (padded(x, 1), wg, wu)])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(700, 8200), (600, 16400), (300, 40_001), (3, 2_100_000)])
def test_norm_backward_of_rows_that_no_registers_hold(dense, dtype, rows, cols):
    norm_grad_check(dense, dtype, dtype, rows, cols)


def test_ffn_of_one_feature_or_one_unit_and_views(dense):
    """One column of wider weights, one row: both weights of one layout are read as they lie, others are refused."""
    from quickrank_amd import QrError
    x, dh = rand(1, 40, 1), rand(2, 40, 50)
    wide = rand(3, 2, 50, 64)
    wg, wu = wide[0][:, 5:6], wide[1][:, 5:6]
    want = dense.gated_ffn(x, wg.contiguous(), wu.contiguous(), save=True)
    got = dense.gated_ffn(x, wg, wu, save=True)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    back = [dense.gated_ffn_backward(dh, x, *w, *want[1:]) for w in ((wg, wu), (wg.contiguous(), wu.contiguous()))]
    assert all(torch.equal(p, q) for p, q in zip(*back))
    row = rand(4, 8, 2)
    y, dh1 = rand(5, 40, 8), rand(6, 40, 1)
    bad = [(x, wg, wu.contiguous(), dh), (x, wg.contiguous(), wu, dh), (y, row.t()[:1].contiguous(), row.t()[:1], dh1)]
    for v, a, b, d in bad:
        for call in (lambda: dense.gated_ffn(v, a, b), lambda: dense.gated_ffn_backward(d, v, a, b, d, d)):
            with pytest.raises(QrError):
                call()


# (m, k, n; scales of dh, x, the weights, gate, up): the gradients of the products lie far below f16's normal numbers or above
# its largest, the results do not
F16_RANGE = [(0, 2.0 ** -20, 2.0 ** 8, 2.0 ** -8, 1.0, 1.0), (1, 2.0 ** -20, 2.0 ** -8, 2.0 ** 8, 1.0, 1.0),
             (2, 2.0 ** -23, 2.0 ** 10, 2.0 ** -3, 1.0, 2.0 ** -6), (3, 300.0, 2.0 ** -12, 2.0 ** -12, 4.0, 400.0),
             (4, 2.0 ** 13, 2.0 ** -14, 2.0 ** -14, 2.0 ** 6, 2.0 ** -8)]


def f16_gradient(dh, x, wg, wu, g, u, act="silu"):
    """The gradients in 64 bits and what rounding dg and du once, to 11 bits or 2^-39 of the largest, and one rounding of the
    result may do to them."""
    dh, x, wg, wu, g, u = (t.double() for t in (dh, x, wg, wu, g, u))
    a, d = act64(act, g)
    dg, du = dh * u * d, dh * a
    te = ACT_STEPS * U32 * (1 + g.abs())
    big = max(float(dg.abs().max()), float(du.abs().max()))
    tg, tu = (2.0 ** -11 * 1.01 * v.abs() + te * w.abs() + 4 * U32 * v.abs() + 2.0 ** -39 * big for v, w in ((dg, dh * u), (du, dh)))
    m, n = dh.shape
    dx = dg @ wg + du @ wu
    tx = tg @ wg.abs() + tu @ wu.abs() + 2 * U32 * (2 * n + 8) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    dw = [v.T @ x for v in (dg, du)]
    tw = [t.T @ x.abs() + 2 * U32 * (m + 8) * (v.abs().T @ x.abs()) for t, v in ((tg, dg), (tu, du))]
    return (dx, *dw), (tx, *tw)


@pytest.mark.parametrize("m,k,n", [(20000, 64, 32), (70, 33, 31), (3000, 136, 512), (2048, 2040, 1032)])
@pytest.mark.parametrize("number,sdh,sx,sw,sg,su", F16_RANGE)
def test_ffn_backward_of_f16_keeps_what_f16_cannot_hold(dense, m, k, n, number, sdh, sx, sw, sg, su):
    t = torch.float16
    x, wg, wu = rand(1, m, k, dtype=t, scale=sx), rand(2, n, k, dtype=t, scale=sw), rand(3, n, k, dtype=t, scale=sw)
    dh, g, u = rand(4, m, n, dtype=t, scale=sdh), rand(5, m, n, dtype=t, scale=sg), rand(6, m, n, dtype=t, scale=su)
    want, tol = f16_gradient(dh, x, wg, wu, g, u)
    got = dense.gated_ffn_backward(dh, x, wg, wu, g, u)
    for i, what in enumerate(("dx", "dw_gate", "dw_up")):
        assert want[i].abs().max() < 60000
        close(got[i], want[i], tol[i], t, what)
        # as a whole: two roundings of 2^-11 / 3^1/2 each where the results are normal numbers, within 2 of that
        normal = want[i].abs() > 2.0 ** -14
        if normal.double().mean() > 0.5:
            e = (got[i].double() - want[i])[normal].norm() / want[i][normal].norm()
            assert e < 2 * 2 ** 0.5 * 2.0 ** -11 / 3 ** 0.5, (what, float(e))


def test_ffn_backward_of_f16_with_broken_and_zero_gradients(dense):
    """The scale comes from the finite numbers: what is not finite stays in its row and column, and zeros stay zeros."""
    t, m, k, n = torch.float16, 600, 72, 96
    x, wg, wu = ffn_inputs(1, m, k, n, t)
    g, u, dh = rand(2, m, n, dtype=t), rand(3, m, n, dtype=t), rand(4, m, n, dtype=t, scale=1e-5)
    ref = dense.gated_ffn_backward(dh, x, wg, wu, g, u)
    bad = dh.clone()
    bad[17, 5], bad[400, 90] = float("inf"), float("nan")
    got = dense.gated_ffn_backward(bad, x, wg, wu, g, u)
    rows, cols = torch.ones(m, dtype=torch.bool), torch.ones(n, dtype=torch.bool)
    rows[[17, 400]], cols[[5, 90]] = False, False
    assert torch.equal(got[0][rows], ref[0][rows]) and not torch.isfinite(got[0][~rows]).any()
    for p, q in zip(got[1:], ref[1:]):
        assert torch.equal(p[cols], q[cols]) and not torch.isfinite(p[~cols]).any()
    none = dense.gated_ffn_backward(torch.zeros_like(dh), x, wg, wu, g, u)
    assert not any(v.any() for v in none)


def test_ffn_backward_of_f16_captured(dense):
    """Replayed on gradients of other sizes, each time among eager work: the scale is made anew."""
    t = torch.float16
    x, wg, wu = ffn_inputs(1, 900, 136, 200, t)
    _, g, u = dense.gated_ffn(x, wg, wu, save=True)
    base, dh = rand(4, 900, 200), torch.zeros(900, 200, dtype=t, device="cuda")
    dense.gated_ffn_backward(dh, x, wg, wu, g, u)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = dense.gated_ffn_backward(dh, x, wg, wu, g, u)
    for scale in (1.0, 2.0 ** -18, 2.0 ** 9, 0.0, 2.0 ** -3):
        dh.copy_(base * scale)
        want = [v.clone() for v in dense.gated_ffn_backward(dh, x, wg, wu, g, u)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), scale


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
def test_ffn_backward_of_far_activations(dense, dtype, act):
    """Gates of up to 2^100 on either side of zero: the derivative is 0 or 1 (a sigmoid's 0) there, whatever its factors are."""
    far = [s * 2.0 ** e for e in (5, 6, 7, 20, 43, 44, 50, 62, 63, 65, 100) for s in (1, -1)]
    n, m = len(far), 40
    g = torch.tensor(far, device="cuda").expand(m, n).contiguous().to(dtype)
    u, dh = rand(1, m, n, dtype=dtype), rand(2, m, n, dtype=dtype)
    x, w = torch.eye(m, device="cuda", dtype=dtype), torch.eye(n, device="cuda", dtype=dtype)[:, :n]
    # (products with unit matrices: dw_gate^T is dg, dw_up^T is du, each rounded once)
    _, dwg, dwu = dense.gated_ffn_backward(dh, x, torch.zeros(n, m, device="cuda", dtype=dtype), torch.zeros(n, m, device="cuda", dtype=dtype),
                                           g, u, act)
    s, one = (g > 0).double(), dh.double() * u.double()
    slope = torch.zeros_like(s) if act == "sigmoid" else s
    value = s if act == "sigmoid" else s * g.double()
    # (2^5 and beyond: 1 - sigmoid, erf's tail and the like are below 2^-45, far under a rounding of 1)
    close(dwg.T.contiguous(), one * slope, 4 * U32 * one.abs() + 2.0 ** -40, dtype, "dg")
    close(dwu.T.contiguous(), dh.double() * value, 4 * U32 * (dh.double() * value).abs() + 2.0 ** -35, dtype, "du")


@pytest.mark.parametrize("act", ACTS)
def test_ffn_forward_of_far_activations(dense, act):
    """The same gates forward, by the few-rows kernel and by tiles, f32."""
    far = [s * 2.0 ** e for e in (5, 7, 20, 44, 62, 65, 100) for s in (1, -1)]
    n = len(far)
    for m in (3, 40000):
        x = rand(1, m, 1).abs() + 0.5
        wg, wu = torch.tensor(far, device="cuda").view(n, 1), torch.ones(n, 1, device="cuda")
        h = dense.gated_ffn(x, wg, wu, act)
        g = x.double() @ wg.double().T
        a = (g > 0).double() if act == "sigmoid" else g.clamp(min=0)
        close(h, a * x.double(), 16 * U32 * (a * x.double()).abs() + 2.0 ** -16, torch.float32, "h")


def f32_products(dense, m, k, n):
    """(result, the one product it is, in 64 bits) of the forward pass, dx and both dW: every other term of the sums is zero,
    every factor has 24 bits, all sizes above the few-rows kernel's."""
    g = torch.Generator(device="cuda")
    g.manual_seed(m + k + n)

    def full(*shape):  # in 1 .. 2, either sign
        return (1 + torch.rand(shape, generator=g, device="cuda")) * (1 - 2 * torch.randint(0, 2, shape, generator=g, device="cuda"))
    x, wg, wu = torch.zeros(m, k, device="cuda"), torch.zeros(n, k, device="cuda"), torch.zeros(n, k, device="cuda")
    x[:, k // 2], wg[:, k // 2], wu[:, k // 2] = full(m), full(n), full(n)
    _, gate, up = dense.gated_ffn(x, wg, wu, "relu", save=True)
    for got, w in ((gate, wg), (up, wu)):
        yield "forward", got, x[:, k // 2].double()[:, None] * w[:, k // 2].double()
    x, wg, wu = full(m, k), full(n, k), full(n, k)
    one, none = torch.ones(m, n, device="cuda"), torch.zeros(m, n, device="cuda")
    for gate, up, w, i in ((one, none, wu, 2), (none + 2.0 ** -30, one, wg, 1)):  # du = dh, dg = 0; dg = dh, du as good as 0
        dh = torch.zeros(m, n, device="cuda")
        dh[:, n // 3] = full(m)
        dx, *_ = dense.gated_ffn_backward(dh, x, wg if i == 1 else torch.zeros_like(wg), wu if i == 2 else torch.zeros_like(wu), gate, up, "relu")
        yield "dx", dx, dh[:, n // 3].double()[:, None] * w[n // 3].double()
        dh.zero_()
        dh[m // 2] = full(n)
        got = dense.gated_ffn_backward(dh, x, wg, wu, gate, up, "relu")[i]
        yield "dW", got, dh[m // 2].double()[:, None] * x[m // 2].double()


@pytest.mark.parametrize("m,k,n", [(4096, 256, 1024), (4096, 64, 1024), (9000, 96, 1000), (9000, 160, 1000), (3001, 129, 999)])
def test_f32_products_of_the_tiled_kernels_are_as_near_as_f32(dense, m, k, n):
    """One product of two numbers of 24 bits each.  To the nearest, the parts of a number of 1 .. 2 are at most 2, 2^-8 and
    2^-16, so what is left out is at most 2 x 2^-24 + 2^-32, of a product of 1 at least: 2.1 units of 2^-24.  The six that are
    taken are added smallest first: one rounding of the result (1 unit, 2 if an addition cuts off) and two of terms below 2^-6
    of it.  5 in all; and nothing of it leans to one side: the mean over all products within a tenth of a unit.  (Parts cut
    off instead have one sign and left out 7 units at most, 0.63 on average.)"""
    for what, got, want in f32_products(dense, m, k, n):
        assert got.dtype == torch.float32 and want.abs().min() >= 1
        e = (got.double() - want) / want * 2.0 ** 24
        assert e.abs().max() <= 5 and abs(float(e.mean())) <= 0.1, (what, float(e.abs().max()), float(e.mean()))
        assert e.square().mean().sqrt() <= 0.6, (what, float(e.square().mean().sqrt()))


@pytest.mark.parametrize("m,n", [(3, 50), (100, 512), (4000, 512), (4001, 200)])
def test_ffn_f32_of_infinite_factors(dense, m, n):
    """An infinite feature or weight: its row or column is not finite, whichever kernel makes it, and no other element changes.
    Few rows: what f32 arithmetic gives."""
    k = 72
    x, wg, wu = ffn_inputs(m, m, k, n, torch.float32)
    x2, wg2 = x.clone(), wg.clone()
    x2[m // 2, 7], wg2[n // 3, 70] = float("inf"), float("-inf")
    ref, got = dense.gated_ffn(x, wg, wu, "sigmoid", save=True), dense.gated_ffn(x2, wg2, wu, "sigmoid", save=True)
    rows, cols = torch.ones(m, dtype=torch.bool), torch.ones(n, dtype=torch.bool)
    rows[m // 2], cols[n // 3] = False, False
    for i, (p, q) in enumerate(zip(got, ref)):
        assert torch.equal(p[rows][:, cols], q[rows][:, cols])
        if i:  # gate and up; up does not see w_gate
            assert not torch.isfinite(p[~rows]).any() and (i == 2 or not torch.isfinite(p[:, ~cols]).any())
    if m <= 100:
        g = x2.double() @ wg2.double().T
        assert torch.equal(got[1].isnan(), g.isnan()) and torch.equal(got[1].isinf(), g.isinf())
        assert torch.equal(got[1][g.isinf()].double(), g[g.isinf()])
    dh = rand(9, m, n)
    a, b = dense.gated_ffn_backward(dh, x, wg, wu, *ref[1:], "sigmoid"), dense.gated_ffn_backward(dh, x2, wg, wu, *ref[1:], "sigmoid")
    keep = torch.arange(k) != 7
    for i in (1, 2):  # the sums over rows: only the feature's own column
        assert torch.equal(a[i][:, keep], b[i][:, keep]) and not torch.isfinite(b[i][:, 7]).any()
    assert torch.equal(a[0], b[0])


def test_an_earlier_failed_call_of_the_runtime_is_not_ours(dense):
    """A HIP call that failed before on this thread does not make an enqueued operator fail, and its error is still there for
    whom it concerns."""
    L = raw(dense)
    L.hipSetDevice.argtypes, L.hipSetDevice.restype, L.hipGetLastError.restype = [C.c_int], C.c_int, C.c_int
    x, w = rand(1, 30, 8), rand(2, 6, 8)
    h, g, u = dense.gated_ffn(x, w, w, save=True)
    _, mean, rstd = dense.layer_norm(x)
    for call in (lambda: dense.layer_norm(x), lambda: dense.layer_norm_backward(x, x, None, mean, rstd), lambda: dense.dropout(x, 0.5, 1),
                 lambda: dense.gated_ffn(x, w, w), lambda: dense.gated_ffn_backward(h, x, w, w, g, u)):
        want = call()
        e = L.hipSetDevice(4096)
        try:
            got = call()
        finally:
            left = L.hipGetLastError()
        assert e != 0 and left == e
        pairs = [(want, got)] if isinstance(want, torch.Tensor) else zip(want, got)
        assert all(torch.equal(p, q) for p, q in pairs)


def test_tangents_of_any_argument_are_refused(dense):
    from torch.autograd import forward_ad
    from quickrank_amd import QrError
    x, wg, wu = ffn_inputs(1, 4, 8, 6, torch.float32)
    w = rand(1, 8)
    want, mean, rstd = dense.layer_norm(x, w)
    h, g, u = dense.gated_ffn(x, wg, wu, save=True)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: dense.layer_norm(x, dual(w)), lambda: dense.layer_norm(x, None, dual(w)),
                     lambda: dense.layer_norm_backward(dual(x), x, w, mean, rstd), lambda: dense.layer_norm_backward(x, x, w, dual(mean), rstd),
                     lambda: dense.dropout(x, 0.1, 1, residual=dual(x)), lambda: dense.gated_ffn(x, dual(wg), wu),
                     lambda: dense.gated_ffn(x, wg, dual(wu)), lambda: dense.gated_ffn_backward(dual(h), x, wg, wu, g, u),
                     lambda: dense.gated_ffn_backward(h, x, wg, wu, g, dual(u))):
            with pytest.raises(QrError) as e:
                call()
            assert "tangent" in str(e.value)
        assert torch.equal(dense.layer_norm(x, w)[0], want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(37, 45, 21), (3000, 64, 200), (5000, 136, 264)])
def test_outputs_beside_the_inputs_in_one_buffer(dense, dtype, m, k, n):
    """x in the first columns of a buffer and h in the next, dx beside dh, y beside x: the C calls write their columns only."""
    L, code, s = raw(dense), dense.TYPES[dtype], torch.cuda.current_stream().cuda_stream
    x, wg, wu = ffn_inputs(1, m, k, n, dtype)
    e, need = x.element_size(), C.c_size_t()

    def space():
        return torch.empty(need.value, dtype=torch.uint8, device="cuda")
    buf = torch.full((m, k + n + 3), 7.0, dtype=dtype, device="cuda")
    buf[:, :k] = x
    ld = k + n + 3
    g, u = torch.empty(2, m, n, dtype=dtype, device="cuda")
    assert L.qr_gated_ffn_workspace(code, m, k, n, C.byref(need)) == 0
    ws = space()
    assert L.qr_gated_ffn_async(0, s, code, 0, m, k, n, buf.data_ptr(), ld, wg.data_ptr(), wu.data_ptr(), k, buf.data_ptr() + k * e, ld,
                                g.data_ptr(), u.data_ptr(), ws.data_ptr(), need.value) == 0
    want = dense.gated_ffn(buf[:, :k], wg, wu, save=True)
    assert torch.equal(buf[:, k:k + n], want[0]) and torch.equal(g, want[1]) and torch.equal(u, want[2])
    assert torch.equal(buf[:, :k], x) and (buf[:, k + n:] == 7).all()
    # dh in the first n columns, dx in the next k
    buf[:, :n] = rand(2, m, n, dtype=dtype)
    dh = buf[:, :n].clone()
    dw = torch.empty(2, n, k, dtype=dtype, device="cuda")
    assert L.qr_gated_ffn_backward_workspace(code, m, k, n, C.byref(need)) == 0
    ws = space()
    assert L.qr_gated_ffn_backward_async(0, s, code, 0, m, k, n, buf.data_ptr(), ld, x.data_ptr(), k, wg.data_ptr(), wu.data_ptr(), k,
                                         g.data_ptr(), u.data_ptr(), buf.data_ptr() + n * e, ld, dw.data_ptr(), dw[1].data_ptr(),
                                         ws.data_ptr(), need.value) == 0
    want = dense.gated_ffn_backward(dh, x, wg, wu, g, u)
    assert torch.equal(buf[:, n:n + k], want[0]) and torch.equal(dw[0], want[1]) and torch.equal(dw[1], want[2])
    assert torch.equal(buf[:, :n], dh) and (buf[:, k + n:] == 7).all()
    # y, dropout's y beside x
    two = torch.full((m, 2 * k + 1), 7.0, dtype=dtype, device="cuda")
    two[:, :k] = x
    assert L.qr_layer_norm_async(0, s, code, code, m, k, two.data_ptr(), 2 * k + 1, None, None, 1e-5, two.data_ptr() + k * e, 2 * k + 1,
                                 None, None) == 0
    assert torch.equal(two[:, k:2 * k], dense.layer_norm(two[:, :k])[0]) and torch.equal(two[:, :k], x)
    assert L.qr_dropout_async(0, s, code, m, k, two.data_ptr(), 2 * k + 1, None, 0, two.data_ptr() + k * e, 2 * k + 1, 0.3, 1, 2, None) == 0
    assert torch.equal(two[:, k:2 * k], dense.dropout(x, 0.3, 1, 2)) and torch.equal(two[:, :k], x) and (two[:, 2 * k:] == 7).all()
