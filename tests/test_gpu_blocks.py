"""GPU parity of the token-block operators (sga_amd.blocks) against their definitions in 64 bits.

Tolerances, derived from the arithmetic and not from runs: a result is rounded once to its type (half a step, eps / 2 of its
value); a sum of K products in float32 is off by at most K * 2^-23 of the sum of their magnitudes (every product and every
addition by one step at most); an activation by a few float32 steps of its argument's scale; dz is rounded to the type before
it enters the products."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import sga_amd  # noqa: E402,F401
from oracle import philox  # noqa: E402

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -23
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
SEED, OFFSET = 0x1234567890ABCDEF, (5 << 32) + 9


def blocks():
    from sga_amd import blocks as b
    return b


def rand(rng, shape, t, scale=1.0, shift=0.0):
    return torch.from_numpy((rng.standard_normal(shape) * scale + shift).astype(np.float32)).to(t).cuda()


def half(t):
    """half a step of the type, relative; and the smallest step of float16's subnormal values, absolute"""
    return torch.finfo(t).eps / 2, (2.0 ** -25 if t == torch.float16 else 2.0 ** -126)


def keep_mask(n, p, seed=SEED, offset=OFFSET, first=0):
    """keep of elements first .. first + n, from the oracle's generator"""
    g0, g1 = first // 4, (first + n + 3) // 4
    g = np.arange(g0, g1, dtype=np.uint64)
    w = philox.philox4x32_10(g & np.uint64(0xFFFFFFFF), g >> np.uint64(32), offset & 0xFFFFFFFF, offset >> 32, seed & 0xFFFFFFFF, seed >> 32)
    words = np.stack(w, 1).reshape(-1).astype(np.uint64)
    return (words >= np.uint64(round(p * 2.0 ** 32)))[first - 4 * g0:first - 4 * g0 + n]


def gain(rows, cols, p):
    if not p:
        return torch.ones(rows, cols, dtype=torch.float64)
    return torch.from_numpy(keep_mask(rows * cols, p).reshape(rows, cols)).double() / (1.0 - p if p < 1 else 1.0)


def act64(z, act):
    if act == "relu":
        return torch.relu(z)
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2.0))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, act):
    """by central differences where the function is smooth"""
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    h = 1e-5
    return (act64(z + h, act) - act64(z - h, act)) / (2 * h)


def check(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    d = (got - want).abs()
    bad = ~(d <= tol)
    assert not bad.any(), "%s: %d of %d off; worst |d| %.3e where %.3e is allowed, at %s" % (
        what, int(bad.sum()), bad.numel(), d[bad].max(), (tol + 0 * d)[bad].max(), np.argwhere(bad.numpy())[0])


def linear_want(x, w, bias, act, residual, p, t):
    """-> out, its tolerance, pre, its tolerance (float64 on the host)"""
    K = x.shape[-1]
    x, w = x.cpu().double().reshape(-1, K), w.cpu().double()
    z, mag = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, mag = z + bias.cpu().double(), mag + bias.cpu().double().abs()
    eps, tiny = half(t)
    dz = (K + 1) * U * mag
    g = gain(*z.shape, p)
    y = act64(z, act) * g
    dy = (1.2 * dz + 16 * U * (z.abs() + 1) * (act != "none")) * g + 2 * U * y.abs()
    out = y if residual is None else y + residual.cpu().double().reshape(y.shape)
    return out, dy + (eps + U) * (out.abs() + dy) + tiny, z, dz + (eps + U) * (z.abs() + dz) + tiny


LINEAR = [  # rows, in, out: single tokens, a few, every side of a tile's edge, sizes that divide by nothing
    (1, 1, 1), (1, 7, 5), (1, 64, 16), (1, 520, 257), (1, 4096, 100), (2, 129, 300), (3, 1000, 16), (5, 8, 1), (7, 65, 1000), (8, 513, 24),
    (12, 640, 129), (15, 40, 33), (16, 256, 256), (17, 72, 100), (31, 96, 64), (33, 64, 129), (63, 200, 17), (64, 64, 64), (65, 31, 65),
    (100, 3, 200), (127, 128, 128), (129, 65, 127), (130, 520, 257), (200, 192, 300), (257, 136, 520), (300, 1001, 77), (513, 40, 250)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,inn,out", LINEAR)
def test_linear(rows, inn, out, dtype):
    t = TYPES[dtype]
    rng = np.random.RandomState(rows * 31 + inn * 7 + out)
    act = ACTS[(rows + inn + out) % 5]
    x, w = rand(rng, (rows, inn), t), rand(rng, (out, inn), t, inn ** -0.5)
    bias = rand(rng, (out,), t, 0.3) if (rows + out) % 3 else None
    res = rand(rng, (rows, out), t, 2.0) if (inn + out) % 2 else None
    p = 0.3 if (rows + inn) % 3 == 0 else 0.0
    got, pre = blocks().linear(x, w, bias, act=act, residual=res, dropout=(p, SEED, OFFSET) if p else None, want_pre=True)
    want, tol, z, tolz = linear_want(x, w, bias, act, res, p, t)
    assert got.dtype == t and pre.dtype == t
    check(pre, z, tolz, "pre")
    check(got, want, tol, "out")
    again = blocks().linear(x, w, bias, act=act, residual=res, dropout=(p, SEED, OFFSET) if p else None)
    assert torch.equal(got, again)                     # the same without `pre`, and from run to run


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows", [1, 40])
def test_linear_activations_with_everything(rows, act, dtype):
    t = TYPES[dtype]
    rng = np.random.RandomState(7)
    x, w, bias, res = rand(rng, (rows, 96), t, 3.0), rand(rng, (90, 96), t, 0.2), rand(rng, (90,), t), rand(rng, (rows, 90), t)
    got, pre = blocks().linear(x, w, bias, act=act, residual=res, dropout=(0.4, SEED, OFFSET), want_pre=True)
    want, tol, z, tolz = linear_want(x, w, bias, act, res, 0.4, t)
    check(pre, z, tolz, "pre")
    check(got, want, tol, "out")


def strided(rng, rows, n, t, kind):
    """[rows, n] as part of something else: wider rows, a start off the 16-byte grid, one row for all, all three dimensions of a batch"""
    if kind == "wide":
        return rand(rng, (rows, n + 24), t)[:, 8:8 + n]
    if kind == "odd":
        return rand(rng, (rows, n + 3), t)[:, 1:1 + n]
    if kind == "one":
        return rand(rng, (1, n), t).expand(rows, n)
    if kind == "every other":
        return rand(rng, (2 * rows, n), t)[::2]
    return rand(rng, (rows, n), t)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,inn,out", [(1, 264, 72), (9, 65, 130), (70, 264, 136), (140, 131, 66)])
@pytest.mark.parametrize("kind", ["wide", "odd", "one", "every other"])
def test_linear_rows_of_wider_buffers(kind, rows, inn, out, dtype):
    t = TYPES[dtype]
    rng = np.random.RandomState(rows + inn)
    x, w, res = strided(rng, rows, inn, t, kind), strided(rng, out, inn, t, kind if kind != "one" else "odd"), strided(rng, rows, out, t, kind)
    w.mul_(inn ** -0.5)
    want, tol, _, _ = linear_want(x, w, None, "silu", res, 0.0, t)
    check(blocks().linear(x, w, act="silu", residual=res), want, tol, "out")
    room = torch.full((rows, out + 5), 7.0, dtype=t, device="cuda")
    blocks().linear(x, w, act="silu", residual=res, out=room[:, 2:2 + out])
    check(room[:, 2:2 + out], want, tol, "out of a wider buffer")
    assert (room[:, :2] == 7).all() and (room[:, 2 + out:] == 7).all()
    g = strided(rng, rows, out, t, kind)
    wants, tols = linear_grad_want(g, x, w, None, "none", 0.0, t)
    for got, a, b, what in zip(blocks().linear_grad(g, x, w), wants, tols, ("g_x", "g_weight", "g_bias")):
        check(got, a, b, what)


def test_linear_leading_dimensions_and_in_place_residual():
    rng = np.random.RandomState(0)
    t = torch.bfloat16
    x, w = rand(rng, (2, 3, 5, 64), t), rand(rng, (64, 64), t, 0.1)
    want, tol, _, _ = linear_want(x, w, None, "none", x, 0.0, t)
    got = blocks().linear(x, w, residual=x)
    assert got.shape == x.shape
    check(got.reshape(-1, 64), want, tol, "out")
    y = rand(rng, (30, 64), t)
    want, tol, _, _ = linear_want(x, w, None, "none", y, 0.0, t)
    assert blocks().linear(x.reshape(30, 64), w, residual=y, out=y) is y
    check(y, want, tol, "in place")


@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_inf_and_nan_stay_in_their_rows_and_columns(dtype):
    """A row of x with inf / NaN reaches its own row of the product only, a row of w its own column; what dropout takes away is 0."""
    t = TYPES[dtype]
    for rows, inn, out in ((3, 70, 40), (50, 70, 40), (150, 136, 260)):
        rng = np.random.RandomState(1)
        x, w = rand(rng, (rows, inn), t), rand(rng, (out, inn), t, 0.1)
        x[rows // 2, inn - 1] = float("nan")
        x[0, 0] = float("inf")
        w[out - 1, 3] = float("-inf")
        got = blocks().linear(x, w, dropout=(0.5, SEED, OFFSET)).cpu()
        keep = torch.from_numpy(keep_mask(rows * out, 0.5).reshape(rows, out))
        assert (got[~keep] == 0).all()
        assert torch.isnan(got[rows // 2][keep[rows // 2]]).all()
        assert not torch.isfinite(got[0][keep[0]]).any()
        assert not torch.isfinite(got[:, out - 1][keep[:, out - 1]]).any()
        rest = keep.clone()
        rest[rows // 2] = False
        rest[0] = False
        rest[:, out - 1] = False
        assert torch.isfinite(got[rest].float()).all()


def linear_grad_want(g, x, w, pre, act, p, t):
    K, N = x.shape[-1], g.shape[-1]
    g, x, w = g.cpu().double().reshape(-1, N), x.cpu().double().reshape(-1, K), w.cpu().double()
    M = g.shape[0]
    eps, tiny = half(t)
    d = g * gain(M, N, p)
    off = 4 * U * d.abs()
    if act != "none":
        z = pre.cpu().double().reshape(M, N)
        off = off + 40 * U * d.abs() * (1 + z.abs()) + 1e-9 * d.abs()
        d = d * slope64(z, act)
    gb = d.sum(0)
    tb = off.sum(0) + M * U * d.abs().sum(0)
    changed = act != "none" or p > 0
    off = off + (eps * (d.abs() + off) + tiny if changed else 0.0)
    gx, tx = d @ w, off @ w.abs() + (N + 1) * U * ((d.abs() + off) @ w.abs())
    gw, tw = d.t() @ x, off.t() @ x.abs() + (M + 1) * U * ((d.abs() + off).t() @ x.abs())
    return (gx, gw, gb), tuple(a + (eps + U) * (v.abs() + a) + tiny for v, a in ((gx, tx), (gw, tw), (gb, tb)))


GRADS = [(1, 1, 1), (1, 64, 40), (2, 9, 300), (5, 130, 16), (16, 64, 64), (17, 200, 33), (33, 8, 129), (64, 128, 96), (65, 65, 65), (100, 257, 31),
         (129, 72, 260), (200, 33, 520), (300, 136, 64), (520, 264, 77), (1030, 40, 50)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,inn,out", GRADS)
def test_linear_grad(rows, inn, out, dtype):
    t = TYPES[dtype]
    rng = np.random.RandomState(rows + 3 * inn + out)
    act, p = ACTS[(rows + out) % 5], 0.3 if (rows + inn) % 2 else 0.0
    g, x, w = rand(rng, (rows, out), t, 0.5), rand(rng, (rows, inn), t), rand(rng, (out, inn), t, out ** -0.5)
    pre = rand(rng, (rows, out), t, 1.5) if act != "none" else None
    drop = (p, SEED, OFFSET) if p else None
    got = blocks().linear_grad(g, x, w, pre=pre, act=act, dropout=drop)
    wants, tols = linear_grad_want(g, x, w, pre, act, p, t)
    for a, b, tol, what in zip(got, wants, tols, ("g_x", "g_weight", "g_bias")):
        assert a.dtype == t
        check(a, b, tol, what)
    for i in range(3):                                   # each alone is the same
        alone = blocks().linear_grad(g, x, w, pre=pre, act=act, dropout=drop, want=tuple(j == i for j in range(3)))
        assert [v is None for v in alone] == [j != i for j in range(3)]
        assert torch.equal(alone[i], got[i])


@pytest.mark.parametrize("act", ACTS)
def test_linear_grad_of_each_activation_far_out(act):
    """Arguments to +-30, zero and the type's smallest: slopes 0, 1 and 1/2 without NaN"""
    t = torch.float32
    z = torch.tensor([[-30.0, -12.0, -6.0, -1.0, -1e-38, 0.0, 1e-38, 1.0, 6.0, 12.0, 30.0, 88.0, -88.0, -104.0, 3e38, -3e38]], device="cuda")
    g = torch.ones_like(z)
    _, _, gb = blocks().linear_grad(g, torch.ones(1, 1, device="cuda"), torch.ones(16, 1, device="cuda"), pre=z, act=act)
    zz = z.cpu().double().clamp(-60, 60)
    want = slope64(zz, act)[0]
    if act in ("gelu", "silu", "gelu_tanh"):
        want[5] = 0.5
    check(gb, want, 1e-6 * (1 + zz[0].abs().clamp(max=12)) + (act == "none") * 0 + 1e-8, "slope")
    out = blocks().linear(z.t().contiguous(), torch.ones(1, 1, device="cuda"), act=act).cpu().double()[:, 0]
    zf = z.cpu().double()[0]
    good = torch.where(zf.abs() < 60, act64(zf.clamp(-60, 60), act), zf if act == "none" else zf.clamp_min(0))
    check(out, good, 4 * U * zf.abs() + 1e-6 * (zf.abs() < 20), "value")


# ---- layer norm ---------------------------------------------------------------------------------------------------------------

NORMS = [(1, 1), (1, 8), (1, 1000), (1, 4096), (2, 63), (3, 64), (4, 65), (5, 256), (7, 257), (9, 511), (33, 96), (64, 192), (65, 1024), (130, 1025),
         (17, 2047), (6, 4097), (3, 8200), (2, 16384), (2, 20001), (257, 40), (1025, 24), (300, 3)]


def norm_want(x, w, b, eps, t):
    C = x.shape[-1]
    x = x.cpu().double().reshape(-1, C)
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    h = (x - mean) * rstd
    w_ = w.cpu().double() if w is not None else torch.ones(C, dtype=torch.float64)
    y = h * w_ + (b.cpu().double() if b is not None else 0.0)
    e, tiny = half(t)
    dm = C * U * x.abs().mean(1, keepdim=True)                       # the mean's sum
    dr = (C + 4) * U + 2 * (dm * rstd) ** 2 + 4 * U                # rstd's, relative; a mean that is off by dm adds dm^2 to the variance
    dh = (dm + 2 * U * x.abs()) * rstd + h.abs() * dr
    dy = dh * w_.abs() + 2 * U * (y.abs() + (h * w_).abs())
    return y, dy + (e + U) * (y.abs() + dy) + tiny, mean[:, 0], dm[:, 0] + U * mean[:, 0].abs(), rstd[:, 0], (rstd * dr)[:, 0]


@pytest.mark.parametrize("dtype,param", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("rows,cols", NORMS)
def test_layer_norm_and_its_gradients(rows, cols, dtype, param):
    t, tp = TYPES[dtype], TYPES[param]
    rng = np.random.RandomState(rows * 13 + cols)
    x = rand(rng, (rows, cols), t, 2.0, 1.0)
    w, b = rand(rng, (cols,), tp, 0.3, 1.0), rand(rng, (cols,), tp)
    y, mean, rstd = blocks().layer_norm(x, w, b, want_stats=True)
    wy, ty, wm, tm, wr, tr = norm_want(x, w, b, 1e-5, t)
    assert y.dtype == t and mean.dtype == rstd.dtype == torch.float32 and mean.shape == (rows,)
    check(y, wy, ty, "y")
    check(mean, wm, tm, "mean")
    check(rstd, wr, tr, "rstd")
    assert torch.equal(y, blocks().layer_norm(x, w, b))
    add = rand(rng, (rows, cols), t) if (rows + cols) % 2 else None
    g = rand(rng, (rows, cols), t)
    got = blocks().layer_norm_grad(g, x, mean, rstd, w, g_add=add)
    wants, tols = norm_grad_want(g, x, mean, rstd, w, add, t, tp)
    for a, want, tol, what in zip(got, wants, tols, ("g_x", "g_weight", "g_bias")):
        check(a, want, tol, what)
    assert got[0].dtype == t and got[1].dtype == got[2].dtype == tp
    for i in range(3):
        alone = blocks().layer_norm_grad(g, x, mean, rstd, w, g_add=add, want=tuple(j == i for j in range(3)))
        assert [v is None for v in alone] == [j != i for j in range(3)] and torch.equal(alone[i], got[i])


def norm_grad_want(g, x, mean, rstd, w, add, t, tp):
    C = x.shape[-1]
    g, x = g.cpu().double().reshape(-1, C), x.cpu().double().reshape(-1, C)
    M = x.shape[0]
    mean, rstd = mean.cpu().double().reshape(-1, 1), rstd.cpu().double().reshape(-1, 1)
    w_ = w.cpu().double() if w is not None else torch.ones(C, dtype=torch.float64)
    h, gw_ = (x - mean) * rstd, g * w_
    c1, c2 = gw_.mean(1, keepdim=True), (gw_ * h).mean(1, keepdim=True)
    gx = rstd * (gw_ - c1 - h * c2)
    a1, a2 = gw_.abs().mean(1, keepdim=True), (gw_ * h).abs().mean(1, keepdim=True)
    dh = 2 * U * (x.abs() + mean.abs()) * rstd
    d1 = (C + 2) * U * a1
    d2 = (C + 4) * U * a2 + (gw_.abs() * dh).mean(1, keepdim=True)
    dx = rstd * (4 * U * (gw_.abs() + a1 + h.abs() * a2) + d1 + h.abs() * d2 + dh * c2.abs())
    if add is not None:
        gx = gx + add.cpu().double().reshape(gx.shape)
    (e, tiny), (ep, tinyp) = half(t), half(tp)
    gw, gb = (g * h).sum(0), g.sum(0)
    dw = (M + 2) * U * (g * h).abs().sum(0) + (g.abs() * dh).sum(0)
    db = (M + 2) * U * g.abs().sum(0)
    return (gx, gw, gb), (dx + (e + U) * (gx.abs() + dx) + tiny, dw + (ep + U) * (gw.abs() + dw) + tinyp, db + (ep + U) * (gb.abs() + db) + tinyp)


def test_layer_norm_gradient_against_differences():
    """The kernel's gradient against central differences of the 64-bit definition (statistics recomputed at every point)."""
    rng = np.random.RandomState(3)
    t = torch.float32
    x, w, b, g = rand(rng, (6, 40), t, 2.0), rand(rng, (40,), t), rand(rng, (40,), t), rand(rng, (6, 40), t)
    _, mean, rstd = blocks().layer_norm(x, w, b, want_stats=True)
    gx, gw, gb = (v.cpu().double() for v in blocks().layer_norm_grad(g, x, mean, rstd, w))

    def loss(x_, w_, b_):
        d = x_ - x_.mean(1, keepdim=True)
        return float(((d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5) * w_ + b_) * g.cpu().double()).sum())

    base = [v.cpu().double() for v in (x, w, b)]
    for k, grad in enumerate((gx, gw, gb)):
        d = torch.from_numpy(np.random.RandomState(k).standard_normal(tuple(grad.shape)))
        up, down = [v.clone() for v in base], [v.clone() for v in base]
        up[k] += 1e-4 * d
        down[k] -= 1e-4 * d
        diff = (loss(*up) - loss(*down)) / 2e-4
        # 240 terms of size ~1 at float32 steps, and the third derivative (~100 here) times step^2 / 6
        assert abs(diff - float((grad * d).sum())) < 240 * 16 * U + 1e-5, k


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(5, 72), (40, 264), (9, 1031), (3, 5000)])
@pytest.mark.parametrize("kind", ["wide", "odd", "one", "every other"])
def test_layer_norm_rows_of_wider_buffers(kind, rows, cols, dtype):
    t = TYPES[dtype]
    rng = np.random.RandomState(rows)
    x, g, add = (strided(rng, rows, cols, t, kind) for _ in range(3))
    y, mean, rstd = blocks().layer_norm(x, want_stats=True)
    wy, ty, *_ = norm_want(x, None, None, 1e-5, t)
    check(y, wy, ty, "y")
    got = blocks().layer_norm_grad(g, x, mean, rstd, g_add=add)
    wants, tols = norm_grad_want(g, x, mean, rstd, None, add, t, t)
    for a, want, tol, what in zip(got, wants, tols, ("g_x", "g_weight", "g_bias")):
        check(a, want, tol, what)
    assert got[1].dtype == t and blocks().layer_norm_grad(g, x, mean, rstd, param_dtype=torch.float32)[1].dtype == torch.float32


def test_layer_norm_of_constant_and_far_rows():
    """A constant row has variance 0 (y = bias exactly); a row far from 0 keeps its spread: the variance is not a difference of squares."""
    t = torch.float32
    x = torch.full((3, 1000), 7.25, device="cuda")
    x[1] = 1e4 + torch.arange(1000, device="cuda") % 2           # mean 10000.5, variance 1/4: both exact in float32 sums of these
    b = torch.linspace(-1, 1, 1000, device="cuda")
    y, mean, rstd = blocks().layer_norm(x, None, b, want_stats=True)
    assert torch.equal(y[0], b) and torch.equal(y[2], b)
    assert float((mean[1] - 10000.5).abs()) <= 1000 * U * 10000.5
    assert abs(float(rstd[1]) / (1 / math.sqrt(0.25 + 1e-5)) - 1) < 1e-4
    z = torch.zeros(2, 50, device="cuda")
    assert torch.equal(blocks().layer_norm(z, eps=0.5), z)
    bad = torch.randn(3, 64, device="cuda")
    bad[1, 5] = float("nan")
    y = blocks().layer_norm(bad)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2]).all()


# ---- dropout ------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 3), (1, 4), (2, 5), (3, 8), (7, 33), (64, 64), (5, 1001), (130, 257), (33, 520), (1000, 40)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(p, rows, cols, dtype):
    t = TYPES[dtype]
    rng = np.random.RandomState(cols)
    x, res = rand(rng, (rows, cols), t), rand(rng, (rows, cols), t)
    keep = torch.from_numpy(keep_mask(rows * cols, p).reshape(rows, cols))
    eps, tiny = half(t)
    for r in (None, res):
        y = blocks().dropout(x, p, SEED, OFFSET, residual=r)
        want = x.cpu().double() * gain(rows, cols, p) + (r.cpu().double() if r is not None else 0.0)
        check(y, want, (eps + 4 * U) * want.abs() + 4 * U * (want.abs() + (x.cpu().double() * gain(rows, cols, p)).abs()) + tiny, "y")
        if r is None:
            assert torch.equal(y.cpu() != 0, keep & (x.cpu() != 0) if p else x.cpu() != 0)
    if p == 0.0:
        assert torch.equal(blocks().dropout(x, p, SEED, OFFSET), x)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["wide", "odd", "one", "every other"])
def test_dropout_of_wider_buffers_and_bad_values(kind, dtype):
    t = TYPES[dtype]
    rng = np.random.RandomState(5)
    for rows, cols in ((6, 40), (3, 1003)):
        x, r = strided(rng, rows, cols, t, kind), strided(rng, rows, cols, t, kind)
        y = blocks().dropout(x, 0.5, SEED, OFFSET, residual=r)
        assert torch.equal(y, blocks().dropout(x.contiguous(), 0.5, SEED, OFFSET, residual=r.contiguous()))
    x = torch.full((50, 50), float("nan"), dtype=t, device="cuda")
    y = blocks().dropout(x, 0.5, SEED, OFFSET).cpu()
    keep = torch.from_numpy(keep_mask(2500, 0.5).reshape(50, 50))
    assert torch.isnan(y[keep]).all() and (y[~keep] == 0).all()


def test_dropout_mask_of_a_product_is_the_mask_of_dropout():
    rng = np.random.RandomState(2)
    for rows, out in ((1, 50), (9, 70), (70, 130), (300, 264)):
        x, w = rand(rng, (rows, 32), torch.float32), rand(rng, (out, 32), torch.float32)
        a = blocks().linear(x, w, dropout=(0.4, SEED, OFFSET))
        b = blocks().dropout(blocks().linear(x, w), 0.4, SEED, OFFSET)
        assert torch.equal(a, b)


def test_dropout_seed_offset_and_state():
    x = torch.ones(64, 64, device="cuda")
    a = blocks().dropout(x, 0.5, 1, 0)
    for other in ((1, 1), (2, 0), (1 + (1 << 32), 0), (1, 1 << 32)):
        assert not torch.equal(a, blocks().dropout(x, 0.5, *other))
    state = torch.tensor([1, 0], dtype=torch.int64, device="cuda")
    assert torch.equal(a, blocks().dropout(x, 0.5, state))
    assert torch.equal(blocks().linear(x, x, dropout=(0.5, 1, 0)), blocks().linear(x, x, dropout=(0.5, state)))
    kept = (a != 0).float().mean()
    assert abs(float(kept) - 0.5) < 6 * 0.5 / 64                  # six standard deviations of 4096 fair draws


def test_elements_past_32_bits():
    """More than 2^32 elements: the counter's and the addresses' upper halves."""
    rows, cols = 4200000, 1032
    assert rows * cols > 2 ** 32
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device="cuda")
    y = blocks().dropout(x, 0.25, SEED, OFFSET)
    for first in (0, 2 ** 31 // cols, 2 ** 32 // cols, rows - 3):
        keep = keep_mask(3 * cols, 0.25, first=first * cols).reshape(3, cols)
        assert np.array_equal((y[first:first + 3] != 0).cpu().numpy(), keep), first
    x[rows - 2] = torch.arange(cols, device="cuda") % 7
    z, mean, rstd = blocks().layer_norm(x, want_stats=True)
    wy, ty, *_ = norm_want(x[rows - 3:], None, None, 1e-5, torch.bfloat16)
    check(z[rows - 3:], wy, ty, "norm")
    del z
    w = torch.zeros(8, cols, dtype=torch.bfloat16, device="cuda")
    w[3, 5] = 1.0
    out = blocks().linear(x, w)
    assert torch.equal(out[:, 3], x[:, 5]) and float(out[:, :3].abs().max()) == 0.0
    g = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda")
    g[rows - 2, 1] = 1.0
    g_x, g_w, g_b = blocks().linear_grad(g, x, w)
    assert torch.equal(g_w[1], x[rows - 2]) and float(g_w[0].abs().max()) == 0.0 and float(g_b.sum()) == 1.0
    assert float(g_x.abs().max()) == 0.0


# ---- no rows, several streams, graphs, a block -----------------------------------------------------------------------------------

def test_no_rows():
    b = blocks()
    x, w, g = torch.empty(0, 24, device="cuda"), torch.ones(8, 24, device="cuda"), torch.empty(0, 8, device="cuda")
    assert b.linear(x, w).shape == (0, 8)
    g_x, g_w, g_b = b.linear_grad(g, x, w, pre=g, act="silu")
    assert g_x.shape == (0, 24) and torch.equal(g_w, torch.zeros_like(w)) and torch.equal(g_b, torch.zeros(8, device="cuda"))
    y, mean, rstd = b.layer_norm(x, want_stats=True)
    assert y.shape == (0, 24) and mean.shape == (0,)
    _, g_w, g_b = b.layer_norm_grad(x, x, mean, rstd)
    assert torch.equal(g_w, torch.zeros(24, device="cuda")) and torch.equal(g_b, g_w)
    assert b.dropout(x, 0.5, 1).shape == (0, 24)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("inn,out", [(5, 12), (12, 33), (33, 5), (1, 1), (24, 8), (130, 257)])
@pytest.mark.parametrize("act,p", [("none", 0.0), ("silu", 0.0), ("none", 0.5), ("relu", 0.5)])
def test_no_rows_of_any_width(act, p, inn, out, dtype):
    """Weight gradients of no rows are zeros at widths that fill no 16-byte piece too, and the call writes nothing else: empty tensors
    without memory, and empty cuts of a wider buffer (whose rows start anywhere)."""
    b, t = blocks(), TYPES[dtype]
    w = torch.ones(out, inn + 3, dtype=t, device="cuda")[:, 1:1 + inn]
    room = torch.full((4, max(inn, out) + 3), 7.0, dtype=t, device="cuda")
    drop = (p, SEED, OFFSET) if p else None
    for x, g in ((torch.empty(0, inn, dtype=t, device="cuda"), torch.empty(0, out, dtype=t, device="cuda")), (room[2:2, 1:1 + inn], room[2:2, 1:1 + out])):
        pre = torch.empty(0, out, dtype=t, device="cuda")
        g_x, g_w, g_b = b.linear_grad(g, x, w, pre=pre, act=act, dropout=drop)
        assert g_x.shape == (0, inn) and g_w.shape == (out, inn) and g_w.dtype == t
        assert torch.equal(g_w, torch.zeros_like(g_w)) and torch.equal(g_b, torch.zeros_like(g_b))
        assert torch.equal(b.linear_grad(g, x, w, pre=pre, act=act, dropout=drop, want=(False, True, False))[1], g_w)
    assert (room == 7).all()


def block64(x, nw, nb, w1, b1, w2, b2, p):
    C = x.shape[-1]
    d = x - x.mean(1, keepdim=True)
    h = d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5) * nw + nb
    a = act64(h @ w1.t() + b1, "gelu")
    return x + (a @ w2.t() + b2) * gain(x.shape[0], C, p)


def block_run(b, x, nw, nb, w1, b1, w2, b2, g, drop):
    h, mean, rstd = b.layer_norm(x, nw, nb, want_stats=True)
    a, pre = b.linear(h, w1, b1, act="gelu", want_pre=True)
    y = b.linear(a, w2, b2, residual=x, dropout=drop)
    g_a, g_w2, g_b2 = b.linear_grad(g, a, w2, dropout=drop)
    g_h, g_w1, g_b1 = b.linear_grad(g_a, h, w1, pre=pre, act="gelu")
    g_x, g_nw, g_nb = b.layer_norm_grad(g_h, x, mean, rstd, nw, g_add=g)
    return y, g_x, g_nw, g_nb, g_w1, g_b1, g_w2, g_b2


def block_inputs(rows, C, H, t, seed=0):
    rng = np.random.RandomState(seed)
    return [rand(rng, (rows, C), t), rand(rng, (C,), t, 0.2, 1.0), rand(rng, (C,), t, 0.1), rand(rng, (H, C), t, C ** -0.5), rand(rng, (H,), t, 0.1),
            rand(rng, (C, H), t, H ** -0.5), rand(rng, (C,), t, 0.1), rand(rng, (rows, C), t)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,C,H", [(1, 64, 256), (96, 192, 768), (150, 100, 330)])
def test_a_block_and_its_gradient(rows, C, H, dtype):
    """The operators as they are used together, against 64-bit autograd of the block's formula.  Errors pass through six roundings to
    the type (h, pre, a, g_a, dz, g_h) of relative size eps / 2 each, which add up over sums of random signs: 2-norm within
    6 * eps / 2 + the float32 part (sums of up to max(H, rows) terms, same argument: well under 2^-18)."""
    t = TYPES[dtype]
    args = block_inputs(rows, C, H, t)
    got = block_run(blocks(), *args, (0.2, SEED, OFFSET))
    leaves = [v.cpu().double().requires_grad_(True) for v in args[:-1]]
    y = block64(*leaves, 0.2)
    wants = [y.detach()] + list(torch.autograd.grad(y, leaves, args[-1].cpu().double()))
    bound = 6 * torch.finfo(t).eps / 2 + 2.0 ** -18
    for k, (a, want) in enumerate(zip(got, wants)):
        rel = float((a.cpu().double() - want).norm() / want.norm())
        assert rel < bound, (k, rel, bound)


def test_two_streams_at_once():
    """Calls of two streams at the same time share nothing: each gives what it gives alone."""
    b = blocks()
    sets = [block_inputs(200, 136, 264, torch.bfloat16, seed=s) for s in range(2)]
    alone = [block_run(b, *a, (0.2, s, 0)) for s, a in enumerate(sets)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = [None, None]
        for s in range(2):
            streams[s].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[s]):
                got[s] = block_run(b, *sets[s], (0.2, s, 0))
        torch.cuda.synchronize()
        for s in range(2):
            assert all(torch.equal(u, v) for u, v in zip(got[s], alone[s]))


def test_captured_and_replayed():
    """Two captured graphs (a block's forward and backward pass each) replayed in turn with eager work between: new inputs, new
    dropout numbers through the state tensor, every replay equal to the eager result."""
    b = blocks()
    made = []
    for s in range(2):
        args = block_inputs(100 + 50 * s, 72, 200, torch.bfloat16, seed=s)
        state = torch.tensor([s, 0], dtype=torch.int64, device="cuda")
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            block_run(b, *args, (0.2, state))
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = block_run(b, *args, (0.2, state))
        made.append((graph, args, state, outs))
    for it in range(4):
        for s, (graph, args, state, outs) in enumerate(made):
            fresh = block_inputs(100 + 50 * s, 72, 200, torch.bfloat16, seed=10 * it + s)
            for a, f in zip(args, fresh):
                a.copy_(f)
            state.copy_(torch.tensor([s, it], dtype=torch.int64))
            graph.replay()
        torch.cuda.synchronize()
        for s, (graph, args, state, outs) in enumerate(made):
            for u, v in zip(outs, block_run(b, *args, (0.2, s, it))):
                assert torch.equal(u, v), (it, s)


# ---- sizes that take every tile, K split and fetch -------------------------------------------------------------------------------

def check_on_gpu(got, want, tol, what):
    d = (got.double() - want).abs()
    bad = ~(d <= tol)
    assert not bool(bad.any()), "%s: %d of %d off, worst |d| %.3e" % (what, int(bad.sum()), bad.numel(), float(d[bad].max()))


BIG = [(4096, 520, 4104), (2048, 264, 4096), (2048, 1032, 2048), (1537, 1001, 777), (300, 4096, 512), (100, 8192, 264), (520, 130, 1000), (70, 2050, 4100),
       (200, 6, 300), (90, 62, 130), (640, 126, 96), (130, 2, 70), (1000, 9, 65), (257, 4103, 129), (96, 640, 64), (97, 644, 68)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,inn,out", BIG)
def test_linear_and_its_gradients_over_the_plans(rows, inn, out, dtype):
    """The same definitions and tolerances as above, with the 64-bit products on the device."""
    t = TYPES[dtype]
    g = torch.Generator(device="cuda")
    g.manual_seed(rows + inn + out)

    def rnd(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)

    x, w, res = rnd(rows, inn), rnd(out, inn, scale=inn ** -0.5), rnd(rows, out)
    eps, tiny = half(t)
    xd, wd = x.double(), w.double()
    z, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    want = torch.relu(z) + res.double()
    dz = (inn + 1) * U * mag
    check_on_gpu(blocks().linear(x, w, act="relu", residual=res), want, dz + (eps + U) * (want.abs() + dz) + tiny, "out")
    go = rnd(rows, out)
    gd = go.double()
    g_x, g_w, g_b = blocks().linear_grad(go, x, w)
    for got, want, mag, n, what in ((g_x, gd @ wd, gd.abs() @ wd.abs(), out, "g_x"), (g_w, gd.t() @ xd, gd.abs().t() @ xd.abs(), rows, "g_weight"),
                                    (g_b, gd.sum(0), gd.abs().sum(0), rows, "g_bias")):
        off = (n + 1) * U * mag
        check_on_gpu(got, want, off + (eps + U) * (want.abs() + off) + tiny, what)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("inn,ld,start", [(131, 132, 0), (129, 134, 2), (65, 72, 4), (70, 74, 2), (33, 40, 8), (1, 2, 0), (7, 12, 4), (136, 140, 2)])
def test_linear_rows_on_every_4_bytes(inn, ld, start, dtype):
    """Rows that start at multiples of 4 bytes only, with a K that ends inside a 16-byte piece; what lies behind it is NaN."""
    t = TYPES[dtype]
    rng = np.random.RandomState(inn)
    for rows, out in ((200, 130), (20, 24)):
        x, w = (torch.full((n, ld + start), float("nan"), dtype=t, device="cuda")[:, start:start + inn] for n in (rows, out))
        x.copy_(rand(rng, (rows, inn), t))
        w.copy_(rand(rng, (out, inn), t, inn ** -0.5))
        want, tol, _, _ = linear_want(x, w, None, "none", None, 0.0, t)
        check(blocks().linear(x, w), want, tol, "out")
        g = rand(rng, (rows, out), t)
        wants, tols = linear_grad_want(g, x, w, None, "none", 0.0, t)
        for got, a, b, what in zip(blocks().linear_grad(g, x, w), wants, tols, ("g_x", "g_weight", "g_bias")):
            check(got, a, b, what)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_inputs_at_the_end_of_their_memory(dtype):
    """The last row ends where its allocation ends, odd sizes: results as of a copy in the middle of a larger one."""
    t = TYPES[dtype]
    rng = np.random.RandomState(4)
    for rows, inn, out in ((1, 4097, 33), (70, 259, 67), (300, 131, 257)):
        total = rows * inn + 8
        x = torch.empty(total, dtype=t, device="cuda")[total - rows * inn:].view(rows, inn)
        x.copy_(rand(rng, (rows, inn), t))
        w = rand(rng, (out, inn), t, 0.1)
        roomy = torch.zeros(rows + 2, inn, dtype=t, device="cuda")
        roomy[1:-1] = x
        assert torch.equal(blocks().linear(x, w), blocks().linear(roomy[1:-1], w))
        g = rand(rng, (rows, out), t)
        for a, b in zip(blocks().linear_grad(g, x, w), blocks().linear_grad(g, roomy[1:-1], w)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("out", [3, 8, 12, 24, 2047, 2048, 2049, 2056])
@pytest.mark.parametrize("rows,inn,gap", [(1, 200, 0), (16, 1031, 0), (13, 75, 1), (33, 300, 2), (50, 129, 1), (2, 7, 1), (5, 8, 1)])
def test_linear_of_few_rows(rows, inn, gap, out, dtype):
    """Few rows on every alignment, rows that end inside a piece, and column blocks of 8 and 16 whose last one is short; NaN in the gaps."""
    t = TYPES[dtype]
    rng = np.random.RandomState(rows + inn + out)
    x, w = (torch.full((n, inn + gap), float("nan"), dtype=t, device="cuda")[:, :inn] for n in (rows, out))
    x.copy_(rand(rng, (rows, inn), t))
    w.copy_(rand(rng, (out, inn), t, inn ** -0.5))
    bias, res = rand(rng, (out,), t), rand(rng, (rows, out), t)
    want, tol, _, _ = linear_want(x, w, bias, "none", res, 0.0, t)
    check(blocks().linear(x, w, bias, residual=res), want, tol, "out")


def test_linear_with_an_output_over_its_input_is_refused():
    x = torch.zeros(64, 64, device="cuda")
    w = torch.zeros(64, 64, device="cuda")
    for out in (x, w):
        with pytest.raises(ValueError, match="overlaps"):
            blocks().linear(x, w, out=out)
    wide = torch.zeros(64, 80, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        blocks().linear(x, w, residual=wide[:, :64], out=wide[:, 8:72])
    blocks().linear(x, w, residual=wide[:, :64], out=wide[:, :64])
    blocks().linear(wide[:32, :64], w, out=wide[32:, :64])
    both = torch.randn(64, 128, device="cuda")                   # columns side by side in one buffer
    want = blocks().linear(both[:, :64].contiguous(), w)
    assert torch.equal(blocks().linear(both[:, :64], w, out=both[:, 64:]), want)


def test_linear_with_an_output_is_a_change_in_place():
    """Autograd notices that a tensor it saved was written to, through any view of it; an `out` that requires a gradient is refused."""
    x, w = torch.randn(4, 64, device="cuda"), torch.randn(64, 64, device="cuda")
    y = torch.randn(4, 64, device="cuda", requires_grad=True).exp()      # its backward pass needs y
    for out in (y.detach(), y.detach()[:, 0:64]):
        before = y._version
        assert blocks().linear(x, w, out=out) is out and y._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    leaf = torch.zeros(4, 64, device="cuda", requires_grad=True)
    for out in (y, leaf):
        before = out.detach().clone()
        with pytest.raises(ValueError, match="requires a gradient"):
            blocks().linear(x, w, out=out)
        assert torch.equal(out.detach(), before)
    with torch.no_grad():
        blocks().linear(x, w, out=leaf)
    assert torch.equal(leaf.detach(), blocks().linear(x, w))
    with torch.inference_mode():
        assert torch.equal(blocks().linear(x, w, out=torch.empty(4, 64, device="cuda")), leaf.detach())


def test_wrong_parameter_types_are_refused():
    x, w, out = torch.ones(4, 8, device="cuda"), torch.ones(8, 8, device="cuda"), torch.zeros(4, 8, device="cuda")
    for bad in (torch.ones(8, device="cuda", dtype=torch.float64), torch.ones(8, device="cuda", dtype=torch.int32), [1.0] * 8, torch.ones(8)):
        error = ValueError if isinstance(bad, torch.Tensor) and bad.dtype == torch.float32 else TypeError      # right type, wrong device
        for call in (lambda: blocks().layer_norm(x, None, bad), lambda: blocks().layer_norm(x, bad), lambda: blocks().layer_norm(x, x[0], bad),
                     lambda: blocks().linear(x, w, bad), lambda: blocks().linear(x, w, bad, out=out)):
            with pytest.raises(error):
                call()
    assert float(out.abs().max()) == 0.0


def test_linear_of_the_most_rows():
    """A launch counts its lanes in 32 bits: with as many rows as are allowed, every one of them is written."""
    rows = 2 ** 31 - 256
    x = torch.arange(256, device="cuda").to(torch.bfloat16).repeat(rows // 256).view(rows, 1)
    w = torch.full((1, 1), 2.0, dtype=torch.bfloat16, device="cuda")
    y = blocks().linear(x, w)
    for first in range(0, rows, 2 ** 28):
        part = slice(first, first + 2 ** 28)
        assert torch.equal(y[part], x[part] * 2), first
    del y
    g_x, _, _ = blocks().linear_grad(x, x, w, want=(True, False, False))
    for first in range(0, rows, 2 ** 28):
        part = slice(first, first + 2 ** 28)
        assert torch.equal(g_x[part], x[part] * 2), first
    with pytest.raises(RuntimeError, match="UNSUPPORTED"):
        blocks().linear(torch.zeros(1, 1, dtype=torch.bfloat16, device="cuda").expand(rows + 1, 1), w)
