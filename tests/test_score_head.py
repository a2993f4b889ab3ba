"""The score head's operators (layer norm, linear products, softmax loss) against their formulas in 64 bits.

Tolerances are bounds, not fits.  U = 2^-24 is half a step of float32; a result of type t is off by finfo(t).eps / 2 of its value
for the one rounding to t (at least half of the smallest subnormal); a float32 sum of n products is off by at most (n + 2) U times
the sum of their absolute values, in whatever order it is taken."""
import ctypes as C
import os
import subprocess
import sys
import zlib

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24
A, B = 1.5957691216057308, 0.044715


@pytest.fixture(scope="module")
def eng():
    import opal_amd
    e = opal_amd.Engine(0)
    yield e
    e.close()


def rounding(ref, t):
    """What one rounding of ref to t may change."""
    f = torch.finfo(t)
    return ref.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def close(got, ref, tol, what=""):
    assert tuple(got.shape) == tuple(ref.shape), (what, got.shape, ref.shape)
    if not ref.numel():
        return
    off = (got.double().cpu() - ref.cpu()).abs() - tol.cpu()
    bad = ~(off <= 0)
    assert not bad.any(), "%s: %d of %d off, worst by %g at %s" % (what, int(bad.sum()), ref.numel(), float(off[bad].max()), bad.nonzero()[0].tolist())


def rows(g, n, cols, t, ld=None, scale=1.0, base=0):
    """Random [n, cols] with the row stride ld (NaN between the rows) that begins `base` elements into its memory."""
    ld = cols if ld is None else ld
    full = torch.full((base + max(n, 1) * ld,), float("nan"), dtype=t)
    x = full[base:].view(max(n, 1), ld)[:n, :cols]
    x.copy_((torch.randn(n, cols, generator=g, dtype=torch.float64) * scale).to(t))
    dev = full.cuda()
    return dev[base:].view(max(n, 1), ld)[:n, :cols], x.double()


def gen(*key):
    g = torch.Generator()
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


def act64(v, a):
    return {"none": v, "relu": v.clamp(min=0), "silu": v * torch.sigmoid(v), "gelu": v * torch.sigmoid(A * (v + B * v ** 3))}[a]


def slope64(v, a):
    if a == "none":
        return torch.ones_like(v)
    if a == "relu":
        return (v > 0).double()
    z, dz = (v, torch.ones_like(v)) if a == "silu" else (A * (v + B * v ** 3), A * (1 + 3 * B * v ** 2))
    p = torch.sigmoid(z)
    return p + v * p * (1 - p) * dz


# every product: sizes around the tiles' and steps' edges, one row, odd sizes, strides that break the 16-byte alignment
SHAPES = [(1, 1, 1), (1, 356, 64), (3, 7, 5), (64, 64, 64), (65, 63, 66), (130, 129, 127), (17, 355, 100), (200, 1563, 33), (129, 40, 1564), (700, 72, 260), (2049, 130, 129), (4500, 130, 66), (5003, 33, 65)]


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("n,k,m", SHAPES)
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_linear(eng, t, n, k, m, pad):
    g = gen("linear", n, k, m, pad)
    step = 16 // torch.empty(0, dtype=t).element_size()
    ldk = k if pad == 0 else k + 1 if pad == 1 else -(-k // step) * step + step      # 8: aligned rows with a gap
    x, x64 = rows(g, n, k, t, ldk, base=1 if pad == 1 else 0)
    w, w64 = rows(g, m, k, t, ldk, scale=k ** -0.5)
    act = ["none", "relu", "silu", "gelu"][(n + k + m + pad) % 4]
    bias = torch.randn(m, generator=g) if pad != 1 else None
    res, res64 = rows(g, n, m, [F32, t][pad % 2], m + 3) if pad else (None, 0.0)
    out = F32 if (n + pad) % 2 else t
    y, pre = eng.linear(x, w, bias.cuda() if bias is not None else None, activation=act, residual=res, out_dtype=out, want_pre=True)
    p = x64 @ w64.t() + (bias.double() if bias is not None else 0.0)
    dp = (k + 3) * U * (x64.abs() @ w64.abs().t() + (bias.double().abs() if bias is not None else 0.0))
    close(pre, p, dp + rounding(p.abs() + dp, t), "pre")
    a = act64(p, act)
    # |slope| <= 1.13; v_exp / v_rcp and the argument's rounding: a few U of the value, |z| U of the sigmoid
    da = 1.13 * dp + U * (8 + 4 * p.abs() + 2 * p.abs() ** 3) * a.abs() + 1e-37
    ref = a + res64
    d = da + U * (ref.abs() + a.abs() + da)
    close(y, ref, d + rounding(ref.abs() + d, out), "y")
    y2, none = eng.linear(x, w, bias.cuda() if bias is not None else None, activation=act, residual=res, out_dtype=out)
    assert none is None and torch.equal(y, y2)                                        # the same bits with and without pre


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("n,k,m", SHAPES)
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_linear_gradients(eng, t, n, k, m, pad):
    g = gen("grad", n, k, m, pad)
    step = 16 // torch.empty(0, dtype=t).element_size()
    up = (lambda c: c) if pad == 0 else (lambda c: c + 1) if pad == 1 else (lambda c: -(-c // step) * step + step)
    dy, dy64 = rows(g, n, m, t, up(m), scale=0.1)
    x, x64 = rows(g, n, k, t, up(k), base=1 if pad == 1 else 0)
    w, w64 = rows(g, m, k, t, up(k), scale=k ** -0.5)
    pre, pre64 = rows(g, n, k, t, k + pad)
    act = ["none", "relu", "silu", "gelu"][(n + k + m + pad) % 4]
    res, res64 = rows(g, n, k, [F32, t][pad % 2], k + 3) if pad else (None, 0.0)
    out = F32 if (n + pad) % 2 else t
    dx = eng.linear_grad_input(dy, w, pre=pre if act != "none" else None, activation=act, residual=res, out_dtype=out)
    s = slope64(pre64, act)
    p = dy64 @ w64
    d = s.abs() * (m + 2) * U * (dy64.abs() @ w64.abs())
    ds = U * (16 + 16 * pre64.abs() + 8 * pre64.abs() ** 3) if act in ("silu", "gelu") else 0.0
    ref = p * s + res64
    d = d + p.abs() * ds + 2 * U * (ref.abs() + (p * s).abs())
    close(dx, ref, d + rounding(ref.abs() + d, out), "dx")
    dw, db = eng.linear_grad_weight(dy, x)
    assert dw.dtype == F32 and db.dtype == F32
    close(dw, dy64.t() @ x64, (n + 2) * U * (dy64.abs().t() @ x64.abs()) + 1e-38, "dw")
    close(db, dy64.sum(0), (n + 2) * U * dy64.abs().sum(0) + 1e-38, "db")
    dw2, none = eng.linear_grad_weight(dy, x, want_bias=False)
    assert none is None and torch.equal(dw, dw2)


# enough rows and columns for the larger tiles of 16-bit products: sums that end inside a step, a chunk, a stage of 64; columns that
# end inside a group of eight; several tiles a block (every epilogue of every kernel: test_score_head_kernels.py)
BIG_SHAPES = [(16700, 100, 520), (33000, 71, 250), (11000, 40, 1563), (16500, 1, 512), (8200, 355, 1030), (70001, 33, 257), (16400, 192, 511), (9000, 1563, 1040), (33000, 1027, 500), (131000, 259, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("n,k,m", BIG_SHAPES)
@pytest.mark.parametrize("out", [F32, None, "other"])
def test_large_products(eng, t, n, k, m, out):
    """A thousand rows of the result, the first and the last ones among them, and its gradients."""
    g = torch.Generator(device="cuda").manual_seed(n + k + m)
    rnd = lambda a, b, s=1.0: (torch.randn(a, -(-b // 8) * 8, device="cuda", generator=g) * s).to(t)[:, :b]  # noqa: E731
    x, w, dy, pre = rnd(n, k), rnd(m, k, k ** -0.5), rnd(n, m, 0.1), rnd(n, k)
    out = {None: t, "other": F16 if t == BF16 else BF16}.get(out, out)
    act = ["none", "relu", "silu", "gelu"][(n + m + (out == F32)) % 4]
    bias = torch.randn(m, device="cuda", generator=g) if m % 2 == 0 else None
    res = rnd(n, m).to([F32, t, out][n % 3]) if k % 2 else None
    at = torch.cat([torch.arange(300), torch.randint(0, n, (400,), generator=gen("rows")), torch.arange(n - 300, n)])
    y, saved = eng.linear(x, w, bias, activation=act, residual=res, out_dtype=out, want_pre=True)
    x64, w64 = x[at.cuda()].double().cpu(), w.double().cpu()
    p = x64 @ w64.t()
    dp = (k + 3) * U * (x64.abs() @ w64.abs().t())
    if bias is not None:
        p, dp = p + bias.double().cpu(), dp + (k + 3) * U * bias.double().abs().cpu()
    close(saved[at.cuda()], p, dp + rounding(p.abs() + dp, t), "pre")
    a = act64(p, act)
    da = 1.13 * dp + U * (8 + 4 * p.abs() + 2 * p.abs() ** 3) * a.abs() + 1e-37
    ref = a + (res[at.cuda()].double().cpu() if res is not None else 0.0)
    d = da + U * (ref.abs() + a.abs() + da)
    close(y[at.cuda()], ref, d + rounding(ref.abs() + d, out), "y")
    assert torch.isfinite(y.float()).all()
    res = rnd(n, k).to([F32, t, out][n % 3]) if m % 2 else None
    dx = eng.linear_grad_input(dy, w, pre=pre if act != "none" else None, activation=act, residual=res, out_dtype=out)
    dy64, pre64 = dy[at.cuda()].double().cpu(), pre[at.cuda()].double().cpu()
    s = slope64(pre64, act)
    p = dy64 @ w64
    d = s.abs() * (m + 2) * U * (dy64.abs() @ w64.abs())
    ds = U * (16 + 16 * pre64.abs() + 8 * pre64.abs() ** 3) if act in ("silu", "gelu") else 0.0
    ref = p * s + (res[at.cuda()].double().cpu() if res is not None else 0.0)
    d = d + p.abs() * ds + 2 * U * (ref.abs() + (p * s).abs())
    close(dx[at.cuda()], ref, d + rounding(ref.abs() + d, out), "dx")
    assert torch.isfinite(dx.float()).all()
    if out == F32:
        dw, db = eng.linear_grad_weight(dy, x)
        dy64, x64 = dy.double().cpu(), x.double().cpu()
        close(dw, dy64.t() @ x64, (n + 2) * U * (dy64.abs().t() @ x64.abs()) + 1e-38, "dw")
        close(db, dy64.sum(0), (n + 2) * U * dy64.abs().sum(0) + 1e-38, "db")


@pytest.mark.gpu
def test_large_products_keep_nans_behind_the_edge_out(eng):
    """What lies between the rows is NaN: it must not reach a sum, also where the last chunk of a row is cut."""
    n, k, m = 16700, 99, 515
    for t in (F16, BF16):
        full = [torch.full((r, c), float("nan"), device="cuda", dtype=t) for r, c in ((n, 104), (m, 112), (n, 520))]
        x, w, dy = full[0][:, :k], full[1][:, :k], full[2][:, :m]
        for v in (x, w, dy):
            v.copy_(torch.randn(v.shape, device="cuda"))
        y, _ = eng.linear(x, w, out_dtype=F32)
        assert torch.isfinite(y).all()
        assert torch.isfinite(eng.linear_grad_input(dy, w, out_dtype=F32)).all()
        dw, db = eng.linear_grad_weight(dy, x)
        assert torch.isfinite(dw).all() and torch.isfinite(db).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("n,k,m", [(16700, 99, 515), (33000, 1027, 257), (70001, 40, 130), (3000, 33, 63)])
@pytest.mark.parametrize("wide", [True, False])
def test_large_products_in_place_and_their_edges(eng, t, n, k, m, wide):
    """The residual's place may be the result's: the bits are those of a result elsewhere, and what lies between the rows and behind the
    last one (all NaN) stays what it is."""
    from opal_amd._lib import check
    g = torch.Generator(device="cuda").manual_seed(n + k)
    code, out = {F16: 1, BF16: 2}[t], F32 if wide else t

    def framed(r, c, dt):
        full = torch.full((r + 2, -(-c // 8) * 8 + 8), float("nan"), device="cuda", dtype=dt)
        full[:r, :c] = torch.randn(r, c, device="cuda", generator=g)
        return full, full[:r, :c]

    def untouched(full, r, c):
        return bool(full[r:].isnan().all()) and bool(full[:, c:].isnan().all())
    x, w, dy = framed(n, k, t)[1], framed(m, k, t)[1], framed(n, m, t)[1]
    for a, b, cols, entry in ((x, w, m, "opal_linear"), (dy, w, k, "opal_linear_grad_input")):
        full, res = framed(n, cols, out)
        want = eng.linear(a, b, residual=res, out_dtype=out)[0] if entry == "opal_linear" else eng.linear_grad_input(a, b, residual=res, out_dtype=out)
        oc, ld = {F32: 0, F16: 1, BF16: 2}[out], full.stride(0)
        if entry == "opal_linear":
            check(eng._lib.opal_linear(eng._h, a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), code, None, 0, full.data_ptr(), oc, ld, n, k, m,
                                       full.data_ptr(), oc, ld, None, 0), eng._h)
        else:
            check(eng._lib.opal_linear_grad_input(eng._h, a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), code, None, 0, 0, full.data_ptr(), oc, ld, n, k, m,
                                                  full.data_ptr(), oc, ld), eng._h)
        assert torch.isfinite(want).all() and torch.equal(res, want) and untouched(full, n, cols)
    full, dw = framed(m, k, F32)
    want, db = eng.linear_grad_weight(dy, x)
    work = torch.empty(max(eng._lib.opal_linear_grad_weight_workspace(n, k, m, code), 16), dtype=torch.uint8, device="cuda")
    check(eng._lib.opal_linear_grad_weight(eng._h, dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), code, n, k, m, full.data_ptr(), full.stride(0), None,
                                           work.data_ptr(), work.numel()), eng._h)
    assert torch.isfinite(want).all() and torch.isfinite(db).all() and torch.equal(dw, want) and untouched(full, m, k)


@pytest.mark.gpu
def test_products_of_no_rows(eng):
    w = torch.randn(5, 7, device="cuda")
    x = torch.empty(0, 7, device="cuda")
    y, pre = eng.linear(x, w, want_pre=True)
    assert y.shape == (0, 5) and pre.shape == (0, 5)
    assert eng.linear_grad_input(torch.empty(0, 5, device="cuda"), w).shape == (0, 7)
    dw, db = eng.linear_grad_weight(torch.empty(0, 5, device="cuda"), x)
    assert torch.equal(dw, torch.zeros(5, 7, device="cuda")) and torch.equal(db, torch.zeros(5, device="cuda"))
    y, mean, rstd = eng.layer_norm(x, want_stats=True)
    assert y.shape == (0, 7) and mean.shape == (0,)
    dx, dg, db = eng.layer_norm_backward(x, x, None, mean, rstd)
    assert dx.shape == (0, 7) and torch.equal(dg, torch.zeros(7, device="cuda")) and torch.equal(db, torch.zeros(7, device="cuda"))
    loss, grad = eng.softmax_loss(x, torch.empty(0, dtype=torch.int32, device="cuda"))
    assert loss.shape == (0,) and grad.shape == (0, 7)
    assert [v.shape for v in eng.softmax_class(x)] == [(0,), (0,)]


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16])
def test_products_keep_infinities_in_their_place(eng, t):
    """A NaN or an infinity reaches the results whose sums it is part of, and no other."""
    g = gen("inf")
    x, x64 = rows(g, 70, 41, t, 48)
    w, w64 = rows(g, 90, 41, t, 48)
    x[3, 40] = float("inf")
    w[5, 2] = float("nan")
    y, _ = eng.linear(x, w, out_dtype=F32)
    bad = torch.zeros(70, 90, dtype=torch.bool)
    bad[3], bad[:, 5] = True, True
    assert torch.equal(~torch.isfinite(y.cpu()), bad)
    dy, _ = rows(g, 70, 90, t, 96)
    dy[69, 89] = float("nan")
    dw, db = eng.linear_grad_weight(dy, x)
    bad = torch.zeros(90, 41, dtype=torch.bool)
    bad[89], bad[:, 40] = True, True
    assert torch.equal(~torch.isfinite(dw.cpu()), bad) and torch.isfinite(db).sum() == 89


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16])
def test_residual_may_be_the_result(eng, t):
    """C level: y == res and dx == res, in place; what lies between the rows stays."""
    from opal_amd._lib import check, lib
    g = gen("inplace")
    n, k, m = 130, 70, 66
    x, x64 = rows(g, n, k, t, 72)
    w, w64 = rows(g, m, k, t, 72)
    res, r64 = rows(g, n, m, F32, 70)
    before = res.as_strided((n, 70), (70, 1)).clone()
    code = {F32: 0, BF16: 2}[t]
    check(lib().opal_linear(eng._h, x.data_ptr(), 72, w.data_ptr(), 72, code, None, 0, res.data_ptr(), 0, 70, n, k, m, res.data_ptr(), 0, 70, None, 0), eng._h)
    ref = x64 @ w64.t() + r64
    close(res, ref, (k + 4) * U * (x64.abs() @ w64.abs().t() + r64.abs()))
    after = res.as_strided((n, 70), (70, 1))
    assert torch.equal(after[:, m:].isnan(), before[:, m:].isnan()) and after[:, m:].isnan().all()


# ------------------------------------------------------------------------------ layer norm
NORM_SHAPES = [(1, 1), (1, 356), (5, 2), (3, 255), (9, 256), (33, 257), (100, 355), (7, 1563), (70, 1564), (11, 2048), (6, 2049), (13, 5000), (5, 8192), (3, 8193), (70, 9001)]


def norm64(x, gamma, beta, eps):
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = ((d * d).mean(1, keepdim=True) + eps) ** -0.5
    xh = d * rstd
    return xh * gamma + beta, mean, rstd, xh


@pytest.mark.gpu
@pytest.mark.parametrize("tx,ty", [(F32, BF16), (F32, F32), (BF16, F16), (F16, F32)])
@pytest.mark.parametrize("n,cols", NORM_SHAPES)
def test_layer_norm(eng, tx, ty, n, cols):
    g = gen("norm", n, cols)
    x, x64 = rows(g, n, cols, tx, cols + (n % 3), base=n % 2, scale=0.5)
    plain = n % 2 == 0
    gamma, beta = (None, None) if plain else (torch.randn(cols, generator=g), torch.randn(cols, generator=g))
    eps = 1e-5
    y, mean, rstd = eng.layer_norm(x, None if plain else gamma.cuda(), None if plain else beta.cuda(), eps=eps, out_dtype=ty, want_stats=True)
    ga, be = (1.0, torch.zeros(cols, dtype=torch.float64)) if plain else (gamma.double(), beta.double())
    ref, m64, r64, xh = norm64(x64, ga, be, eps)
    dm = (cols + 2) * U * x64.abs().mean(1, keepdim=True)
    # variance: each difference off by dm + U of itself; its relative error halves in the root; 1 / sqrt a few U
    var = r64 ** -2
    dvar = (cols + 4) * U * (var - eps).clamp(min=0) + 2 * (var ** 0.5) * (dm + U * x64.abs().amax(1, keepdim=True)) + dm ** 2
    dr = r64 * (0.5 * dvar / (var - dvar).clamp(min=eps / 2) + 4 * U)
    close(mean, m64[:, 0], (dm + 2 * U * m64.abs())[:, 0], "mean")
    close(rstd, r64[:, 0], dr[:, 0], "rstd")
    d = (dr / r64 * xh.abs() + r64 * (dm + 2 * U * (x64.abs() + m64.abs())) + 3 * U * xh.abs()) * (1.0 if plain else ga.abs()) + 2 * U * (ref.abs() + be.abs())
    close(y, ref, d + rounding(ref.abs() + d, ty), "y")
    y2, a, b = eng.layer_norm(x, None if plain else gamma.cuda(), None if plain else beta.cuda(), eps=eps, out_dtype=ty)
    assert a is None and b is None and torch.equal(y, y2)


@pytest.mark.gpu
def test_layer_norm_of_constant_rows(eng):
    """No spread: the root of eps alone; far from zero the difference to the mean is exact where the mean is."""
    x = torch.tensor([[3.0] * 356, [0.0] * 356, [-1.0] * 356], device="cuda")
    y, mean, rstd = eng.layer_norm(x, want_stats=True, eps=1e-5)
    assert torch.equal(mean.cpu(), torch.tensor([3.0, 0.0, -1.0])) and torch.equal(y, torch.zeros_like(y))
    assert (rstd.cpu().double() * 1e-5 ** 0.5 - 1).abs().max() < 4 * U + 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("td,tx", [(BF16, F32), (F32, F32), (F16, BF16), (F32, F16)])
@pytest.mark.parametrize("n,cols", NORM_SHAPES + [(4099, 355), (9000, 63)])
def test_layer_norm_backward(eng, td, tx, n, cols):
    g = gen("back", n, cols)
    x, x64 = rows(g, n, cols, tx, cols + (n % 3), scale=0.5)
    dy, dy64 = rows(g, n, cols, td, cols + (n % 2))
    gamma = torch.randn(cols, generator=g) if n % 2 else None
    ga = gamma.double() if gamma is not None else torch.ones(cols, dtype=torch.float64)
    _, m64, r64, _ = norm64(x64, ga, 0.0, 1e-3)
    mean, rstd = m64[:, 0].float(), r64[:, 0].float()
    xh = (x64 - mean.double()[:, None]) * rstd.double()[:, None]                     # the definition, at the given statistics
    h = dy64 * ga
    c0, c1 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
    ref = rstd.double()[:, None] * (h - c0 - xh * c1)
    dxh = U * (3 * xh.abs() + 2 * rstd.double()[:, None] * (x64.abs() + mean.double().abs()[:, None]))
    dc0 = (cols + 3) * U * h.abs().mean(1, keepdim=True)
    dc1 = (cols + 4) * U * (h * xh).abs().mean(1, keepdim=True) + (h.abs() * dxh).mean(1, keepdim=True)
    d = rstd.double()[:, None] * (dc0 + dc1 * xh.abs() + dxh * c1.abs() + 4 * U * (h.abs() + c0.abs() + (xh * c1).abs()))
    gc = gamma.cuda() if gamma is not None else None
    dx, dg, db = eng.layer_norm_backward(dy, x, gc, mean.cuda(), rstd.cuda(), out_dtype=F32)
    close(dx, ref, d + U * ref.abs() + 1e-38, "dx")
    close(dg, (dy64 * xh).sum(0), ((n + 3) * U * (dy64 * xh).abs() + dy64.abs() * dxh).sum(0) + 1e-38, "dgamma")
    close(db, dy64.sum(0), (n + 2) * U * dy64.abs().sum(0) + 1e-38, "dbeta")
    dx2, a, b = eng.layer_norm_backward(dy, x, gc, mean.cuda(), rstd.cuda(), out_dtype=F32, want_params=False)
    assert a is None and b is None and torch.equal(dx, dx2)
    none, dg2, db2 = eng.layer_norm_backward(dy, x, gc, mean.cuda(), rstd.cuda(), want_dx=False)
    assert none is None and torch.equal(dg, dg2) and torch.equal(db, db2)


# ------------------------------------------------------------------------------ softmax
SOFT_SHAPES = [(1, 1), (1, 356), (4, 2), (9, 255), (33, 256), (50, 355), (20, 1563), (301, 1564), (3, 2048), (5, 2049), (3, 8192), (3, 9001)]


@pytest.mark.gpu
@pytest.mark.parametrize("tx,tg", [(F32, BF16), (F32, F32), (BF16, F16), (F16, F32)])
@pytest.mark.parametrize("n,K", SOFT_SHAPES)
def test_softmax(eng, tx, tg, n, K):
    g = gen("soft", n, K)
    s, s64 = rows(g, n, K, tx, K + (n % 3), scale=4.0, base=n % 2)
    labels = torch.randint(0, K + 1, (n,), generator=g, dtype=torch.int32)
    labels[0] = K
    scale = 0.37
    loss, grad = eng.softmax_loss(s, labels.cuda(), scale=scale, out_dtype=tg)
    lse = torch.logsumexp(s64, 1)
    p = torch.exp(s64 - lse[:, None])
    known = (labels > 0).double()
    at = (labels.long() - 1).clamp(min=0)
    ref = (lse - s64.gather(1, at[:, None])[:, 0]) * known
    spread = s64.amax(1) - s64.amin(1)
    # exp: 2 U and the rounding of its argument; the sum K U; the logarithm and two sums a few U of what they hold
    dz = (K + 6) * U + U * spread
    close(loss, ref, (dz + 4 * U * (lse.abs() + s64.abs().amax(1) + s64.gather(1, at[:, None])[:, 0].abs())) * known, "loss")
    one = torch.nn.functional.one_hot(labels.long(), K + 1)[:, 1:]
    sc = float(np.float32(scale))
    gref = (p - one) * sc * known[:, None]
    d = p * (dz[:, None] + 6 * U + U * spread[:, None]) * sc + 2 * U * sc * one
    close(grad, gref, d + rounding(gref.abs() + d, tg), "grad")
    cls, prob = eng.softmax_class(s)
    best = s64.amax(1)
    assert torch.equal(cls.cpu().long() - 1, (s64 == best[:, None]).int().argmax(1))
    pb = torch.exp(best - lse)
    close(prob, pb, pb * (dz + 4 * U), "prob")
    only, none = eng.softmax_loss(s, labels.cuda(), want_grad=False)
    assert none is None and torch.equal(only, loss)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [10, 300, 2500, 9000])
@pytest.mark.parametrize("t", [F32, BF16])
def test_softmax_of_ruled_out_classes(eng, t, K):
    inf, nan, low = float("inf"), float("nan"), torch.finfo(t).min
    s = torch.zeros(8, K)
    s[0] = -inf                                    # nothing is left
    s[1] = -inf
    s[1, K - 1] = 2.0                              # one class is left, and it is the label
    s[2] = -inf
    s[2, 4] = -3.0                                 # one class is left, and the label is another
    s[3, 5] = nan
    s[4] = low                                     # the type's lowest value everywhere: an ordinary row, all equal
    s[5, 7] = inf
    s[6] = -inf                                    # nothing left, no label
    s[7, 3] = low
    s[7, 2] = -inf
    labels = torch.tensor([1, K, 1, 1, 2, 8, 0, 1], dtype=torch.int32)
    loss, grad = eng.softmax_loss(s.to(t).cuda(), labels.cuda(), out_dtype=F32)
    loss, grad = loss.cpu(), grad.cpu()
    assert loss[0] == inf and torch.equal(grad[0], torch.zeros(K))
    assert loss[1] == 0 and torch.equal(grad[1], torch.zeros(K))
    want = torch.zeros(K)
    want[0], want[4] = -1, 1
    assert loss[2] == inf and torch.equal(grad[2], want)
    assert loss[3].isnan() and grad[3].isnan().all()
    assert abs(float(loss[4]) - np.log(K)) < 8 * U * np.log(K) + (K + 8) * U and abs(float(grad[4, 0]) * K - 1) < (K + 8) * U
    assert loss[5].isnan()
    assert loss[6] == 0 and torch.equal(grad[6], torch.zeros(K))
    assert abs(float(loss[7]) - np.log(K - 2)) < 8 * U * np.log(K) + (K + 8) * U and grad[7, 3] == 0 and grad[7, 2] == 0
    cls, prob = eng.softmax_class(s.to(t).cuda())
    assert cls.tolist() == [1, K, 5, 1, 1, 8, 1, 1]
    prob = prob.cpu()
    assert prob[0] == 0 and prob[1] == 1 and prob[2] == 1 and prob[3].isnan() and prob[5].isnan() and prob[6] == 0


@pytest.mark.gpu
def test_labels_that_are_no_class_are_reported(eng):
    import opal_amd
    s = torch.randn(6, 20, device="cuda")
    labels = torch.tensor([1, 21, -1, 20, 0, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    loss, grad = eng.softmax_loss(s, labels)
    with pytest.raises(opal_amd.OpalError, match=r"3 label\(s\)"):
        eng.sync()
    eng.sync()                                     # reported once
    for i in (1, 2, 4, 5):
        assert loss[i] == 0 and torch.equal(grad[i], torch.zeros(20, device="cuda"))
    assert loss[0] > 0 and loss[3] > 0


# ------------------------------------------------------------------------------ together
def head_step(eng, s, labels, gamma, beta, w1, b1, w2, b2, t, scale):
    """Forward and backward of the head, as a training step makes them."""
    z, mean, rstd = eng.layer_norm(s, gamma, beta, out_dtype=t, want_stats=True)
    h, pre = eng.linear(z, w1, b1, activation="gelu", want_pre=True)
    logits, _ = eng.linear(h, w2, b2, residual=z, out_dtype=F32)
    loss, dl = eng.softmax_loss(logits, labels, scale=scale, out_dtype=t)
    dw2, db2 = eng.linear_grad_weight(dl, h)
    dpre = eng.linear_grad_input(dl, w2, pre=pre, activation="gelu")
    dw1, db1 = eng.linear_grad_weight(dpre, z)
    dz = eng.linear_grad_input(dpre, w1, residual=dl)
    ds, dg, db = eng.layer_norm_backward(dz, s, gamma, mean, rstd)
    return loss, ds, dg, db, dw1, db1, dw2, db2


def head_inputs(n, K, H, t, seed=3):
    g = torch.Generator().manual_seed(seed)
    r = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    return (r(n, K) * 0.3, torch.randint(0, K + 1, (n,), generator=g, dtype=torch.int32), 1 + 0.1 * r(K), 0.1 * r(K), (r(H, K) * K ** -0.5).to(t), 0.1 * r(H),
            (r(K, H) * H ** -0.5).to(t), 0.1 * r(K))


def head_loss64(s, labels, gamma, beta, w1, b1, w2, b2):
    z = norm64(s, gamma, beta, 1e-5)[0]
    logits = act64(z @ w1.t() + b1, "gelu") @ w2.t() + b2 + z
    known = (labels > 0).double()
    return ((torch.logsumexp(logits, 1) - logits.gather(1, (labels.long() - 1).clamp(min=0)[:, None])[:, 0]) * known)


@pytest.mark.gpu
@pytest.mark.parametrize("n,K,H", [(1, 10, 16), (37, 63, 33), (300, 356, 128)])
def test_head_gradients_against_the_formula_and_differences(eng, n, K, H):
    """The chain in 32 bits against autograd of the formula in 64, and along a direction against differences."""
    vals = head_inputs(n, K, H, F32)
    dev = [v.cuda() for v in vals]
    got = head_step(eng, *dev, F32, 1.0 / n)
    leaf = [v.double().requires_grad_(i != 1) if i != 1 else v for i, v in enumerate(vals)]
    loss = head_loss64(*leaf)
    total = loss.sum() / n
    order = [0, 2, 3, 4, 5, 6, 7]
    grads = torch.autograd.grad(total, [leaf[i] for i in order])
    # a chain of five stages, each off by at most (length + 16) U of sums of absolute values; of all stages together the norm of
    # a gradient is off by less than 5 (K + H + n + 64) U of the norm times the largest gain in absolute values (below 64 here)
    tol = 5 * (K + H + n + 64) * U * 64
    close(got[0], loss.detach(), torch.full((n,), tol) * (1 + loss.detach().abs()), "loss")
    for name, a, b in zip(("ds", "dgamma", "dbeta", "dw1", "db1", "dw2", "db2"), got[1:], [grads[0]] + list(grads[1:3]) + list(grads[3:])):
        assert float((a.double().cpu() - b).norm()) <= tol * float(b.norm()), name
    g = torch.Generator().manual_seed(9)
    direction = [torch.randn(leaf[i].shape, generator=g, dtype=torch.float64) for i in order]
    step = 1e-5
    moved = lambda sgn: [v.double() + sgn * step * direction[order.index(i)] if i in order else v for i, v in enumerate(vals)]  # noqa: E731
    slope = float((head_loss64(*moved(1)).sum() - head_loss64(*moved(-1)).sum()) / n / (2 * step))
    along = sum(float((a.double().cpu() * d).sum()) for a, d in zip(got[1:], direction))
    size = sum(float(a.double().norm()) * float(d.norm()) for a, d in zip(got[1:], direction))
    assert abs(slope - along) <= (tol + 1e-6) * size


@pytest.mark.gpu
@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("n,K,H", [(515, 355, 72), (3, 10, 16), (70001, 512, 256)])
def test_head_step_is_the_same_every_time_and_in_a_graph(eng, t, n, K, H):
    """Equal bits on repetition; captured and replayed with new inputs, with eager work between the replays."""
    import opal_amd
    vals = head_inputs(n, K, H, t)
    want = head_step(eng, *[v.cuda() for v in vals], t, 1.0 / n)
    again = head_step(eng, *[v.cuda() for v in vals], t, 1.0 / n)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        e = opal_amd.Engine(0)
        dev = [v.cuda() for v in vals]
        head_step(e, *dev, t, 1.0 / n)
    side.synchronize()
    graphs = []
    for _ in range(2):                             # two graphs of one engine: neither may lean on the other's memory
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = head_step(e, *dev, t, 1.0 / n)
        graphs.append((graph, out))
    for seed in (4, 5, 3):
        other = head_inputs(n, K, H, t, seed)
        ref = head_step(eng, *[v.cuda() for v in other], t, 1.0 / n)
        for a, b in zip(dev, other):
            a.copy_(b)
        torch.cuda.synchronize()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, ref))
    del graphs
    e.close()


@pytest.mark.gpu
def test_two_engines_at_once(eng):
    """Two engines on two streams, one of them with large products and one with small ones, side by side: nothing is shared."""
    import opal_amd
    sizes = [(70001, 512, 256), (900, 355, 128)]
    vals = [[v.cuda() for v in head_inputs(n, K, H, BF16, seed=n)] for n, K, H in sizes]
    want = [head_step(eng, *v, BF16, 1.0 / n) for v, (n, _, _) in zip(vals, sizes)]
    torch.cuda.synchronize()
    streams, engines = [torch.cuda.Stream() for _ in sizes], []
    for st in streams:
        with torch.cuda.stream(st):
            engines.append(opal_amd.Engine(0))
    got = [None, None]
    for _ in range(4):
        for j, times in ((0, 1), (1, 8)):
            with torch.cuda.stream(streams[j]):
                for _ in range(times):
                    got[j] = head_step(engines[j], *vals[j], BF16, 1.0 / sizes[j][0])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    for e in engines:
        e.close()


@pytest.mark.gpu
def test_calls_from_another_stream_are_ordered(eng):
    """Inputs made on a stream of their own, results used there at once; memory is not handed out again too early."""
    n, K = 20000, 700
    side = torch.cuda.Stream()
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(512, K, device="cuda", generator=g).to(BF16)
    x0 = torch.randn(n, K, device="cuda", generator=g).to(BF16)
    want = eng.linear(x0, w, activation="silu")[0].float().sum(1)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(5):
            x = x0.float().mul(2).to(BF16).float().mul(0.5).to(BF16)              # work that the call has to wait for
            y, _ = eng.linear(x, w, activation="silu")
            del x
            junk = torch.full((n, K), float("nan"), device="cuda", dtype=BF16)    # may take x's memory once that is free
            got = y.float().sum(1)
            del y, junk
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_rows_beyond_32_bits(eng):
    """A matrix of more than 2^32 bytes: its last rows are found."""
    n, K = 1_400_003, 1564
    x = torch.zeros(n, K, dtype=BF16, device="cuda")
    tail = torch.randn(300, K, device="cuda").to(BF16)
    x[-300:] = tail
    w = (torch.randn(65, K, device="cuda") * 0.02).to(BF16)
    y, _ = eng.linear(x, w)
    # against the sums themselves: the kernel, and with it the order of a sum, goes by the number of rows
    ref = tail.double().cpu() @ w.double().cpu().t()
    d = (K + 2) * U * (tail.double().abs().cpu() @ w.double().abs().cpu().t())
    close(y[-300:], ref, d + rounding(ref.abs() + d, BF16))
    assert not y[:-300].any()
    z, mean, _ = eng.layer_norm(x, out_dtype=BF16, want_stats=True)
    assert torch.equal(z[-300:], eng.layer_norm(tail, out_dtype=BF16)[0])
    cls, _ = eng.softmax_class(x)
    assert torch.equal(cls[-300:], eng.softmax_class(tail)[0])
    dy = torch.zeros(n, 65, dtype=BF16, device="cuda")
    dy[-300:] = torch.randn(300, 65, device="cuda").to(BF16)
    dw, db = eng.linear_grad_weight(dy, x)
    ref = dy[-300:].double().t().cpu() @ tail.double().cpu()
    close(dw, ref, (302 + n / 64) * U * (dy[-300:].double().abs().t().cpu() @ tail.double().abs().cpu()) + 1e-38)


# ------------------------------------------------------------------------------ refusals
@pytest.mark.gpu
def test_more_rows_than_one_launch_holds(eng):
    """2^28 + 17 rows for teams of 16 lanes, 2^30 + 300 for a product: the results of the rows around the seam and at both ends are
    those of the same rows alone (a row's arithmetic does not look at the others)."""
    n = (1 << 28) + 17
    x = torch.empty(n, 2, dtype=BF16, device="cuda")
    x.view(torch.int32)[:, 0] = torch.arange(n, dtype=torch.int32, device="cuda") * 40503 & 0x3fff3fff        # finite pairs of bf16
    gamma, beta = torch.tensor([0.5, 2.0], device="cuda"), torch.tensor([0.25, -1.0], device="cuda")
    parts = [(0, 3000), ((1 << 28) - 100, n)]
    y, mean, rstd = eng.layer_norm(x, gamma, beta, want_stats=True)
    for a, b in parts:
        py, pm, pr = eng.layer_norm(x[a:b], gamma, beta, want_stats=True)
        assert torch.equal(y[a:b], py) and torch.equal(mean[a:b], pm) and torch.equal(rstd[a:b], pr)
    del y, mean, rstd
    labels = (torch.arange(n, dtype=torch.int32, device="cuda") % 3)
    loss, grad = eng.softmax_loss(x, labels)
    cls, prob = eng.softmax_class(x)
    for a, b in parts:
        pl, pg = eng.softmax_loss(x[a:b], labels[a:b])
        pc, pp = eng.softmax_class(x[a:b])
        assert torch.equal(loss[a:b], pl) and torch.equal(grad[a:b, :], pg) and torch.equal(cls[a:b], pc) and torch.equal(prob[a:b], pp)
    del x, loss, grad, cls, prob, labels
    n = (1 << 30) + 300
    x = torch.empty(n, 1, dtype=BF16, device="cuda")
    x.copy_((torch.arange(n, dtype=torch.int32, device="cuda") % 251 - 125)[:, None])
    w, bias = torch.tensor([[0.75]], dtype=BF16, device="cuda"), torch.tensor([0.5], device="cuda")
    y = torch.empty_strided((n, 1), (1, 1), dtype=BF16, device="cuda")
    from opal_amd._lib import check
    check(eng._lib.opal_linear(eng._h, x.data_ptr(), 1, w.data_ptr(), 1, 2, bias.data_ptr(), 0, None, 0, 0, n, 1, 1, y.data_ptr(), 2, 1, None, 0), eng._h)
    for a, b in [(0, 3000), ((1 << 30) - 200, n)]:                  # 0.75 k + 0.5: exact in 32 bits, one rounding
        assert torch.equal(y[a:b], (x[a:b].float() * 0.75 + 0.5).to(BF16))


@pytest.mark.gpu
def test_engine_refuses(eng):
    x, w = torch.randn(4, 8, device="cuda"), torch.randn(6, 8, device="cuda")
    lab = torch.ones(4, dtype=torch.int32, device="cuda")
    one = torch.ones(8, device="cuda")
    for call in (lambda: eng.linear(x, w.half()), lambda: eng.linear(x, w[:, :7]), lambda: eng.linear(x.t(), w), lambda: eng.linear(x.cpu(), w),
                 lambda: eng.linear(x, w, one), lambda: eng.linear(x, w, activation="tanh"), lambda: eng.linear(x, w, residual=x), lambda: eng.linear(x, None),
                 lambda: eng.linear(x.double(), w.double()), lambda: eng.linear(x, w, out_dtype=torch.int32), lambda: eng.linear(x[0], w),
                 lambda: eng.linear(x[:1].expand(4, 8), w),
                 lambda: eng.linear_grad_input(x, w), lambda: eng.linear_grad_input(x[:, :6], w, activation="relu"),
                 lambda: eng.linear_grad_weight(x, x[:3]), lambda: eng.linear_grad_weight(None, x), lambda: eng.layer_norm(x, one[:7]),
                 lambda: eng.layer_norm(x, one.half()), lambda: eng.layer_norm_backward(x, x, None, None, None), lambda: eng.layer_norm_backward(x[:3], x, None, one[:4], one[:4]),
                 lambda: eng.softmax_loss(x, lab.long()), lambda: eng.softmax_loss(x, lab[:3]), lambda: eng.softmax_loss(x, None), lambda: eng.softmax_class(x[:, :0])):
        with pytest.raises(ValueError):
            call()
    import opal_amd
    long = torch.zeros((1 << 20) + 1, 8, device="cuda")           # more outputs than a product has
    for call in (lambda: eng.layer_norm(x, eps=0.0), lambda: eng.layer_norm(x, eps=float("nan")), lambda: eng.linear(x[:1], long), lambda: eng.softmax_class(long.view(1, -1)[:, :(1 << 20) + 1])):
        with pytest.raises(opal_amd.OpalError):
            call()


def test_c_entries_refuse(tmp_path):
    """Every refusal happens on the host before anything touches a GPU: a plain C++ client with a ctx of its own making."""
    exe = str(tmp_path / "refuse")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I%s/include" % ROOT, "-I%s/opal_amd/csrc" % ROOT,
                           "%s/tests/native/head_refusals.cpp" % ROOT, "-o", exe, "-L%s/opal_amd" % ROOT, "-lopal_hip", "-L/opt/rocm/lib", "-lamdhip64",
                           "-Wl,-rpath,%s/opal_amd" % ROOT, "-Wl,-rpath,/opt/rocm/lib"])
    run = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout + run.stderr
    assert "head refusals: ok" in run.stdout


def test_workspace_sizes():
    from opal_amd._lib import lib
    L = lib()
    assert L.opal_layer_norm_backward_workspace(0, 10) == 0
    for n in (1, 7, 1000, 10 ** 6):
        for cols in (1, 355, 1564, 2049, 9000):
            size = L.opal_layer_norm_backward_workspace(n, cols)
            assert 8 * cols * (n >= 1000) <= size <= 8 * cols * 1024
    assert L.opal_linear_grad_weight_workspace(0, 5, 7, 2) == 0
    assert L.opal_linear_grad_weight_workspace(100, 5, 7, 9) == 0
    for n in (1, 100, 10 ** 6):
        for k, m in ((1, 1), (355, 63), (1564, 512)):
            assert L.opal_linear_grad_weight_workspace(n, k, m, 2) < 1 << 30


def test_binding_refuses_without_a_gpu():
    """The extension module loads where there is no GPU, and refuses what is no matrix on one."""
    from opal_amd._lib import bind
    b = bind()
    x = torch.zeros(2, 8)
    for call in (lambda: b.softmax_class(0, 0, x), lambda: b.softmax_class(0, 0, None), lambda: b.softmax_class(0, 0, [1.0]), lambda: b.linear(0, 0, x, x, None, None, 0, None, False),
                 lambda: b.layer_norm(0, 0, x.double(), None, None, 1e-5, None, False), lambda: b.linear_grad_weight(0, 0, x[0], x, True)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: b.softmax_class(0, 0), lambda: b.linear(0, 0, x, x), lambda: b.softmax_class("ctx", 0, x)):
        with pytest.raises(TypeError):
            call()
