"""
The read-out of several latent fields (gptools_amd.glm: layer norm, categorical_logit_glm_lpmf, their reverse modes) against
their formulas in 64 bits (plain torch operations on the same inputs), at the sizes, masks and strides where they can go wrong.

Tolerances are error bounds, worked out entry by entry from the inputs: `eps / 2` of the element type for every rounding to it
(the result; for 16-bit data also the entries of r = lpbar ([v = y] - softmax), which the products take in that type), and
`eps` of the accumulator's type times the number of operations that a value passes through for everything else.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = {"f64": 0.0, "f32": 2.0**-126, "f16": 2.0**-25, "bf16": 2.0**-126}  # half a step among the smallest numbers


@pytest.fixture(scope="module")
def glm(gpu_lib):
    from gptools_amd import glm as g

    return g


def _wide(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def _eps(dtype):
    return torch.finfo(dtype).eps


def _rng(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, scale=1.0, offset=0.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float64) * scale + offset).to(dtype)


def _within(what, got, want, tol):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    worst = ((got - want).abs() - tol).max() if got.numel() else torch.zeros(())
    assert bool(worst <= 0), f"{what}: off by up to {float((got - want).abs().max()):.3e}, {float(worst):.3e} over the bound"


# ---- layer norm --------------------------------------------------------------------------------------------------------
def _norm_want(x, w, b, eps, core):
    dims = tuple(range(x.ndim - core, x.ndim))
    x = x.double()
    mean = x.mean(dims, keepdim=True)
    c = x - mean
    rstd = 1 / torch.sqrt((c * c).mean(dims, keepdim=True) + eps)
    h = c * rstd
    y = h * (1 if w is None else w.double()) + (0 if b is None else b.double())
    return y, mean, rstd, h


# adds that a value passes through in a sum over a row: in one thread up to 32 (its registers) + a sweep or a piece at a
# time up to 32, across lanes, waves and pieces up to 6 + 16 + 10; a bound that leaves room for the products
DEPTH = 128


def _check_norm(glm, name, rows, core, affine=True, seed=0, eps=1e-5, scale=1.7, offset=0.4):
    dtype = DTYPES[name]
    g = _rng(seed)
    x = _normal(g, (*rows, *core), dtype, scale, offset)
    w = _normal(g, core, dtype, 0.2, 1.0) if affine else None
    b = _normal(g, core, dtype, 0.3) if affine else None
    ybar = _normal(g, (*rows, *core), dtype)
    nc = len(core)
    y, mean, rstd = glm.layer_norm(x, w, b, eps=eps, core_ndim=nc)
    wy, wm, wr, h = _norm_want(x, w, b, eps, nc)
    assert y.dtype == dtype and mean.dtype == rstd.dtype == _wide(dtype)
    dims = tuple(range(len(rows), len(rows) + nc))
    ea, et, tiny = _eps(_wide(dtype)), _eps(dtype), TINY[name]
    xa = x.double().abs().mean(dims, keepdim=True)
    dm = DEPTH * ea * xa  # of the mean
    # of the variance: relative DEPTH eps, and the square of the mean's error; of rstd: half of that, and the root's own
    dr = wr * (DEPTH * ea + 0.5 * (dm * wr) ** 2)
    _within("mean", mean, wm.reshape(rows), dm.reshape(rows))
    _within("rstd", rstd, wr.reshape(rows), dr.reshape(rows))
    dh = wr * (dm + ea * (x.double().abs() + wm.abs())) + h.abs() * (dr / wr + 4 * ea)
    wa = 1.0 if w is None else w.double().abs()
    _within("y", y, wy, dh * wa + 4 * ea * (h.abs() * wa + wy.abs()) + et / 2 * wy.abs() * (1 + et) + tiny)

    xbar, wbar, bbar = glm.layer_norm_vjp(x, w, mean, rstd, ybar, core_ndim=nc)
    yb = ybar.double()
    gw = yb * (1 if w is None else w.double())
    c0, c1 = gw.mean(dims, keepdim=True), (gw * h).mean(dims, keepdim=True)
    want = wr * (gw - c0 - h * c1)
    d0 = DEPTH * ea * gw.abs().mean(dims, keepdim=True)
    d1 = DEPTH * ea * (gw * h).abs().mean(dims, keepdim=True) + (gw.abs() * dh).mean(dims, keepdim=True)
    tol = wr * (d0 + h.abs() * d1 + dh * c1.abs() + 4 * ea * (gw.abs() + c0.abs() + (h * c1).abs())) + want.abs() * dr / wr
    _within("xbar", xbar, want, tol * (1 + et) + et / 2 * want.abs() * (1 + et) + tiny)
    lead = tuple(range(len(rows)))
    n = math.prod(rows)
    many = (min(n, 64) + n / 64 + 64) * ea  # rows added up one by one by a workgroup, then across workgroups
    want = (yb * h).sum(lead) if rows else yb * h
    tol = ((yb * h).abs() * many + yb.abs() * dh).sum(lead) if rows else yb.abs() * (h.abs() * many + dh)
    _within("weightbar", wbar, want, tol * (1 + et) + et / 2 * want.abs() * (1 + et) + tiny)
    want = yb.sum(lead) if rows else yb
    tol = yb.abs().sum(lead) * many if rows else yb.abs() * many
    _within("biasbar", bbar, want, tol + et / 2 * want.abs() * (1 + et) + tiny)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("rows,width", [((1,), 1), ((3,), 2), ((5,), 7), ((2, 3), 64), ((67,), 129), ((9,), 511), ((6,), 1001),
                                        ((700,), 96), ((33,), 2100), ((4,), 4096), ((3,), 8193), ((2,), 16384), ((), 100)])
def test_layer_norm_rows(glm, name, rows, width):
    _check_norm(glm, name, rows, (width,), seed=width)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("rows,core", [((4,), (35, 60)), ((3,), (257, 301)), ((2, 2), (256, 512)), ((70,), (200, 201)),
                                       ((1,), (1000, 1001))])
def test_layer_norm_lattices(glm, name, rows, core):
    _check_norm(glm, name, rows, core, seed=core[1])


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("rows,core", [((300,), (2049,)), ((270,), (4095,)), ((520,), (8191,)), ((260,), (10001,)), ((300,), (16001,)),
                                       ((300,), (5,)), ((3000,), (17,)), ((2048,), (600,)), ((50,), (1900,)), ((3,), (40961,)), ((290,), (40961,)), ((64,), (300, 1000))])
def test_layer_norm_several_rows_a_workgroup(glm, name, rows, core):
    """More rows than workgroups, at lengths that a part vector, a part sweep or one value ends; lattices that share weights."""
    _check_norm(glm, name, rows, core, seed=core[0])


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("width", [40, 3000, 70001])
def test_layer_norm_without_parameters(glm, name, width):
    _check_norm(glm, name, (5,), (width,), affine=False, seed=width)


@pytest.mark.parametrize("width", [300, 5000, 100000])
def test_layer_norm_far_from_zero(glm, width):
    # a level a thousand times the spread: the variance is not a difference of two large sums
    _check_norm(glm, "f32", (7,), (width,), seed=width, scale=1.0, offset=1000.0)
    _check_norm(glm, "f64", (7,), (width,), seed=width, scale=1.0, offset=1e6)


def test_layer_norm_constant_rows_and_spoilt_rows(glm):
    x = torch.full((4, 100), 3.0, device="cuda")
    x[1, 7] = float("nan")
    x[2, 3] = float("inf")
    y, mean, rstd = glm.layer_norm(x, eps=0.25)
    assert torch.equal(y[[0, 3]], torch.zeros(2, 100, device="cuda"))
    assert torch.equal(rstd[[0, 3]], torch.full((2,), 2.0, device="cuda"))
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[2]).any())


def test_layer_norm_views_empty_batches_and_no_parameter_gradients(glm):
    g = _rng(5)
    wide = _normal(g, (50, 6, 40), torch.float32)
    view = wide.transpose(0, 1)[:, ::2, 3:30]  # (6, 25, 27), no dimension as it lies in memory
    y, mean, rstd = glm.layer_norm(view)
    y2, mean2, rstd2 = glm.layer_norm(view.contiguous())
    assert torch.equal(y, y2) and torch.equal(mean, mean2) and torch.equal(rstd, rstd2)
    off = wide.flatten()[1:1 + 27 * 25].view(25, 27)  # not aligned to 16 bytes
    assert torch.equal(glm.layer_norm(off)[0], glm.layer_norm(off.clone())[0])
    ybar = torch.ones_like(y)
    a = glm.layer_norm_vjp(view, None, mean, rstd, ybar)
    b = glm.layer_norm_vjp(view, None, mean, rstd, ybar, need_param_grad=False)
    assert torch.equal(a[0], b[0]) and b[1] is None and b[2] is None
    empty = wide[:0]
    y, mean, rstd = glm.layer_norm(empty)
    assert y.shape == (0, 6, 40) and mean.shape == (0, 6)
    xbar, wbar, bbar = glm.layer_norm_vjp(empty, None, mean, rstd, empty)
    assert xbar.shape == empty.shape and not bool(wbar.any()) and not bool(bbar.any())


def test_layer_norm_of_very_many_rows(glm):
    """More threads than a grid's dimension counts (2^32), and more values than 32 bits."""
    rows, width = (1 << 26) + 1001, 65
    x = torch.randint(-100, 100, (rows, width), dtype=torch.int8, device="cuda").to(torch.bfloat16)
    y, mean, rstd = glm.layer_norm(x)
    for at in (0, 1 << 25, rows - 700):
        some = x[at:at + 700].clone()
        want = glm.layer_norm(some)
        assert torch.equal(y[at:at + 700], want[0]) and torch.equal(mean[at:at + 700], want[1]) and torch.equal(rstd[at:at + 700], want[2])
    xbar = glm.layer_norm_vjp(x, None, mean, rstd, y, need_param_grad=False)[0]
    for at in (0, 1 << 25, rows - 700):
        c = slice(at, at + 700)
        assert torch.equal(xbar[c], glm.layer_norm_vjp(x[c].clone(), None, mean[c], rstd[c], y[c], need_param_grad=False)[0])


# ---- categorical log density -------------------------------------------------------------------------------------------
def _class_want(y, x, alpha, beta, lpbar, seen):
    xd = torch.where(seen.unsqueeze(1), x.double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    bd, ad = beta.double(), (torch.zeros(beta.shape[0], device="cuda") if alpha is None else alpha).double()
    eta = xd @ bd.T + ad
    lse = torch.logsumexp(eta, 1)
    at = y.clamp(0, beta.shape[0] - 1).unsqueeze(1)
    lp = torch.where(seen, eta.gather(1, at).squeeze(1) - lse, torch.zeros_like(lse))
    scale = torch.where(seen, torch.ones_like(lse) if lpbar is None else lpbar.double(), torch.zeros_like(lse))
    p = torch.exp(eta - lse.unsqueeze(1))
    r = -p * scale.unsqueeze(1)
    r.scatter_add_(1, at, scale.unsqueeze(1))
    return xd, bd, eta, lse, lp, scale, p, r


def _check_class(glm, name, y, x, alpha, beta, lpbar=None):
    dtype = DTYPES[name]
    ea, et, tiny = _eps(_wide(dtype)), _eps(dtype), TINY[name]
    d, v = x.shape[1], beta.shape[0]
    seen = y >= 0
    xd, bd, eta, lse, lp, scale, p, r = _class_want(y, x, alpha, beta, lpbar, seen)
    got_lp = glm.categorical_logit_glm_lpmf(y, x, alpha, beta)
    lp2, xbar, alphabar, betabar = glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta, lpbar=lpbar)
    assert got_lp.dtype == _wide(dtype) and xbar.dtype == betabar.dtype == dtype
    # eta: d products added up one after the other, and alpha; the exponential's and the logarithm's own errors are a few
    # eps, of the argument too; the sum passes through its tile's registers and lanes and through the tiles
    fin = torch.where(torch.isfinite(eta), eta.abs(), torch.zeros_like(eta))
    de = (d + 2) * ea * (xd.abs() @ bd.abs().T + fin) + 4 * ea * (fin + lse.abs().unsqueeze(1))
    top = de.max(1).values
    dlp = 2 * top + (96 + v / 2048) * ea + 2 * ea * (lse.abs() + lp.abs())
    _within("lp", got_lp, lp, dlp)
    _within("lp of the reverse mode", lp2, lp, dlp)
    # r: the probability's relative error, and its rounding to the element type
    dr = scale.abs().unsqueeze(1) * p * (de + dlp.unsqueeze(1) + 4 * ea) + 4 * ea * r.abs()
    if dtype != torch.float64:
        # fp32's exponential gives 0 for results below its smallest normal number 2^-126 (a logit 87.3 below the sum's
        # logarithm): the probability is then off by itself, less than 2^-126, and each entry of r by that times its cotangent
        dr = dr + 2.0**-126 * scale.abs().unsqueeze(1)
    if et > ea:
        dr = dr + et / 2 * r.abs() * (1 + et)
        if name == "f16":  # r is stored times 2^13 / max |lpbar| at least
            dr = dr + 2.0**-25 * 2.0**-13 * scale.abs().max()
    ra = r.abs() + dr
    n = x.shape[0]
    want = r @ bd
    _within("xbar", xbar, want, (dr @ bd.abs()) + (v + 4) * ea * (ra @ bd.abs()) + et / 2 * want.abs() * (1 + et) + tiny * 1.01)
    want = r.T @ xd
    _within("betabar", betabar, want, (dr.T @ xd.abs()) + (n + 4) * ea * (ra.T @ xd.abs()) + et / 2 * want.abs() * (1 + et) + tiny * 1.01)
    if alpha is None:
        assert alphabar is None
    else:
        want = r.sum(0)
        tol = dr.sum(0) + (n + 4) * ea * ra.sum(0)
        _within("alphabar", alphabar, want, tol + et / 2 * (want.abs() + tol) + tiny)
    assert not bool(xbar[~seen].any()), "a row without an observation has a gradient"


def _class_data(name, n, d, v, seed, masked=0.0, alpha=True, spread=1.5):
    dtype = DTYPES[name]
    g = _rng(seed)
    x = _normal(g, (n, d), dtype)
    beta = _normal(g, (v, d), dtype, spread / d**0.5)
    al = _normal(g, (v,), dtype, 0.5) if alpha else None
    y = torch.randint(0, v, (n,), generator=g, device="cuda")
    y[torch.rand(n, generator=g, device="cuda") < masked] = -1
    return y, x, al, beta


SIZES = [(1, 1, 1), (1, 1, 2), (2, 3, 5), (5, 8, 3), (1, 64, 1000), (3, 1000, 130), (17, 129, 300), (127, 64, 128), (128, 65, 129),
         (129, 30, 257), (256, 256, 256), (300, 200, 513), (2100, 8, 300), (1000, 33, 70), (61, 520, 2051)]


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("n,d,v", SIZES)
def test_class_sizes(glm, name, n, d, v):
    _check_class(glm, name, *_class_data(name, n, d, v, seed=n + d + v))


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("n,d,v", [(700, 128, 8192), (520, 200, 8300), (1030, 65, 5003), (300, 1000, 13001), (9000, 130, 700),
                                   (5000, 100, 1300)])
def test_class_large_sizes(glm, name, n, d, v):
    """Products of enough tiles for the large ones; aligned and not."""
    _check_class(glm, name, *_class_data(name, n, d, v, seed=n + d + v, masked=0.1))


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("n,d,v", [(40, 16, 20), (333, 100, 1000), (16, 256, 4000), (1500, 96, 6000)])
@pytest.mark.parametrize("masked", [0.3, 1.0])
def test_class_masked_rows(glm, name, n, d, v, masked):
    y, x, alpha, beta = _class_data(name, n, d, v, 7, masked)
    y[y < 0] = torch.where(torch.rand(int((y < 0).sum()), device="cuda") < 0.5, -1, -100)
    x[y < 0] = float("nan")  # such rows may hold anything
    x[(y < 0).nonzero()[::2].squeeze(1)] = float("inf")
    lpbar = _normal(_rng(3), (n,), _wide(DTYPES[name]))
    lpbar[y < 0] = float("nan")
    _check_class(glm, name, y, x, alpha, beta, lpbar)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("size", [1.0, -1e-4, 300.0])
def test_class_cotangents(glm, name, size):
    y, x, _, beta = _class_data(name, 200, 72, 700, 11, alpha=False)
    lpbar = size * (0.5 + torch.rand(200, generator=_rng(1), device="cuda", dtype=_wide(DTYPES[name])))
    _check_class(glm, name, y, x, None, beta, lpbar)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("n,d,v", [(50, 20, 30), (70, 200, 700), (800, 80, 7000)])
def test_class_excluded_classes(glm, name, n, d, v):
    y, x, alpha, beta = _class_data(name, n, d, v, 13)
    alpha[1::2] = -float("inf")
    y = y // 2 * 2
    _check_class(glm, name, y, x, alpha, beta)
    # an excluded class observed: -inf, and the gradient of the others as ever
    y[3] = 1
    lp, xbar, alphabar, betabar = glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta)
    assert float(lp[3]) == -float("inf") and bool(torch.isfinite(lp[:3]).all())
    assert bool(torch.isfinite(xbar).all()) and bool(torch.isfinite(betabar).all())
    # the lowest finite value excludes a class too
    alpha[1::2] = torch.finfo(alpha.dtype).min / 2
    y[3] = 2
    _check_class(glm, name, y, x, alpha, beta)
    # nothing possible at all: lp is -inf, no gradient
    alpha[:] = -float("inf")
    lp, xbar, alphabar, betabar = glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta)
    assert bool((lp == -float("inf")).all()) and not bool(xbar.any()) and not bool(alphabar.any()) and not bool(betabar.any())


@pytest.mark.parametrize("name", list(DTYPES))
def test_class_large_logits(glm, name):
    # logits of some hundreds: one class takes nearly everything
    y, x, alpha, beta = _class_data(name, 100, 40, 300, 17, spread=100.0)
    _check_class(glm, name, y, x, alpha, beta)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("n,d,v", [(30, 7, 50), (65, 160, 300), (800, 80, 7000)])
def test_class_spoilt_rows(glm, name, n, d, v):
    y, x, alpha, beta = _class_data(name, n, d, v, 19)
    y[4] = v  # no class: refused, or NaN where the check is left out
    with pytest.raises(ValueError, match="class"):
        glm.categorical_logit_glm_lpmf(y, x, alpha, beta)
    with pytest.raises(ValueError, match="class"):
        glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta)
    lp, xbar, _, betabar = glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta, check=False)
    assert bool(torch.isnan(lp[4])) and bool(torch.isnan(xbar[4]).all()) and bool(torch.isnan(betabar).all())
    rest = torch.arange(n, device="cuda") != 4
    assert bool(torch.isfinite(lp[rest]).all()) and bool(torch.isfinite(xbar[rest]).all())
    y[4] = 0
    x[4, 0] = float("nan")
    lp, xbar, _, _ = glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta)
    assert bool(torch.isnan(lp[4])) and bool(torch.isfinite(lp[rest]).all()) and bool(torch.isfinite(xbar[rest]).all())


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("n,v", [(30, 210), (90, 210), (900, 6300)])
@pytest.mark.parametrize("d", [8, 64, 100, 131])
def test_class_strides_and_shapes(glm, name, d, n, v):
    dtype = DTYPES[name]
    g = _rng(23)
    wide_x, wide_b = _normal(g, (n, d + 9), dtype), _normal(g, (v, d + 5), dtype, 1 / d**0.5)
    y = torch.randint(0, v, (n,), generator=g, device="cuda")
    x, beta = wide_x[:, 3:3 + d], wide_b[:, 1:1 + d]  # rows apart, not aligned to 16 bytes
    _check_class(glm, name, y, x, None, beta)
    base = glm.categorical_logit_glm_lpmf_vjp(y, x.contiguous(), None, beta.contiguous())
    for got in (glm.categorical_logit_glm_lpmf_vjp(y, x, None, beta),
                glm.categorical_logit_glm_lpmf_vjp(y.int(), x.T.contiguous().T, None, beta.T.contiguous().T),
                glm.categorical_logit_glm_lpmf_vjp(y.view(2, 3, -1), x.reshape(2, 3, -1, d), None, beta)):
        for a, b in zip(got, base):
            # (rows that do not start on 16 bytes may be added up in another order: the bound above holds for both)
            assert (a is None and b is None) or torch.allclose(a.reshape(b.shape).double(), b.double(), rtol=4 * _eps(b.dtype),
                                                               atol=64 * _eps(b.dtype) * float(b.double().abs().max()))


@pytest.mark.parametrize("name,n,d,v", [("f64", 262144 + 300, 3, 300), ("f64", 262144 + 1, 90, 129), ("bf16", 262144 + 129, 130, 1100)])
def test_class_many_rows(glm, name, n, d, v):
    """More rows than are taken at a time, and (with that many) several pieces of the classes."""
    y, x, alpha, beta = _class_data(name, n, d, v, 29, masked=0.1)
    lpbar = torch.full((n,), 1 / 1024, dtype=_wide(DTYPES[name]), device="cuda")
    _check_class(glm, name, y, x, alpha, beta, lpbar)


def test_class_of_very_many_rows(glm):
    """More threads than a grid's dimension counts (2^32)."""
    n = (1 << 29) + 77
    x = torch.zeros(n, 1, dtype=torch.float64, device="cuda")
    x[-5:, 0] = torch.arange(1.0, 6.0, dtype=torch.float64, device="cuda")
    y = torch.zeros(n, dtype=torch.int64, device="cuda")
    y[: n - 3 : 2] = -1
    beta = torch.tensor([[0.5], [-0.25]], dtype=torch.float64, device="cuda")
    lp = glm.categorical_logit_glm_lpmf(y, x, None, beta)
    want = glm.categorical_logit_glm_lpmf(y[-100:].clone(), x[-100:].clone(), None, beta)
    assert torch.allclose(lp[-100:], want, rtol=16 * 2.0**-53, atol=16 * 2.0**-53)
    some = torch.arange(0, n - 5, 1001, device="cuda")
    some_lp = -math.log(2) * (y[some] >= 0).double()
    assert torch.allclose(lp[some], some_lp, rtol=16 * 2.0**-53, atol=0)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("n,d,v", [(100, 72, 50000), (257, 72, 25000), (384, 72, 25000), (385, 72, 25000), (1100, 1000, 24680)])
def test_class_last_rows_and_classes_fill_part_of_a_tile(glm, name, n, d, v):
    _check_class(glm, name, *_class_data(name, n, d, v, seed=n + v))


@pytest.mark.parametrize("name", list(DTYPES))
def test_class_observed_rows_fill_part_of_a_tile(glm, name):
    for masked in (0.5, 0.6, 0.9):  # of 700 rows, about 350, 280, 70
        y, x, alpha, beta = _class_data(name, 700, 72, 20000, 5, masked)
        x[y < 0] = float("nan")
        _check_class(glm, name, y, x, alpha, beta)


@pytest.mark.parametrize("name,n,d,v", [("bf16", 16500, 768, 18000), ("f16", 16500, 800, 18000), ("f32", 4100, 170, 80000), ("f64", 2000, 70, 90000)])
def test_class_some_logits_are_kept(glm, name, n, d, v):
    """Several pieces of the classes, the logits of some of them kept and of the others computed again."""
    y, x, alpha, beta = _class_data(name, n, d, v, 31, masked=0.1)
    alpha[v // 2 : v // 2 + 300] = -float("inf")
    y[(y >= v // 2) & (y < v // 2 + 300)] = 0
    lpbar = torch.full((n,), -1 / 1024, dtype=_wide(DTYPES[name]), device="cuda")
    _check_class(glm, name, y, x, alpha, beta, lpbar)


@pytest.mark.parametrize("name", list(DTYPES))
def test_class_kept_logits_of_rows_without_any(glm, name):
    """Rows whose classes are all excluded, or whose values are spoilt, where the logits are kept."""
    y, x, alpha, beta = _class_data(name, 300, 800, 1500, 37, masked=0.2)
    lp, xbar, alphabar, betabar = glm.categorical_logit_glm_lpmf_vjp(y, x, torch.full_like(alpha, -float("inf")), beta)
    seen = y >= 0
    assert bool((lp[seen] == -float("inf")).all()) and not bool(lp[~seen].any())
    assert not bool(xbar.any()) and not bool(alphabar.any()) and not bool(betabar.any())
    want = glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta)
    row = int(seen.nonzero()[3])
    x[row, 5] = float("nan")
    got = glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta)
    rest = torch.arange(300, device="cuda") != row
    assert bool(torch.isnan(got[0][row])) and torch.equal(got[0][rest], want[0][rest])
    assert bool(torch.isnan(got[1][row]).all()) and torch.equal(got[1][rest], want[1][rest])


def test_class_empty(glm):
    for name, dtype in DTYPES.items():
        x, beta = torch.empty(0, 5, dtype=dtype, device="cuda"), torch.ones(7, 5, dtype=dtype, device="cuda")
        y, alpha = torch.empty(0, dtype=torch.int64, device="cuda"), torch.ones(7, dtype=dtype, device="cuda")
        lp, xbar, alphabar, betabar = glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta)
        assert lp.shape == (0,) and xbar.shape == (0, 5) and not bool(alphabar.any()) and not bool(betabar.any())
        assert glm.categorical_logit_glm_lpmf(y, x, alpha, beta).shape == (0,)


def test_class_gradient_against_differences(glm):
    y, x, alpha, beta = _class_data("f64", 40, 6, 9, 31, masked=0.2)
    w = torch.rand(40, dtype=torch.float64, device="cuda", generator=_rng(2))
    _, xbar, alphabar, betabar = glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta, lpbar=w)
    h = 1e-5
    g = _rng(3)
    for which, grad in enumerate((xbar, alphabar, betabar)):
        u = torch.randn(grad.shape, dtype=torch.float64, device="cuda", generator=g)
        u = u / u.norm()
        val = []
        for s in (h, -h):
            args = [x, alpha, beta]
            args[which] = args[which] + s * u
            val.append(float((w * glm.categorical_logit_glm_lpmf(y, *args)).sum()))
        # central differences: h^2 / 6 times the third derivative (of 40 rows, each below 10 here), and 2^-53 |sum| / h
        assert abs((val[0] - val[1]) / (2 * h) - float((grad * u).sum())) < 40 * 10 * h * h + 400 * 2.0**-52 / h


def test_host_arguments_are_taken_in_fp64(glm):
    import numpy as np

    rng = np.random.default_rng(0)
    x, beta, alpha = rng.normal(size=(4, 3)), rng.normal(size=(5, 3)), rng.normal(size=5)
    lp = glm.categorical_logit_glm_lpmf([0, 4, -1, 2], x, alpha, beta)
    eta = x @ beta.T + alpha
    want = eta - np.log(np.exp(eta).sum(1, keepdims=True))
    want = np.array([want[0, 0], want[1, 4], 0.0, want[3, 2]])
    assert lp.dtype == torch.float64 and float(np.abs(lp.cpu().numpy() - want).max()) < 64 * 2.0**-53 * (1 + np.abs(eta).max())
    y, mean, rstd = glm.layer_norm(x)
    assert y.dtype == torch.float64 and y.is_cuda and mean.shape == (4,)


# ---- as they are used --------------------------------------------------------------------------------------------------
def test_fields_to_classes_and_back(glm):
    """Fields from white noise, standardised, read out as classes: the log density's gradient with respect to the white noise
    through all four reverse modes, against differences."""
    from gptools_amd import fft

    g = _rng(41)
    d, h, w, v = 3, 12, 10, 6
    cov = fft.gp_periodic_matern_cov_rfft2(1.5, h, w, 1.3, [2.0, 3.0], [float(h), float(w)]) + 0.01
    z = torch.randn(d, h, w, generator=g, dtype=torch.float64, device="cuda")
    beta, alpha = _normal(g, (v, d), torch.float64), _normal(g, (v,), torch.float64)
    scale = _normal(g, (h, w), torch.float64, 0.1, 1.0)
    y = torch.randint(0, v, (h, w), generator=g, device="cuda")
    y[torch.rand(h, w, generator=g, device="cuda") < 0.2] = -1

    def density(z):
        f = fft.gp_inv_rfft2(z, 0.3, cov)
        s, mean, rstd = glm.layer_norm(f, scale, core_ndim=2)
        return f, s, mean, rstd, glm.categorical_logit_glm_lpmf(y, s.movedim(0, -1), alpha, beta).sum()

    f, s, mean, rstd, lp = density(z)
    lps, sbar, alphabar, betabar = glm.categorical_logit_glm_lpmf_vjp(y, s.movedim(0, -1), alpha, beta)
    assert abs(float(lps.sum() - lp)) <= 1e-12 * abs(float(lp))
    fbar, scalebar, _ = glm.layer_norm_vjp(f, scale, mean, rstd, sbar.movedim(-1, 0), core_ndim=2)
    zbar, _ = fft.gp_inv_rfft2_vjp(z, cov, fbar)
    u = torch.randn(z.shape, generator=g, dtype=torch.float64, device="cuda")
    u = u / u.norm()
    step = 1e-5
    slope = float(density(z + step * u)[-1] - density(z - step * u)[-1]) / (2 * step)
    # h^2 / 6 times the third derivative along a unit direction (120 sites, each term's below 10) and rounding over h
    assert abs(slope - float((zbar * u).sum())) < 120 * 10 * step**2 + abs(float(lp)) * 2.0**-48 / step
    up = torch.randn(h, w, generator=g, dtype=torch.float64, device="cuda")
    up = up / up.norm()
    vals = []
    for sgn in (step, -step):
        s2 = glm.layer_norm(f, scale + sgn * up, core_ndim=2)[0]
        vals.append(float(glm.categorical_logit_glm_lpmf(y, s2.movedim(0, -1), alpha, beta).sum()))
    assert abs((vals[0] - vals[1]) / (2 * step) - float((scalebar * up).sum())) < 120 * 10 * step**2 + abs(float(lp)) * 2.0**-48 / step


def _training_calls(glm, name, x, weight, bias, alpha, beta, y):
    s, mean, rstd = glm.layer_norm(x, weight, bias)
    lp, sbar, alphabar, betabar = glm.categorical_logit_glm_lpmf_vjp(y, s, alpha, beta, check=False)
    xbar, wbar, bbar = glm.layer_norm_vjp(x, weight, mean, rstd, sbar)
    return [lp, alphabar, betabar, xbar, wbar, bbar]


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("n,d,v", [(60, 16, 50), (150, 192, 1000), (1000, 128, 6500)])
def test_captured_and_replayed(glm, name, n, d, v):
    """A training step's calls in a graph, replayed on new data, with eager calls of other sizes in between; two graphs alive."""
    dtype = DTYPES[name]
    g = _rng(43)
    y, x, alpha, beta = _class_data(name, n, d, v, 47, masked=0.1)
    weight, bias = _normal(g, (d,), dtype, 0.1, 1.0), _normal(g, (d,), dtype, 0.1)
    args = (x, weight, bias, alpha, beta, y)
    _training_calls(glm, name, *args)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _training_calls(glm, name, *args)
        graphs.append((graph, out))
    other = _class_data(name, 333, d, 1500, 53)
    for i in range(4):
        x.copy_(_normal(g, (n, d), dtype))
        y.copy_(torch.randint(-1, v, (n,), generator=g, device="cuda"))
        want = [t.clone() for t in _training_calls(glm, name, *args)]
        glm.categorical_logit_glm_lpmf_vjp(*other)
        torch.cuda.synchronize()
        for graph, out in graphs if i % 2 else reversed(graphs):
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_on_another_stream(glm):
    y, x, alpha, beta = _class_data("bf16", 500, 128, 3000, 59)
    want = glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta)
    nwant = glm.layer_norm(x)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for s in streams:  # two calls at once, each with a workspace of its own
        with torch.cuda.stream(s):
            got.append((glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta, check=False), glm.layer_norm(x)))
    torch.cuda.synchronize()
    for c, n in got:
        assert all(torch.equal(a, b) for a, b in zip(c, want)) and all(torch.equal(a, b) for a, b in zip(n, nwant))


# ---- refusals ----------------------------------------------------------------------------------------------------------
def test_refusals(glm):
    from gptools_amd.fft import get_context

    x = torch.zeros(4, 6, device="cuda")
    beta, alpha, y = torch.zeros(5, 6, device="cuda"), torch.zeros(5, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    bad = [
        lambda: glm.layer_norm(x, weight=torch.zeros(5, device="cuda")),
        lambda: glm.layer_norm(x, bias=torch.zeros(6, device="cuda", dtype=torch.float64)),
        lambda: glm.layer_norm(x, core_ndim=0),
        lambda: glm.layer_norm(x, core_ndim=3),
        lambda: glm.layer_norm(x[:, :0]),
        lambda: glm.layer_norm(x, eps=-1.0),
        lambda: glm.layer_norm(x, eps=float("nan")),
        lambda: glm.layer_norm(x.int()),
        lambda: glm.layer_norm_vjp(x, None, torch.zeros(4, device="cuda"), torch.zeros(3, device="cuda"), x),
        lambda: glm.layer_norm_vjp(x, None, torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda").double(), x),
        lambda: glm.layer_norm_vjp(x, None, torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda"), x[:3]),
        lambda: glm.categorical_logit_glm_lpmf(y, x, alpha, beta[:, :5]),
        lambda: glm.categorical_logit_glm_lpmf(y, x, alpha, beta.half()),
        lambda: glm.categorical_logit_glm_lpmf(y, x, alpha, beta[:0]),
        lambda: glm.categorical_logit_glm_lpmf(y, x, alpha[:4], beta),
        lambda: glm.categorical_logit_glm_lpmf(y[:3], x, alpha, beta),
        lambda: glm.categorical_logit_glm_lpmf(y.double(), x, alpha, beta),
        lambda: glm.categorical_logit_glm_lpmf(y + 5, x, alpha, beta),
        lambda: glm.categorical_logit_glm_lpmf(y, x.half(), alpha, beta),
        lambda: glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta, lpbar=torch.zeros(3, device="cuda")),
        lambda: glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta, lpbar=torch.zeros(4, device="cuda").half()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("call", i, "went through")
    # the C entry points refuse too: nothing is launched
    ctx = get_context(x.device)
    p = [t.data_ptr() for t in (y, x, alpha, beta)]
    out = torch.zeros(64, device="cuda")
    need = glm._space("gpt_categorical_logit_glm_workspace", 1, 4, 6, 5, 1)
    ws = torch.zeros(need + 256, dtype=torch.uint8, device="cuda")
    vjp = ("gpt_categorical_logit_glm_lpmf_vjp", 1, p[0], p[1], 6, p[2], p[3], 6, None, 4, 6, 5, out.data_ptr(), out.data_ptr(),
           out.data_ptr(), out.data_ptr(), ws.data_ptr(), need)
    for at, value, error in [(1, 4, NotImplementedError), (1, -1, NotImplementedError), (2, None, ValueError), (3, None, ValueError),
                             (4, 5, ValueError), (6, None, ValueError), (7, 5, ValueError), (9, -1, ValueError), (9, 1 << 32, ValueError),
                             (10, 0, ValueError), (11, 0, ValueError), (12, None, ValueError), (13, None, ValueError),
                             (15, None, ValueError), (16, None, ValueError), (16, ws.data_ptr() + 8, ValueError),
                             (17, need - 1, ValueError)]:
        args = list(vjp)
        args[at] = value
        with pytest.raises(error):
            ctx.call(*args)
    many, sums = torch.zeros(3000, 6, device="cuda"), torch.zeros(3000, device="cuda")
    need = glm._space("gpt_layer_norm_workspace", 1, 3000, 6, 1)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    norm = ("gpt_layer_norm_vjp", 1, many.data_ptr(), None, sums.data_ptr(), sums.data_ptr(), many.data_ptr(), 3000, 6, sums.data_ptr(),
            sums.data_ptr(), sums.data_ptr(), ws.data_ptr(), need)
    assert need > 0
    for at, value, error in [(1, 9, NotImplementedError), (2, None, ValueError), (4, None, ValueError), (6, None, ValueError),
                             (7, -1, ValueError), (8, 0, ValueError), (9, None, ValueError), (10, None, ValueError),
                             (11, None, ValueError), (12, None, ValueError), (13, 0, ValueError)]:
        args = list(norm)
        args[at] = value
        with pytest.raises(error):
            ctx.call(*args)
    torch.cuda.synchronize()
    assert not bool(out.any()) and not bool(sums.any())
