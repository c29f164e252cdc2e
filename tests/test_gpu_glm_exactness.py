"""
Where the read-out of several latent fields (gptools_amd.glm) loses digits by cancellation, or a whole value: rows whose class is
predicted with confidence, probabilities far below the likeliest class's, a level common to all classes, infinite coefficients,
the largest calls. Inputs, formulas and bounds are those of test_gpu_glm.py unless a test says otherwise.
"""
import pytest
import torch

from test_gpu_glm import DTYPES, _check_class, _class_data, _class_want, _eps, _normal, _rng, _wide, glm  # noqa: F401

pytestmark = pytest.mark.gpu


def _towards(name, n, d, v, sure, seed):
    """Rows that lean towards their class, as a fitted model's do: x = t beta_y + noise, with the first t of a geometric series at
    which the median probability of the rows' classes reaches `sure`. beta's rows have length 1."""
    dtype = DTYPES[name]
    g = _rng(seed)
    beta = torch.randn(v, d, generator=g, device="cuda", dtype=torch.float64)
    beta = (beta / beta.norm(dim=1, keepdim=True)).to(dtype)
    y = torch.randint(0, v, (n,), generator=g, device="cuda")
    noise = 0.3 * torch.randn(n, d, generator=g, device="cuda", dtype=torch.float64)
    some = slice(0, 256)
    for k in range(60):
        x = (1.2**k * beta.double()[y] + noise).to(dtype)
        eta = x[some].double() @ beta.double().T
        p = torch.softmax(eta, 1).gather(1, y[some].unsqueeze(1))
        if float(p.median()) >= sure:
            break
    return y, x, beta


# rows: for which the workgroups' waves share a row's classes, and so many that a wave has rows of its own
SURE = [(150, 8, 300), (150, 32, 70), (300, 64, 300), (150, 32, 1000), (1000, 32, 4000), (66000, 32, 300), (66000, 64, 70)]


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("n,d,v", SURE)
@pytest.mark.parametrize("sure", [0.5, 0.9, 0.99])
def test_rows_predicted_with_confidence(glm, name, n, d, v, sure):
    """xbar is about (1 - p_y) beta there: a probability's rounding to the element type, taken for y's as well, would be as large."""
    y, x, beta = _towards(name, n, d, v, sure, seed=n + d + v)
    alpha = _normal(_rng(1), (v,), DTYPES[name], 0.1)
    y[::7] = -1
    lpbar = 0.5 + torch.rand(n, generator=_rng(2), device="cuda", dtype=_wide(DTYPES[name]))
    _check_class(glm, name, y, x, alpha, beta, lpbar)


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("n,d,v", [(150, 32, 1000), (66000, 8, 1000), (30, 100, 1000), (300, 100, 1000)])
@pytest.mark.parametrize("lead", [8.0, 14.0, 17.5])
def test_probabilities_far_below_the_likeliest(glm, name, n, d, v, lead):
    """One class `lead` above all others, which alone have a coefficient: xbar is minus the sum of many small probabilities."""
    dtype, wide = DTYPES[name], _wide(DTYPES[name])
    x = torch.zeros(n, d, dtype=dtype, device="cuda")
    for likely in (0, v // 2):
        beta = torch.zeros(v, d, dtype=dtype, device="cuda")
        beta[:, 0] = 1
        beta[likely, 0] = 0
        alpha = torch.zeros(v, dtype=dtype, device="cuda")
        alpha[likely] = lead
        y = torch.full((n,), likely, dtype=torch.int64, device="cuda")
        lpbar = torch.full((n,), 1000.0, dtype=wide, device="cuda")
        xbar = glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta, lpbar=lpbar)[1]
        p = torch.softmax(alpha.double(), 0)
        want = -1000.0 * float(p.sum() - p[likely])
        # a half step of the element type for r or p, one for the result; the exponential of `lead`, v additions; in fp16 what is
        # stored times 2^13 at least is off by half of its smallest step 2^-24 besides
        rel = 2 * (_eps(dtype) / 2) * 1.01 + (4 * lead + v + 16) * _eps(wide)
        off = v * 1000.0 * 2.0**-38 + 2.0**-25 if name == "f16" else 0.0
        assert not bool(xbar[:, 1:].any())
        assert float((xbar[:, 0].double() - want).abs().max()) <= rel * abs(want) + off


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("n,d,v", [(60, 16, 70), (66, 17, 70), (100, 64, 300), (66000, 20, 70), (64, 65, 700), (65, 65, 700), (300, 128, 3000),
                                   (700, 100, 9000)])
def test_classes_excluded_by_their_coefficients(glm, name, n, d, v):
    """An intercept column of ones whose coefficient is -inf for some classes: their probability is zero, at all sizes alike."""
    dtype = DTYPES[name]
    g = _rng(n + d + v)
    x, beta = _normal(g, (n, d), dtype), _normal(g, (v, d), dtype, 1.5 / d**0.5)
    x[:, 0] = 1
    out = torch.zeros(v, dtype=torch.bool, device="cuda")
    out[1::3] = True
    y = torch.randint(0, v // 3, (n,), generator=g, device="cuda") * 3
    finite = beta.clone()
    finite[out, 0] = 0
    beta[out, 0] = -float("inf")
    alpha = torch.where(out, -float("inf"), 0.0).to(dtype)
    want = glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, finite)  # (tested elsewhere)
    want_lp = glm.categorical_logit_glm_lpmf(y, x, alpha, finite)
    lp = glm.categorical_logit_glm_lpmf(y, x, None, beta)
    got = glm.categorical_logit_glm_lpmf_vjp(y, x, torch.zeros_like(alpha), beta)
    # the same products, with zeros for the excluded classes' probabilities. (xbar's first column holds 0 times -inf)
    assert torch.equal(lp, want_lp) and torch.equal(got[0], want[0])
    assert torch.equal(got[1][:, 1:], want[1][:, 1:])
    assert torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])
    # both infinite, and an infinity times zero: as in any product
    x[2, 0], x[3, 0] = float("inf"), 0
    lp = glm.categorical_logit_glm_lpmf(y, x, None, beta)
    assert bool(torch.isnan(lp[3])) and torch.equal(lp[4:], want_lp[4:])


@pytest.mark.parametrize("name", list(DTYPES))
@pytest.mark.parametrize("n,d,v", [(1, 1000, 40), (40, 100, 2000), (64, 4096, 500), (17, 200, 40000), (150, 32, 300), (150, 8, 70),
                                   (66000, 64, 70), (66000, 8, 300), (300, 100, 700), (700, 256, 9000)])
def test_log_probabilities_are_at_most_zero(glm, name, n, d, v):
    """The logit of a row's class is the one that the sum over the classes holds, not another rounding of it."""
    y, x, beta = _towards(name, n, d, v, 0.999999, seed=n + d + v)
    alpha = _normal(_rng(4), (v,), DTYPES[name], 0.1)
    for al in (None, alpha):
        assert bool((glm.categorical_logit_glm_lpmf(y, x, al, beta) <= 0).all())
        assert bool((glm.categorical_logit_glm_lpmf_vjp(y, x, al, beta)[0] <= 0).all())


@pytest.mark.parametrize("name", ["f64", "f32"])
@pytest.mark.parametrize("n,d,v", [(40, 100, 2000), (300, 8, 300), (300, 40, 77), (66000, 8, 300), (300, 100, 700), (600, 100, 24680)])
@pytest.mark.parametrize("level", [0.0, 1024.0, -1024.0])
def test_a_level_common_to_all_classes(glm, name, n, d, v, level):
    """It cancels in the probabilities, which are 1 / v here, and may not cost them digits."""
    dtype, ea = DTYPES[name], _eps(DTYPES[name])
    x = torch.zeros(n, d, dtype=dtype, device="cuda")
    x[:, 0] = 1
    beta = torch.zeros(v, d, dtype=dtype, device="cuda")
    beta[:, 1] = 1  # (x is zero there)
    alpha = torch.full((v,), level, dtype=dtype, device="cuda")
    y = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    y[7:27] = 3
    lp, xbar, alphabar, betabar = glm.categorical_logit_glm_lpmf_vjp(y, x, alpha, beta)
    want = torch.full((v,), -20.0 / v, dtype=torch.float64, device="cuda")
    want[3] += 20
    # the logits are all equal, their exponentials about the largest are 1 and add up to v exactly; 1 / v, the product and the
    # difference are rounded, and 20 additions of them
    assert bool(((alphabar.double() - want).abs() <= 24 * ea * want.abs()).all())
    assert bool(((betabar[:, 0].double() - want).abs() <= 24 * ea * want.abs()).all())
    # one entry of size 1, v of 1 / v and their sum in any order
    assert float(xbar[:, 1].abs().max()) <= (v + 8) * ea


@pytest.mark.parametrize("name,v", [("f64", 1 << 20), ("bf16", 2100001)])
def test_more_tiles_than_a_grid_counts_threads(glm, name, v):
    """Rows x classes whose tiles have more threads than a grid's first dimension counts (2^32)."""
    n, d = 1 << 18, 65
    y, x, alpha, beta = _class_data(name, n, d, v, 3)
    lp = glm.categorical_logit_glm_lpmf(y, x, alpha, beta)
    ea = _eps(_wide(DTYPES[name]))
    for at in (0, n // 2 + 3, n - 50):
        some = slice(at, at + 50)
        xd, bd, eta, lse, want, *_ = _class_want(y[some], x[some], alpha, beta, None, y[some] >= 0)
        # as in _check_class
        de = (d + 2) * ea * (xd.abs() @ bd.abs().T + eta.abs()) + 4 * ea * (eta.abs() + lse.abs().unsqueeze(1))
        tol = 2 * de.max(1).values + (96 + v / 2048) * ea + 2 * ea * (lse.abs() + want.abs())
        assert bool(((lp[some].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("name,n,d,v", [("f64", 64, 66, 1100001), ("f64", 3, 66, 6000001), ("f32", 64, 71, 2200001), ("f16", 50, 72, 3900001),
                                        ("bf16", 64, 67, 3200001)])
def test_few_rows_of_very_many_classes(glm, name, n, d, v):
    """So many that the logits and r of all classes at once would be more than is held per row and class."""
    y, x, alpha, beta = _class_data(name, n, d, v, 5)
    y[n // 3] = -1
    x[n // 3] = float("nan")
    _check_class(glm, name, y, x, alpha, beta)
