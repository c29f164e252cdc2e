"""
Where the read-out of several latent fields (gptools_amd.glm) loses digits by cancellation, or a whole value: rows whose class is
predicted with confidence, probabilities far below the likeliest class's, a level common to all classes, infinite coefficients,
the largest calls. Inputs, formulas and bounds are those of test_gpu_glm.py unless a test says otherwise.
"""
import pytest
import torch

from test_gpu_glm import DTYPES, _check_class, _class_want, _eps, _normal, _rng, _wide, glm  # noqa: F401

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
