"""CPU-only: what the read-out operators say without a GPU -- workspace sizes (host arithmetic), argument checks."""
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from gptools_amd import _lib

    return _lib.load()


@pytest.mark.parametrize("dtype", range(4))
def test_workspace_sizes(lib, dtype):
    norm, glm = lib.gpt_layer_norm_workspace, lib.gpt_categorical_logit_glm_workspace
    for bad in [(-1, 5), (0, 5), (5, 0), (1 << 31, 5), (5, 1 << 41)]:
        assert norm(dtype, *bad, 1) == 0
    for bad in [(0, 5, 5), (5, 0, 5), (5, 5, 0), (-1, 5, 5), (1 << 31, 5, 5), (5, 1 << 22, 5), (5, 5, (1 << 31) - 1)]:
        assert glm(dtype, *bad, 1) == 0
    assert norm(dtype, 1, 64, 0) == 0 and norm(dtype, 1, 64, 1) == 0 and norm(dtype, 10000, 64, 1) > 0
    assert glm(dtype, 1, 1, 1, 1) > glm(dtype, 1, 1, 1, 0) >= 0 and glm(dtype, 100, 100, 100, 1) > glm(dtype, 100, 100, 100, 0) > 0
    # the logits are not in it: 4096 rows of 128000 classes would take 2 GiB in fp32 (a copy of beta may be, 6 bytes a value in fp32)
    assert glm(dtype, 4096, 512, 128000, 0) < 512 << 20
    # r, for a piece of the classes and a block of the rows, is bounded; the rest grows with the rows or with the classes
    for rows in (1, 100, 4096, 100000, 1 << 20, 1 << 24):
        assert glm(dtype, rows, 64, 1000, 1) < (4 << 30)
    assert norm(9, 4, 4, 1) == 0 and glm(9, 4, 4, 4, 1) == 0


def test_null_context_is_refused(lib):
    assert lib.gpt_layer_norm(None, 1, None, None, None, 1, 1, 0.0, None, None, None, None, 0) == 2
    assert lib.gpt_layer_norm_vjp(None, 1, None, None, None, None, None, 1, 1, None, None, None, None, 0) == 2
    assert lib.gpt_categorical_logit_glm_lpmf(None, 1, None, None, 1, None, None, 1, 1, 1, 1, None, None, 0) == 2
    assert lib.gpt_categorical_logit_glm_lpmf_vjp(None, 1, None, None, 1, None, None, 1, None, 1, 1, 1, None, None, None, None,
                                                  None, 0) == 2


def test_shapes_without_a_gpu():
    from gptools_amd import glm

    x = torch.zeros(4, 3, 5)
    assert glm._core(x, 1) == ((4, 3), (5,), 5) and glm._core(x, 2) == ((4,), (3, 5), 15) and glm._core(x, 3) == ((), (4, 3, 5), 60)
    for bad in (0, 4, -1):
        with pytest.raises(ValueError):
            glm._core(x, bad)
    with pytest.raises(ValueError):
        glm._core(x[..., :0], 1)
    m, ld = glm._matrix(x)
    assert m.shape == (12, 5) and ld == 5
    m, ld = glm._matrix(torch.zeros(6, 9)[:, 2:7])
    assert m.shape == (6, 5) and ld == 9
    m, ld = glm._matrix(torch.zeros(5, 6).T)
    assert m.is_contiguous() and ld == 5
    m, ld = glm._matrix(torch.zeros(1, 5).expand(6, 5))
    assert m.is_contiguous() and ld == 5
    for kw in (dict(shape=(3,)), dict(dtype=torch.float64)):
        with pytest.raises(ValueError, match="weight"):
            glm._alike("weight", torch.zeros(5), kw.get("shape", (5,)), kw.get("dtype", torch.float32), torch.device("cpu"))


@pytest.mark.parametrize("dtype,size,acc", [(0, 8, 8), (1, 4, 4), (2, 2, 4), (3, 2, 4)])
@pytest.mark.parametrize("rows", [1, 20, 64, 65, 3000])
def test_workspace_per_row_and_class_is_bounded(lib, dtype, size, acc, rows):
    """1.5 GB of logits and r, however many classes there are; beside it a maximum and a sum for every row and 128 classes (up to 64 rows: 64, 32 in
    fp64), in fp32 three planes of beta, and what does not grow with the classes (transposes of a piece, sums for xbar)."""
    features = 64
    tile = 128 if rows > 64 else 32 if size == 8 else 64
    for classes in (1 << 20, 1 << 22, 1 << 24, 1 << 26):
        rest = 2 * acc * rows * (classes // tile + 1) + (6 * features * (classes + 64) if size == 4 else 0) + (256 << 20)
        assert lib.gpt_categorical_logit_glm_workspace(dtype, rows, features, classes, 1) <= (3 << 29) + rest


@pytest.mark.parametrize("dtype", range(4))
@pytest.mark.parametrize("rows", [20000, 1 << 20, 1 << 28])
def test_few_features_take_one_number_a_row(lib, dtype, rows):
    """The log density of many rows needs their order, a count for every 4096 of them and one in all, in pieces of 256 bytes."""
    assert lib.gpt_categorical_logit_glm_workspace(dtype, rows, 8, 300, 0) <= 4 * rows + 4 * (rows // 4096 + 1) + 3 * 256
