"""
Read-out of several latent fields: standardisation and the log probability of observed classes.

A model with classes as data (species, land-cover types) reads them off several Gaussian-process fields at each site. The
fields come from :func:`gptools_amd.fft.gp_inv_rfft2`; each is standardised over its lattice (:func:`layer_norm` with
``core_ndim=2``: its level and scale are confounded with ``alpha`` and ``beta``), and the classes' log odds at a site are linear
in the fields' values there (:func:`categorical_logit_glm_lpmf`, Stan's function of that name, row by row). The ``_vjp``
functions are the reverse modes; those of the chain end in :func:`gptools_amd.fft.gp_inv_rfft2_vjp`.

Device tensors in fp64, fp32, fp16 or bf16 (all floating arguments of a call alike), results in the same type; statistics,
log probabilities and their cotangents are fp32, or fp64 for fp64 data. Other arguments (NumPy arrays, lists, host tensors)
are taken to the GPU in fp64, as in :mod:`gptools_amd.fft`. Every call runs on torch's current stream, takes its workspace from
torch's allocator and may be captured into a graph (``check=False`` where a function has that argument: the check waits for the
GPU). The same call on the same data gives the same bits.
"""
from __future__ import annotations

import functools
import math

import numpy as np
import torch

from . import _lib
from .fft import get_context

_TYPES = {torch.float64: _lib.GPT_F64, torch.float32: _lib.GPT_F32, torch.float16: _lib.GPT_F16,
          torch.bfloat16: _lib.GPT_BF16}


def _given(x, like=None):
    """A device tensor of a supported type as it is; anything else as fp64 on the GPU."""
    if isinstance(x, torch.Tensor) and x.is_cuda:
        if x.dtype not in _TYPES:
            raise ValueError(f"unsupported type {x.dtype}: expected float64, float32, float16 or bfloat16")
        return x
    device = like.device if like is not None else torch.device("cuda", torch.cuda.current_device())
    if isinstance(x, torch.Tensor):
        return x.to(device, torch.float64)
    return torch.as_tensor(np.asarray(x, dtype=np.float64)).to(device)


def _alike(what, t, shape, dtype, device):
    if t.shape != shape:
        raise ValueError(f"{what} has shape {tuple(t.shape)}; expected {tuple(shape)}")
    if t.dtype is not dtype:
        raise ValueError(f"{what} has type {t.dtype}; expected {dtype}")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}; expected {device}")
    return t.contiguous()


def _at(t):
    return None if t is None else t.data_ptr()


def _wide(dtype):
    return torch.float64 if dtype is torch.float64 else torch.float32


@functools.lru_cache(maxsize=1024)
def _space(name, *sizes):
    return getattr(_lib.load(), name)(*sizes)


def _workspace(device, name, *sizes):
    n = _space(name, *sizes)
    return (torch.empty(n, dtype=torch.uint8, device=device) if n else None), n


def _core(x, core_ndim):
    if core_ndim < 1 or x.ndim < core_ndim:
        raise ValueError(f"core_ndim must lie between 1 and the number of dimensions of x ({x.ndim})")
    shape = tuple(x.shape)
    core = shape[x.ndim - core_ndim:]
    width = math.prod(core)
    if width < 1:
        raise ValueError("layer norm needs at least one value in a row")
    return shape[: x.ndim - core_ndim], core, width


def layer_norm(x, weight=None, bias=None, eps=1e-5, core_ndim=1):
    """Standardise over the last ``core_ndim`` dimensions (1: the features of a site; 2: a whole lattice):
    ``y = (x - mean) * rstd * weight + bias`` with ``rstd = 1 / sqrt(var + eps)``, ``var`` the mean squared deviation.
    ``weight`` and ``bias`` have the shape of these dimensions. Returns ``(y, mean, rstd)``; ``mean`` and ``rstd`` (fp32, or
    fp64 for fp64 data) have the leading dimensions' shape and are what :func:`layer_norm_vjp` takes."""
    x = _given(x).contiguous()
    bshape, core, width = _core(x, core_ndim)
    if weight is not None:
        weight = _alike("weight", _given(weight, x), core, x.dtype, x.device)
    if bias is not None:
        bias = _alike("bias", _given(bias, x), core, x.dtype, x.device)
    rows = math.prod(bshape)
    y = torch.empty_like(x)
    mean, rstd = torch.empty((2, *bshape), dtype=_wide(x.dtype), device=x.device).unbind(0)
    kind = _TYPES[x.dtype]
    ws, n = _workspace(x.device, "gpt_layer_norm_workspace", kind, rows, width, 0)
    get_context(x.device).call("gpt_layer_norm", kind, x.data_ptr(), _at(weight), _at(bias), rows, width, eps, y.data_ptr(),
                               mean.data_ptr(), rstd.data_ptr(), _at(ws), n)
    return y, mean, rstd


def layer_norm_vjp(x, weight, mean, rstd, ybar, core_ndim=1, need_param_grad=True):
    """Reverse mode of :func:`layer_norm` from its ``mean`` and ``rstd``: ``ybar -> (xbar, weightbar, biasbar)``. The gradients of
    ``weight`` and ``bias`` are summed over all leading dimensions (``None`` with ``need_param_grad=False``)."""
    x = _given(x).contiguous()
    bshape, core, width = _core(x, core_ndim)
    if weight is not None:
        weight = _alike("weight", _given(weight, x), core, x.dtype, x.device)
    ybar = _alike("ybar", _given(ybar, x), x.shape, x.dtype, x.device)
    wide = _wide(x.dtype)
    mean = _alike("mean", _given(mean, x), bshape, wide, x.device)
    rstd = _alike("rstd", _given(rstd, x), bshape, wide, x.device)
    rows = math.prod(bshape)
    xbar = torch.empty_like(x)
    wbar = bbar = None
    if need_param_grad:
        wbar, bbar = torch.empty((2, *core), dtype=x.dtype, device=x.device).unbind(0)
    kind = _TYPES[x.dtype]
    ws, n = _workspace(x.device, "gpt_layer_norm_workspace", kind, rows, width, 1)
    get_context(x.device).call("gpt_layer_norm_vjp", kind, x.data_ptr(), _at(weight), mean.data_ptr(), rstd.data_ptr(),
                               ybar.data_ptr(), rows, width, xbar.data_ptr(), _at(wbar), _at(bbar), _at(ws), n)
    return xbar, wbar, bbar


def _matrix(t):
    """Two-dimensional with the last dimension contiguous, and the distance of its rows (a slice of wider rows is taken as it is)."""
    if t.ndim != 2:
        t = t.reshape(-1, t.shape[-1])
    rows, cols = t.shape
    ld, one = t.stride()
    if rows > 1 and one == 1 and ld >= cols:
        return t, ld
    return t.contiguous(), cols


def _glm(y, x, alpha, beta, check):
    x = _given(x)
    beta = _given(beta, x)
    shape = tuple(x.shape)
    if not shape or beta.ndim != 2 or beta.shape[1] != shape[-1] or beta.numel() == 0:
        raise ValueError(f"x has shape {tuple(x.shape)} and beta {tuple(beta.shape)}; expected (..., features) and (classes, features)")
    if beta.dtype is not x.dtype or beta.device != x.device:
        raise ValueError(f"beta is {beta.dtype} on {beta.device}; expected {x.dtype} on {x.device}")
    bshape = shape[:-1]
    if alpha is not None:
        alpha = _alike("alpha", _given(alpha, x), (beta.shape[0],), x.dtype, x.device)
    if not isinstance(y, torch.Tensor):
        y = torch.as_tensor(np.asarray(y))
    if y.dtype is not torch.int64 and y.dtype not in (torch.int32, torch.int16, torch.int8):
        raise ValueError(f"y has type {y.dtype}; expected integers")
    if y.shape != bshape:
        raise ValueError(f"y has shape {tuple(y.shape)}; expected {bshape}")
    if y.is_cuda and y.device != x.device:
        raise ValueError(f"y is on {y.device}; expected {x.device}")
    y = (y if y.is_cuda and y.dtype is torch.int64 else y.to(x.device, torch.int64)).contiguous()
    if check and y.numel():
        most = int(y.max())
        if most >= beta.shape[0]:
            raise ValueError(f"y holds class {most}; there are {beta.shape[0]}, counted from 0")
    return y, x, alpha, beta, bshape


def categorical_logit_glm_lpmf(y, x, alpha, beta, check=True):
    """Log probability of the class ``y`` of each row of ``x`` (Stan's ``categorical_logit_glm_lpmf``, not summed):
    ``eta[v] = alpha[v] + beta[v] . x``, ``lp = eta[y] - log(sum(exp(eta)))``. ``x`` is ``(..., features)``, ``y`` has its leading
    dimensions, ``beta`` is ``(classes, features)``, ``alpha`` ``(classes,)`` or ``None``. Classes count from 0; a negative ``y`` is a
    row without an observation (``lp = 0``; that row of ``x`` may hold anything). An ``alpha`` of ``-inf`` excludes a class. The
    matrix of logits is never stored. ``check``: refuse a ``y`` that is no class (waits for the GPU); without it such a row is NaN."""
    y, x, alpha, beta, bshape = _glm(y, x, alpha, beta, check)
    xm, ldx = _matrix(x)
    bm, ldb = _matrix(beta)
    rows, (classes, features) = xm.shape[0], beta.shape
    lp = torch.empty(bshape, dtype=_wide(x.dtype), device=x.device)
    kind = _TYPES[x.dtype]
    ws, n = _workspace(x.device, "gpt_categorical_logit_glm_workspace", kind, rows, features, classes, 0)
    get_context(x.device).call("gpt_categorical_logit_glm_lpmf", kind, y.data_ptr(), xm.data_ptr(), ldx, _at(alpha),
                               bm.data_ptr(), ldb, rows, features, classes, lp.data_ptr(), ws.data_ptr() if n else None, n)
    return lp


def categorical_logit_glm_lpmf_vjp(y, x, alpha, beta, lpbar=None, check=True):
    """:func:`categorical_logit_glm_lpmf` and its reverse mode in one call: ``(lp, xbar, alphabar, betabar)`` for the cotangent
    ``lpbar`` of the log probabilities (``None``: ones, the gradients of their sum). ``alphabar`` and ``betabar`` are summed over all
    leading dimensions (``alphabar`` is ``None`` where ``alpha`` is). A row without an observation has no gradient. The classes are
    taken in pieces: what is held per row and class (logits and their gradients) stays below 1.61 GB (1.5 * 2**30), however many there are,
    and a maximum and a sum for every row and 128 or 256 classes (up to 64 rows: 16 to 64) beside it."""
    y, x, alpha, beta, bshape = _glm(y, x, alpha, beta, check)
    xm, ldx = _matrix(x)
    bm, ldb = _matrix(beta)
    rows, (classes, features) = xm.shape[0], beta.shape
    wide = _wide(x.dtype)
    if lpbar is not None:
        lpbar = _alike("lpbar", _given(lpbar, x), bshape, wide, x.device)
    lp = torch.empty(bshape, dtype=wide, device=x.device)
    xbar = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    alphabar = None if alpha is None else torch.empty(classes, dtype=x.dtype, device=x.device)
    betabar = torch.empty((classes, features), dtype=x.dtype, device=x.device)
    kind = _TYPES[x.dtype]
    ws, n = _workspace(x.device, "gpt_categorical_logit_glm_workspace", kind, rows, features, classes, 1)
    get_context(x.device).call("gpt_categorical_logit_glm_lpmf_vjp", kind, y.data_ptr(), xm.data_ptr(), ldx, _at(alpha),
                               bm.data_ptr(), ldb, _at(lpbar), rows, features, classes, lp.data_ptr(), xbar.data_ptr(),
                               _at(alphabar), betabar.data_ptr(), ws.data_ptr() if n else None, n)
    return lp, xbar, alphabar, betabar
