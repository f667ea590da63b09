"""Operators of a graph network's training step around the aggregation.

- ``group_norm``: group norm with its activation over channels-last features,
  the layout that the aggregation writes (rows of nodes, channels last);
- ``linear_cross_entropy``: the softmax cross entropy of a linear classifier,
  over many classes without the logits in memory, with its gradients;
- ``orthogonalize``: an update matrix orthogonalised by Newton-Schulz products,
  the step of ``mask_amd.optim.OrthogonalMomentum``.

Hand-written gfx950 kernels behind the C ABI (include/srbcrs.h); torch
supplies memory, the current stream and autograd.  Tensors are float32,
bfloat16 or float16 on one GPU; sums and statistics are 32 bits.  There is no
other implementation: a host tensor raises.  No reference counterparts.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import _capi
from .SRBCRSSpMM import _raw_stream

Tensor = torch.Tensor

__all__ = ["group_norm", "linear_cross_entropy", "orthogonalize"]

_DTYPE = {torch.float32: _capi.DTYPE_CODES["float32"], torch.bfloat16: _capi.DTYPE_CODES["bfloat16"],
          torch.float16: _capi.DTYPE_CODES["float16"]}


def _check(t: Tensor, name: str, like: Optional[Tensor] = None) -> None:
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dtype not in _DTYPE:
        raise TypeError(f"{name} must be float32, bfloat16 or float16")
    if like is not None and t.device != like.device:
        raise RuntimeError(f"{name} is on {t.device}, expected {like.device}")


class _on_device:
    """The tensor's device current, without a device context where it is."""

    def __new__(cls, t: Tensor):
        return _HERE if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


class _Here:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def _like(t: Tensor) -> Tensor:
    """Memory for a contiguous tensor like t."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _dense(t: Optional[Tensor]) -> Optional[Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _workspace(n: int, like: Tensor) -> Optional[Tensor]:
    return torch.empty(n, dtype=torch.uint8, device=like.device) if n > 1 else None


# Descriptions and workspace sizes by shape, type and strides: both follow from
# these alone, and asking the library again costs as much as a small launch.
_PLANS: dict = {}


def _plan(key, make, size):
    """(description's address, workspace bytes) of a call with this key."""
    got = _PLANS.get(key)
    if got is None:
        if len(_PLANS) >= 1024:
            _PLANS.clear()
        desc = make()
        ref = ctypes.byref(desc)
        n = ctypes.c_size_t(0)
        _capi.check(size(ref, ctypes.byref(n)))
        got = _PLANS[key] = (ref, n.value)
    return got


def _once(backward):
    """A backward pass without a derivative of its own: refused when one is asked for.  The
    wrapper that does so costs as much as a launch, so it is there only where the pass runs with gradients enabled."""
    checked = torch.autograd.function.once_differentiable(backward)
    return staticmethod(lambda ctx, g: checked(ctx, g) if torch.is_grad_enabled() else backward(ctx, g))


# Hooks of saved tensors may give them back in another layout (save_on_cpu makes slices dense).  The
# forward pass notes what its features are, and a backward pass that gets others describes them anew.  What is
# looked at is kept short: on the engine's thread each of these costs a part of a launch.

def _kind(t: Tensor):
    return t.shape, t.stride(), t.dtype, t.is_cuda


def _same_values(t: Tensor, kind) -> None:
    """Raises where a saved tensor is not what it was but for its layout."""
    if (t.shape, t.dtype, t.is_cuda) != (kind[0], kind[2], kind[3]):
        raise RuntimeError(f"a saved tensor came back as {tuple(t.shape)}, {t.dtype} on {t.device}")


# ---- group norm ---------------------------------------------------------------

def _rows(t: Tensor):
    """(tensor, batch stride, row stride) of (batch, ..., channels) features with the
    dimensions between as rows one stride apart; a copy where they are not."""
    if t.dim() == 2:
        if t.stride(1) == 1 or t.shape[1] == 1:
            return t, t.stride(0), t.shape[1]
    elif t.stride(-1) == 1 or t.shape[-1] == 1:
        ld, ok, span = None, True, None
        for d in range(t.dim() - 2, 0, -1):
            if t.shape[d] == 1:
                continue
            if ld is None:
                ld = span = t.stride(d)
            ok = ok and t.stride(d) == span
            span *= t.shape[d]
        if ok:
            return t, t.stride(0), t.shape[-1] if ld is None else ld
    t = t.contiguous()
    rows = 1
    for d in range(1, t.dim() - 1):
        rows *= t.shape[d]
    return t, rows * t.shape[-1], t.shape[-1]


def _norm_plan(x, xs, dys, groups, params, eps, act, backward):
    key = (0, x.shape, xs, dys, x.dtype, groups, None if params is None else params.dtype, eps, act, backward)

    def make():
        length = 1
        for d in range(1, x.dim() - 1):
            length *= x.shape[d]
        return _capi.NormDesc(x.shape[0], length, x.shape[-1], groups, *xs, *dys, _DTYPE[x.dtype],
                              _DTYPE[params.dtype] if params is not None else 0, act, eps)

    return _plan(key, make, lambda d, n: _capi.lib().srbcrs_group_norm_workspace(d, backward, n))


def _norm_forward(x, sb, ld, weight, bias, groups, eps, act):
    with _on_device(x):
        desc, n = _norm_plan(x, (sb, ld), (0, 0), groups, weight if weight is not None else bias, eps, act, 0)
        y = _like(x)
        stats = torch.empty((x.shape[0], groups, 4), dtype=torch.float32, device=x.device)
        ws = _workspace(n, x)
        _capi.check(_capi.lib().srbcrs_group_norm(
            desc, x.data_ptr(), _capi.ptr(weight), _capi.ptr(bias), y.data_ptr(), stats.data_ptr(), _capi.ptr(ws), n,
            _raw_stream(x.device.index)))
    return y, stats


def _norm_backward(ctx, dy):
    # the engine runs this on the device and the stream of the forward pass
    x, weight, bias, stats = ctx.saved_tensors
    groups, eps, act, xs, (desc, n) = ctx.args
    weight, bias, stats = _dense(weight), _dense(bias), _dense(stats)
    same = _kind(x) == ctx.kind
    if not same:
        _same_values(x, ctx.kind)
        x, *xs = _rows(x)
    if not same or not dy.is_contiguous():
        dy, dsb, dld = _rows(dy)
        desc, n = _norm_plan(x, tuple(xs), (dsb, dld), groups, weight if weight is not None else bias, eps, act, 1)
    dx = _like(x)
    dw = _like(weight) if weight is not None and ctx.needs_input_grad[1] else None
    db = _like(bias) if bias is not None and ctx.needs_input_grad[2] else None
    ws = _workspace(n, x)
    _capi.check(_capi.lib().srbcrs_group_norm_backward(
        desc, dy.data_ptr(), x.data_ptr(), _capi.ptr(weight), _capi.ptr(bias), stats.data_ptr(),
        dx.data_ptr(), _capi.ptr(dw), _capi.ptr(db), _capi.ptr(ws), n, _raw_stream(x.device.index)))
    return dx, dw, db, None, None, None


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        x, sb, ld = _rows(x)
        y, stats = _norm_forward(x, sb, ld, weight, bias, groups, eps, act)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.kind = _kind(x)
        # the description for a contiguous gradient, found here: the backward pass's thread is the slower one
        ctx.args = (groups, eps, act, (sb, ld), _norm_plan(x, (sb, ld), (y.stride(0), y.shape[-1]), groups,
                                                           weight if weight is not None else bias, eps, act, 1))
        return y

    backward = _once(_norm_backward)


def group_norm(x: Tensor, num_groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
               eps: float = 1e-5, activation: str = "none") -> Tensor:
    """``activation((x - mean) / sqrt(var + eps) * weight + bias)`` of features
    ``x`` (samples, ..., channels), channels last: mean and biased variance over
    all rows of a sample and the ``channels / num_groups`` consecutive channels of a
    group.  With two dimensions every row is a sample; a whole graph as one sample is
    ``x.unsqueeze(0)``.

    ``activation``: "none", "relu", "silu" or "gelu" (the exact one).  ``weight`` and
    ``bias`` have one value a channel, of x's type or another of the three.  Any
    strides; rows that are not one stride apart, or channels that are not next to
    each other, are copied first.  The result is contiguous.  Differentiable once in
    x, weight and bias.

    Elements are computed in 32 bits (gelu to a few 2^-24 of itself, in its negative
    tail as far as exp is), sums are joined in 64, results rounded once."""
    _check(x, "x")
    if x.dim() < 2:
        raise ValueError("x must have samples, and channels last: at least two dimensions")
    channels = x.shape[-1]
    groups = int(num_groups)
    if groups < 1 or channels % groups:
        raise ValueError(f"{channels} channels do not split into {num_groups} groups")
    if activation not in _capi.ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r} ({', '.join(_capi.ACTIVATIONS)})")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        _check(p, name, x)
        if p.shape != (channels,):
            raise ValueError(f"{name} must have one value a channel")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one type")
    weight, bias = _dense(weight), _dense(bias)
    act = _capi.ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _GroupNorm.apply(x, weight, bias, groups, float(eps), act)
    return _norm_forward(*_rows(x), weight, bias, groups, float(eps), act)[0]


# ---- linear cross entropy -------------------------------------------------------

def _matrix(t: Tensor) -> Tensor:
    """Rows of contiguous values; a copy where they are not (a transposed view)."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _xent_plan(h, weight, ignore, reduction, backward):
    row = lambda t: t.stride(0) if t.shape[0] > 1 else t.shape[1]  # noqa: E731
    # of the pointers only their alignment matters
    hp, wp = h.data_ptr() & 15, weight.data_ptr() & 15
    key = (1, h.shape, weight.shape, row(h), row(weight), h.dtype, ignore, reduction, hp, wp, backward)
    return _plan(key, lambda: _capi.XentDesc(h.shape[0], h.shape[1], weight.shape[0], row(h), row(weight), ignore,
                                             _DTYPE[h.dtype], reduction),
                 lambda d, n: _capi.lib().srbcrs_linear_xent_workspace(d, hp, wp, backward, n))


def _xent_forward(h, weight, target, ignore, reduction):
    with _on_device(h):
        desc, n = _xent_plan(h, weight, ignore, reduction, 0)
        rows = h.shape[0]
        loss = torch.empty((rows,) if reduction == 0 else (), dtype=torch.float32, device=h.device)
        state = torch.empty(2 * rows + 1, dtype=torch.float32, device=h.device)
        ws = _workspace(n, h)
        _capi.check(_capi.lib().srbcrs_linear_xent(
            desc, h.data_ptr(), weight.data_ptr(), target.data_ptr(), loss.data_ptr(), state.data_ptr(), _capi.ptr(ws), n,
            _raw_stream(h.device.index)))
    return loss, state


def _xent_kinds(h, weight):
    # operands that are not aligned are copied to the workspace
    return _kind(h), _kind(weight), h.data_ptr() & 15, weight.data_ptr() & 15


def _xent_backward(ctx, dloss):
    # the engine runs this on the device and the stream of the forward pass
    h, weight, target, state = ctx.saved_tensors
    ignore, reduction, (desc, n) = ctx.args
    target, state, dloss = _dense(target), _dense(state), _dense(dloss)
    if _xent_kinds(h, weight) != ctx.kinds:
        _same_values(h, ctx.kinds[0])
        _same_values(weight, ctx.kinds[1])
        h, weight = _matrix(h), _matrix(weight)
        desc, n = _xent_plan(h, weight, ignore, reduction, 1)
    dh = _like(h) if ctx.needs_input_grad[0] else None
    dw = _like(weight) if ctx.needs_input_grad[1] else None
    ws = _workspace(n, h)
    _capi.check(_capi.lib().srbcrs_linear_xent_backward(
        desc, h.data_ptr(), weight.data_ptr(), target.data_ptr(), state.data_ptr(), dloss.data_ptr(),
        _capi.ptr(dh), _capi.ptr(dw), _capi.ptr(ws), n, _raw_stream(h.device.index)))
    return dh, dw, None, None, None


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, weight, target, ignore, reduction):
        hm, wm = _matrix(h), _matrix(weight)
        loss, state = _xent_forward(hm, wm, target, ignore, reduction)
        ctx.save_for_backward(hm, wm, target, state)
        ctx.kinds = _xent_kinds(hm, wm)
        ctx.args = (ignore, reduction, _xent_plan(hm, wm, ignore, reduction, 1))
        return loss

    backward = _once(_xent_backward)


def linear_cross_entropy(h: Tensor, weight: Tensor, target: Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> Tensor:
    """Softmax cross entropy of the logits ``h @ weight.T`` (``h`` rows x
    features, ``weight`` classes x features, one int64 class in ``target`` a row)
    in float32, with gradients in h and weight; the logits are never in memory as a whole.

    ``reduction``: "mean" over the rows whose target is not ``ignore_index`` (0 if
    there is none), "sum", or "none": one loss a row, 0 for ignored ones.  Ignored
    rows get a gradient of 0 whatever they hold.  A target that is neither a class
    nor ``ignore_index`` gives NaN (nothing is checked on the host).  A weight that is
    stored features x classes is passed as ``w.t()`` and copied.

    Sums are 32 bits; logits are at no time rounded to fewer.  The operands of the products: 16-bit inputs are
    used as they are, and ``dz = softmax - onehot`` keeps 11 bits (16 and more up to 128 classes or rows).
    float32 keeps 22 bits of every value (24 with up to 128 classes or rows against many of the other), in
    the logits of values down to 2^-29 of the largest in their own row of ``h`` or ``weight``,
    in the gradients down to 2^-29 of the largest ``h`` times its upstream gradient and of the
    largest weight; of what is smaller an absolute error of 2^-40 of those is left."""
    _check(h, "h")
    _check(weight, "weight", h)
    if h.dim() != 2 or weight.dim() != 2 or h.shape[1] != weight.shape[1]:
        raise ValueError("h must be rows x features, weight classes x features")
    if h.dtype != weight.dtype:
        raise TypeError("h and weight must have one type")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError("at least one class and one feature are needed")
    if not isinstance(target, Tensor) or target.dtype != torch.int64 or target.shape != (h.shape[0],):
        raise ValueError("target must be int64, one class a row")
    if target.device != h.device:
        raise RuntimeError(f"target is on {target.device}, expected {h.device}")
    if reduction not in _capi.REDUCTIONS:
        raise ValueError(f"unknown reduction {reduction!r} ({', '.join(_capi.REDUCTIONS)})")
    target = _dense(target)
    code = _capi.REDUCTIONS[reduction]
    if torch.is_grad_enabled() and (h.requires_grad or weight.requires_grad):
        return _LinearCrossEntropy.apply(h, weight, target, int(ignore_index), code)
    return _xent_forward(_matrix(h), _matrix(weight), target, int(ignore_index), code)[0]


# ---- orthogonalised updates -------------------------------------------------------

def orthogonalize(update: Tensor, steps: int = 5, coefficients: Sequence[float] = (3.4445, -4.7750, 2.0315),
                  eps: float = 1e-7) -> Tensor:
    """The update matrix (or each of a batch: ..., rows, cols) with its
    singular values driven towards 1: ``X = update / (norm + eps)``, then ``steps`` times
    ``X <- a X + (b K + c K K) X`` with ``K = X X^T`` and ``coefficients = (a, b, c)``.

    Products keep 22 bits of every value and sum in 32; the result has the
    update's type.  The coefficients must keep singular values of [0, 1] below 1.4.
    Not differentiable: an optimiser's step."""
    _check(update, "update")
    if update.dim() < 2:
        raise ValueError("update must be a matrix, or a batch of matrices")
    if len(coefficients) != 3:
        raise ValueError("coefficients are three numbers")
    g = update.detach()
    if g.dim() > 3:
        g = g.reshape(-1, *g.shape[-2:])
    if g.stride(-1) != 1 and g.shape[-1] != 1:
        g = g.contiguous()
    rows, cols = g.shape[-2:]
    batch = g.shape[0] if g.dim() == 3 else 1
    a, b, c = (float(v) for v in coefficients)
    strides = (g.stride(0) if g.dim() == 3 else 0, g.stride(-2) if rows > 1 else cols)
    with _on_device(g):
        desc, n = _plan((2, batch, rows, cols, strides, g.dtype, steps, a, b, c, eps),
                        lambda: _capi.OrthoDesc(batch, rows, cols, *strides, _DTYPE[g.dtype], int(steps), a, b, c, float(eps)),
                        _capi.lib().srbcrs_orthogonalize_workspace)
        out = _like(update.detach())
        ws = _workspace(n, g)
        _capi.check(_capi.lib().srbcrs_orthogonalize(desc, g.data_ptr(), out.data_ptr(), _capi.ptr(ws), n,
                                                     _raw_stream(g.device.index)))
    return out
