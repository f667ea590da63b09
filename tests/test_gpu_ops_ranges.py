"""The training operators over the range of their values: rows that hold garbage beside rows that count, rows and
classes of very unlike magnitude.  What one row holds must not cost another row's digits."""
from __future__ import annotations

import pytest

from tests.test_gpu_ops import DTYPES, U32, _say, _xent_case

pytestmark = pytest.mark.gpu

# few classes and rows, few rows, tiles (their sums whole and split), and few classes
XENT_FORMS = [(90, 64, 70), (90, 64, 300), (300, 64, 300), (700, 2500, 400), (300, 72, 70)]


def _garbage(dtype):
    """What an ignored row may hold, finite and not."""
    import torch
    lim = torch.finfo(getattr(torch, dtype))
    some = [lim.min, lim.max, float("nan"), float("inf"), -float("inf")]
    return some + ([6e4, -3e4] if dtype == "float16" else [1e10, -1e15])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", XENT_FORMS)
def test_ignored_rows_change_no_loss(gpu, shape, dtype):
    """Equal bits: a row's logits are scaled by its own values alone."""
    import torch
    from mask_amd import ops
    h, w, t = _xent_case(*shape, dtype, seed=21, labelled=0.5)
    off = (t == -100).nonzero().squeeze(1)
    for value in _garbage(dtype):
        _say("ignored rows", shape, dtype, value)
        bad = h.clone()
        bad[off[::2]] = value
        bad[off[1], 3] = value
        for reduction in ("none", "mean", "sum"):
            assert torch.equal(ops.linear_cross_entropy(bad, w, t, reduction=reduction),
                               ops.linear_cross_entropy(h, w, t, reduction=reduction)), (value, reduction)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", XENT_FORMS)
def test_a_large_row_leaves_the_others_losses(gpu, shape, dtype):
    """A labelled row of 1e15, and one of 1e-15: the others' losses keep their bits, its own is that of 64 bits (a
    logit's error is 2^-21 of its terms' magnitudes for the operands, 2^-24 of them a sum, twice a loss)."""
    import torch
    from mask_amd import ops
    rows, dim, _ = shape
    h, w, t = _xent_case(*shape, dtype, seed=22, labelled=1.0)
    ref = ops.linear_cross_entropy(h, w, t, reduction="none")
    for size in (1e15, 1e-15):
        _say("large row", shape, dtype, size)
        other = h.clone()
        other[7] = (h[7].float() * size).to(h.dtype)
        got = ops.linear_cross_entropy(other, w, t, reduction="none")
        keep = torch.arange(rows, device="cuda") != 7
        assert torch.equal(got[keep], ref[keep])
        z = other[7].double() @ w.double().t()
        want = torch.logsumexp(z, 0) - z[t[7]]
        ez = (2.0 ** -21 + (dim + 8) * U32) * (other[7].double().abs() @ w.double().abs().t()).max()
        assert (got[7].double() - want).abs() <= 2 * ez + 16 * U32 * (z.abs().max() + 1)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", XENT_FORMS)
def test_a_large_class_leaves_the_others_logits(gpu, shape, dtype):
    """A class of weights of -1e15 over positive features has no probability anywhere: the losses are those without
    it, up to the order in which the statistics are joined (a rounding of log and exp each time)."""
    import torch
    from mask_amd import ops
    h, w, t = _xent_case(*shape, dtype, seed=23, labelled=1.0)
    h = h.abs()
    more = torch.cat((w, torch.full_like(w[:1], -1e15)))
    _say("large class", shape, dtype)
    ref = ops.linear_cross_entropy(h, w, t, reduction="none").double()
    got = ops.linear_cross_entropy(h, more, t, reduction="none").double()
    lse = torch.logsumexp(h.double() @ w.double().t(), 1)
    ez = (h.shape[1] + 8) * U32 * (h.double().abs() @ w.double().abs().t()).max(dim=1).values   # sums in another order
    assert ((got - ref).abs() <= 2 * ez + 32 * U32 * (lse.abs() + ref + 1)).all()
