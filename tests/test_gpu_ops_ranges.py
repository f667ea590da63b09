"""The training operators over the range of their values: rows that hold garbage beside rows that count, rows and
classes of very unlike magnitude.  What one row holds must not cost another row's digits."""
from __future__ import annotations

import pytest

from tests.test_gpu_ops import DTYPES, HALF_ULP, TINY, U32, _check_norm, _check_xent, _norm64, _norm_case, _say, _within, _xent_case

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


def _gradients(h, w, t, reduction="mean", up=None):
    import torch
    from mask_amd import ops
    hl, wl = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = ops.linear_cross_entropy(hl, wl, t, reduction=reduction)
    return torch.autograd.grad(loss, (hl, wl), torch.ones_like(loss) if up is None else up)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", XENT_FORMS)
def test_ignored_rows_change_no_gradient(gpu, shape, dtype):
    """Equal bits: rows that do not count have no say in an operand's scale."""
    import torch
    h, w, t = _xent_case(*shape, dtype, seed=24, labelled=0.5)
    off = (t == -100).nonzero().squeeze(1)
    clean = _gradients(h, w, t)
    assert clean[1].any() and not clean[0][off].any()
    for value in _garbage(dtype):
        _say("ignored rows, gradients", shape, dtype, value)
        bad = h.clone()
        bad[off[::2]] = value
        bad[off[1], 3] = value
        for a, b in zip(_gradients(bad, w, t), clean):
            assert torch.equal(a, b), value


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", XENT_FORMS)
def test_a_large_row_of_a_small_gradient(gpu, shape, dtype):
    """A row of 1e6 whose upstream gradient is 1e-6 is a row like the others in the weight's gradient: 64 bits' within
    the bound of its products (2^-21 of a 32-bit operand, 2^-11 of dz and of a row times its factor in 16 bits)."""
    import torch
    rows, _, classes = shape
    h, w, t = _xent_case(*shape, dtype, seed=25, labelled=1.0)
    h = h / 16          # logits that stay soft times 1e6 would be one-hot: that row's are made small by its weight below
    w = w.clone()
    w[:, 0] = 0
    h[7] = 0
    h[7, 0] = 1e6       # the only large feature meets weights of 0: the row's softmax is flat
    up = torch.ones(rows, device="cuda")
    up[7] = 1e-6
    _say("large row of a small gradient", shape, dtype)
    _, dw = _gradients(h, w, t, "none", up)
    z = h.double() @ w.double().t()
    dz = torch.softmax(z, 1)
    dz.scatter_add_(1, t.unsqueeze(1), -torch.ones_like(t, dtype=torch.float64).unsqueeze(1))
    dz *= up.double().unsqueeze(1)
    want = dz.t() @ h.double()
    size = dz.abs().t() @ h.double().abs()
    ez = (2.0 ** -21 + (h.shape[1] + 8) * U32) * (h.double().abs() @ w.double().abs().t()).max()
    half = 2.0 ** -24 if dtype == "float32" else 2.0 ** -8
    keep = 2.0 ** -19 if dtype == "float32" else 2.0 ** -10 + 2.0 ** -20   # dz, a row times its factor, the other operand
    # operands: 2^-40 of the largest entry (1e6 times 1e-6 and h's own) times the gradients' sum
    edge = 2.0 ** -39 * (h[:7].double().abs().max() + 1) * dz.abs().sum(0).unsqueeze(1) + rows * 2.0 ** -38
    bound = half * want.abs() + (keep + 2 * ez + (4 * rows ** 0.5 + 96) * U32) * size + edge
    assert ((dw.double() - want).abs() <= bound).all(), ((dw.double() - want).abs() / bound).max().item()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", XENT_FORMS)
def test_rows_of_no_upstream_gradient_change_no_gradient(gpu, shape, dtype):
    """A labelled row whose loss has an upstream gradient of 0 is a row of zeros in every gradient, whatever it holds
    (its own loss is what it is)."""
    import torch
    h, w, t = _xent_case(*shape, dtype, seed=26, labelled=1.0)
    off = torch.arange(0, shape[0], 3, device="cuda")
    up = torch.linspace(0.5, 2.0, shape[0], device="cuda")
    up[off] = 0
    clean = _gradients(h, w, t, "none", up)
    assert clean[1].any() and not clean[0][off].any()
    for value in _garbage(dtype):
        _say("no upstream gradient", shape, dtype, value)
        bad = h.clone()
        bad[off[::2]] = value
        bad[off[1], 3] = value
        for a, b in zip(_gradients(bad, w, t, "none", up), clean):
            assert torch.equal(a, b), value


# ---- saved tensors that come back in another layout ------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
def test_saved_tensors_may_come_back_in_another_layout(gpu, dtype):
    """save_on_cpu makes a slice dense, and another hook gives back a slice of something wider or something that starts
    elsewhere: the gradients keep their bits.  A tensor of another type or shape is refused."""
    import torch
    from mask_amd import ops

    def wider(t):
        if t.dim() < 2 or not t.is_floating_point():
            return t.clone()
        out = torch.zeros((*t.shape[:-1], t.shape[-1] + 24), dtype=t.dtype, device=t.device)[..., 8:8 + t.shape[-1]]
        return out.copy_(t)

    def shifted(t):
        return torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].copy_(t.reshape(-1)).view(t.shape)

    hooks = {"plain": None, "save_on_cpu": torch.autograd.graph.save_on_cpu(),
             "wider": torch.autograd.graph.saved_tensors_hooks(lambda t: t, wider),
             "dense": torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.contiguous()),
             # matrices only: statistics are aligned by contract, and group norm's loads, so the order of its sums, go by alignment
             "shifted": torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: shifted(t) if t.dim() == 2 else t.clone())}
    calls = []
    for shape in ((130, 64, 300), (300, 64, 300), (90, 64, 70), (90, 64, 300)):
        h, w, t = _xent_case(*shape, dtype, seed=31)
        hw = torch.zeros(shape[0], 3 * shape[1], dtype=h.dtype, device="cuda")
        ww = torch.zeros(shape[2], 2 * shape[1], dtype=h.dtype, device="cuda")
        hc, wc = hw[:, 64:128].copy_(h), ww[:, 64:].copy_(w)
        calls.append((shape, (hc, wc), lambda a, b, t=t: ops.linear_cross_entropy(a, b, t)))
    for shape, groups in (((3, 40, 32), 4), ((2, 3000, 24), 6), ((500, 1, 64), 8), ((1, 9000, 16), 2)):
        x, w, b, dy = _norm_case(shape, groups, "silu", dtype, seed=32)
        wide = torch.zeros(shape[0], 2 * shape[1], shape[2] + 8, dtype=x.dtype, device="cuda")
        xc = wide[:, shape[1]:, 8:].copy_(x)
        calls.append((shape, (xc, w, b), lambda a, g, o, groups=groups, dy=dy:
                      (ops.group_norm(a, groups, g, o, activation="silu") * dy).sum()))
    for shape, ins, fn in calls:
        want = None
        for name, hook in hooks.items():
            _say("saved tensors", shape, dtype, name)
            leaves = [v.detach().requires_grad_() for v in ins]
            if hook is None:
                out = fn(*leaves)
            else:
                with hook:
                    out = fn(*leaves)
            got = torch.autograd.grad(out, leaves)
            want = got if want is None else want
            for a, b in zip(got, want):
                assert torch.equal(a, b), name
    for bad in (lambda t: t.double() if t.is_floating_point() else t, lambda t: t[:-1]):
        for shape, ins, fn in (calls[0], calls[-1]):
            leaves = [v.detach().requires_grad_() for v in ins]
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, bad):
                out = fn(*leaves) if len(ins) == 2 else ops.group_norm(leaves[0], 2, leaves[1], leaves[2])
            out = out.sum()
            with pytest.raises(RuntimeError, match="came back as"):
                torch.autograd.grad(out, leaves)


# ---- group norm of many samples --------------------------------------------------

@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape, groups", [((2048, 50, 320), 32), ((2048, 50, 320), 2), ((600, 130, 256), 256), ((70, 700, 200), 1)])
def test_group_norm_of_many_split_samples(gpu, shape, groups, dtype):
    """Samples of a chunk or a few each: groups of few parts, parameters of many."""
    x, w, b, dy = _norm_case(shape, groups, "silu", dtype, seed=41)
    _say("many split samples", shape, groups, dtype)
    _check_norm(x, groups, w, b, dy, "silu", what=f"{shape} {groups} {dtype}")


@pytest.mark.parametrize("shape, groups, rows", [((1, 1000003, 8), 8, 4), ((3000000, 1, 4), 2, 23), ((65536, 30, 8), 2, 8)])
def test_group_norm_parameter_gradients_of_many_rows(gpu, shape, groups, rows):
    """Sums over millions of rows for few channels, a shape for each form: a thread adds `rows` values in 32 bits, the
    threads' sums are joined in 64, what a workgroup has is rounded once and so is the result.  In units of 2^-24 of
    the root of the sum of squares, roundings of random sign then come to sqrt((rows / 2 + 2) / 3); the root mean
    square over channels and seeds stays below 1.5 times that (a chain of 128 threads in 32 bits: 4.6 and more).  Of the
    weight's gradient as well, whose terms have two roundings more."""
    import torch
    from mask_amd import ops
    units = {"dweight": [], "dbias": []}
    for seed in range(4):
        _say("parameter gradients", shape, seed)
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        x = torch.randn(shape, generator=gen, device="cuda")
        dy = torch.randn(shape, generator=gen, device="cuda")
        w = torch.ones(shape[-1], device="cuda", requires_grad=True)
        b = torch.zeros(shape[-1], device="cuda", requires_grad=True)
        dw, db = torch.autograd.grad(ops.group_norm(x, groups, w, b, eps=0.1), (w, b), dy)
        d = dy.double()
        units["dbias"].append((db.double() - d.sum(dim=(0, 1))) / (U32 * (d * d).sum(dim=(0, 1)).sqrt()))
        if shape[1] > 1:
            v = x.double().reshape(shape[0], shape[1], groups, -1)
            var, mean = torch.var_mean(v, dim=(1, 3), unbiased=False, keepdim=True)
            d = d * ((v - mean) / (var + 0.1).sqrt()).reshape(shape)
            units["dweight"].append((dw.double() - d.sum(dim=(0, 1))) / (U32 * (d * d).sum(dim=(0, 1)).sqrt()))
    for (what, u), more in zip(units.items(), (2, 0)):
        if u:
            rms = torch.stack(u).square().mean().sqrt().item()
            assert rms <= 1.5 * ((rows / 2 + 2 + more) / 3) ** 0.5, (what, rms)


@pytest.mark.parametrize("shape, groups", [((70, 1, 4096), 512), ((3, 1, 768), 256), ((5, 1, 500), 1), ((1, 1, 8192), 8)])
def test_group_norm_relu_knows_its_side(gpu, shape, groups):
    """Single float32 rows: biases that take u to the rounding of a 32-bit number away from 0, about 1e-8, on either
    side.  y is positive where 64 bits say so, and so the slope: no gradient is masked.  What 64 bits themselves leave
    open (1e-12) is left out."""
    import torch
    from mask_amd import ops
    n, _, c = shape
    gen = torch.Generator().manual_seed(51)
    x = (torch.randn(1, 1, c, generator=gen) + 3.0).cuda().expand(shape).contiguous()
    w = (1 + 0.3 * torch.randn(c, generator=gen)).cuda()
    dy = torch.randn(shape, generator=gen).cuda()
    _, _, hat, _, rstd = _norm64(x.double(), groups, w.double(), torch.zeros_like(w).double(), 1e-5, "none")
    b = (-hat[0, 0] * w.double()).float()
    _, u, _, _, _ = _norm64(x.double(), groups, w.double(), b.double(), 1e-5, "relu")
    open_ = u.abs() < 1e-12
    assert (u.abs() < 1e-6).all() and (u > 1e-12).any() and (u < -1e-12).any() and open_.float().mean() < 0.05
    dy = torch.where(open_, torch.zeros_like(dy), dy)
    _say("relu's side", shape, groups)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = ops.group_norm(leaves[0], groups, leaves[1], leaves[2], activation="relu")
    assert ((y > 0) == (u > 0))[~open_].all()
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    # with the right slopes what is left are roundings: 64 of them of each term
    du = torch.where(u > 0, dy.double(), torch.zeros_like(u))
    g = du * w.double()
    mean = lambda t: t.reshape(n, groups, -1).mean(dim=2, keepdim=True).expand(n, groups, c // groups).reshape(shape)  # noqa: E731
    want = rstd * (g - mean(g) - hat * mean(g * hat))
    size = rstd * (g.abs() + mean(g.abs()) + hat.abs() * mean((g * hat).abs()))
    # xhat is off by the rounding of x - mean
    ehat = 4 * U32 * (x.double().abs() * rstd + 1)
    _within(dx, want, 64 * U32 * size + rstd * (ehat * mean((g * hat).abs()) + (hat.abs() + ehat) * mean(g.abs() * ehat)), "dx")
    _within(db, du.sum(dim=(0, 1)), 64 * U32 * du.abs().sum(dim=(0, 1)) + 1e-38, "dbias")
    _within(dw, (du * hat).sum(dim=(0, 1)), (du.abs() * (64 * U32 * hat.abs() + ehat)).sum(dim=(0, 1)) + 1e-38, "dweight")


@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm_gelu_keeps_its_negative_tail(gpu, dtype):
    """Weights of 0 make u the bias, exactly: gelu's value and slope from 0 to -9 to a relative error, where y comes down
    to 1e-18.  exp's argument has three roundings (3 U32 u^2 / 2 of the result), the rest 40; the slope's two terms
    count each.  Then the result's type."""
    import torch
    from mask_amd import ops
    c = 4096
    u = torch.linspace(-9.0, 3.0, c).cuda()
    x = torch.randn(1, 1, c, generator=torch.Generator().manual_seed(61)).to(getattr(torch, dtype)).cuda()
    w = torch.zeros(c, device="cuda")
    b = u.clone().requires_grad_()
    _say("gelu's tail", dtype)
    y = ops.group_norm(x, 8, w, b, activation="gelu")
    (db,) = torch.autograd.grad(y, b, torch.ones_like(y))
    u = u.double()
    cdf = 0.5 * torch.special.erfcx(u.abs() / 2 ** 0.5) * torch.exp(-0.5 * u * u)
    cdf = torch.where(u < 0, cdf, 1 - cdf)
    pdf = torch.exp(-0.5 * u * u) * 0.3989422804014327
    rel = U32 * (1.5 * u * u + 40)
    _within(y[0, 0], u * cdf, (u * cdf).abs() * (HALF_ULP[dtype] + rel) + TINY[dtype], "gelu")
    _within(db, cdf + u * pdf, (cdf + (u * pdf).abs()) * (U32 + rel), "gelu's slope")


# ---- where the forms of the cross entropy change -----------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(4607, 520, 9), (4608, 520, 9), (1000, 511, 9), (5631, 260, 40), (5632, 260, 40), (1000, 255, 40),
                                   (12287, 70, 100), (12288, 70, 100), (9, 520, 4607), (9, 520, 4608), (40, 260, 5632),
                                   (100, 70, 12287), (100, 70, 12288), (49152, 24, 64), (49151, 24, 64), (65536, 24, 9),
                                   (70, 1024, 90), (70, 1025, 90), (20000, 1024, 20), (19999, 1024, 20)])
def test_linear_cross_entropy_where_its_forms_change(gpu, shape, dtype):
    """On both sides of the sizes from which the long matrix is streamed, of the features from which it counts, and of
    the tiles of a wave; workgroups whose last waves have no rows."""
    _say("forms", shape, dtype)
    h, w, t = _xent_case(*shape, dtype, seed=71)
    _check_xent(h, w, t, "mean", what=f"{shape} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape, groups", [((90, 1, 728), 8), ((70, 1, 1023), 1), ((70, 1, 1023), 3), ((80, 1, 992), 32), ((66, 1, 1025), 5),
                                           ((70, 3, 1023), 1), ((65, 7, 777), 7), ((600, 1, 1024), 1024), ((70, 9, 1001), 1001)])
def test_group_norm_of_many_odd_channels(gpu, shape, groups, dtype):
    """More than 512 channels that no vector divides: a channel a thread, up to 1024 of them, and one more."""
    x, w, b, dy = _norm_case(shape, groups, "gelu", dtype, seed=42)
    _say("odd channels", shape, groups, dtype)
    _check_norm(x, groups, w, b, dy, "gelu", what=f"{shape} {groups} {dtype}")
