"""Group norm with an activation on channels-last tensors (ops.nn.group_norm,
csrc/group_norm.hip) against its formulas in 64 bits.

Tolerances.  A result is rounded to its type once: at most eps / 2 of its value.
Before that everything is fp32: a statistic over M values is summed in runs of
at most M / 64 + 64 terms, so with u = 2^-24 the normalised value xh is off by at
most (M / 64 + 64) u (1 + |xh| + |mean| / std), and an activation multiplies
that by at most 1.1 (its largest slope).  Gradients are sums of such terms; a factor of 4 covers
the product rule (e, gamma, xh and r each carry the error once).  Where ReLU's
argument is within 1e-4 of a kink the incoming gradient is zero, so no gate
depends on a rounding.
"""

import pytest
import torch

from kf_benchmarks_amd.ops import _native as N
from kf_benchmarks_amd.ops import nn as F

U = 2.0 ** -24
ACTS = [None, "relu", "relu6", "tanh", "silu"]


def act_and_slope(u, act):
    if act == "relu":
        return u.clamp(min=0), (u > 0).double()
    if act == "relu6":
        return u.clamp(0, 6), ((u > 0) & (u < 6)).double()
    if act == "tanh":
        return torch.tanh(u), 1 - torch.tanh(u) ** 2
    if act == "silu":
        s = torch.sigmoid(u)
        return u * s, s * (1 + u * (1 - s))
    return u, torch.ones_like(u)


def oracle(x, gamma, beta, groups, eps, act, dy=None):
    """The formulas in 64 bits: {name: (value, fp32 error bound)}."""
    shape, C = x.shape, x.shape[-1]
    v = x.double().reshape(shape[0], -1, groups, C // groups)
    M = v.shape[1] * v.shape[3]
    ga = (gamma if gamma is not None else torch.ones(C, device=x.device)).double().view(groups, -1)
    be = (beta if beta is not None else torch.zeros(C, device=x.device)).double().view(groups, -1)
    mu = v.mean((1, 3), keepdim=True)
    r = 1 / torch.sqrt(((v - mu) ** 2).mean((1, 3), keepdim=True) + eps)
    xh = (v - mu) * r
    u = xh * ga + be
    exh = (M / 64 + 64) * U * (1 + xh.abs() + mu.abs() * r)
    y, slope = act_and_slope(u, act)
    out = {"y": (y, 1.1 * (exh * ga.abs() + 4 * U * u.abs()))}
    if dy is not None:
        g = dy.double().view(v.shape)
        e, size = g * slope, g.abs() * 1.1 * ga.abs()
        eg = e * ga
        dx = r * (eg - eg.mean((1, 3), keepdim=True) - xh * (eg * xh).mean((1, 3), keepdim=True))
        part = size * exh * (1 + xh.abs())
        bound = r * (part + part.mean((1, 3), keepdim=True) * (1 + xh.abs())
                     + (size * xh.abs()).mean((1, 3), keepdim=True) * exh)
        out["x"] = (dx, 4 * bound)
        rows = v.shape[0] * v.shape[1]
        w = (rows / 16 + 64) * U
        out["gamma"] = ((e * xh).sum((0, 1)), 4 * ((w + exh) * g.abs() * 1.1 * (1 + xh.abs()) * (1 + ga.abs())).sum((0, 1)))
        out["beta"] = (e.sum((0, 1)), 4 * ((w + exh) * g.abs() * 1.1 * (1 + ga.abs())).sum((0, 1)))
    full = {"y": shape, "x": shape, "gamma": (C,), "beta": (C,)}
    return {k: tuple(t.reshape(full[k]) for t in p) for k, p in out.items()}


def check(got, want, name):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    fi = torch.finfo(got.dtype)
    half = fi.eps / 2 if got.dtype != torch.float32 else U
    lim = half * value.abs() + bound + fi.smallest_normal * fi.eps
    off = (got.double() - value).abs()
    worst = (off / lim).max().item()
    assert worst <= 1, "%s: %.3g times the bound" % (name, worst)


def inputs(shape, groups, act, dtype, dev, seed=0, affine=True, offset=1.0):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(shape, generator=g) * 1.5 + offset * torch.randn(C, generator=g)).to(dtype)
    gamma = 1 + 0.2 * torch.randn(C, generator=g) if affine else None
    beta = 0.2 * torch.randn(C, generator=g) if affine else None
    dy = torch.randn(shape, generator=g).to(dtype)
    if act in ("relu", "relu6"):
        u = oracle(x, gamma, beta, groups, 1e-5, None)["y"][0]
        dy[(u.abs() < 1e-4) | ((u - 6).abs() < 1e-4)] = 0
    return tuple(t.to(dev) if t is not None else None for t in (x, gamma, beta, dy))


def run(x, gamma, beta, groups, act, dy, eps=1e-5):
    leaves = {k: t.detach().requires_grad_() for k, t in (("x", x), ("gamma", gamma), ("beta", beta))
              if t is not None}
    y = F.group_norm(leaves["x"], leaves.get("gamma"), leaves.get("beta"), groups, eps, act)
    return {"y": y.detach(), **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))}


def compare(shape, groups, act, dtype, dev, **kw):
    x, gamma, beta, dy = inputs(shape, groups, act, dtype, dev, **kw)
    want = oracle(x, gamma, beta, groups, 1e-5, act, dy)
    got = run(x, gamma, beta, groups, act, dy)
    for name, t in got.items():
        check(t, want[name], name)
    with torch.no_grad():
        assert torch.equal(F.group_norm(x, gamma, beta, groups, 1e-5, act), got["y"])


# ------------------------------------------------------------------- CPU
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape,groups", [((2, 3, 5, 12), 4), ((3, 8), 2), ((1, 7, 6), 6)])
def test_group_norm_cpu(shape, groups, act):
    compare(shape, groups, act, torch.float32, "cpu")


@pytest.mark.parametrize("act", ACTS)
def test_oracle_gradients_against_differences(act):
    x, gamma, beta, dy = (t.double() for t in inputs((2, 3, 2, 6), 3, act, torch.float32, "cpu"))
    want = oracle(x, gamma, beta, 3, 1e-5, act, dy)
    for name, t in (("x", x), ("gamma", gamma), ("beta", beta)):
        flat = t.view(-1)
        for i in range(0, flat.numel(), 5):
            old, h, f = flat[i].item(), 1e-6, []
            for s in (1, -1):
                flat[i] = old + s * h
                f.append((oracle(x, gamma, beta, 3, 1e-5, act)["y"][0] * dy).sum())
            flat[i] = old
            assert abs((f[0] - f[1]) / (2 * h) - want[name][0].view(-1)[i]) < 1e-6


def test_group_norm_refusals():
    x, p = torch.randn(2, 4, 6), torch.ones(6)
    for call in (lambda: F.group_norm(x, p, p, 4), lambda: F.group_norm(x, p, p, 0),
                 lambda: F.group_norm(x, p[:5], p, 2), lambda: F.group_norm(x, p.double(), p, 2),
                 lambda: F.group_norm(x, p, torch.ones(12)[::2], 2),
                 lambda: F.group_norm(x[:0], p, p, 2), lambda: F.group_norm(torch.ones(6), p, p, 2)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(KeyError):
        F.group_norm(x, p, p, 2, activation="swoosh")


# ------------------------------------------------------------------- GPU
SHAPES = [((1, 14, 14, 256), 32), ((3, 5, 7, 288), 32), ((2, 9, 9, 30), 6), ((4, 33, 17, 64), 1),
          ((5, 1, 1, 1600), 8), ((37, 200), 8), ((3, 1, 1, 5), 5), ((2, 11, 13, 7), 7), ((2, 6, 6, 2500), 1),
          ((1, 3, 40000), 2), ((2, 56, 56, 64), 32), ((70, 3, 3, 24), 3), ((300, 48), 1), ((1, 1, 1, 1), 1),
          ((2, 130, 3, 40), 4), ((1, 112, 112, 66), 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_group_norm_gpu(cuda, shape, groups, dtype):
    compare(shape, groups, "silu", dtype, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape,groups", [((2, 9, 9, 48), 6), ((1, 40, 40, 512), 32)])
def test_group_norm_activations_gpu(cuda, shape, groups, act):
    compare(shape, groups, act, torch.bfloat16, cuda)
    compare(shape, groups, act, torch.float32, cuda, affine=False)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((1, 40, 40, 64), 8), ((6, 7, 7, 64), 8), ((200, 1, 1, 256), 8)])
def test_group_norm_far_mean_gpu(cuda, shape, groups):
    """Values whose mean is 300 standard deviations off: the variance is that of the centred values."""
    compare(shape, groups, None, torch.float32, cuda, offset=300.0)


@pytest.mark.gpu
def test_group_norm_extremes_gpu(cuda):
    """A constant group gives beta; NaN stays in its own group; infinities give NaN like the formula."""
    x = torch.randn(2, 8, 8, 64, device=cuda)
    x[0, :, :, :8] = 3.0
    x[1, 2, 3, 16] = float("nan")
    x[1, 4, 4, 40] = float("inf")
    beta = torch.randn(64, device=cuda)
    y = F.group_norm(x, None, beta, 8)
    assert torch.equal(y[0, :, :, :8], beta[:8].expand(8, 8, 8))
    bad = torch.zeros(2, 8, 8, 64, dtype=torch.bool, device=cuda)
    bad[1, :, :, 16:24] = True
    bad[1, :, :, 40:48] = True
    assert torch.equal(~torch.isfinite(y), bad)


@pytest.mark.gpu
def test_group_norm_strided_and_unaligned_gpu(cuda):
    wide = torch.randn(4, 6, 6, 80, device=cuda).to(torch.bfloat16)
    flat = torch.randn(4 * 36 * 64 + 1, device=cuda).to(torch.bfloat16)
    for x in (wide[..., 8:72], wide[::2, :, 1:, :64], flat[1:].view(4, 6, 6, 64), wide.transpose(1, 3)[..., :6, :].transpose(1, 3)):
        C = x.shape[-1]
        G = 8 if C % 8 == 0 else 2
        gamma, beta = torch.rand(C, device=cuda), torch.rand(C, device=cuda)
        dy = torch.randn(x.shape, device=cuda).to(torch.bfloat16)
        want = oracle(x, gamma, beta, G, 1e-5, "silu", dy)
        for name, t in run(x, gamma, beta, G, "silu", dy).items():
            check(t, want[name], name)
        gap = torch.randn(x.shape[:-1] + (2 * C,), device=cuda).to(torch.bfloat16)[..., ::2]
        want = oracle(x, gamma, beta, G, 1e-5, "silu", gap)
        for name, t in run(x, gamma, beta, G, "silu", gap).items():
            check(t, want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((2, 9, 9, 48), 6), ((8, 30, 30, 256), 32), ((500, 96), 3)])
def test_group_norm_same_bits_and_sinks_gpu(cuda, shape, groups):
    """Two runs give the same bits; a flat-buffer gradient is added to."""
    x, gamma, beta, dy = inputs(shape, groups, "relu", torch.bfloat16, cuda)
    a, b = (run(x, gamma, beta, groups, "relu", dy) for _ in range(2))
    assert all(torch.equal(a[k], b[k]) for k in a)
    ps = [t.clone().requires_grad_() for t in (gamma, beta)]
    for p in ps:
        p._kfb_grad_sink = torch.full_like(p, 2.0)
    F.group_norm(x.clone().requires_grad_(), ps[0], ps[1], groups, 1e-5, "relu").backward(dy)
    assert ps[0].grad is None and ps[1].grad is None
    torch.testing.assert_close(ps[0]._kfb_grad_sink, a["gamma"] + 2, rtol=1e-6, atol=1e-5)
    torch.testing.assert_close(ps[1]._kfb_grad_sink, a["beta"] + 2, rtol=1e-6, atol=1e-5)


@pytest.mark.gpu
def test_group_norm_large_offsets_gpu(cuda):
    """More than 2^31 values: the last image equals the same image alone."""
    n, c = 2050, 1 << 20
    x = torch.empty((n, 1, 1, c), dtype=torch.bfloat16, device=cuda)
    x[0].normal_()
    x[-1].normal_()
    x[1:-1] = x[0]
    y = F.group_norm(x, None, None, 1 << 15, activation="silu")
    assert torch.equal(y[-1:], F.group_norm(x[-1:].clone(), None, None, 1 << 15, activation="silu"))
    assert torch.equal(y[:1], F.group_norm(x[:1].clone(), None, None, 1 << 15, activation="silu"))


@pytest.mark.gpu
def test_group_norm_refuses_other_types_gpu(cuda):
    with pytest.raises(N.NativeError):
        F.group_norm(torch.ones(2, 3, 4, device=cuda, dtype=torch.float64), None, None, 2)
    with pytest.raises(ValueError):
        F.group_norm(torch.ones(2, 3, 4, device=cuda), torch.ones(4), None, 2)
    x = torch.randn(2, 3, 4, device=cuda, requires_grad=True)
    (g,) = torch.autograd.grad(F.group_norm(x, None, None, 2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [N.BF16, N.F32])
@pytest.mark.parametrize("C,groups", [(4096, 1), (2048, 1), (4096, 8), (8192, 1), (1600, 8)])
@pytest.mark.parametrize("at", [0, 4])
def test_workspace_does_not_grow_with_the_rows(dtype, C, groups, at):
    """At most 2048 slabs of 2 C channel sums for any number of rows, wide groups and unaligned tensors among them."""
    for rows in (1, 1000, 32768, 1 << 24):
        assert 0 < N.query("kfb_gn_bwd_ws", dtype, rows, 1, C, groups, at) <= 2048 * 2 * C
        assert N.query("kfb_gn_fwd_ws", dtype, rows, 1, C, groups, at) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups,dtype", [((2100, 2052), 1, torch.float32), ((2060, 4104), 1, torch.bfloat16),
                                                ((1100, 2, 1026), 2, torch.float16), ((1030, 8208), 2, torch.bfloat16)])
def test_group_norm_more_images_than_slabs_gpu(cuda, shape, groups, dtype):
    compare(shape, groups, "silu", dtype, cuda)


FAR = [((1, 40, 40, 64), 8), ((2, 56, 56, 64), 32), ((6, 7, 7, 64), 8), ((200, 256), 8), ((3, 9, 2052), 1)]


def far_inputs(shape, groups):
    """Inputs whose groups' means are 1000 and more of their standard deviations."""
    x, gamma, beta, dy = inputs(shape, groups, None, torch.float32, "cpu", offset=0.0)
    g = torch.Generator().manual_seed(2)
    x = x + 3000.0 * (1 + 0.2 * torch.rand(groups, generator=g)).repeat_interleave(shape[-1] // groups)
    v = x.double().reshape(shape[0], -1, groups, shape[-1] // groups)
    assert (v.mean((1, 3)).abs() / v.std((1, 3))).min() > 1000
    return x, gamma, beta, dy


@pytest.mark.parametrize("shape,groups", FAR)
def test_far_mean_tells_variances_apart(shape, groups):
    """The bound passes the variance of centred fp32 values and not the mean square minus the squared mean."""
    x, gamma, beta, _ = far_inputs(shape, groups)
    v = x.reshape(shape[0], -1, groups, shape[-1] // groups)
    mu = v.mean((1, 3), keepdim=True)
    want = oracle(x, None, None, groups, 1e-5, None)["y"]
    centred = ((v - mu) ** 2).mean((1, 3), keepdim=True)
    one_pass = (v * v).mean((1, 3), keepdim=True) - mu * mu
    check(((v - mu) / torch.sqrt(centred + 1e-5)).reshape(shape), want, "y")
    with pytest.raises(AssertionError):
        check(((v - mu) / torch.sqrt(one_pass.clamp(min=0) + 1e-5)).reshape(shape), want, "y")


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", FAR)
def test_group_norm_of_far_means_gpu(cuda, shape, groups):
    x, gamma, beta, dy = (t.to(cuda) for t in far_inputs(shape, groups))
    want = oracle(x, gamma, beta, groups, 1e-5, None, dy)
    for name, t in run(x, gamma, beta, groups, None, dy).items():
        check(t, want[name], name)
