"""The causal convolution and the selective scan (ops.ssm, csrc/causal_conv.hip,
csrc/ssm.hip) against their formulas in 64 bits.

Tolerances.  A result is rounded to its type once: at most eps / 2 of its value.
Before that everything is fp32.  ``oracle(..., size=True)`` evaluates the same
formulas on absolute values, so its results bound every sum of magnitudes on the
way.  With u = 2^-24 each step of a recurrence multiplies in at most 8 roundings (the decay
and its argument, the step size, the products, the additions) and a sum of n terms
adds at most n: a result after T steps of B sequences over N states or D
channels is off by at most 8 (T + B + N + D / 16 + 16) u times its size.  (Decays
only shrink an error; the absolute error of exp(v), v <= 0, is below 4 u.)
"""

import pytest
import torch

from kf_benchmarks_amd.ops import _native as N
from kf_benchmarks_amd.ops import ssm

U = 2.0 ** -24


def positions(T, B, lengths, reverse, dev):
    s = torch.arange(T, device=dev)[:, None].expand(T, B)
    n = torch.full((B,), T, device=dev) if lengths is None else lengths.long().clamp(0, T)
    return torch.where((s < n) & reverse, n - 1 - s, s), (s < n)[..., None], n


def gather(x, pos):
    return torch.gather(x, 0, pos[..., None].expand(-1, -1, x.shape[2]))


def silu(u):
    return u * torch.sigmoid(u)


def dsilu(u):
    p = torch.sigmoid(u)
    return p * (1 + u * (1 - p))


def scan_oracle(i, dy=None, dh=None, size=False):
    """The scan's formulas in 64 bits, one step after the other; size: on absolute values."""
    mag = (lambda t: t.abs()) if size else (lambda t: t)
    dev = i["x"].device
    T, B, D = i["x"].shape
    pos, inside, _ = positions(T, B, i["lengths"], i["reverse"], dev)
    zero = torch.zeros((), dtype=torch.float64, device=dev)

    def take(t):
        return torch.where(inside, gather(t.double(), pos), zero)

    x, Bm, C = (mag(take(i[k])) for k in ("x", "B", "C"))
    A = -torch.exp(i["A"].double()) if i.get("log_A") else i["A"].double()
    raw = take(i["delta"]) + (i["bias"].double() if i["bias"] is not None else 0)
    dt = torch.where(inside, raw.clamp(min=0) + torch.log1p(torch.exp(-raw.abs())) if i["softplus"] else raw, zero)
    slope = torch.sigmoid(raw) if i["softplus"] else torch.ones_like(raw)
    skip = mag(i["D"].double()) if i["D"] is not None else torch.zeros(D, device=dev, dtype=torch.float64)
    h = mag(i["state"].double()) if i["state"] is not None else torch.zeros(B, A.shape[0], D, device=dev, dtype=torch.float64)
    a, before, after = [], [], []
    for t in range(T):
        before.append(h)
        a.append(torch.exp(dt[t][:, None] * A))
        h = a[t] * h + (mag(dt[t]) * x[t])[:, None] * Bm[t][:, :, None]
        after.append(h)
    v = torch.stack([(after[t] * C[t][:, :, None]).sum(1) for t in range(T)]) + skip * x
    z = take(i["z"]) if i["z"] is not None else None
    gate = mag(silu(z)) if z is not None else torch.ones_like(v)
    inv = lambda t: gather(torch.where(inside, t, zero), pos)  # noqa: E731
    out = {"y": inv(v * gate), "state_out": h}
    if dy is None:
        return out
    g0 = mag(take(dy))
    e = g0 * gate
    carry = mag(dh.double()) if dh is not None else torch.zeros_like(h)
    dA, dx, dd, dB, dC = torch.zeros_like(A), [0] * T, [0] * T, [0] * T, [0] * T
    for t in reversed(range(T)):
        g = carry + C[t][:, :, None] * e[t][:, None]
        k = g * a[t] * before[t]
        p = (g * Bm[t][:, :, None]).sum(1)
        dx[t] = mag(dt[t]) * p + skip * e[t]
        dd[t] = (k * mag(A)).sum(1) + x[t] * p
        dA = dA + (k * mag(dt[t])[:, None]).sum(0)
        dB[t] = (g * (mag(dt[t]) * x[t])[:, None]).sum(2)
        dC[t] = (e[t][:, None] * after[t]).sum(2)
        carry = g * a[t]
    dd = torch.stack(dd) * slope
    out |= {"x": inv(torch.stack(dx)), "delta": inv(dd), "A": dA * mag(A) if i.get("log_A") else dA, "B": inv(torch.stack(dB)),
            "C": inv(torch.stack(dC)), "D": (e * x).sum((0, 1)), "bias": torch.where(inside, dd, zero).sum((0, 1)), "state": carry}
    if z is not None:
        # silu'(z) = p (1 + z (1 - p)) cancels at z = -1.278: the magnitudes on the way are p (1 + |z| (1 - p)),
        # whose roundings (u each) stay where the sum itself is near zero
        slope = torch.sigmoid(z) * (1 + z.abs() * (1 - torch.sigmoid(z))) if size else dsilu(z)
        out["z"] = inv(g0 * v * slope)
    return out


def act_of(u, act):
    if act == "silu":
        return silu(u), dsilu(u)
    if act == "tanh":
        return torch.tanh(u), 1 - torch.tanh(u) ** 2
    return u, torch.ones_like(u)


def conv_oracle(i, dy=None, dlast=None, size=False):
    mag = (lambda t: t.abs()) if size else (lambda t: t)
    dev = i["x"].device
    T, B, D = i["x"].shape
    K = i["w"].shape[0]
    pos, inside, n = positions(T, B, i["lengths"], i["reverse"], dev)
    zero = torch.zeros((), dtype=torch.float64, device=dev)

    def seen_of(t):
        head = torch.zeros(K - 1, B, D, device=dev, dtype=torch.float64) if i["state"] is None else i["state"].double()
        return torch.cat([head, torch.where(inside, gather(t.double(), pos), zero)])

    w, seen = i["w"].double(), seen_of(i["x"])
    b = i["b"].double() if i["b"] is not None else torch.zeros(D, device=dev, dtype=torch.float64)
    u = sum(w[k] * seen[k:k + T] for k in range(K)) + b
    usize = sum(w[k].abs() * seen[k:k + T].abs() for k in range(K)) + b.abs()
    y, slope = act_of(u, i["act"])
    if size:
        y, slope, w, seen = 1.1 * usize, 1.1 * (1 + usize), w.abs(), seen.abs()
    inv = lambda t: gather(torch.where(inside, t, zero), pos)  # noqa: E731
    at = n[None, :] + torch.arange(K - 1, device=dev)[:, None]
    out = {"y": inv(y), "state_out": gather(seen, at)}
    if dy is None:
        return out
    e = torch.where(inside, mag(gather(dy.double(), pos)) * slope, zero)
    after = torch.cat([e, e.new_zeros(K - 1, B, D)])
    full = torch.cat([e.new_zeros(K - 1, B, D), after])  # e at s - (K - 1) .. s + K - 1
    dseen = sum(w[k] * full[K - 1 - k:K - 1 - k + T + K - 1] for k in range(K))  # of the inputs 1 - K .. T - 1
    if dlast is not None:
        dseen = dseen.scatter_add(0, at[..., None].expand(-1, -1, D), mag(dlast.double()))
    out |= {"x": inv(dseen[K - 1:]), "state": dseen[:K - 1], "b": e.sum((0, 1)),
            "w": torch.stack([(e * seen[k:k + T]).sum((0, 1)) for k in range(K)])}
    return out


def check(got, value, bound, name):
    assert got.shape == value.shape, (name, got.shape, value.shape)
    if not got.numel():
        return
    fi = torch.finfo(got.dtype)
    half = fi.eps / 2 if got.dtype != torch.float32 else U
    lim = half * value.abs() + bound + fi.smallest_normal * fi.eps
    off = (got.double() - value).abs()
    worst = (off / lim).max().item()
    assert worst <= 1, "%s: %.3g times the bound" % (name, worst)


def scan_inputs(T, B, D, n, dtype, dev, seed=0, z=True, skip=True, bias=True, softplus=True, ragged=False,
                state=False, reverse=False, slices=False, poison=False, log_A=False):
    g = torch.Generator().manual_seed(seed)

    def rand(*s):
        return torch.randn(*s, generator=g)

    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
        lengths[:3] = torch.tensor([T, 0, 1], dtype=torch.int32)[:min(3, B)]
    x, zz = rand(T, B, D), rand(T, B, D)
    wide = torch.cat([x, zz], 2).to(dtype)
    delta = (0.7 * rand(T, B, D)).to(dtype) if softplus else (0.3 * rand(T, B, D).abs()).to(dtype)
    small = rand(T, B, 3 + 2 * n).to(dtype)
    if poison and ragged:  # what padding holds does not count
        bad = torch.arange(T)[:, None] >= lengths[None, :]
        for t in (wide, delta, small):
            t[bad] = float("nan")
    wide, delta, small = wide.to(dev), delta.to(dev), small.to(dev)
    i = {"x": wide[..., :D], "z": wide[..., D:] if z else None, "delta": delta, "B": small[..., 3:3 + n],
         "C": small[..., 3 + n:]}
    if not slices:
        i = {k: t.contiguous() if t is not None else None for k, t in i.items()}
    i |= {"A": -(0.2 + 2 * torch.rand(n, D, generator=g)).to(dev), "D": rand(D).to(dev) if skip else None,
          "bias": (rand(D) - 1).to(dev) if bias and softplus else None, "state": rand(B, n, D).to(dev) if state else None}
    i |= {"lengths": lengths.to(dev) if ragged else None, "softplus": softplus, "reverse": reverse, "log_A": log_A}
    if log_A:
        i["A"] = torch.log(-i["A"])
    dy, dh = rand(T, B, D).to(dtype).to(dev), rand(B, n, D).to(dev)
    return i, dy, dh


SCAN_LEAVES = ("x", "delta", "A", "B", "C", "D", "z", "bias", "state")


def scan_run(i, dy=None, dh=None):
    i = dict(i)
    if dy is not None:
        for k in SCAN_LEAVES:
            i[k] = i[k].detach().requires_grad_() if i[k] is not None else None
    y, h = ssm.selective_scan(i["x"], i["delta"], i["A"], i["B"], i["C"], i["D"], i["z"], i["bias"], i["softplus"],
                              i["lengths"], i["state"], True, i["reverse"], i["log_A"])
    out = {"y": y.detach(), "state_out": h.detach()}
    if dy is not None:
        names = [k for k in SCAN_LEAVES if i[k] is not None]
        outs, grads = ((y, h), (dy, dh)) if dh is not None else ((y,), (dy,))
        out |= dict(zip(names, torch.autograd.grad(outs, [i[k] for k in names], grads)))
    return out


def scan_compare(T, B, D, n, dtype, dev, state_grad=True, **kw):
    i, dy, dh = scan_inputs(T, B, D, n, dtype, dev, **kw)
    dh = dh if state_grad else None
    dyc = torch.nan_to_num(dy)
    want, size = scan_oracle(i, dyc, dh), scan_oracle(i, dyc, dh, size=True)
    u = 8 * (T + B + n + D / 16 + 16) * U
    got = scan_run(i, dy, dh)
    for k, t in got.items():
        check(t, want[k], u * size[k], k)
    with torch.no_grad():
        again = scan_run(i)
    assert torch.equal(again["y"], got["y"]) and torch.equal(again["state_out"], got["state_out"])


def conv_inputs(T, B, D, K, dtype, dev, seed=0, bias=True, act="silu", ragged=False, state=False, reverse=False,
                slices=False, poison=False):
    g = torch.Generator().manual_seed(seed)

    def rand(*s):
        return torch.randn(*s, generator=g)

    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
        lengths[:3] = torch.tensor([T, 0, 1], dtype=torch.int32)[:min(3, B)]
    wide = rand(T, B, 2 * D + 1).to(dtype)
    if poison and ragged:
        wide[torch.arange(T)[:, None] >= lengths[None, :]] = float("nan")
    wide = wide.to(dev)
    x = wide[..., :D]
    i = {"x": x if slices else x.contiguous(), "w": rand(K, D).to(dev) / K ** 0.5, "b": rand(D).to(dev) if bias else None,
         "state": rand(K - 1, B, D).to(dtype).to(dev) if state else None, "act": act, "reverse": reverse,
         "lengths": lengths.to(dev) if ragged else None}
    return i, rand(T, B, D).to(dtype).to(dev), rand(K - 1, B, D).to(dtype).to(dev)


CONV_LEAVES = ("x", "w", "b", "state")


def conv_run(i, dy=None, dlast=None):
    i = dict(i)
    if dy is not None:
        for k in CONV_LEAVES:
            i[k] = i[k].detach().requires_grad_() if i[k] is not None else None
    y, last = ssm.causal_conv(i["x"], i["w"], i["b"], i["act"], i["lengths"], i["state"], True, i["reverse"])
    out = {"y": y.detach(), "state_out": last.detach()}
    if dy is not None:
        names = [k for k in CONV_LEAVES if i[k] is not None]
        outs, grads = ((y, last), (dy, dlast)) if dlast is not None and last.numel() else ((y,), (dy,))
        out |= dict(zip(names, torch.autograd.grad(outs, [i[k] for k in names], grads)))
    return out


def conv_compare(T, B, D, K, dtype, dev, state_grad=True, **kw):
    i, dy, dlast = conv_inputs(T, B, D, K, dtype, dev, **kw)
    dlast = dlast if state_grad and K > 1 else None
    want, size = conv_oracle(i, dy, dlast), conv_oracle(i, dy, dlast, size=True)
    u = 8 * (T + B + K + 16) * U
    got = conv_run(i, dy, dlast)
    for k, t in got.items():
        check(t, want[k], u * size[k] if k != "state_out" else 0 * size[k], k)
    with torch.no_grad():
        again = conv_run(i)
    assert torch.equal(again["y"], got["y"]) and torch.equal(again["state_out"], got["state_out"])


# ------------------------------------------------------------------------- CPU
OPTIONS = [{}, {"ragged": True, "poison": True}, {"state": True}, {"reverse": True},
           {"ragged": True, "state": True, "reverse": True}]
SCAN_OPTIONS = OPTIONS + [{"log_A": True}]


@pytest.mark.parametrize("kw", SCAN_OPTIONS)
def test_selective_scan_cpu(kw):
    scan_compare(7, 4, 6, 3, torch.float32, "cpu", **kw)


@pytest.mark.parametrize("kw", OPTIONS + [{"act": None, "bias": False}, {"act": "tanh"}])
@pytest.mark.parametrize("K", [1, 2, 4, 8])
def test_causal_conv_cpu(K, kw):
    conv_compare(6, 4, 5, K, torch.float32, "cpu", **kw)


def _differences(oracle, i, leaves, out_grads, kw):
    want = oracle(i, *out_grads)
    for name in leaves:
        if i[name] is None:
            continue
        flat = i[name].view(-1)
        for j in range(0, flat.numel(), max(1, flat.numel() // 7)):
            old, f = flat[j].item(), []
            for s in (1, -1):
                flat[j] = old + s * 1e-6
                o = oracle(i)
                f.append((o["y"] * out_grads[0]).sum() + (o["state_out"] * out_grads[1]).sum())
            flat[j] = old
            assert abs((f[0] - f[1]) / 2e-6 - want[name].reshape(-1)[j]) < 1e-6 * (1 + abs(want[name].reshape(-1)[j])), name


@pytest.mark.parametrize("kw", OPTIONS[:1] + OPTIONS[2:] + [{"softplus": False}, {"z": False, "skip": False}, {"log_A": True}])
def test_scan_oracle_gradients_against_differences(kw):
    i, dy, dh = scan_inputs(5, 4, 3, 2, torch.float64, "cpu", **kw)
    i = {k: t.double() if torch.is_tensor(t) and t.is_floating_point() else t for k, t in i.items()}
    _differences(scan_oracle, i, SCAN_LEAVES, (dy.double(), dh.double()), kw)


@pytest.mark.parametrize("kw", OPTIONS[:1] + OPTIONS[2:])
def test_conv_oracle_gradients_against_differences(kw):
    i, dy, dl = conv_inputs(5, 4, 3, 3, torch.float64, "cpu", **kw)
    i = {k: t.double() if torch.is_tensor(t) and t.is_floating_point() else t for k, t in i.items()}
    _differences(conv_oracle, i, CONV_LEAVES, (dy.double(), dl.double()), kw)


def _steps(dev, dtype, T=6, B=3, D=20, n=5, K=4, n_bytes=None):
    """A prompt and then single tokens give what the whole sequence gives."""
    i, _, _ = scan_inputs(T, B, D, n, dtype, dev, seed=3, slices=True)
    c, _, _ = conv_inputs(T, B, D, K, dtype, dev, seed=4, slices=True)
    with torch.no_grad():
        want, cwant = scan_run(i), conv_run(c)
        cut = lambda t, a, b: t[a:b] if t is not None else None  # noqa: E731
        for P in (1, T - 2):
            p = scan_run({k: cut(t, 0, P) if k in ("x", "delta", "B", "C", "z") else t for k, t in i.items()})
            q = conv_run({k: cut(t, 0, P) if k == "x" else t for k, t in c.items()})
            h, s = p["state_out"], q["state_out"]
            ys, cs = [], []
            for t in range(P, T):
                ys.append(ssm.selective_scan_step(i["x"][t], i["delta"][t], i["A"], i["B"][t], i["C"][t], h, i["D"],
                                                  i["z"][t], i["bias"], i["softplus"]))
                cs.append(ssm.causal_conv_step(c["x"][t], s, c["w"], c["b"], c["act"]))
            size = scan_oracle(i, size=True)
            u = 8 * (T + n + 32) * U
            fi = torch.finfo(dtype)
            half = fi.eps if dtype != torch.float32 else 0.0  # two roundings, one on each side
            y = torch.stack(ys).double()
            assert ((y - want["y"][P:].double()).abs() <= half * y.abs() + 2 * u * size["y"][P:]).all()
            assert ((h - want["state_out"]).double().abs() <= 2 * u * size["state_out"]).all()
            assert torch.equal(s, cwant["state_out"])
            csize = conv_oracle(c, size=True)["y"][P:]
            y = torch.stack(cs).double()
            assert ((y - cwant["y"][P:].double()).abs() <= half * y.abs() + 2 * u * csize).all()


def test_steps_cpu():
    _steps("cpu", torch.float32)


def _refusals(dev):
    T, B, D, n = 3, 2, 4, 2
    mk = lambda *s: torch.randn(*s, device=dev)  # noqa: E731
    x, A, bm, w = mk(T, B, D), -torch.ones(n, D, device=dev), mk(T, B, n), mk(3, D)
    scan, conv = ssm.selective_scan, ssm.causal_conv
    st = mk(B, n, D)
    calls = [lambda: scan(x[0], x, A, bm, bm), lambda: scan(x, x[:2], A, bm, bm), lambda: scan(x, x, A.t(), bm, bm),
             lambda: scan(x, x, A, bm[..., :1], bm), lambda: scan(x, x, A, bm, bm.half()), lambda: scan(x, x, A, bm, bm, D=mk(D + 1)),
             lambda: scan(x, x, A, bm, bm, z=mk(T, B, D + 1)), lambda: scan(x, x, A, bm, bm, lengths=torch.ones(B, device=dev)),
             lambda: scan(x, x, A, bm, bm, lengths=torch.ones(B + 1, device=dev, dtype=torch.int32)),
             lambda: scan(x, x, A, bm, bm, initial_state=mk(B, D, n)), lambda: scan(x, x, A.double(), bm, bm),
             lambda: scan(x[:0], x[:0], A, bm[:0], bm[:0]), lambda: scan(x, x, -torch.ones(65, D, device=dev), mk(T, B, 65), mk(T, B, 65)),
             lambda: ssm.selective_scan_step(x[0], x[0], A, bm[0], bm[0], st.half()),
             lambda: ssm.selective_scan_step(x[0], x[0], A, bm[0], bm[0], st.transpose(1, 2).contiguous().transpose(1, 2)),
             lambda: ssm.selective_scan_step(x[0].clone().requires_grad_(), x[0], A, bm[0], bm[0], st),
             lambda: conv(x, mk(9, D)), lambda: conv(x, mk(3, D + 1)), lambda: conv(x, w.half()), lambda: conv(x[0], w),
             lambda: conv(x, w, mk(D + 1)), lambda: conv(x, w, initial_state=mk(3, B, D)),
             lambda: conv(x, w, initial_state=mk(2, B, D).half()), lambda: conv(x[:, :0], w),
             lambda: ssm.causal_conv_step(x[0], mk(2, D, B).transpose(1, 2), w), lambda: ssm.causal_conv_step(x, mk(2, B, D), w),
             lambda: ssm.causal_conv_step(x[0], mk(2, B, D), w.clone().requires_grad_())]
    for k, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail("call %d was taken" % k)
    with pytest.raises(KeyError):
        conv(x, w, activation="swoosh")


def test_refusals_cpu():
    _refusals("cpu")


# ------------------------------------------------------------------------- GPU
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,D,K", [(1, 1, 1, 2), (3, 2, 8, 4), (19, 5, 24, 4), (33, 3, 203, 3), (40, 2, 520, 8),
                                     (16, 1, 64, 1), (17, 4, 72, 5), (130, 7, 40, 2), (5, 70, 16, 4)])
def test_causal_conv_gpu(cuda, T, B, D, K, dtype):
    conv_compare(T, B, D, K, dtype, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", OPTIONS + [{"act": None, "bias": False}, {"act": "tanh", "slices": True},
                                          {"state": True, "state_grad": False}])
@pytest.mark.parametrize("T,B,D,K", [(37, 4, 24, 4), (2, 3, 16, 8), (35, 5, 33, 3)])
def test_causal_conv_options_gpu(cuda, T, B, D, K, kw):
    conv_compare(T, B, D, K, torch.bfloat16, cuda, **kw)
    conv_compare(T, B, D, K, torch.float32, cuda, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,D,n", [(1, 1, 1, 1), (1, 3, 64, 16), (16, 2, 64, 16), (17, 2, 68, 16), (50, 3, 203, 8),
                                     (33, 2, 130, 5), (40, 1, 96, 24), (21, 2, 70, 33), (23, 2, 64, 64), (9, 5, 200, 32)])
def test_selective_scan_gpu(cuda, T, B, D, n, dtype):
    scan_compare(T, B, D, n, dtype, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", SCAN_OPTIONS + [{"z": False}, {"skip": False, "bias": False}, {"softplus": False},
                                          {"slices": True}, {"state_grad": False, "z": False}])
@pytest.mark.parametrize("T,B,D,n", [(37, 4, 72, 16), (2, 3, 33, 6), (70, 4, 64, 40)])
def test_selective_scan_options_gpu(cuda, T, B, D, n, kw):
    scan_compare(T, B, D, n, torch.bfloat16, cuda, **kw)
    scan_compare(T, B, D, n, torch.float32, cuda, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("T,B,D,n", [(1500, 1, 64, 16), (700, 2, 130, 4), (515, 3, 64, 48)])
@pytest.mark.parametrize("kw", [{}, {"ragged": True, "state": True, "reverse": True, "poison": True}])
def test_selective_scan_long_gpu(cuda, T, B, D, n, kw):
    scan_compare(T, B, D, n, torch.bfloat16, cuda, **kw)
    scan_compare(T, B, D, n, torch.float32, cuda, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_gpu(cuda, dtype):
    _steps(cuda, dtype)
    _steps(cuda, dtype, T=5, B=9, D=136, n=33, K=8)


@pytest.mark.gpu
def test_refusals_gpu(cuda):
    _refusals(cuda)
    x = torch.ones(2, 2, 4, device=cuda, dtype=torch.float64)
    with pytest.raises(N.NativeError):
        ssm.causal_conv(x, torch.ones(2, 4, device=cuda))
    with pytest.raises(ValueError):
        ssm.causal_conv(x.float(), torch.ones(2, 4))


@pytest.mark.gpu
def test_same_bits_and_sinks_gpu(cuda):
    """Two runs give the same bits; flat-buffer gradients are added to."""
    i, dy, dh = scan_inputs(300, 3, 200, 16, torch.bfloat16, cuda)
    a, b = scan_run(i, dy, dh), scan_run(i, dy, dh)
    assert all(torch.equal(a[k], b[k]) for k in a)
    c, cdy, cdl = conv_inputs(300, 3, 200, 4, torch.bfloat16, cuda)
    ca, cb = conv_run(c, cdy, cdl), conv_run(c, cdy, cdl)
    assert all(torch.equal(ca[k], cb[k]) for k in ca)
    ps = {k: i[k].clone().requires_grad_() for k in ("A", "D", "bias")} | {k: c[k].clone().requires_grad_() for k in ("w", "b")}
    for p in ps.values():
        p._kfb_grad_sink = torch.full_like(p, 3.0)
    y, h = ssm.selective_scan(i["x"].clone().requires_grad_(), i["delta"], ps["A"], i["B"], i["C"], ps["D"], i["z"], ps["bias"],
                              return_state=True)
    torch.autograd.backward((y, h), (dy, dh))
    y, s = ssm.causal_conv(c["x"].clone().requires_grad_(), ps["w"], ps["b"], "silu", return_state=True)
    torch.autograd.backward((y, s), (cdy, cdl))
    for k, p in ps.items():
        assert p.grad is None
        torch.testing.assert_close(p._kfb_grad_sink, (a if k in a and k != "w" and k != "b" else ca)[k] + 3, rtol=1e-6, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [2, 4, 6])
def test_causal_conv_infinite_inputs_gpu(cuda, K):
    """An infinite input reaches the outputs and gradients of its own channel and window alone."""
    T, B, D = 37, 2, 24
    i, dy, _ = conv_inputs(T, B, D, K, torch.float32, cuda, act=None)
    i["lengths"] = torch.tensor([20, 37], dtype=torch.int32, device=cuda)
    clean = conv_run(i, dy)
    x = i["x"].clone()
    x[19, 0, 3], x[5, 1, 7] = float("inf"), float("nan")
    i["x"] = x
    got = conv_run(i, dy)
    bad = torch.zeros(T, B, D, dtype=torch.bool, device=cuda)
    bad[19:20, 0, 3] = True
    bad[5:5 + K, 1, 7] = True
    assert torch.equal(~torch.isfinite(got["y"]), bad)
    assert torch.equal(got["x"], clean["x"]) and torch.equal(got["b"], clean["b"])
    bad = torch.zeros(K, D, dtype=torch.bool, device=cuda)
    bad[:, 7] = True
    bad[K - 1, 3] = True  # of sequence 0 only its last row sees the infinity, through the last tap
    assert torch.equal(~torch.isfinite(got["w"]), bad)
    assert torch.equal(got["w"][~bad], clean["w"][~bad])


@pytest.mark.gpu
def test_causal_conv_many_short_runs_gpu(cuda):
    """2^20 positions of one narrow sequence: as many runs as a launch takes."""
    x = torch.randn(1 << 20, 1, 8, device=cuda)
    w = torch.randn(2, 8, device=cuda)
    y, last = ssm.causal_conv(x, w, return_state=True)
    want = w[1] * x
    want[1:] += w[0] * x[:-1]
    torch.testing.assert_close(y, want, rtol=1e-6, atol=1e-6)
    assert torch.equal(last, x[-1:])
    with pytest.raises(ValueError):
        ssm.causal_conv(torch.zeros((1 << 20) + 1, 1, 1, device=cuda), w[:, :1].contiguous())


@pytest.mark.gpu
def test_one_parameter_twice_gpu(cuda):
    """One tensor given as skip and as bias: its flat-buffer gradient is the sum of both."""
    i, dy, _ = scan_inputs(40, 2, 72, 5, torch.float32, cuda)
    p = i["D"].clone().requires_grad_()
    want = torch.autograd.grad(ssm.selective_scan(i["x"], i["delta"], i["A"], i["B"], i["C"], p, i["z"], p), p, dy)[0]
    q = i["D"].clone().requires_grad_()
    q._kfb_grad_sink = torch.zeros_like(q)
    y = ssm.selective_scan(i["x"], i["delta"], i["A"], i["B"], i["C"], q, i["z"], q)
    y.backward(dy)
    torch.testing.assert_close(q._kfb_grad_sink + q.grad, want, rtol=1e-6, atol=1e-6)


def test_split_columns_too_many_slices():
    n = ssm.F_ops._CAT_MAX + 1
    with pytest.raises(ValueError, match="at most"):
        ssm.split_columns(torch.zeros(2, n), (1,) * n)


def test_scalar_parameters_are_refused():
    x, s = torch.zeros(2, 3, 4), torch.zeros(())
    with pytest.raises(ValueError):
        ssm.selective_scan(x, x, s, x[..., :1], x[..., :1])
    with pytest.raises(ValueError):
        ssm.selective_scan_step(x[0], x[0], s, x[0, :, :1], x[0, :, :1], torch.zeros(3, 1, 4))
    with pytest.raises(ValueError):
        ssm.causal_conv(x, s)
    with pytest.raises(ValueError):
        ssm.causal_conv_step(x[0], x[:1].contiguous(), s)


@pytest.mark.parametrize("T,B,D", [(1, 1, 1), (16, 1, 64), (40, 3, 130), (1024, 64, 2048), (874, 16, 1600)])
def test_scan_reads_inside_its_saved_states(T, B, D):
    """Every wave of the backward, also one without states, reads inside the saved states (the numbers are the
    kernel's own, evaluated on the host)."""
    for n in range(1, ssm.MAX_STATES + 1):
        size, at = N.query("kfb_ssm_floats", 1, T, B, D, n), N.query("kfb_ssm_furthest_state", T, B, D, n)
        assert size // 2 <= at < size, (n, at, size)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 3, 7, 9, 10, 11, 12, 36])
def test_selective_scan_partly_filled_waves_gpu(cuda, n):
    scan_compare(35, 3, 72, n, torch.bfloat16, cuda)
    scan_compare(70, 2, 33, n, torch.float32, cuda, ragged=True, poison=True, state=True, reverse=True)


def _steps_count_as_changes(dev):
    """A step is an in-place change of its state that autograd knows of."""
    i, _, _ = scan_inputs(3, 2, 8, 4, torch.float32, dev)
    c, _, _ = conv_inputs(3, 2, 8, 4, torch.float32, dev, state=True)
    h, s = torch.zeros(2, 4, 8, device=dev), c["state"]
    w = c["w"].clone().requires_grad_()
    y = ssm.causal_conv(c["x"], w, c["b"], "silu", initial_state=s)
    versions = s._version, h._version

    def steps():
        ssm.causal_conv_step(c["x"][0], s, c["w"], c["b"], "silu")
        ssm.selective_scan_step(i["x"][0], i["delta"][0], i["A"], i["B"][0], i["C"][0], h)

    with torch.no_grad():
        steps()
    assert s._version > versions[0] and h._version > versions[1]
    with torch.inference_mode():  # tensors made here count no changes
        h, s = torch.zeros(2, 4, 8, device=dev), torch.zeros(3, 2, 8, device=dev)
        steps()
        assert torch.equal(s[-1], c["x"][0]) and h.abs().sum() > 0
    return y


def test_steps_count_as_changes_of_their_state_cpu():
    _steps_count_as_changes("cpu")


@pytest.mark.gpu
def test_steps_count_as_changes_of_their_state_gpu(cuda):
    y = _steps_count_as_changes(cuda)
    with pytest.raises(RuntimeError, match="inplace"):  # the state was kept for the filter's gradient
        y.sum().backward()


INF = float("inf")


def _mask(shape, dev, *at):
    m = torch.zeros(shape, dtype=torch.bool, device=dev)
    for a in at:
        m[a] = True
    return m


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, {"skip": False, "z": False}, {"skip": False}])
@pytest.mark.parametrize("n", [1, 3, 4, 5, 8, 9, 16, 33, 40])
def test_selective_scan_infinite_input_gpu(cuda, n, kw):
    """An infinite input gives infinities, not NaN, and only in what it reaches (with maps and skip of one sign, so that
    no infinities of opposite signs meet)."""
    T, B, D, t = 37, 2, 72, 20
    i, dy, dh = scan_inputs(T, B, D, n, torch.float32, cuda, state=True, **kw)
    for k in ("B", "C", "D"):
        i[k] = i[k].abs() if i[k] is not None else None
    clean = scan_run(i, dy, dh)
    i["x"] = i["x"].clone()
    i["x"][t, 0, 3] = INF
    got = scan_run(i, dy, dh)
    after, there, row = (slice(t, None), 0, 3), (t, 0, 3), (t, 0)
    bad = {"y": _mask((T, B, D), cuda, after), "x": _mask((T, B, D), cuda), "delta": _mask((T, B, D), cuda, after),
           "z": _mask((T, B, D), cuda, after), "A": _mask((n, D), cuda, (slice(None), 3)),
           "B": _mask((T, B, n), cuda, row), "C": _mask((T, B, n), cuda, (slice(t, None), 0)),
           "D": _mask((D,), cuda, 3), "bias": _mask((D,), cuda, 3), "state": _mask((B, n, D), cuda),
           "state_out": _mask((B, n, D), cuda, (0, slice(None), 3))}
    for k, v in got.items():
        assert torch.equal(~torch.isfinite(v), bad[k]), k
        assert torch.equal(v[~bad[k]], clean[k][~bad[k]]), k
    gate = 1.0 if i["z"] is None else i["z"][after]
    assert torch.equal(got["y"][after], torch.full((T - t,), INF, device=cuda) * gate)
    if i["z"] is not None:
        z = i["z"][after].double()
        s = torch.sigmoid(z)
        assert torch.equal(got["z"][after].double(), INF * dy[after].double() * (s * (1 + z * (1 - s))))
    assert (got["state_out"][0, :, 3] == INF).all()


def _infinite_last_input(dev, n, state_grad):
    """What stands behind a sequence's end, in its tile or in padding, adds nothing, not even zero times infinity."""
    T, B, D = 37, 2, 72
    i, dy, dh = scan_inputs(T, B, D, n, torch.float32, dev)
    dh = dh if state_grad else None
    i["lengths"] = torch.tensor([20, 37], dtype=torch.int32, device=dev)
    clean = scan_run(i, dy, dh)
    i["x"] = i["x"].clone()
    i["x"][19, 0, 3], i["x"][36, 1, 7] = INF, -INF
    got = scan_run(i, dy, dh)
    at, rows, ch = ((19, 0, 3), (36, 1, 7)), ((19, 0), (36, 1)), (3, 7)
    m = lambda *s: _mask(s, dev)  # noqa: E731
    bad = {"y": _mask((T, B, D), dev, *at), "x": m(T, B, D), "delta": _mask((T, B, D), dev, *at),
           "z": _mask((T, B, D), dev, *at), "A": m(n, D), "B": _mask((T, B, n), dev, *rows),
           "C": _mask((T, B, n), dev, *rows), "D": _mask((D,), dev, *ch), "bias": _mask((D,), dev, *ch),
           "state_out": _mask((B, n, D), dev, (0, slice(None), 3), (1, slice(None), 7))}
    for k, v in got.items():
        assert torch.equal(~torch.isfinite(v), bad[k]), k
        assert torch.equal(v[~bad[k]], clean[k][~bad[k]]), k


@pytest.mark.parametrize("state_grad", [True, False])
def test_selective_scan_infinite_last_input_cpu(state_grad):
    _infinite_last_input("cpu", 5, state_grad)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 5, 16, 40])
@pytest.mark.parametrize("state_grad", [True, False])
def test_selective_scan_infinite_last_input_gpu(cuda, n, state_grad):
    _infinite_last_input(cuda, n, state_grad)


@pytest.mark.gpu
def test_selective_scan_infinite_state_over_chunks_gpu(cuda):
    """An infinite state stays infinite where the decays of a whole chunk multiply to zero."""
    T, D, n, t = 1500, 64, 16, 100
    i, _, _ = scan_inputs(T, 1, D, n, torch.float32, cuda, z=False, skip=False)
    i["A"], i["B"], i["C"] = 8 * i["A"], i["B"].abs(), i["C"].abs()
    i["x"][t, 0, 3] = INF
    with torch.no_grad():
        got = scan_run(i)
    assert torch.equal(~torch.isfinite(got["y"]), _mask((T, 1, D), cuda, (slice(t, None), 0, 3)))
    assert (got["y"][t:, 0, 3] == INF).all() and (got["state_out"][0, :, 3] == INF).all()


@pytest.mark.gpu
@pytest.mark.parametrize("K", [2, 4, 6])
def test_causal_conv_infinite_gradient_gpu(cuda, K):
    """An infinite gradient of y gives infinities, not NaN, and only in what it reaches, wherever in a run it stands."""
    T, B, D = 64, 2, 24
    i, dy, _ = conv_inputs(T, B, D, K, torch.float32, cuda, act=None)
    i["x"], i["w"] = i["x"].abs() + 0.1, i["w"].abs() + 0.1
    clean = conv_run(i, dy)
    for t in range(K, 20):
        bad = dy.clone()
        bad[t, 1, 5] = INF
        got = conv_run(i, bad)
        dx, dw, db = (torch.zeros_like(got[k], dtype=torch.bool) for k in ("x", "w", "b"))
        dx[t - K + 1:t + 1, 1, 5] = True
        dw[:, 5] = True
        db[5] = True
        for k, m in (("x", dx), ("w", dw), ("b", db)):
            assert (got[k][m] == INF).all() and torch.equal(got[k][~m], clean[k][~m]), (t, k)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3, 4, 5, 8, 9, 16, 33, 40])
def test_selective_scan_infinite_gradient_gpu(cuda, n):
    """An infinite gradient of y gives infinities, not NaN, and only in what it reaches (inputs, maps and skip of one sign)."""
    T, B, D, t = 37, 2, 72, 20
    i, dy, dh = scan_inputs(T, B, D, n, torch.float32, cuda, state=True, z=False)
    for k in ("x", "B", "C", "D", "state"):
        i[k] = i[k].abs()
    clean = scan_run(i, dy, dh)
    dy = dy.clone()
    dy[t, 0, 3] = INF
    got = scan_run(i, dy, dh)
    before, ch, m = (slice(0, t + 1), 0, 3), (slice(None), 3), lambda *s: _mask(s, cuda)  # noqa: E731
    bad = {"y": m(T, B, D), "state_out": m(B, n, D), "x": _mask((T, B, D), cuda, before), "delta": _mask((T, B, D), cuda, before),
           "A": _mask((n, D), cuda, ch), "B": _mask((T, B, n), cuda, (slice(0, t + 1), 0)), "C": _mask((T, B, n), cuda, (t, 0)),
           "D": _mask((D,), cuda, 3), "bias": _mask((D,), cuda, 3), "state": _mask((B, n, D), cuda, (0, slice(None), 3))}
    for k, v in got.items():
        assert torch.equal(~torch.isfinite(v), bad[k]), k
        assert torch.equal(v[~bad[k]], clean[k][~bad[k]]), k
    for k in ("x", "B", "C", "D", "state"):
        assert (got[k][bad[k]] == INF).all(), k


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, {"ragged": True, "poison": True}, {"state_grad": False, "reverse": True}])
def test_causal_conv_of_one_tap_with_its_empty_state_gpu(cuda, kw):
    conv_compare(9, 3, 24, 1, torch.bfloat16, cuda, state=True, **kw)
