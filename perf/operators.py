"""The sequence and normalisation operators as they are measured: group norm with an activation on channels-last
tensors, the short causal convolution over time, and the selective state space scan, for training, for prompts and
for single tokens.

``own`` is false: the operators in elementary torch operations in 32 bits, from their formulas.  ``own`` is true: the
framework's calls (``ops.nn.group_norm``, ``ops.ssm``).

Layouts are the framework's: images [N, H, W, C], sequences time-major [T, B, D]; parameters in 32 bits.  The inputs of
the sequence operators are column slices of the projections' outputs, as a layer has them.
"""

import math
import random  # noqa: F401  (the generator that draw() takes)

import torch

own = False

EPS = 1e-5
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one small image through a norm at inference: latency
        dict(name="norm one image", op="norm", mode="infer", n=1, h=14, w=14, c=256, groups=32, act="silu", dtype="bf16"),
        # the wide early layers of a residual net in training, a batch as data-parallel ranks hold it
        dict(name="norm 56x56x256 train", op="norm", mode="train", n=32, h=56, w=56, c=256, groups=32, act="relu",
             dtype="bf16"),
        # an inception block's width: nine channels a group, odd images, fp32
        dict(name="norm 35x35x288 train", op="norm", mode="train", n=7, h=35, w=35, c=288, groups=32, act="silu",
             dtype="fp32"),
        # the norm of every token of a speech batch between two sequence layers
        dict(name="norm tokens", op="norm", mode="infer", n=874 * 16, h=1, w=1, c=1600, groups=8, act="linear",
             dtype="bf16"),
        # a speech batch (874 frames after the convolutions) in training
        dict(name="conv speech train", op="conv", mode="train", t=874, b=16, d=1600, k=4, act="silu", ragged=False,
             dtype="bf16"),
        # padded prompts of odd width, with the state that serving goes on from
        dict(name="conv prompts", op="conv", mode="prompt", t=333, b=3, d=805, k=3, act="silu", ragged=True,
             dtype="fp32"),
        # one token for each of 64 streams
        dict(name="conv step", op="conv", mode="step", t=1, b=64, d=1600, k=4, act="silu", ragged=False, dtype="bf16"),
        # one token for each of 64 streams
        dict(name="scan step", op="scan", mode="step", t=1, b=64, d=1600, s=16, gate=True, ragged=False, dtype="bf16"),
        # one long recording: few channels, many frames
        dict(name="scan long prompt", op="scan", mode="prompt", t=8192, b=1, d=1600, s=16, gate=True, ragged=False,
             dtype="bf16"),
        # a speech batch through the scan at inference
        dict(name="scan speech prompt", op="scan", mode="prompt", t=874, b=16, d=1600, s=16, gate=True, ragged=True,
             dtype="bf16"),
        # a speech batch through the scan in training
        dict(name="scan speech train", op="scan", mode="train", t=874, b=16, d=1600, s=16, gate=True, ragged=False,
             dtype="bf16"),
        # a small padded batch of odd width in fp32, without the gate
        dict(name="scan small train", op="scan", mode="train", t=201, b=5, d=203, s=8, gate=False, ragged=True,
             dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "conv", "scan"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "norm":
        tokens = rng.random() < 0.3  # one token a row: groups of 16 values and more
        groups, per = rng.choice([1, 2, 4, 8, 16, 32]), _log(rng, 16, 200) if tokens else _log(rng, 1, 80)
        c = groups * per
        most = 25_000_000 // c
        if tokens:
            n, h, w = max(1, min(_log(rng, 1, 20000), most)), 1, 1
        else:
            h, w = _log(rng, 4, 112), _log(rng, 4, 112)
            n = max(1, min(_log(rng, 1, 64), most // (h * w)))
        return dict(op=op, mode=rng.choice(["infer", "train"]), n=n, h=h, w=w, c=c, groups=groups,
                    act=rng.choice(["linear", "relu", "silu"]), dtype=dtype)
    mode = rng.choice(["train", "prompt", "step"])
    b, d, ragged = _log(rng, 1, 64), _log(rng, 16, 2048), rng.random() < 0.5 and mode != "step"
    if op == "conv":
        t = 1 if mode == "step" else max(1, min(_log(rng, 1, 16384), 22_000_000 // (b * d)))
        return dict(op=op, mode=mode, t=t, b=b, d=d, k=rng.randint(2, 8), act=rng.choice(["linear", "silu"]), ragged=ragged,
                    dtype=dtype)
    s = rng.choice([4, 8, 16, 16, 16, 24, 32, 64])
    t = 1 if mode == "step" else max(1, min(_log(rng, 1, 16384), 350_000_000 // (b * d * s)))
    return dict(op=op, mode=mode, t=t, b=b, d=d, s=s, gate=rng.random() < 0.7, ragged=ragged, dtype=dtype)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    train = case["mode"] == "train"
    if case["op"] == "norm":
        values, c = case["n"] * case["h"] * case["w"] * case["c"], case["c"]
        return {"bytes": values * size * (4 if train else 2) + 4 * c * (4 if train else 2), "flops": values * (30 if train else 10)}
    values, rows = case["t"] * case["b"] * case["d"], case["t"] * case["b"]
    if case["op"] == "conv":
        k = case["k"]
        small = 4 * case["d"] * (k + 1) * (2 if train else 1)
        state = 0 if train else (k - 1) * case["b"] * case["d"] * size * (2 if case["mode"] == "step" else 1)
        return {"bytes": values * size * (4 if train else 2) + small + state, "flops": values * (6 * k + 12 if train else 2 * k + 4)}
    s, gate = case["s"], int(case["gate"])
    wide = (6 + 2 * gate) if train else (3 + gate)  # x, delta, (z), y; in training their gradients and that of y too
    state = 0 if train else case["b"] * s * case["d"] * 4 * (2 if case["mode"] == "step" else 1)
    small = 4 * case["d"] * (s + 2) * (2 if train else 1)
    return {"bytes": values * size * wide + rows * 2 * s * size * (2 if train else 1) + state + small,
            "flops": values * (s * (26 if train else 8) + 20)}


# ------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, train = _TYPES[case["dtype"]], case["mode"] == "train"

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["op"] == "norm":
        n, h, w, c = case["n"], case["h"], case["w"], case["c"]
        s = {"x": (rand(n, h, w, c) * 1.5 + rand(c)).to(dt), "gamma": 1 + 0.1 * rand(c), "beta": 0.1 * rand(c),
             "dy": rand(n, h, w, c).to(dt) if train else None}
        leaves = ("x", "gamma", "beta")
    else:
        t, b, d = case["t"], case["b"], case["d"]
        both = rand(t, b, 2 * d).to(dt)  # the input projection: the channels and their gate
        s = {"x": both[..., :d], "dy": rand(t, b, d).to(dt) if train else None, "lengths": None}
        if case["ragged"]:
            lengths = torch.randint(0, t + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
            lengths[b - 1] = t
            s["lengths"] = lengths
        if case["op"] == "conv":
            k = case["k"]
            s |= {"w": rand(k, d) / math.sqrt(k), "bias": 0.1 * rand(d)}
            s["state"] = rand(k - 1, b, d).to(dt) if case["mode"] == "step" else None
            leaves = ("x", "w", "bias")
        else:
            n = case["s"]
            rank = max(1, d // 16)
            small = rand(t, b, rank + 2 * n).to(dt)  # the projection that gives the step's rank, B and C
            step = torch.exp(torch.rand(d, generator=g, device="cuda") * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
            s |= {"delta": (0.5 * rand(t, b, d)).to(dt), "A": -(torch.arange(1, n + 1, device="cuda").float()[:, None] * (1 + 0.1 * rand(n, d).abs())),
                  "B": small[..., rank:rank + n], "C": small[..., rank + n:], "skip": 1 + 0.1 * rand(d),
                  "z": both[..., d:] if case["gate"] else None,
                  "bias": step + torch.log(-torch.expm1(-step))}  # softplus(bias) = step
            s["state"] = rand(b, n, d) if case["mode"] == "step" else None
            leaves = ("x", "delta", "A", "B", "C", "skip", "bias") + (("z",) if case["gate"] else ())
    s = {name: v.detach() if v is not None else None for name, v in s.items()}
    if train:
        for name in leaves:
            s[name].requires_grad_()
    return {"case": case, "leaves": leaves, **s}


# ------------------------------------------------------------------------------------------------------- plain forms
def _silu(u):
    return u * torch.sigmoid(u)


def _dsilu(u):
    p = torch.sigmoid(u)
    return p * (1 + u * (1 - p))


def _act(u, act):
    return u.clamp(min=0) if act == "relu" else _silu(u) if act == "silu" else u


def _dact(u, act):
    return (u > 0).to(u.dtype) if act == "relu" else _dsilu(u) if act == "silu" else torch.ones_like(u)


def _inside(s, t):
    """[T, B, 1]: whether a row is inside its sequence; None: every row is."""
    return None if s["lengths"] is None else (torch.arange(t, device="cuda")[:, None] < s["lengths"][None, :])[..., None]


def _only(v, inside):
    return v if inside is None else torch.where(inside, v, torch.zeros((), device=v.device, dtype=v.dtype))


def _norm_plain(s):
    case, dt = s["case"], s["x"].dtype
    n, c, groups = case["n"], case["c"], case["groups"]
    x = s["x"].detach().float().view(n, -1, groups, c // groups)
    gamma, beta = (s[p].detach().view(groups, -1) for p in ("gamma", "beta"))
    off = x - x.mean((1, 3), keepdim=True)
    r = torch.rsqrt((off * off).mean((1, 3), keepdim=True) + EPS)
    xh = off * r
    u = xh * gamma + beta
    y = _act(u, case["act"]).view(s["x"].shape).to(dt)
    if s["dy"] is None:
        return {"y": y}
    e = s["dy"].float().view(x.shape) * _dact(u, case["act"])
    eg = e * gamma
    dx = r * (eg - eg.mean((1, 3), keepdim=True) - xh * (eg * xh).mean((1, 3), keepdim=True))
    return {"y": y, "x": dx.view(s["x"].shape).to(dt), "gamma": (e * xh).sum((0, 1)).view(c), "beta": e.sum((0, 1)).view(c)}


def _conv_plain(s):
    case = s["case"]
    t, k, dt = case["t"], case["k"], s["x"].dtype
    x, w, bias = (s[p].detach().float() for p in ("x", "w", "bias"))
    inside = _inside(s, t)
    before = torch.zeros_like(x[:1]).expand(k - 1, -1, -1) if s["state"] is None else s["state"].float()
    seen = torch.cat([before, _only(x, inside)])  # row t + K - 1 is x_t
    pre = bias + sum(w[j] * seen[j:j + t] for j in range(k))
    y = _only(_act(pre, case["act"]), inside).to(dt)
    if case["mode"] == "step":
        s["state"].copy_(seen[t:])
        return {"y": y[0], "state": s["state"]}
    if case["mode"] == "prompt":
        if inside is None:
            return {"y": y, "state": seen[t:].to(dt)}
        at = s["lengths"].long()[None, :] + torch.arange(k - 1, device="cuda")[:, None]
        return {"y": y, "state": torch.gather(seen, 0, at[..., None].expand(-1, -1, x.shape[2])).to(dt)}
    e = _only(s["dy"].float() * _dact(pre, case["act"]), inside)
    after = torch.cat([e, torch.zeros_like(e[:1]).expand(k - 1, -1, -1)])
    dx = _only(sum(w[j] * after[k - 1 - j:k - 1 - j + t] for j in range(k)), inside).to(dt)
    dw = torch.stack([(e * seen[j:j + t]).sum((0, 1)) for j in range(k)])
    return {"y": y, "x": dx, "w": dw, "bias": e.sum((0, 1))}


def _recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 0 from h = 0: in each of log2(T) rounds every row takes in twice as many before it."""
    step = 1
    while step < len(b):
        b = torch.cat([b[:step], b[step:] + a[step:] * b[:-step]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _scan_plain(s):
    case = s["case"]
    t, dt = case["t"], s["x"].dtype
    x, delta, B, C = (s[p].detach().float() for p in ("x", "delta", "B", "C"))
    A, skip, bias = (s[p].detach() for p in ("A", "skip", "bias"))
    inside = _inside(s, t)
    raw = delta + bias
    d = _only(raw.clamp(min=0) + torch.log1p(torch.exp(-raw.abs())), inside)
    a = torch.exp(d[:, :, None] * A)  # [T, B, N, D]
    h = (d * x)[:, :, None] * B[..., None]
    if s["state"] is not None:
        h = torch.cat([h[:1] + a[:1] * s["state"], h[1:]])
    h = _recurrence(a, h)
    v = (h * C[..., None]).sum(2) + skip * x
    gate = _silu(s["z"].detach().float()) if case["gate"] else None
    y = _only(v * gate if case["gate"] else v, inside).to(dt)
    if case["mode"] == "step":
        s["state"].copy_(h[0])
        return {"y": y[0], "state": s["state"]}
    if case["mode"] == "prompt":
        return {"y": y, "state": h[t - 1]}
    dy = _only(s["dy"].float(), inside)
    out = {"y": y}
    if case["gate"]:
        out["z"] = (dy * v * _dsilu(s["z"].detach().float())).to(dt)
        dy = dy * gate
    g = (dy[:, :, None] * C[..., None]).flip(0)
    g = _recurrence(torch.cat([torch.zeros_like(a[:1]), a[1:].flip(0)]), g).flip(0)
    kept = a * torch.cat([torch.zeros_like(h[:1]), h[:-1]])  # a_t h_{t-1}
    gk, gb = g * kept, (g * B[..., None]).sum(2)
    dd = (gk * A).sum(2) + gb * x
    ddelta = _only(dd * torch.sigmoid(raw), inside)
    return out | {"x": (gb * d + skip * dy).to(dt), "delta": ddelta.to(dt), "A": (gk * d[:, :, None]).sum((0, 1)),
                  "B": (g * (d * x)[:, :, None]).sum(3).to(dt), "C": (dy[:, :, None] * h).sum(3).to(dt),
                  "skip": (dy * x).sum((0, 1)), "bias": ddelta.sum((0, 1))}


# ------------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    from kf_benchmarks_amd.ops import nn, ssm

    case, mode = s["case"], s["case"]["mode"]
    if case["op"] == "norm":
        y = nn.group_norm(s["x"], s["gamma"], s["beta"], case["groups"], EPS, case["act"])
    elif case["op"] == "conv":
        if mode == "step":
            return {"y": ssm.causal_conv_step(s["x"][0], s["state"], s["w"], s["bias"], case["act"]), "state": s["state"]}
        y = ssm.causal_conv(s["x"], s["w"], s["bias"], case["act"], lengths=s["lengths"], return_state=mode == "prompt")
    else:
        if mode == "step":
            z = s["z"][0] if case["gate"] else None
            y = ssm.selective_scan_step(s["x"][0], s["delta"][0], s["A"], s["B"][0], s["C"][0], s["state"], s["skip"], z,
                                        s["bias"], softplus=True)
            return {"y": y, "state": s["state"]}
        y = ssm.selective_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], s["skip"], s["z"], s["bias"], softplus=True,
                               lengths=s["lengths"], return_state=mode == "prompt")
    if mode == "prompt":
        return {"y": y[0], "state": y[1]}
    if mode == "train":
        return {"y": y.detach()} | dict(zip(s["leaves"], torch.autograd.grad(y, [s[p] for p in s["leaves"]], s["dy"])))
    return {"y": y}


def run(state):
    if own:
        return _own(state)
    return {"norm": _norm_plain, "conv": _conv_plain, "scan": _scan_plain}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits, one row after the other; the gradients by differentiating them."""
    s = prepare(case, seed)
    v = {p: t.detach().double() if t is not None and t.is_floating_point() else t for p, t in s.items()
         if p not in ("case", "leaves")}
    train = case["mode"] == "train"
    if train:
        for p in s["leaves"]:
            v[p].requires_grad_()
    with torch.set_grad_enabled(train):
        if case["op"] == "norm":
            n, c, groups = case["n"], case["c"], case["groups"]
            x = v["x"].reshape(n, case["h"] * case["w"], groups, c // groups).transpose(1, 2).reshape(n, groups, -1)
            x = (x - x.mean(2, keepdim=True)) / (x.var(2, unbiased=False, keepdim=True) + EPS).sqrt()
            x = x.view(n, groups, case["h"] * case["w"], c // groups).transpose(1, 2).reshape(s["x"].shape)
            u = x * v["gamma"] + v["beta"]
            out = {"y": torch.nn.functional.silu(u) if case["act"] == "silu" else torch.relu(u) if case["act"] == "relu" else u}
        else:
            out = (_conv_rows if case["op"] == "conv" else _scan_rows)(case, v)
    if train:
        out |= dict(zip(s["leaves"], torch.autograd.grad(out["y"], [v[p] for p in s["leaves"]], v["dy"])))
    return {p: t.detach() for p, t in out.items()}


def _conv_rows(case, v):
    t, b, d, k = (case[p] for p in "tbdk")
    lengths = v["lengths"].long() if v["lengths"] is not None else torch.full((b,), t, device="cuda")
    state = v["state"] if v["state"] is not None else torch.zeros(k - 1, b, d, device="cuda", dtype=torch.float64)
    on = torch.arange(t, device="cuda")[:, None, None] < lengths[None, :, None]
    x = torch.cat([state, v["x"].masked_fill(~on, 0)]).permute(1, 2, 0)
    u = (x.unfold(2, k, 1) @ v["w"].t().unsqueeze(2)).squeeze(3).permute(2, 0, 1) + v["bias"]
    y = (torch.nn.functional.silu(u) if case["act"] == "silu" else u).masked_fill(~on, 0)
    last = torch.stack([x[i, :, n:n + k - 1].t() for i, n in enumerate(lengths.tolist())], 1)
    return {"y": y} if case["mode"] == "train" else {"y": y[0] if case["mode"] == "step" else y, "state": last}


def _scan_rows(case, v):
    t, b, d, n = (case[p] for p in "tbds")
    h = v["state"] if v["state"] is not None else torch.zeros(b, n, d, device="cuda", dtype=torch.float64)
    dt = torch.nn.functional.softplus(v["delta"] + v["bias"], threshold=100)
    rows = []
    for i in range(t):
        new = torch.exp(dt[i][:, None] * v["A"]) * h + (dt[i] * v["x"][i])[:, None] * v["B"][i][:, :, None]
        row = (new * v["C"][i][:, :, None]).sum(1) + v["skip"] * v["x"][i]
        if v["lengths"] is not None:
            on = (i < v["lengths"])[:, None]
            new, row = torch.where(on[:, None], new, h), torch.where(on, row, 0.0)
        h = new
        rows.append(row)
    y = torch.stack(rows)
    if case["gate"]:
        y = y * torch.nn.functional.silu(v["z"])
    return {"y": y} if case["mode"] == "train" else {"y": y[0] if case["mode"] == "step" else y, "state": h}
