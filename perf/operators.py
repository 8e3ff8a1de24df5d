"""Timing cases of the token-block operators: layer norm, the gated feed-forward block and the
gated linear recurrence, each in its plain form (elementary torch operations in 32 bits) and, with
`own` set, as the calls a user's program makes of this package (`mragan_hip.ops`)."""
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5


def listed():
    return [
        # one position of a streamed volume: two rows of a 256-channel bottleneck, launch latency
        dict(name="norm_step", op="norm", mode="forward", rows=2, channels=256, dtype="float32"),
        # every voxel of a 64^3 patch at batch 2 with the generator's 32 channels, training
        dict(name="norm_volume", op="norm", mode="train", rows=2 * 64 ** 3, channels=32, dtype="float32"),
        # a wide token batch, training
        dict(name="norm_tokens", op="norm", mode="train", rows=8192, channels=2048, dtype="bfloat16"),
        # an odd token count and a channel count that no vector width divides, inference
        dict(name="norm_odd", op="norm", mode="forward", rows=20011, channels=1001, dtype="float16"),
        # one token through the block, inference: the weights' bytes
        dict(name="ffn_token", op="ffn", mode="forward", tokens=1, channels=1024, hidden=4096, dtype="bfloat16", act="silu",
             bias=False),
        # the ResnetBlock section of a 64^3 patch at batch 2 (16^3 voxels, 128 channels), fp32 training
        dict(name="ffn_bottleneck", op="ffn", mode="train", tokens=2 * 16 ** 3, channels=128, hidden=512, dtype="float32",
             act="gelu", bias=True),
        # odd sizes throughout, inference
        dict(name="ffn_odd", op="ffn", mode="forward", tokens=1009, channels=515, hidden=1333, dtype="float16", act="sigmoid",
             bias=True),
        # a large training step
        dict(name="ffn_large", op="ffn", mode="train", tokens=16384, channels=2048, hidden=8192, dtype="bfloat16", act="silu",
             bias=False),
        # one step of a stream: every sequence's state moves by one position
        dict(name="recur_step", op="recur", mode="forward", batch=64, steps=1, channels=1024, dtype="bfloat16", gate=True,
             reverse=False),
        # a flattened 32^3 section at batch 2, 128 channels, fp32 training
        dict(name="recur_volume", op="recur", mode="train", batch=2, steps=32 ** 3, channels=128, dtype="float32", gate=False,
             reverse=False),
        # few channels over a whole flattened 64^3 patch, backwards in time, inference
        dict(name="recur_long", op="recur", mode="forward", batch=1, steps=64 ** 3, channels=64, dtype="bfloat16", gate=False,
             reverse=True),
        # a batch of ordinary sequences with the output gate, training
        dict(name="recur_batch", op="recur", mode="train", batch=16, steps=2048, channels=1024, dtype="bfloat16", gate=True,
             reverse=False),
    ]


def _log_uniform(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm; one in three is made odd."""
    n = int(round(lo * (hi / lo) ** rng.random()))
    if rng.random() < 1 / 3:
        n |= 1
    return max(lo, min(hi, n))


def _rounded(rng, n, step):
    """n, or with even chance the nearest positive multiple of `step`: channel counts are mostly that."""
    return max(step, (n + step // 2) // step * step) if rng.random() < 0.5 else n


def draw(rng):
    dtype = rng.choice(sorted(DTYPES))
    op = rng.choice(("norm", "ffn", "recur"))
    if op == "norm":
        channels = _rounded(rng, _log_uniform(rng, 16, 8192), 16)
        rows = _log_uniform(rng, 1, min(1 << 20, (1 << 25) // channels))
        return dict(op=op, mode=rng.choice(("forward", "train")), rows=rows, channels=channels, dtype=dtype)
    if op == "ffn":
        channels = _rounded(rng, _log_uniform(rng, 32, 2048), 32)
        hidden = _rounded(rng, _log_uniform(rng, 64, 8192), 64)
        mode = rng.choice(("forward", "train"))
        most = 16384 if dtype != "float32" else max(1, min(16384, (1 << 34) // (channels * hidden)))
        return dict(op=op, mode=mode, tokens=_log_uniform(rng, 1 if mode == "forward" else 16, max(16, most)), channels=channels,
                    hidden=hidden, dtype=dtype, act=rng.choice(("silu", "gelu", "sigmoid")), bias=rng.random() < 0.5)
    channels = _rounded(rng, _log_uniform(rng, 8, 4096), 8)
    steps = 1 if rng.random() < 0.2 else _log_uniform(rng, 2, min(1 << 18, (1 << 25) // channels))
    batch = _log_uniform(rng, 1, max(1, min(64, (1 << 25) // (channels * steps))))
    return dict(op=op, mode=rng.choice(("forward", "train")), batch=batch, steps=steps, channels=channels, dtype=dtype,
                gate=rng.random() < 0.5, reverse=rng.random() < 0.5)


def prepare(case, seed):
    dt = DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).add_(shift).to(dtype)

    train = case["mode"] == "train"
    s = dict(case=dict(case))
    if case["op"] == "norm":
        R, C = case["rows"], case["channels"]
        s.update(x=normal(R, C, scale=2.0, shift=0.5), weight=normal(C, scale=0.2, shift=1.0), bias=normal(C, scale=0.2))
        if train:
            s["dy"] = normal(R, C)
    elif case["op"] == "ffn":
        M, C, F = case["tokens"], case["channels"], case["hidden"]
        s.update(x=normal(M, C), w_gate=normal(F, C, scale=C ** -0.5), w_up=normal(F, C, scale=C ** -0.5),
                 w_down=normal(C, F, scale=F ** -0.5))
        for k, n in (("b_gate", F), ("b_up", F), ("b_down", C)):
            s[k] = normal(n, scale=0.1) if case["bias"] else None
        if train:
            s["dy"] = normal(M, C)
    else:
        B, T, C = case["batch"], case["steps"], case["channels"]
        # decays between about 0.5 and 0.999: memories of a few to a thousand steps
        s.update(x=normal(B, T, C), decay=normal(B, T, C, scale=1.5, shift=3.0),
                 gate=normal(B, T, C) if case["gate"] else None, h0=normal(B, C, dtype=torch.float32))
        if train:
            s.update(dy=normal(B, T, C), dlast=normal(B, C, dtype=torch.float32))
    return s


# ---- plain forms ------------------------------------------------------------------------------


def _plain_norm(s):
    dt = s["x"].dtype
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).mean(1, keepdim=True) + EPS)
    xh = xc * rstd
    y = (xh * w + b).to(dt)
    if "dy" not in s:
        return {"y": y}
    dy = s["dy"].float()
    p = dy * w
    dx = rstd * (p - p.mean(1, keepdim=True) - xh * (p * xh).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(dt), "dweight": (dy * xh).sum(0).to(dt), "dbias": dy.sum(0).to(dt)}


def _act(g, act):
    """act(g) and act'(g)."""
    if act == "gelu":
        phi = 0.5 * (1.0 + torch.erf(g * 0.5 ** 0.5))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * 0.3989422804014327
    sg = torch.sigmoid(g)
    if act == "sigmoid":
        return sg, sg * (1.0 - sg)
    return g * sg, sg * (1.0 + g * (1.0 - sg))


def _plain_ffn(s):
    dt, act = s["x"].dtype, s["case"]["act"]
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.t(), x @ wu.t()
    if s["b_gate"] is not None:
        g, u = g + s["b_gate"].float(), u + s["b_up"].float()
    ag, dag = _act(g, act)
    h = ag * u
    y = h @ wd.t()
    if s["b_down"] is not None:
        y = y + s["b_down"].float()
    out = {"y": y.to(dt)}
    if "dy" in s:
        dy = s["dy"].float()
        dh = dy @ wd
        dg, du = dh * u * dag, dh * ag
        out.update(dx=(dg @ wg + du @ wu).to(dt), dw_gate=(dg.t() @ x).to(dt), dw_up=(du.t() @ x).to(dt),
                   dw_down=(dy.t() @ h).to(dt))
        if s["b_gate"] is not None:
            out.update(db_gate=dg.sum(0).to(dt), db_up=du.sum(0).to(dt), db_down=dy.sum(0).to(dt))
    return out


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1 from h = 0, by doubling the span that a pair (a, b) stands for."""
    k = 1
    while k < b.shape[1]:
        b = torch.cat((b[:, :k], a[:, k:] * b[:, :-k] + b[:, k:]), 1)
        a = torch.cat((a[:, :k], a[:, k:] * a[:, :-k]), 1)
        k *= 2
    return b


def _plain_recur(s):
    dt, rev = s["x"].dtype, s["case"]["reverse"]

    def seq(t):
        return t.float().flip(1) if rev else t.float()

    x, d, h0 = seq(s["x"]), seq(s["decay"]), s["h0"]
    a, i = torch.sigmoid(d), torch.sigmoid(-d)
    b = i * x
    b[:, 0] += a[:, 0] * h0
    h = _scan(a, b)
    y = h
    if s["gate"] is not None:
        z = seq(s["gate"])
        sz, dsz = _act(z, "silu")
        y = h * sz
    out = {"y": (y.flip(1) if rev else y).to(dt), "last": h[:, -1].clone()}
    if "dy" in s:
        dy = seq(s["dy"])
        top = dy if s["gate"] is None else dy * sz
        top = torch.cat((top[:, :-1], top[:, -1:] + s["dlast"][:, None]), 1)
        behind = torch.cat((torch.zeros_like(a[:, :1]), a[:, 1:].flip(1)), 1)      # a_{t+1}, last step first
        G = _scan(behind, top.flip(1)).flip(1)
        prev = torch.cat((h0[:, None], h[:, :-1]), 1)
        grads = {"dx": G * i, "ddecay": G * (prev - x) * a * i}
        if s["gate"] is not None:
            grads["dgate"] = dy * h * dsz
        out.update({k: (v.flip(1) if rev else v).to(dt) for k, v in grads.items()})
        out["dh0"] = a[:, 0] * G[:, 0]
    return out


# ---- the package's calls ----------------------------------------------------------------------


def _ops():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mra-gan_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from mragan_hip import ops
    return ops


def _own_norm(ops, s):
    y, mean, rstd = ops.layer_norm_fwd(s["x"], s["weight"], s["bias"], EPS)
    if "dy" not in s:
        return {"y": y}
    dx, dw, db = ops.layer_norm_bwd(s["x"], mean, rstd, s["dy"], s["weight"], bias=True)
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db}


def _own_ffn(ops, s):
    act, train = s["case"]["act"], "dy" in s
    w = (s["w_gate"], s["w_up"], s["w_down"])
    y, kept = ops.gated_ffn_fwd(s["x"], *w, s["b_gate"], s["b_up"], s["b_down"], act=act, keep=train)
    if not train:
        return {"y": y}
    g = ops.gated_ffn_bwd(s["x"], *w, s["dy"], kept, s["b_gate"], s["b_up"], s["b_down"], act=act)
    out = {"y": y, "dx": g[0], "dw_gate": g[1], "dw_up": g[2], "dw_down": g[3]}
    if s["b_gate"] is not None:
        out.update(db_gate=g[4], db_up=g[5], db_down=g[6])
    return out


def _own_recur(ops, s):
    rev = s["case"]["reverse"]
    y, last, carry = ops.linear_recurrence_fwd(s["x"], s["decay"], s["gate"], s["h0"], reverse=rev)
    out = {"y": y, "last": last}
    if "dy" in s:
        dx, dd, dz, dh0 = ops.linear_recurrence_bwd(s["x"], s["decay"], carry, s["dy"], s["gate"], dlast=s["dlast"], reverse=rev)
        out.update(dx=dx, ddecay=dd, dh0=dh0)
        if dz is not None:
            out["dgate"] = dz
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "ffn": _own_ffn, "recur": _own_recur}[op](_ops(), state)
    return {"norm": _plain_norm, "ffn": _plain_ffn, "recur": _plain_recur}[op](state)


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    train = case["mode"] == "train"
    if case["op"] == "norm":
        R, C = case["rows"], case["channels"]
        return {"bytes": (4 if train else 2) * R * C * e + (4 if train else 2) * C * e, "flops": (22 if train else 8) * R * C}
    if case["op"] == "ffn":
        M, C, F = case["tokens"], case["channels"], case["hidden"]
        weights = 3 * C * F + (2 * F + C if case["bias"] else 0)
        return {"bytes": (4 if train else 2) * M * C * e + (2 if train else 1) * weights * e,
                "flops": (3 if train else 1) * 6 * M * C * F}
    B, T, C = case["batch"], case["steps"], case["channels"]
    n = (4 if case["gate"] else 3) + ((4 if case["gate"] else 3) if train else 0)
    return {"bytes": n * B * T * C * e + (4 if train else 2) * B * C * 4, "flops": (40 if train else 12) * B * T * C}


# ---- the definitions in 64 bits ---------------------------------------------------------------


def _exact_norm(s):
    x, w, b = (s[k].double().requires_grad_() for k in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    y = (x - mean) / torch.sqrt(var + EPS) * w + b
    out = {"y": y.detach()}
    if "dy" in s:
        out.update(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, (x, w, b), s["dy"].double())))
    return out


def _exact_ffn(s):
    names = ["x", "w_gate", "w_up", "w_down"] + (["b_gate", "b_up", "b_down"] if s["b_gate"] is not None else [])
    v = {k: s[k].double().requires_grad_() for k in names}
    zero = torch.zeros((), dtype=torch.float64, device=s["x"].device)
    g = torch.mm(v["x"], v["w_gate"].t()) + v.get("b_gate", zero)
    u = torch.mm(v["x"], v["w_up"].t()) + v.get("b_up", zero)
    curve = {"silu": lambda t: t / (1 + torch.exp(-t)), "sigmoid": lambda t: 1 / (1 + torch.exp(-t)),
             "gelu": lambda t: t * torch.special.ndtr(t)}[s["case"]["act"]]
    y = torch.mm(curve(g) * u, v["w_down"].t()) + v.get("b_down", zero)
    out = {"y": y.detach()}
    if "dy" in s:
        grads = torch.autograd.grad(y, [v[k] for k in names], s["dy"].double())
        out.update({"d" + k: t for k, t in zip(names, grads)})
    return out


def _steps(a, b, h):
    """Every h_t = a_t h_{t-1} + b_t along dimension 1 in order, over up to 512 spans at once that are joined in order."""
    B, T, C = b.shape
    n = max(1, min(512, T // 32))
    span = -(-T // n)
    pad = n * span - T
    a = torch.cat((a, a.new_ones(B, pad, C)), 1).reshape(B, n, span, C)
    b = torch.cat((b, b.new_zeros(B, pad, C)), 1).reshape(B, n, span, C)
    local, grown = torch.empty_like(b), torch.empty_like(a)
    state, product = torch.zeros_like(b[:, :, 0]), torch.ones_like(a[:, :, 0])
    for t in range(span):
        state = a[:, :, t] * state + b[:, :, t]
        product = product * a[:, :, t]
        local[:, :, t], grown[:, :, t] = state, product
    for k in range(n):
        local[:, k] += grown[:, k] * h[:, None]
        h = local[:, k, -1]
    return local.reshape(B, n * span, C)[:, :T]


def _exact_recur(s):
    rev = s["case"]["reverse"]
    turn = (lambda t: torch.flip(t, (1,))) if rev else (lambda t: t)
    x, d, h0 = turn(s["x"].double()), turn(s["decay"].double()), s["h0"].double()
    a = 1 / (1 + torch.exp(-d))
    keep = 1 / (1 + torch.exp(d))
    h = _steps(a, keep * x, h0)
    sz = dsz = None
    if s["gate"] is not None:
        z = turn(s["gate"].double())
        sg = 1 / (1 + torch.exp(-z))
        sz, dsz = z * sg, sg + z * sg * (1 - sg)
    out = {"y": turn(h if sz is None else h * sz), "last": h[:, -1].clone()}
    if "dy" in s:
        dy = turn(s["dy"].double())
        top = torch.flip(dy if sz is None else dy * sz, (1,)).contiguous()
        later = torch.cat((torch.ones_like(a[:, :1]), torch.flip(a, (1,))[:, :-1]), 1)
        G = torch.flip(_steps(later, top, s["dlast"].double()), (1,))
        before = torch.cat((h0[:, None], h), 1)[:, :-1]
        out.update(dx=turn(G * keep), ddecay=turn(G * (before - x) * a * keep), dh0=a[:, 0] * G[:, 0])
        if sz is not None:
            out["dgate"] = turn(dy * h * dsz)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"norm": _exact_norm, "ffn": _exact_ffn, "recur": _exact_recur}[case["op"]](s)
