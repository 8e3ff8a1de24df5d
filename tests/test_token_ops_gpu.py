"""Layer norm, gated feed-forward block and gated linear recurrence on the GPU, forward and backward,
against plain float64 forms of their definitions.

Tolerances are bounds on the rounding errors, computed per element in float64 from the inputs:
u(T) = finfo(T).eps / 2 for every rounding to a tensor's type, and e = 2^-24 per fp32 operation, carried
through the absolute values of the terms that a sum is made of.  A sum of n terms in some order is off
by at most n·e·Σ|terms|; the constants below count the operations of a step generously."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
F64 = torch.float64
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """What a rounding into the subnormal range may be off by."""
    return torch.finfo(dtype).smallest_normal * u(dtype) * 2


def close(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / bound).max()):.3g} of the bound"


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    from mragan_hip import ops as m
    import mragan_hip.torch_ops  # noqa: F401
    m.set_conv_precision("f32")
    return m


@pytest.fixture(autouse=True)
def f32_mode(ops):
    ops.set_conv_precision("f32")
    yield
    ops.set_conv_precision("f32")


def randn(seed, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).cuda()


# ---- layer norm ---------------------------------------------------------------------------------

def check_norm(ops, x, w, b, eps=1e-5, dy=None):
    C, T = x.shape[-1], x.dtype
    y, mean, rstd = ops.layer_norm_fwd(x, w, b, eps)
    xd = x.double().reshape(-1, C)
    wd = torch.ones(C, dtype=F64, device="cuda") if w is None else w.double()
    bd = torch.zeros(C, dtype=F64, device="cuda") if b is None else b.double()
    mu = xd.mean(1, keepdim=True)
    xc = xd - mu
    r = (xc.square().mean(1, keepdim=True) + eps).rsqrt()
    n = 64                                                    # additions in a row's sum: ≤ 32 in a lane, the tree, the mean
    if C > 8192:
        n = C // 1024 + 32
    dmu = n * E * xd.abs().mean(1, keepdim=True) + E * mu.abs()
    dxc = dmu + E * xc.abs()
    # relative error of rstd: half that of the mean square, a few of rsqrt
    drel = ((2 * dxc * xc.abs()).mean(1, keepdim=True) + dxc.square().mean(1, keepdim=True) + n * E * xc.square().mean(1, keepdim=True)) * r * r + 4 * E
    close(mean.reshape(-1, 1), mu, dmu + E * mu.abs() + 1e-38, "mean")
    close(rstd.reshape(-1, 1), r, drel * r, "rstd")
    xh = xc * r
    dxh = dxc * r + xh.abs() * (drel + 2 * E)
    want = xh * wd + bd
    close(y.reshape(-1, C), want, (dxh * wd.abs() + 4 * E * (xh * wd).abs() + 2 * E * bd.abs()) * 1.01 + u(T) * want.abs() + tiny(T), "y")
    if dy is None:
        return
    wt = T if w is None else w.dtype
    dx, dw, db = ops.layer_norm_bwd(x, mean, rstd, dy, w, bias=True)
    g = dy.double().reshape(-1, C)
    p = g * wd
    m1, m2 = p.mean(1, keepdim=True), (p * xh).mean(1, keepdim=True)
    want = r * (p - m1 - xh * m2)
    d1 = (n + 2) * E * p.abs().mean(1, keepdim=True)
    d2 = (p.abs() * dxh).mean(1, keepdim=True) + (n + 4) * E * (p * xh).abs().mean(1, keepdim=True)
    bound = r * (d1 + dxh * m2.abs() + xh.abs() * d2 + 4 * E * (p.abs() + m1.abs() + (xh * m2).abs())) + (drel + 2 * E) * want.abs()
    close(dx.reshape(-1, C), want, 1.01 * bound + u(T) * want.abs() + tiny(T), "dx")
    rows = xd.shape[0]
    k = rows / 256 + 160 if C <= 8192 else rows + 8           # rows that one thread adds up, and the joins
    if w is not None:
        want = (g * xh).sum(0)
        close(dw, want, 1.01 * ((g.abs() * dxh).sum(0) + (k + 4) * E * (g * xh).abs().sum(0)) + u(wt) * want.abs() + tiny(wt), "dw")
    else:
        assert dw is None
    want = g.sum(0)
    close(db, want, 1.01 * k * E * g.abs().sum(0) + u(wt) * want.abs() + tiny(wt), "db")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (40, 3), (9, 7), (70, 9), (6, 31), (2, 7, 33), (1, 2, 3, 4, 16), (17, 64), (1300, 72), (5, 1000), (2500, 1001),
                                   (70000, 8), (2, 2048), (1030, 2048), (1500, 1535), (3, 4096), (1100, 4100), (1200, 2051), (2, 8192), (2, 8195), (3, 20000)])
def test_layer_norm(ops, shape, dtype):
    C = shape[-1]
    check_norm(ops, randn(1, *shape, dtype=dtype, scale=2, shift=0.5), randn(2, C, dtype=dtype, scale=0.2, shift=1),
               randn(3, C, dtype=dtype, scale=0.3), dy=randn(4, *shape, dtype=dtype))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(150, 8200), (4500, 8195), (513, 1024), (2000, 512), (260, 2050), (2300, 2048), (33, 8192)])
def test_layer_norm_row_groups(ops, shape, dtype):
    """Row counts on both sides of every split of the rows over blocks and runs."""
    C = shape[-1]
    check_norm(ops, randn(1, *shape, dtype=dtype), randn(2, C, dtype=dtype), randn(3, C, dtype=dtype), dy=randn(4, *shape, dtype=dtype))


def test_layer_norm_more_long_rows_than_blocks(ops):
    x, dy = randn(1, 65600, 8200, dtype=torch.bfloat16), randn(2, 65600, 8200, dtype=torch.bfloat16)
    w, tail = randn(3, 8200, dtype=torch.bfloat16), slice(65500, None)
    whole, part = ops.layer_norm_fwd(x, w), ops.layer_norm_fwd(x[tail], w)
    assert all(torch.equal(a[tail], b) for a, b in zip(whole, part))
    dx = ops.layer_norm_bwd(x, *whole[1:], dy, w)[0]
    assert torch.equal(dx[tail], ops.layer_norm_bwd(x[tail], *part[1:], dy[tail], w)[0])


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=str)
@pytest.mark.parametrize("shape", [(9, 40), (1500, 256), (3, 8195)])
def test_layer_norm_float32_parameters(ops, shape, dtype):
    C = shape[-1]
    x, dy = randn(1, *shape, dtype=dtype), randn(4, *shape, dtype=dtype)
    check_norm(ops, x, randn(2, C), randn(3, C), dy=dy)
    dx, dw, db = ops.layer_norm_bwd(x, *ops.layer_norm_fwd(x)[1:], dy, None, bias=torch.float32)
    assert dw is None and db.dtype == torch.float32


@pytest.mark.parametrize("w,b", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_parameters(ops, w, b):
    check_norm(ops, randn(1, 33, 130), randn(2, 130) if w else None, randn(3, 130) if b else None, dy=randn(4, 33, 130))


def test_layer_norm_hard_rows(ops):
    """Rows far from zero, constant rows (variance 0), and rows with an infinity or a NaN, which stay in their row."""
    x = randn(1, 8, 96)
    x[1] += 3000.0
    x[2] = 7.0
    x[3] *= 1e-12
    check_norm(ops, x, randn(2, 96), randn(3, 96), dy=randn(4, 8, 96))
    x[4, 3], x[5, 7] = float("inf"), float("nan")
    y = ops.layer_norm_fwd(x)[0]
    assert y[4].isnan().any() and y[5].isnan().all()
    assert y[[0, 1, 2, 3, 6, 7]].isfinite().all()


def test_layer_norm_views_and_empty(ops):
    base = randn(1, 20, 300)
    check_norm(ops, base[:, 7:137], randn(2, 260)[::2], randn(3, 130), dy=randn(4, 130, 20).t())
    y, mean, rstd = ops.layer_norm_fwd(base[:0], None, None)
    assert y.shape == (0, 300) and mean.shape == (0,)
    w = randn(2, 300)
    dx, dw, db = ops.layer_norm_bwd(base[:0], mean, rstd, base[:0], w, bias=True)
    assert dx.shape == (0, 300) and not dw.any() and not db.any()


# ---- gated feed-forward -------------------------------------------------------------------------

def act_pair(g, act):
    g = g.detach().requires_grad_()
    f = {"silu": lambda t: t * torch.sigmoid(t), "gelu": lambda t: t * torch.special.ndtr(t), "sigmoid": torch.sigmoid,
         "relu": torch.relu, "lrelu": lambda t: torch.nn.functional.leaky_relu(t, 0.2), "tanh": torch.tanh, "none": lambda t: t}[act](g)
    return f.detach(), torch.autograd.grad(f.sum(), g)[0]


def ffn_inputs(M, C, F, O, dtype, bias=True, seed=0):
    a = [randn(seed + 1, M, C, dtype=dtype), randn(seed + 2, F, C, dtype=dtype, scale=C ** -0.5),
         randn(seed + 3, F, C, dtype=dtype, scale=C ** -0.5), randn(seed + 4, O, F, dtype=dtype, scale=F ** -0.5)]
    b = [randn(seed + 5 + i, n, dtype=dtype, scale=0.3) if bias else None for i, n in enumerate((F, F, O))]
    return a, b, randn(seed + 9, M, O, dtype=dtype)


def check_ffn(ops, a, b, dy, act, mode="f32", keep=True, need=(True,) * 7):
    """Bounds: a product of operands known to relative v (the planes of the mode) with k terms in fp32 is off by
    (2v + k·e)·Σ|terms| plus what its operands bring; h, act'·u, act and dg, du are rounded to the type, by u."""
    ops.set_conv_precision(mode)
    x, wg, wu, wd = (t.double() for t in a)
    bg, bu, bd = ((0.0 if t is None else t.double()) for t in b)
    T, g_out = a[0].dtype, dy.double()
    M, C = x.shape
    F, O = wg.shape[0], wd.shape[0]
    # relative error of an operand as the product takes it: exact for 16-bit tensors; planes of fp32 ones
    v = 0.0 if T != torch.float32 else {"f32": 2.0 ** -24, "bf16x3": 3 * 2.0 ** -18, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}[mode]
    h_v = u(T) if T != torch.float32 else v                    # h, dg, du as operands
    mm = lambda p, q: p @ q
    y, kept = ops.gated_ffn_fwd(*a, *b, act=act, keep=keep)
    k = lambda n: 2 * v + (n + 8) * E
    g, uu = mm(x, wg.t()) + bg, mm(x, wu.t()) + bu
    ag, au = mm(x.abs(), wg.abs().t()), mm(x.abs(), wu.abs().t())
    dg_, du_ = k(C) * ag + 4 * E * g.abs(), k(C) * au + 4 * E * uu.abs()
    f, df = act_pair(g, act)
    kink = (g.abs() <= dg_).double() if act in ("relu", "lrelu") else 0.0
    tr = 16 * E * (1 + g.abs())                                # exp / erf / tanh and what they are made of
    ef = 1.2 * dg_ + tr * (f.abs() + E) + tr * 0.1
    edf = 1.2 * dg_ + tr * 1.2 + kink
    h, P = f * uu, df * uu
    eh = ef * uu.abs() + f.abs() * du_ + ef * du_ + 2 * E * h.abs()
    eP = edf * uu.abs() + df.abs() * du_ + edf * du_ + 2 * E * P.abs()
    t16 = tiny(T) if T != torch.float32 else (tiny(torch.float16) if mode == "fp16" else 0.0)
    want = mm(h, wd.t()) + bd
    ehr = eh + h_v * h.abs() + t16
    by = mm(ehr, wd.abs().t()) + (k(F) * mm(h.abs(), wd.abs().t())) + 4 * E * want.abs()
    close(y, want, 1.02 * by + u(T) * want.abs() + tiny(T), "y")
    grads = ops.gated_ffn_bwd(*a, dy, kept, *b, act=act, need=need)
    dh = mm(g_out, wd)
    edh = k(O) * mm(g_out.abs(), wd.abs())
    kr = E if T == torch.float32 else 2.0 ** -16               # P and f are kept with 24 bits
    dg, du = dh * P, dh * f
    edg = edh * P.abs() + (dh.abs() + edh) * (eP + kr * P.abs() + 1e-38) + (h_v + 2 * E) * dg.abs() + t16
    edu = edh * f.abs() + (dh.abs() + edh) * (ef + kr * f.abs() + 1e-38) + (h_v + 2 * E) * du.abs() + t16
    wants = [mm(dg, wg) + mm(du, wu), mm(dg.t(), x), mm(du.t(), x), mm(g_out.t(), h), dg.sum(0), du.sum(0), g_out.sum(0)]
    ek = eh + (u(T) + h_v) * h.abs() + t16 + tiny(T)             # h as kept, then as an operand
    bounds = [mm(edg, wg.abs()) + mm(edu, wu.abs()) + k(2 * F) * (mm(dg.abs(), wg.abs()) + mm(du.abs(), wu.abs())),
              mm(edg.t(), x.abs()) + k(M) * mm(dg.abs().t(), x.abs()), mm(edu.t(), x.abs()) + k(M) * mm(du.abs().t(), x.abs()),
              mm(g_out.abs().t(), ek) + k(M) * mm(g_out.abs().t(), h.abs()), edg.sum(0) + k(M) * dg.abs().sum(0),
              edu.sum(0) + k(M) * du.abs().sum(0), (v + k(M)) * g_out.abs().sum(0) + M * t16]
    names = ["dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down"]
    for got, want, bound, name, t, n in zip(grads, wants, bounds, names, [*a, *b], need):
        if t is None or not n:
            assert got is None, name
        else:
            close(got, want, 1.03 * bound + u(T) * want.abs() + tiny(T), name)


FFN_SIZES = [(1, 64, 128, 64), (3, 5, 7, 11), (1, 1, 1, 1), (130, 64, 200, 96), (257, 515, 333, 130), (1000, 256, 1024, 256),
             (600, 136, 520, 72), (2048, 64, 4096, 64)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("size", FFN_SIZES)
def test_gated_ffn(ops, size, dtype):
    check_ffn(ops, *ffn_inputs(*size, dtype), "silu")


@pytest.mark.parametrize("act", ["none", "relu", "lrelu", "tanh", "sigmoid", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_gated_ffn_activations(ops, act, dtype):
    check_ffn(ops, *ffn_inputs(70, 72, 136, 40, dtype), act)


@pytest.mark.parametrize("mode", ["bf16x3", "bf16", "fp16"])
@pytest.mark.parametrize("size", [(3, 5, 7, 11), (300, 128, 512, 128), (257, 100, 333, 130)])
def test_gated_ffn_precision_modes(ops, size, mode):
    check_ffn(ops, *ffn_inputs(*size, torch.float32), "gelu", mode=mode)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("size", [(1, 64, 128, 64), (257, 515, 333, 130), (200, 64, 192, 64)])
def test_gated_ffn_recomputed_and_without_bias(ops, size, dtype):
    check_ffn(ops, *ffn_inputs(*size, dtype, bias=False), "silu", keep=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("size", [(1, 1024, 4096, 1024), (1, 8, 8, 8), (2, 72, 200, 24), (16, 264, 136, 33), (17, 1000, 1000, 1000),
                                  (33, 128, 520, 96), (64, 320, 640, 64), (65, 320, 640, 64)])
def test_gated_ffn_few_rows(ops, size, dtype):
    """Inference on up to 64 rows and one more; in fp32 each precision mode's planes."""
    for mode in ("f32", "bf16x3", "bf16", "fp16") if dtype == torch.float32 else ("f32",):
        a, b, dy = ffn_inputs(*size, dtype)
        check_ffn(ops, a, b, dy, "silu", mode=mode, keep=False, need=(False,) * 7)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("size", [(3, 40, 88, 16), (4, 520, 1032, 130), (5, 512, 8, 40), (8, 72, 8192, 64), (9, 72, 8192, 64),
                                  (48, 64, 1368, 64), (64, 64, 1024, 33), (1, 959, 333, 70), (2, 515, 1333, 9),
                                  (4, 9, 11, 5), (3, 8, 15, 3), (7, 13, 517, 33), (30, 101, 77, 9), (64, 35, 100, 20), (20, 40, 1001, 8)])
def test_gated_ffn_few_rows_forms(ops, size, dtype):
    """Rows and hidden channels on both sides of every change of form."""
    check_ffn(ops, *ffn_inputs(*size, dtype), "gelu", keep=False, need=(False,) * 7)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows", [1, 2, 4, 7, 33, 70])
def test_gated_ffn_non_finite_rows_stay_apart(ops, rows, dtype):
    """A row of infinities and NaN changes no other row, and a weight's infinite row only its hidden channel."""
    a, b, _ = ffn_inputs(rows + 1, 40, 88, 24, dtype)
    y, _ = ops.gated_ffn_fwd(*a, *b)
    x = a[0].clone()
    x[rows, ::2], x[rows, 1::2] = float("inf"), float("nan")
    y2, _ = ops.gated_ffn_fwd(x, *a[1:], *b)
    assert torch.equal(y2[:rows], y[:rows]) and not y2[rows].isfinite().any()
    wd = a[3].clone()
    wd[5, 0] = float("inf")
    y3, _ = ops.gated_ffn_fwd(*a[:3], wd, *b)
    keep = [i for i in range(24) if i != 5]
    assert torch.equal(y3[:, keep], y[:, keep]) and not y3[:, 5].isfinite().any()


@pytest.mark.parametrize("need", [(1, 0, 0, 0, 0, 0, 0), (0, 1, 0, 0, 0, 0, 0), (0, 0, 1, 0, 0, 0, 1), (0, 0, 0, 1, 0, 0, 0),
                                  (0, 0, 0, 0, 1, 0, 0), (0, 0, 0, 0, 0, 1, 0), (0,) * 7])
def test_gated_ffn_some_gradients(ops, need):
    check_ffn(ops, *ffn_inputs(150, 64, 96, 32, torch.bfloat16), "silu", need=tuple(map(bool, need)))


def test_gated_ffn_views_and_empty(ops):
    """A slice off the 16-byte boundary, transposed weights, leading dimensions; no rows."""
    (x, wg, wu, wd), b, dy = ffn_inputs(24, 65, 40, 33, torch.bfloat16)
    x4 = torch.cat((x[:, :1], x), 1)[:, 1:].reshape(2, 3, 4, 65)
    y, _ = ops.gated_ffn_fwd(x4, wg.t().contiguous().t(), wu, wd, *b)
    y2, _ = ops.gated_ffn_fwd(x.contiguous(), wg, wu, wd, *b)
    assert y.shape == (2, 3, 4, 33) and torch.equal(y.reshape(24, 33), y2)
    y, kept = ops.gated_ffn_fwd(x[:0], wg, wu, wd, *b, keep=True)
    assert y.shape == (0, 33) and kept.shape == (4, 0, 40)
    grads = ops.gated_ffn_bwd(x[:0], wg, wu, wd, dy[:0], kept, *b)
    assert all(not g.any() for g in grads) and grads[1].shape == wg.shape


# ---- gated linear recurrence --------------------------------------------------------------------

def scan(a, b, h):
    """All h_t = a_t h_{t-1} + b_t along dimension 1, in order, in float64 on the CPU."""
    a, b, h = a.cpu(), b.cpu(), h.cpu()
    out = torch.empty_like(b)
    for t in range(b.shape[1]):
        h = a[:, t] * h + b[:, t]
        out[:, t] = h
    return out.cuda()


def check_recurrence(ops, x, d, z, h0, dy, dlast, reverse, plain=True):
    """Bounds: the errors obey the recurrences themselves: e_t = a_t·e_{t-1} + c·2^-24·(terms of step t), with
    c counting the operations of a step (σ: exp of an argument rounded to |d|·2^-24, product chains)."""
    B, T, C = x.shape
    Ty = x.dtype
    y, last, carry = ops.linear_recurrence_fwd(x, d, z, h0, reverse=reverse)
    turn = (lambda t: t.flip(1)) if reverse else (lambda t: t)
    xd, dd = turn(x.double()), turn(d.double())
    zero = torch.zeros(B, C, dtype=F64, device="cuda")
    s0 = zero if h0 is None else h0.double()
    a, i = torch.sigmoid(dd), torch.sigmoid(-dd)
    h = scan(a, i * xd, s0)
    prev = torch.cat((s0[:, None], h[:, :-1]), 1)
    c = (24 + 4 * dd.abs().clamp(max=104)) * E                # beyond, exp(-|d|) is 0 in fp32 and sigma exactly 0 or 1
    eh = scan(a, c * (a * prev.abs() + (i * xd).abs()), zero)
    eprev = torch.cat((zero[:, None], eh[:, :-1]), 1)
    if z is None:
        f, df, cz = torch.ones_like(h), torch.zeros_like(h), torch.zeros_like(h)
    else:
        zd = turn(z.double())
        sg = torch.sigmoid(zd)
        f, df = zd * sg, sg * (1 + zd * torch.sigmoid(-zd))
        cz = (24 + 4 * zd.abs()) * E
    want = h * f
    close(turn(y), want, 1.02 * (eh * f.abs() + cz * want.abs()) + u(Ty) * want.abs() + tiny(Ty), "y")
    close(last, h[:, -1], 1.02 * eh[:, -1] + E * h[:, -1].abs() + 1e-38, "last")
    if dy is None:
        return
    got = ops.linear_recurrence_bwd(x, d, carry, dy, z, dlast, reverse=reverse)
    g = turn(dy.double())
    q0 = zero if dlast is None else dlast.double()
    top, etop = g * f, cz * (g * f).abs()
    shift = lambda t, fill: torch.cat((t[:, 1:], fill[:, None]), 1)
    one = torch.ones_like(zero)
    back = lambda b, q: scan(shift(a, one).flip(1), b.flip(1), q).flip(1)        # G_t = b_t + a_{t+1} G_{t+1}
    G = back(top, q0)
    later = shift(a, one) * shift(G, q0)
    eG = back(etop + c * (top.abs() + later.abs()) + shift(c, zero) * later.abs(), zero)
    dfz = df.abs() + cz * 2
    wants = [G * i, G * (prev - xd) * a * i, g * h * df, a[:, 0] * G[:, 0]]
    ai = a * i
    bounds = [(eG + c * G.abs()) * i, eG * (prev - xd).abs() * ai + (G.abs() + eG) * ai * (eprev + c * (prev.abs() + xd.abs())),
              g.abs() * (eh * dfz + h.abs() * cz * 2 + c * h.abs() * dfz), (a * (eG + c * G.abs()))[:, 0]]
    for k, name in enumerate(("dx", "ddecay", "dgate")):
        if name == "dgate" and z is None:
            assert got[2] is None
            continue
        close(turn(got[k]), wants[k], 1.03 * bounds[k] + u(Ty) * wants[k].abs() + tiny(Ty), name)
    close(got[3], wants[3], 1.03 * bounds[3] + E * wants[3].abs() + 1e-38, "dh0")


def recurrence_inputs(B, T, C, dtype, gate=True, seed=0):
    return (randn(seed + 1, B, T, C, dtype=dtype), randn(seed + 2, B, T, C, dtype=dtype, scale=1.5, shift=2.5),
            randn(seed + 3, B, T, C, dtype=dtype) if gate else None, randn(seed + 4, B, C), randn(seed + 5, B, T, C, dtype=dtype),
            randn(seed + 6, B, C))


RECUR_SIZES = [(1, 1, 1), (3, 1, 70), (2, 5, 64), (2, 16, 3), (2, 17, 65), (1, 128, 64), (2, 129, 36), (300, 40, 70), (1, 1000, 130),
               (2, 2600, 8), (1, 5000, 64)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("size", RECUR_SIZES)
def test_linear_recurrence(ops, size, dtype):
    x, d, z, h0, dy, dlast = recurrence_inputs(*size, dtype)
    check_recurrence(ops, x, d, z, h0, dy, dlast, False)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("size", [(70, 1, 130), (5, 2, 37), (7, 3, 130), (5, 4, 37), (40, 7, 9), (2, 15, 64), (130, 16, 128)])
def test_linear_recurrence_short(ops, size, reverse, dtype):
    x, d, z, h0, dy, dlast = recurrence_inputs(*size, dtype, gate=not reverse)
    check_recurrence(ops, x, d, z, h0, dy, dlast, reverse)


@pytest.mark.parametrize("size", RECUR_SIZES)
def test_linear_recurrence_reverse_without_gate(ops, size):
    x, d, _, _, dy, _ = recurrence_inputs(*size, torch.float32, gate=False)
    check_recurrence(ops, x, d, None, None, dy, None, True)


@pytest.mark.parametrize("T", [9, 300, 1500])
def test_linear_recurrence_strided(ops, T):
    """Slices of one projection, a decay shared by all positions, a gradient expanded from one value, unit batch strides."""
    B, C = 3, 72
    proj = randn(1, B, T, 3 * C, dtype=torch.bfloat16)
    x, z = proj[..., :C], proj[..., C + 5:2 * C + 5]
    d = randn(2, C, dtype=torch.bfloat16, shift=2).expand(B, T, C)
    check_recurrence(ops, x, d, z, randn(4, B, C), randn(5, 1, 1, 1, dtype=torch.bfloat16).expand(B, T, C), None, False)
    xt = randn(6, T, B, C).transpose(0, 1)                          # time outermost
    check_recurrence(ops, xt, randn(7, B, C, T).transpose(1, 2), None, None, xt, None, True)


@pytest.mark.parametrize("T", [12, 700])
def test_linear_recurrence_pads_and_restarts(ops, T):
    """decay = +inf: the state passes a padded position unchanged; −inf: a packed sequence starts from its x."""
    B, C = 2, 40
    x, d, z, h0, dy, dlast = recurrence_inputs(B, T, C, torch.float32)
    n = T // 2
    pad = d.clone()
    pad[:, n:] = float("inf")
    y, last, _ = ops.linear_recurrence_fwd(x, pad, z, h0)
    assert torch.allclose(last, ops.linear_recurrence_fwd(x[:, :n], d[:, :n], z[:, :n], h0)[1], rtol=1e-5, atol=1e-6)
    check_recurrence(ops, x, pad, z, h0, dy, dlast, False)
    cut = d.clone()
    cut[:, n] = float("-inf")
    check_recurrence(ops, x, cut, z, h0, dy, dlast, False)
    y = ops.linear_recurrence_fwd(x, cut, None, h0)[0]
    assert torch.equal(y[:, n], x[:, n])


def test_linear_recurrence_continues(ops):
    """A sequence cut in pieces, each from the last state of the one before, down to single positions."""
    x, d, z, h0, _, _ = recurrence_inputs(2, 400, 48, torch.float32)
    y, last, _ = ops.linear_recurrence_fwd(x, d, z, h0)
    h, parts = h0, []
    for lo, hi in ((0, 131), (131, 132), (132, 133), (133, 390), (390, 400)):
        p, h, _ = ops.linear_recurrence_fwd(x[:, lo:hi], d[:, lo:hi], z[:, lo:hi], h)
        parts.append(p)
    assert torch.allclose(torch.cat(parts, 1), y, rtol=2e-5, atol=2e-6) and torch.allclose(h, last, rtol=2e-5, atol=2e-6)


def test_linear_recurrence_empty(ops):
    x, d, z, h0, dy, dlast = recurrence_inputs(2, 4, 8, torch.float32)
    y, last, carry = ops.linear_recurrence_fwd(x[:, :0], d[:, :0], z[:, :0], h0)
    assert y.shape == (2, 0, 8) and torch.equal(last, h0)
    dx, dd, dz, dh0 = ops.linear_recurrence_bwd(x[:, :0], d[:, :0], carry, dy[:, :0], z[:, :0], dlast)
    assert dx.shape == (2, 0, 8) and torch.equal(dh0, dlast)
    y, last, _ = ops.linear_recurrence_fwd(x[:0], d[:0])
    assert y.shape == (0, 4, 8) and last.shape == (0, 8)


# ---- registered ops, compositions, streams and graphs -------------------------------------------

def block(p, x, h0, reverse=False):
    """x + R(LN x), then + FFN(LN ·): the operators as a network uses them, on [B, T, C]."""
    m = torch.ops.mragan
    C = x.shape[-1]
    n = m.layer_norm(x, p["w1"], p["b1"], 1e-5)[0]
    proj = n @ p["proj"].t()
    r, last, _ = m.linear_recurrence(proj[..., :C], proj[..., C:2 * C], proj[..., 2 * C:], h0, reverse)
    x = x + r
    n = m.layer_norm(x, p["w2"], p["b2"], 1e-5)[0]
    return x + m.gated_ffn(n, p["wg"], p["wu"], p["wd"], None, None, p["bd"], "silu", True)[0], last


def plain_block(p, x, h0):
    C = x.shape[-1]
    n = torch.nn.functional.layer_norm(x, (C,), p["w1"], p["b1"])
    a, d, z = (n @ p["proj"].t()).split(C, -1)
    h, out = h0, []
    for t in range(x.shape[1]):
        h = torch.sigmoid(d[:, t]) * h + torch.sigmoid(-d[:, t]) * a[:, t]
        out.append(h * torch.nn.functional.silu(z[:, t]))
    x = x + torch.stack(out, 1)
    n = torch.nn.functional.layer_norm(x, (C,), p["w2"], p["b2"])
    return x + (torch.nn.functional.silu(n @ p["wg"].t()) * (n @ p["wu"].t())) @ p["wd"].t() + p["bd"], h


def block_params(C, F, dtype=torch.float32):
    return dict(w1=randn(1, C, shift=1, scale=0.1, dtype=dtype), b1=randn(2, C, scale=0.1, dtype=dtype),
                proj=randn(3, 3 * C, C, scale=C ** -0.5, dtype=dtype), w2=randn(4, C, shift=1, scale=0.1, dtype=dtype),
                b2=randn(5, C, scale=0.1, dtype=dtype), wg=randn(6, F, C, scale=C ** -0.5, dtype=dtype),
                wu=randn(7, F, C, scale=C ** -0.5, dtype=dtype), wd=randn(8, C, F, scale=F ** -0.5, dtype=dtype),
                bd=randn(9, C, scale=0.1, dtype=dtype))


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def test_block_matches_plain(ops):
    """The composed block and every gradient against float64 autograd.  fp32 throughout: about ten chained operations,
    each off by a few 2^-24 of its terms' sum, whose cancellation costs a factor of the order of ten."""
    B, T, C, F = 2, 150, 64, 160
    p = block_params(C, F)
    x, h0 = randn(11, B, T, C), randn(12, B, C)
    dy, dl = randn(13, B, T, C), randn(14, B, C)
    leaves = [x, h0, *p.values()]
    for t in leaves:
        t.requires_grad_()
    y, last = block(p, x, h0)
    got = torch.autograd.grad((y, last), leaves, (dy, dl))
    ref = [t.detach().double().cpu().requires_grad_() for t in leaves]
    yr, lr = plain_block(dict(zip(p, ref[2:])), ref[0], ref[1])
    want = torch.autograd.grad((yr, lr), ref, (dy.double().cpu(), dl.double().cpu()))
    assert rel(y.detach().cpu(), yr.detach()) < 1e-5 and rel(last.detach().cpu(), lr.detach()) < 1e-5
    for name, g, w in zip(["x", "h0", *p], got, want):
        assert rel(g.cpu(), w) < 1e-5, name


def test_gradients_against_differences(ops):
    """Directional derivatives of each registered op in fp32 against central differences of itself: truncation of
    order s² and rounding of order 2^-24/s, at s = 2^-7 both below 1e-3 of a derivative of order one."""
    m = torch.ops.mragan
    cases = [
        (lambda x, w, b: m.layer_norm(x, w, b, 1e-5)[0], [randn(1, 9, 40), randn(2, 40), randn(3, 40)]),
        (lambda *t: m.gated_ffn(*t, "gelu", False)[0], [t for q in ffn_inputs(9, 24, 40, 16, torch.float32)[:2] for t in q]),
        (lambda x, d, z, h: m.linear_recurrence(x, d, z, h, False)[0], list(recurrence_inputs(2, 40, 12, torch.float32)[:4])),
        (lambda x, d, z, h: m.linear_recurrence(x, d, z, h, True)[1], list(recurrence_inputs(2, 40, 12, torch.float32)[:4])),
    ]
    for fn, ts in cases:
        ts = [t.requires_grad_() for t in ts]
        out = fn(*ts)
        w = randn(77, *out.shape)
        grads = torch.autograd.grad(out, ts, w, allow_unused=True)
        for k, (t, g) in enumerate(zip(ts, grads)):
            v = randn(90 + k, *t.shape)
            v /= v.norm()
            s = 2.0 ** -7
            with torch.no_grad():
                f = [(fn(*[q + sg * s * v if q is t else q for q in ts]).double() * w.double()).sum() for sg in (1, -1)]
            num, ana = float(f[0] - f[1]) / (2 * s), 0.0 if g is None else float((g.double() * v.double()).sum())
            assert abs(num - ana) < 2e-3 * max(1.0, abs(ana)), (k, num, ana)


def test_opcheck(ops):
    checks = ("test_schema", "test_autograd_registration", "test_faketensor")
    m = torch.ops.mragan
    x = randn(1, 3, 5, 24).requires_grad_()
    w = randn(2, 24).requires_grad_()
    torch.library.opcheck(m.layer_norm.default, (x, w, None, 1e-5), test_utils=checks)
    (a, b, _) = ffn_inputs(15, 24, 40, 16, torch.float32)
    for keep in (False, True):
        torch.library.opcheck(m.gated_ffn.default, (a[0].requires_grad_(), *a[1:], *b, "silu", keep), test_utils=checks)
    r = recurrence_inputs(2, 20, 12, torch.float32)
    torch.library.opcheck(m.linear_recurrence.default, (r[0].requires_grad_(), r[1], r[2], r[3], True), test_utils=checks)


def everything(ops, s):
    """Each operator once, forward and backward, on the state's tensors."""
    y, mean, rstd = ops.layer_norm_fwd(s["x"], s["w"], s["b"])
    out = [y, *ops.layer_norm_bwd(s["x"], mean, rstd, s["dy"], s["w"], bias=True)]
    y, kept = ops.gated_ffn_fwd(s["x"], s["wg"], s["wu"], s["wd"], act="gelu", keep=True)
    out += [y, *[g for g in ops.gated_ffn_bwd(s["x"], s["wg"], s["wu"], s["wd"], s["dy"], kept, act="gelu") if g is not None]]
    q = [s[k].view(s["B"], -1, s["x"].shape[-1]) for k in ("x", "d", "dy")]
    y, last, carry = ops.linear_recurrence_fwd(q[0], q[1], q[2])
    return out + [y, last, *ops.linear_recurrence_bwd(q[0], q[1], carry, q[2], q[0])]


def state(seed, dtype, rows=1200, C=64, F=192, B=2):
    return dict(B=B, x=randn(seed, rows, C, dtype=dtype), dy=randn(seed + 1, rows, C, dtype=dtype), d=randn(seed + 2, rows, C, dtype=dtype, shift=2),
                w=randn(seed + 3, C, dtype=dtype), b=randn(seed + 4, C, dtype=dtype), wg=randn(seed + 5, F, C, dtype=dtype, scale=0.1),
                wu=randn(seed + 6, F, C, dtype=dtype, scale=0.1), wd=randn(seed + 7, C, F, dtype=dtype, scale=0.1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_repeatable_and_captured(ops, dtype):
    """The same bits from call to call, and from replays of two captured graphs with other work between them."""
    states = [state(100, dtype), state(200, dtype, rows=700, C=96, F=130)]
    want = [[t.clone() for t in everything(ops, s)] for s in states]
    for s, w in zip(states, want):
        assert all(torch.equal(p, q) for p, q in zip(everything(ops, s), w))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(everything(ops, s))
        graphs.append(g)
    side = torch.cuda.Stream()
    for _ in range(3):
        for o in outs:
            for t in o:
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):                              # both graphs at once
            graphs[1].replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(o, w))
        everything(ops, states[1])
        torch.cuda.synchronize()


def test_two_streams_at_once(ops):
    states = [state(300 + 10 * k, torch.bfloat16, rows=4000 + 500 * k) for k in range(2)]
    want = [everything(ops, s) for s in states]
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                got.append(everything(ops, s))
        torch.cuda.synchronize()
        for o, w in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(o, w))


def test_refusals(ops):
    x = randn(1, 4, 8)
    for bad in (x.double(), x.int(), x.cpu()):
        with pytest.raises(ValueError):
            ops.layer_norm_fwd(bad)
    for w in (randn(2, 7), randn(2, 8).bfloat16(), randn(2, 8).cpu(), randn(2, 8).double()):
        with pytest.raises(ValueError):
            ops.layer_norm_fwd(x, w)
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x, randn(2, 8), randn(3, 8), eps=-1.0)
    with pytest.raises(ValueError):
        ops.layer_norm_fwd(x.bfloat16(), randn(2, 8), randn(3, 8).bfloat16())
    _, mean, rstd = ops.layer_norm_fwd(x)
    for dy in (randn(3, 4, 7), x.bfloat16()):
        with pytest.raises(ValueError):
            ops.layer_norm_bwd(x, mean, rstd, dy)
    (a, b, dy) = ffn_inputs(5, 8, 12, 6, torch.float32)
    for k, t in ((0, a[0].half()), (1, a[1].t()), (2, a[2][:11]), (3, a[3].t()), (3, a[3].cpu())):
        with pytest.raises(ValueError):
            ops.gated_ffn_fwd(*[t if q == k else a[q] for q in range(4)])
    with pytest.raises(ValueError):
        ops.gated_ffn_fwd(*a, b[0][:3], b[1], b[2])
    with pytest.raises(ValueError):
        ops.gated_ffn_fwd(*a, act="softplus")
    with pytest.raises(ValueError):
        ops.gated_ffn_bwd(*a, dy[:, :5])
    with pytest.raises(ValueError):
        ops.gated_ffn_bwd(*a, dy, randn(1, 3, 5, 11))
    r = recurrence_inputs(2, 6, 8, torch.float32)
    for bad in ((r[0][0], r[1][0]), (r[0], r[1][:, :5]), (r[0], r[1].half())):
        with pytest.raises(ValueError):
            ops.linear_recurrence_fwd(*bad)
    with pytest.raises(ValueError):
        ops.linear_recurrence_fwd(r[0], r[1], h0=r[3].half())
    _, _, carry = ops.linear_recurrence_fwd(r[0], r[1])
    with pytest.raises(ValueError):
        ops.linear_recurrence_bwd(r[0], r[1], carry[:, :0], r[4])
    from mragan_hip import MraganError
    from mragan_hip._lib import call
    with pytest.raises(MraganError, match="workspace"):
        call("mragan_gated_ffn_fwd", a[0].data_ptr(), 5, 8, 12, 6, 0, a[1].data_ptr(), a[2].data_ptr(), a[3].data_ptr(), None, None,
             None, 5, dy.data_ptr(), None, None, 0, None)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("size", [(2, 140, 1), (3, 300, 2), (2, 200, 15), (2, 300, 33), (2, 400, 63), (3, 1300, 117), (1, 5000, 65),
                                  (2, 300, 129)])
def test_linear_recurrence_last_channels(ops, size, dtype):
    """Channel counts that end inside a tile, in one segment and in several, in both directions."""
    x, d, z, h0, dy, dlast = recurrence_inputs(*size, dtype)
    check_recurrence(ops, x, d, z, h0, dy, dlast, False)
    check_recurrence(ops, x, d, None, h0, dy, dlast, True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("frozen", ["gate", "up"])
@pytest.mark.parametrize("size", [(1024, 512, 1024, 512), (512, 512, 1024, 512), (1000, 136, 1032, 40)])
def test_gated_ffn_one_frozen_weight(ops, size, frozen, dtype):
    """One of the two projections without a gradient, whose product alone splits where the two together do not: its
    gradients, and nothing behind a workspace of the queried size."""
    need = tuple(k != (1 if frozen == "gate" else 2) for k in range(7))
    a, b, dy = ffn_inputs(*size, dtype)
    check_ffn(ops, a, b, dy, "silu", need=need)
    check_ffn(ops, a, b, dy, "silu", need=need, keep=False)
    from mragan_hip._lib import call, query
    M, C, F, O = size
    code = DTYPES.index(dtype)
    nbytes = query("mragan_gated_ffn_workspace", M, C, F, O, code, 1, 1)
    ws = torch.full((nbytes + (64 << 20),), 0xA5, dtype=torch.uint8, device="cuda")
    grads = [torch.empty_like(t) if n else None for t, n in zip([*a, *b], need)]
    p = lambda t: None if t is None else t.data_ptr()
    call("mragan_gated_ffn_bwd", p(a[0]), M, C, F, O, code, *map(p, a[1:]), p(b[0]), p(b[1]), 5, p(dy), None, *map(p, grads),
         p(ws), nbytes, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert bool((ws[nbytes:] == 0xA5).all())
    for got, want in zip(grads, ops.gated_ffn_bwd(*a, dy, None, *b, need=need)):
        assert got is want is None or torch.equal(got, want)


def test_gated_ffn_frozen_weight_registered(ops):
    a, b, dy = ffn_inputs(1024, 512, 1024, 512, torch.bfloat16)
    for k, t in enumerate(a):
        t.requires_grad_(k != 2)
    y = torch.ops.mragan.gated_ffn(*a, *b, "silu", True)[0]
    got = torch.autograd.grad(y, [a[0], a[1], a[3]], dy)
    _, kept = ops.gated_ffn_fwd(*a, *b, keep=True)
    want = ops.gated_ffn_bwd(*a, dy, kept, *b, need=(True, True, False, True) + (False,) * 3)
    assert all(torch.equal(g, w) for g, w in zip(got, (want[0], want[1], want[3])))


@pytest.mark.parametrize("reverse", [False, True])
def test_linear_recurrence_position_of_time_major(ops, reverse):
    """One position of [T, B, C] tensors whose steps are 2^22 elements apart."""
    seqs = [randn(k, 3, 1024, 4096, dtype=torch.bfloat16) for k in range(4)]
    x, d, z, dy = (t[1:2].transpose(0, 1) for t in seqs)
    check_recurrence(ops, x, d, z, randn(4, 1024, 4096), dy, randn(5, 1024, 4096), reverse)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("T,C,dtype", [(9, 1 << 22, torch.float32), (17, 256 * 256 * 64, torch.bfloat16), (130, (1 << 23) + 70, torch.float16)])
def test_linear_recurrence_wide_rows(ops, T, C, dtype, reverse):
    """Scans along the depth of wide volumes, tensors of more than 2^31 bytes among them; channels do not mix, so the
    first and the last ones are compared."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    new = lambda *s, t=dtype, shift=0.0: torch.empty(s, dtype=t, device="cuda").normal_(shift, 1.0, generator=gen)
    x, d, z, dy = new(1, T, C), new(1, T, C, shift=2.0), new(1, T, C), new(1, T, C)
    h0, dlast = new(1, C, t=torch.float32), new(1, C, t=torch.float32)

    class Part:
        """The operator on whole rows, seen through some of their channels."""
        sel = None

        def linear_recurrence_fwd(self, *_, reverse):
            y, last, self.carry = ops.linear_recurrence_fwd(x, d, z, h0, reverse=reverse)
            return y[..., self.sel], last[..., self.sel], None

        def linear_recurrence_bwd(self, *_, reverse):
            return [t[..., self.sel] for t in ops.linear_recurrence_bwd(x, d, self.carry, dy, z, dlast, reverse=reverse)]

    part = Part()
    for part.sel in (slice(0, 66), slice(C - 131, C)):
        check_recurrence(part, *(t[..., part.sel] for t in (x, d, z, h0, dy, dlast)), reverse)


def test_layer_norm_longest_rows(ops):
    """Rows of 2^26 channels, whose parameter sums have more columns than one launch has threads for at 64 a column.
    Bounds as in check_norm, with the additions that one of a block's 1024 threads makes."""
    rows, C = 2, (1 << 26) + 5
    gen = torch.Generator(device="cuda").manual_seed(1)
    new = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda").normal_(0.5, 1.0, generator=gen)
    check_norm(ops, new(rows, C), new(C), new(C), dy=new(rows, C))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_gated_ffn_more_packed_rows_than_blocks(ops, dtype):
    """Rows of odd length whose padded copy is longer than one pass of its launch (2^28 elements)."""
    M, C, F, O = (1 << 20) + 77, 201, 8, 9
    gen = torch.Generator(device="cuda").manual_seed(1)
    new = lambda *s, k=1: (torch.empty(s, device="cuda").normal_(generator=gen) * k ** -0.5).to(dtype)
    a = [new(M, C), new(F, C, k=C), new(F, C, k=C), new(O, F, k=F)]
    check_ffn(ops, a, [new(F), new(F), new(O)], new(M, O), "silu")


def test_second_derivatives_refused(ops):
    """A gradient penalty through one of the operators raises where it would need their second derivative; the first
    one is the same with create_graph as without."""
    m = torch.ops.mragan
    a, b, _ = ffn_inputs(9, 24, 40, 16, torch.float32)
    r = recurrence_inputs(2, 20, 12, torch.float32)
    for x, fn in ((randn(1, 6, 40), lambda t: m.layer_norm(t, randn(2, 40), None, 1e-5)[0]),
                  (a[0], lambda t: m.gated_ffn(t, *a[1:], *b, "silu", True)[0]),
                  (a[0], lambda t: m.gated_ffn(t, *a[1:], *b, "silu", False)[0]),
                  (r[0], lambda t: m.linear_recurrence(t, *r[1:4], False)[0]),
                  (r[0], lambda t: m.linear_recurrence(t, *r[1:4], False)[1])):
        x = x.clone().requires_grad_()
        y = fn(x)
        want = torch.autograd.grad(y.square().sum(), x, retain_graph=True)[0]
        (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        assert torch.equal(g.detach(), want)
        with pytest.raises(RuntimeError, match="second derivative"):
            (y.sum() + g.square().sum()).backward()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("size", [(2, 700, 15), (3, 129, 33), (2, 400, 63), (3, 1300, 117), (1, 5000, 65), (2, 9, 7), (1, 4100, 679)])
def test_linear_recurrence_channels_do_not_depend_on_their_place(ops, size, dtype):
    """An odd channel count moves the last lanes back by one, so that two of them form the same channel in different
    places: each channel has the same bits as in a tensor of one channel more, and from call to call."""
    B, T, C = size
    x, d, z, h0, dy, dlast = recurrence_inputs(B, T, C + 1, dtype)

    def run(n, gated, reverse):
        c = lambda t: t[..., :n].contiguous()
        g = c(z) if gated else None
        y, last, carry = ops.linear_recurrence_fwd(c(x), c(d), g, c(h0), reverse=reverse)
        grads = ops.linear_recurrence_bwd(c(x), c(d), carry, c(dy), g, c(dlast), reverse=reverse)
        return [t[..., :C] for t in (y, last, carry, *grads) if t is not None]

    for gated, reverse in ((True, False), (False, True)):
        odd = run(C, gated, reverse)
        for want in (run(C + 1, gated, reverse), run(C, gated, reverse)):
            assert all(torch.equal(p, q) for p, q in zip(odd, want))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(700, 9), (300, 33), (90, 515), (70, 1001), (20, 2051), (9, 5003)])
def test_layer_norm_columns_do_not_depend_on_their_place(ops, shape, dtype):
    """The last vector of a row of odd length is moved back over columns of the one before, which both write:
    columns that are alike have the same bits wherever they stand, and from call to call."""
    R, C = shape
    x, dy = randn(1, R, 1, dtype=dtype), randn(2, R, 1, dtype=dtype)
    noise, k = randn(3, R, C // 2, dtype=dtype), C // 2
    x = torch.cat((noise, x.expand(R, C - k)), 1)                    # columns k … C − 1 are alike
    dy = torch.cat((noise.flip(0), dy.expand(R, C - k)), 1)
    w, b = (torch.cat((randn(s, k, dtype=dtype), randn(s + 1, 1, dtype=dtype).expand(C - k))) for s in (4, 6))
    for _ in range(3):
        y, mean, rstd = ops.layer_norm_fwd(x, w, b)
        dx, _, _ = ops.layer_norm_bwd(x, mean, rstd, dy, w, True)
        for t in (y, dx):
            assert torch.equal(t[:, k:], t[:, k:k + 1].expand(R, C - k))


def ffn_tiles(run):
    """The products' launches of a call and their tiles, in order."""
    from mragan_hip._lib import lib
    lib().mragan_launch_log(1)
    run()
    return [n[len("ffn_gemm_"):] for n in lib().mragan_launch_log(1).decode().split(";") if n.startswith("ffn_gemm_")]


LARGE = {"one plane": [(torch.bfloat16, "f32"), (torch.float16, "f32"), (torch.float32, "bf16"), (torch.float32, "fp16")],
         "plane pairs": [(torch.float32, "f32"), (torch.float32, "bf16x3")]}


@pytest.mark.parametrize("dtype,mode", LARGE["one plane"] + LARGE["plane pairs"], ids=str)
@pytest.mark.parametrize("size,tiles", [
    ((4100, 3600, 4104, 3592), (256, 256, 256, 256, 256, 256)),
    ((4099, 3601, 4101, 3593), (256, 256, 256, 256, 256, 256)),
    ((4100, 1032, 4104, 1040), (256, 128, 256, 128, 128, 128)),
    ((2801, 1289, 2051, 1801), (128, 128, 128, 128, 128, 128)),
    ((200, 2056, 8200, 1000), (128, 64, 64, 64, 256, 128)),
    ((500, 2056, 8200, 2056), (128, 64, 128, 64, 256, 256)),
], ids=str)
def test_gated_ffn_large_tiles(ops, size, tiles, dtype, mode):
    """Each product (gate and up, down, dg and du, dx, both projections' weights, w_down) on the larger tiles, with
    remainders along all sides."""
    a, b, dy = ffn_inputs(*size, dtype)
    ops.set_conv_precision(mode)
    _, kept = ops.gated_ffn_fwd(*a, *b, keep=True)
    names = ["gate_%d", "%d", "gate_bwd_%d", "%d", "%d", "%d"]
    want = [n % t for n, t in zip(names, tiles)]
    assert ffn_tiles(lambda: ops.gated_ffn_fwd(*a, *b, keep=True)) == want[:2]
    assert ffn_tiles(lambda: ops.gated_ffn_bwd(*a, dy, kept, *b)) == want[2:]
    check_ffn(ops, a, b, dy, "silu", mode=mode)
    if dtype == torch.bfloat16:
        check_ffn(ops, a, b, dy, "gelu", mode=mode, keep=False, need=(True, False, True, True) + (True,) * 3)


# ---- tensors whose offsets pass 32 bits -----------------------------------------------------------
# Each operator on the whole tensors, seen through the rows at their end: only those have a gradient, so the
# sums over all rows are theirs.

def fresh(seed, *shape, dtype=torch.bfloat16, shift=0.0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(shift, scale, generator=gen)


@pytest.mark.parametrize("rows,C", [((1 << 26) + 3, 70), ((1 << 19) + 1, 8200), ((1 << 23) + 5, 515)])
def test_layer_norm_far_rows(ops, rows, C):
    x, w, b = fresh(1, rows, C, scale=2.0), fresh(2, C), fresh(3, C)
    dy, tail = torch.zeros_like(x), slice(rows - 300, None)
    dy[tail] = fresh(4, 300, C)

    class Part:
        def layer_norm_fwd(self, *_):
            y, *self.stats = ops.layer_norm_fwd(x, w, b, 1e-5)
            return y[tail], *[t[tail] for t in self.stats]

        def layer_norm_bwd(self, *_, bias):
            dx, dw, db = ops.layer_norm_bwd(x, *self.stats, dy, w, bias=bias)
            assert not dx[:1000].any()
            return dx[tail], dw, db

    check_norm(Part(), x[tail], w, b, dy=dy[tail])


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("size", [((1 << 20) + 9, 64, 4160, 72), ((1 << 22) + 9, 1032, 40, 1033)])
def test_gated_ffn_far_rows(ops, size, keep):
    M, C, F, O = size
    x, (a, b, _) = fresh(1, M, C), ffn_inputs(1, C, F, O, torch.bfloat16)
    dy, tail = torch.zeros(M, O, dtype=torch.bfloat16, device="cuda"), slice(M - 300, None)
    dy[tail] = fresh(2, 300, O)

    class Part:
        set_conv_precision = staticmethod(ops.set_conv_precision)

        def gated_ffn_fwd(self, *_, act, keep):
            y, self.kept = ops.gated_ffn_fwd(x, *a[1:], *b, act=act, keep=keep)
            return y[tail], None

        def gated_ffn_bwd(self, *_, act, need):
            dx, *rest = ops.gated_ffn_bwd(x, *a[1:], dy, self.kept, *b, act=act, need=need)
            assert not dx[:1000].any()
            return [dx[tail], *rest]

    check_ffn(Part(), [x[tail], *a[1:]], b, dy[tail], "silu", keep=keep)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("C", [66, 5])
def test_linear_recurrence_far_steps(ops, C, reverse):
    """More than 2^32 elements of one sequence.  The checked steps restart the state, so that they depend on no others;
    backwards the first steps taken are the far ones, whose bits are those of a short sequence."""
    T, n = ((1 << 26) if C == 66 else (1 << 28)) + 77, 640
    x, d, dy = fresh(1, 1, T, C), fresh(2, 1, T, C, shift=2.5), fresh(3, 1, T, C)
    h0, dlast = fresh(4, 1, C, dtype=torch.float32), fresh(5, 1, C, dtype=torch.float32)
    sel = slice(0, n) if reverse else slice(T - n, T)
    d[:, n - 1 if reverse else T - n] = float("-inf")

    class Part:
        def linear_recurrence_fwd(self, *_, reverse):
            self.y, last, self.carry = ops.linear_recurrence_fwd(x, d, None, h0, reverse=reverse)
            return self.y[:, sel], last, None

        def linear_recurrence_bwd(self, *_, reverse):
            *grads, _ = ops.linear_recurrence_bwd(x, d, self.carry, dy, None, dlast, reverse=reverse)
            return [t if t is None else t[:, sel] for t in grads] + [torch.zeros(1, C, device="cuda")]   # a restart passes nothing back

    part = Part()
    check_recurrence(part, x[:, sel], d[:, sel], None, h0, dy[:, sel], dlast, reverse)
    if reverse:
        far = slice(T - n, T)
        assert torch.equal(part.y[:, far], ops.linear_recurrence_fwd(x[:, far], d[:, far], None, h0, reverse=True)[0])


LONG = (1 << 22) - 64


@pytest.mark.parametrize("size", [(70, LONG, 24, 8), (70, LONG - 3, 16, 9), (33, 16, LONG, 8), (33, 9, LONG - 5, 8), (70, 16, 24, LONG),
                                  (2, LONG - 1, 9, 8), (300, LONG, 16, 8)])
def test_gated_ffn_longest_sides(ops, size):
    M, C, F, O = size
    a = [fresh(1, M, C), fresh(2, F, C, scale=C ** -0.5), fresh(3, F, C, scale=C ** -0.5), fresh(4, O, F, scale=F ** -0.5)]
    b = [fresh(5, F), fresh(6, F), fresh(7, O)]
    for keep in (True, False):
        check_ffn(ops, a, b, fresh(8, M, O), "silu", keep=keep)
