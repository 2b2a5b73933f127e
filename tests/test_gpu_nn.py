"""The recurrent-block operators (phyz_b200.nn) against their definitions in 64 bits.

Tolerances, all from the arithmetic's own bounds. u is the unit roundoff of an array's type (2^-24, 2^-8, 2^-11). A
sum of K products in f32, in any order and with additions rounded either way, is off by at most (K + 8) 2^-23 times
the sum of the products' magnitudes. An activation is 1.13-Lipschitz and evaluated within a few f32 roundings (16 *
2^-23 of max(1, |z|)). A result is rounded to its type once (u), in f16 with an absolute 2^-25 below its normal range.
"""
import math

import pytest
import torch

from phyz_b200 import nn

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "tanh", "silu", "gelu"]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(g, *shape, dt=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dt)


def act64(z, act):
    return {"none": lambda v: v, "relu": torch.relu, "tanh": torch.tanh, "silu": torch.nn.functional.silu,
            "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[act](z)


def gamma(k):
    return (k + 8) * 2.0 ** -23


def within(got, want, tol):
    off = (got.double() - want).abs() - (tol + 2.0 ** -25)
    assert torch.isfinite(got.double()).all()
    assert off.max() <= 0, f"over the tolerance by {off.max():.3g}, |want| up to {want.abs().max():.3g}"


def near(got, want, u):
    """Over a whole array roundings average out: the relative 2-norm of the error stays under u."""
    n = want.norm()
    assert (got.double() - want).norm() <= u * n


# ── linear ────────────────────────────────────────────────────────────────

def layout(t, how):
    """t's values behind other strides: as they are, feature-major, in rows longer than they are, from an odd offset,
    every second column."""
    r, c = t.shape
    if how == "features":
        return t.t().contiguous().t()
    if how == "padded":
        return torch.cat([t, torch.full((r, 8 if c % 8 == 0 else 3), float("nan"), dtype=t.dtype, device=t.device)],
                         1)[:, :c]
    if how == "odd":
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(r, c)
    if how == "strided":
        wide = torch.full((r, 2 * c), float("nan"), dtype=t.dtype, device=t.device)
        wide[:, ::2] = t
        return wide[:, ::2]
    return t


def check_forward(dt, m, k, n, act, bias, residual, how, seed=0, scale=1.0):
    g = gen(seed)
    x, w = layout(rnd(g, m, k, dt=dt, std=scale), how), layout(rnd(g, n, k, dt=dt, std=1 / math.sqrt(k)), how)
    b = rnd(g, n) if bias else None
    r = layout(rnd(g, m, n, dt=dt), how) if residual else None
    y, pre = nn.linear(x, w, b, activation=act, residual=r, save_pre=True)
    assert y.dtype == dt and y.shape == (m, n)
    assert torch.equal(nn.linear(x, w, b, activation=act, residual=r), y)
    z = x.double() @ w.double().t() + (b.double() if bias else 0)
    mag = x.double().abs() @ w.double().abs().t() + (b.double().abs() if bias else 0)
    ez = gamma(k) * mag
    within(pre, z, ez + U[dt] * (z.abs() + ez))
    a = act64(z, act)
    want = a + (r.double() if residual else 0)
    ey = 1.13 * ez + 16 * 2.0 ** -23 * z.abs().clamp(min=1) + 2.0 ** -23 * (a.abs() + want.abs())
    within(y, want, ey + U[dt] * (want.abs() + ey))
    if m * n >= 1000 and dt != torch.float32:
        near(pre, z, U[dt])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 512, 1024), (3, 30, 64), (17, 33, 129), (128, 64, 128), (129, 65, 127),
                                   (256, 512, 300), (1000, 200, 72), (2049, 136, 264)])
def test_linear_sizes(dt, m, k, n):
    check_forward(dt, m, k, n, "silu", True, True, "rows")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear_activations(dt, act):
    check_forward(dt, 200, 96, 160, act, True, False, "rows", scale=4.0)
    check_forward(dt, 200, 96, 160, act, False, True, "features", scale=0.01)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("how", ["features", "padded", "odd", "strided"])
@pytest.mark.parametrize("m,k,n", [(64, 64, 64), (133, 515, 130), (300, 264, 520)])
def test_linear_layouts(dt, how, m, k, n):
    check_forward(dt, m, k, n, "tanh", True, True, how)


@pytest.mark.parametrize("k,n", [(30, 64), (1, 1), (64, 100), (300, 33), (37, 128)])
@pytest.mark.parametrize("act", ["tanh", "none"])
def test_linear_many_feature_major_rows(k, n, act):
    """The policy history's shape: rows enough to fill the GPU, feature-major."""
    check_forward(torch.float32, 19001, k, n, act, True, True, "features")
    check_forward(torch.float32, 19001, k, n, act, False, False, "features")


@pytest.mark.parametrize("how", ["rows", "features"])
def test_linear_backward_more_rows_than_a_grid_side(how):
    """9 million rows: more blocks of rows than a launch has along its second axis. With x = 1 and w = 1 the gradients
    are sums of dy, whole numbers that f32 and bf16 hold exactly in every order."""
    m = 9_000_000
    dy = torch.zeros(m, 8, device="cuda", dtype=torch.bfloat16)
    dy[::70_001] = 1
    dy[-1] = 1
    dy = layout(dy, how)
    x, w = torch.ones(m, 8, device="cuda", dtype=torch.bfloat16), torch.ones(8, 8, device="cuda", dtype=torch.bfloat16)
    dx, dw, db = nn.linear_backward(dy, x, w)
    hits = float(dy[:, 0].sum(dtype=torch.float64))
    assert (db == hits).all() and (dw == hits).all() and torch.equal(dx, (dy * 8).contiguous())


@pytest.mark.parametrize("dt", TYPES)
def test_linear_large(dt):
    check_forward(dt, 5003, 1032, 1000, "gelu", True, True, "rows")


@pytest.mark.parametrize("dt", TYPES)
def test_linear_no_rows(dt):
    w, b = torch.ones(8, 4, dtype=dt, device="cuda"), torch.ones(8, device="cuda")
    assert nn.linear(torch.empty(0, 4, dtype=dt, device="cuda"), w, b).shape == (0, 8)
    dx, dw, db = nn.linear_backward(torch.empty(0, 8, dtype=dt, device="cuda"),
                                    torch.empty(0, 4, dtype=dt, device="cuda"), w)
    assert dx.shape == (0, 4) and not dw.any() and not db.any()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m", [1, 40, 700])
def test_linear_into_the_residual(dt, m):
    g = gen(3)
    x, w, r = rnd(g, m, 64, dt=dt), rnd(g, 64, 64, dt=dt, std=0.1), rnd(g, m, 64, dt=dt)
    want = nn.linear(x, w, activation="relu", residual=r)
    assert nn.linear(x, w, activation="relu", residual=r, out=r) is r
    assert torch.equal(r, want)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k", [(5, 96), (300, 96), (3000, 640)])
def test_linear_nonfinite_rows_stay_theirs(dt, m, k):
    """A diverged world's row is not finite in its own outputs and changes no other row."""
    g = gen(4)
    x, w = rnd(g, m, k, dt=dt), rnd(g, 72, k, dt=dt, std=0.1)
    clean = nn.linear(x, w)
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    got = nn.linear(x, w)
    keep = torch.ones(m, dtype=torch.bool, device="cuda")
    keep[1:3] = False
    assert torch.equal(got[keep], clean[keep])
    assert got[1].isnan().all() and not got[2].isfinite().any()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_linear_rows_past_32_bit_offsets(dt):
    g = gen(5)
    stride = (1 << 31) // 2 + 64
    store = torch.empty(stride * 3 + 128, dtype=dt, device="cuda")
    x = store.as_strided((4, 128), (stride, 1))
    x.copy_(rnd(g, 4, 128, dt=dt))
    w = rnd(g, 96, 128, dt=dt, std=0.1)
    assert torch.equal(nn.linear(x, w), nn.linear(x.contiguous(), w))
    y = torch.empty(1, dtype=dt, device="cuda")
    del y
    out = store.as_strided((4, 96), (stride, 1))
    want = nn.linear(x.contiguous(), w)
    nn.linear(x.contiguous(), w, out=out)
    assert torch.equal(out, want)


def check_backward(dt, m, k, n, act, bias, how, seed=0, pre_how=None):
    g = gen(seed)
    x, w = layout(rnd(g, m, k, dt=dt), how), layout(rnd(g, n, k, dt=dt, std=1 / math.sqrt(k)), how)
    pre, dy = layout(rnd(g, m, n, dt=dt), pre_how or how), layout(rnd(g, m, n, dt=dt, std=0.5), how)
    dx, dw, db = nn.linear_backward(dy, x, w, pre if act != "none" else None, activation=act, bias=bias)
    z = pre.double().requires_grad_()
    slope = torch.autograd.grad(act64(z, act).sum(), z)[0] if act != "none" else torch.ones_like(z)
    dz = (dy.double() * slope).detach()
    edz = dy.double().abs() * 32 * 2.0 ** -23 * (1 + z.detach().abs())   # the slope's evaluation
    u = U[dt]
    e16 = edz + u * dz.abs() + 2.0 ** -25                     # and its rounding to the type
    for got, want, err, k_ in ((dx, dz @ w.double(), (e16 + gamma(n) * dz.abs()) @ w.double().abs(), n),
                               (dw, dz.t() @ x.double(), (e16 + gamma(m) * dz.abs()).t() @ x.double().abs(), m)):
        assert got.dtype == dt
        within(got, want, err + u * (want.abs() + err))
        if want.numel() >= 1000 and dt != torch.float32:
            near(got, want, u)
    if bias:
        assert db.dtype == torch.float32
        within(db, dz.sum(0), (edz + gamma(m) * dz.abs()).sum(0))
    else:
        assert db is None


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 64, 96), (7, 30, 64), (129, 65, 127), (1000, 200, 72),
                                   (1537, 515, 129), (4096, 128, 256), (3000, 264, 8)])
def test_linear_backward_sizes(dt, m, k, n):
    check_backward(dt, m, k, n, "tanh", True, "rows")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear_backward_activations(dt, act):
    check_backward(dt, 520, 96, 160, act, True, "rows")
    check_backward(dt, 520, 96, 160, act, False, "features")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("how", ["features", "padded", "odd", "strided"])
def test_linear_backward_layouts(dt, how):
    check_backward(dt, 203, 136, 130, "gelu", True, how)
    check_backward(dt, 640, 64, 128, "silu", True, how)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("how,pre_how", [("rows", "features"), ("features", "rows"), ("padded", "features"),
                                         ("features", "odd"), ("strided", "features")])
@pytest.mark.parametrize("m,k,n", [(32, 64, 32), (33, 24, 95), (31, 40, 70), (2049, 96, 130), (4200, 8, 33)])
def test_linear_backward_mixed_orders(dt, how, pre_how, m, k, n):
    check_backward(dt, m, k, n, "gelu", True, how, pre_how=pre_how)
    check_backward(dt, m, k, n, "tanh", False, how, pre_how=pre_how)


@pytest.mark.parametrize("dt", TYPES)
def test_linear_backward_wide(dt):
    check_backward(dt, 9000, 520, 1032, "silu", True, "rows")


def test_linear_backward_parts_and_repeats():
    g = gen(6)
    x, w, dy = rnd(g, 4000, 96, dt=torch.bfloat16), rnd(g, 64, 96, dt=torch.bfloat16), rnd(g, 4000, 64, dt=torch.bfloat16)
    dx, dw, db = nn.linear_backward(dy, x, w)
    for _ in range(3):  # fixed order of every sum
        assert all(torch.equal(a, b) for a, b in zip(nn.linear_backward(dy, x, w), (dx, dw, db)))
    only = nn.linear_backward(dy, x, w, need_dx=False, bias=False)
    assert only[0] is None and only[2] is None and torch.equal(only[1], dw)
    only = nn.linear_backward(dy, x, w, need_dw=False)
    assert only[1] is None and torch.equal(only[0], dx) and torch.equal(only[2], db)


@pytest.mark.parametrize("act", ACTS)
def test_linear_gradient_against_differences(act):
    """Central differences of L = sum(r * y) along random directions, in f32: the loss is summed in 64 bits, so its
    noise is y's rounding, sqrt(m n) 2^-23, over 2 eps; the third derivative (at most 2 |r| |d|^3) gives eps^2."""
    g = gen(7)
    m, k, n, eps = 33, 24, 40, 2.0 ** -7
    x, w, b, r = rnd(g, m, k), rnd(g, n, k, std=0.3), rnd(g, n), rnd(g, m, n)

    def loss(x, w, b):
        return (nn.linear(x, w, b, activation=act).double() * r.double()).sum()

    _, pre = nn.linear(x, w, b, activation=act, save_pre=True)
    if act == "relu":  # differences do not see a kink
        r[pre.abs() < 0.3] = 0
    dx, dw, db = nn.linear_backward(r, x, w, pre, activation=act)
    for i, (grad, v) in enumerate(((dx, x), (dw, w), (db, b))):
        d = rnd(g, *v.shape)
        d = d / d.norm()
        args = [x, w, b]
        up, down = list(args), list(args)
        up[i], down[i] = v + eps * d, v - eps * d
        num = (loss(*up) - loss(*down)) / (2 * eps)
        want = (grad.double() * d.double()).sum()
        noise = math.sqrt(m * n) * 2.0 ** -21 * 8 / eps
        cube = eps * eps * 2 * float(r.abs().max()) * float((d.norm() * max(x.norm(), w.norm())) ** 3) / math.sqrt(m * n)
        assert abs(num - want) <= noise + cube


# ── gated scan ────────────────────────────────────────────────────────────

def scan64(x, gate, h0, reset):
    a = torch.sigmoid(gate.double())
    h = torch.zeros_like(x[:, 0], dtype=torch.float64) if h0 is None else h0.double()
    out = torch.empty_like(x, dtype=torch.float64)
    for t in range(x.shape[1]):
        if reset is not None:
            h = torch.where(reset[:, t] != 0, torch.zeros_like(h), h)
        h = a[:, t] * h + (1 - a[:, t]) * x[:, t].double()
        out[:, t] = h
    return out, h


def seq(t, how):
    """[b, t, c] values behind other strides."""
    if how == "history":
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    if how == "time inside":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if how == "halves":  # one half of a projection that holds x and gate side by side
        return torch.cat([t, torch.full_like(t, float("nan"))], 2)[..., :t.shape[2]]
    if how == "odd":
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)
    return t


def scan_inputs(dt, b, t, c, how, resets, seed=0, mean=2.0):
    g = gen(seed)
    x, gate = seq(rnd(g, b, t, c, dt=dt), how), seq(rnd(g, b, t, c, dt=dt, std=1.5, mean=mean), how)
    h0 = rnd(g, b, c, std=0.7)
    reset = None
    if resets == "rows":
        reset = (torch.rand(b, t, generator=g, device="cuda") < 0.1).to(torch.uint8)
        if b > 1:
            reset[1] = 1  # a sequence that starts again at every step
    elif resets == "each":
        reset = torch.rand(b, t, c, generator=g, device="cuda") < 0.1
    elif resets == "inside":
        reset = torch.rand(1, t, c, generator=g, device="cuda") < 0.1
    return x, gate, h0, reset


def full(reset, shape):
    if reset is None:
        return None
    return (reset.unsqueeze(2) if reset.dim() == 2 else reset).expand(shape)


# a step's update rounds to f32 a few times, and what is carried is damped: a state is off by at most its roundings'
# sum, 1 / (1 - a) steps of 8 * 2^-24 each; gates reach a = sigmoid(7), so about 1000 steps of them, at most t
def scan_err(t):
    return 8 * 2.0 ** -24 * min(t, 1200) + 2.0 ** -22


def check_scan(dt, b, t, c, how="rows", resets=None, h0=True, seed=0):
    x, gate, s0, reset = scan_inputs(dt, b, t, c, how, resets, seed)
    s0 = s0 if h0 else None
    h, last = nn.gated_scan(x, gate, s0, reset)
    assert h.dtype == dt and h.shape == (b, t, c) and last.dtype == torch.float32
    want, end = scan64(x, gate, s0, full(reset, x.shape))
    big = float(want.abs().max()) + 1
    within(h, want, scan_err(t) * big + U[dt] * want.abs())
    within(last, end, scan_err(t) * big)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("b,t,c", [(1, 1, 1), (4, 1, 33), (1, 2, 8), (2, 3, 5), (3, 17, 64), (1, 1000, 3),
                                   (2, 1025, 72), (1, 4099, 256), (5, 64, 1000), (300, 5, 7), (1, 20000, 16)])
def test_scan_sizes(dt, b, t, c):
    check_scan(dt, b, t, c)
    check_scan(dt, b, t, c, resets="rows", h0=False)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("how", ["history", "time inside", "halves", "odd"])
@pytest.mark.parametrize("resets", ["rows", "each", "inside"])
@pytest.mark.parametrize("b,t,c", [(3, 70, 40), (2, 3000, 24)])
def test_scan_layouts_and_resets(dt, how, resets, b, t, c):
    check_scan(dt, b, t, c, how, resets)


@pytest.mark.parametrize("t", [1, 40, 9000])
def test_scan_reset_drops_a_nonfinite_state(t):
    x, gate, h0, _ = scan_inputs(torch.float32, 2, t, 8, "rows", None)
    reset = torch.zeros(2, t, dtype=torch.bool, device="cuda")
    reset[0, 0] = True
    h0[0, 0], h0[1, 1] = float("nan"), float("inf")
    h, last = nn.gated_scan(x, gate, h0, reset)
    assert h[0].isfinite().all() and last[0].isfinite().all()
    assert not h[1, 0, 1].isfinite() and h[1, :, 2:].isfinite().all()
    if t > 30:  # and in the middle: everything from the reset on is clean, everything before is not
        reset[:] = False
        reset[0, t - 7] = True
        h, last = nn.gated_scan(x, gate, h0, reset)
        assert h[0, t - 7:].isfinite().all() and last[0].isfinite().all() and h[0, :t - 7, 0].isnan().all()


def test_scan_saturated_gates():
    """sigmoid at its ends: exactly 1 keeps the state to the bit, exactly 0 replaces it."""
    x = rnd(gen(8), 2, 3000, 16)
    h0 = rnd(gen(9), 2, 16)
    h, last = nn.gated_scan(x, torch.full_like(x, 200.0), h0)
    assert torch.equal(last, h0) and torch.equal(h, h0[:, None].expand_as(h))
    h, _ = nn.gated_scan(x, torch.full_like(x, -200.0), h0)
    assert torch.equal(h, x)


@pytest.mark.parametrize("dt", TYPES)
def test_scan_step_by_step_is_the_scan(dt):
    """Serving one step at a time, the state kept in place, gives the sequence's outputs."""
    x, gate, h0, reset = scan_inputs(dt, 5, 12, 48, "rows", "rows")
    want, end = nn.gated_scan(x, gate, h0, reset)
    state = h0.clone()
    for t in range(12):
        h, state = nn.gated_scan(x[:, t:t + 1], gate[:, t:t + 1], state, reset[:, t:t + 1])
        assert (h.float() - want[:, t:t + 1].float()).abs().max() <= U[dt] * 8 + 2.0 ** -20
    assert (state - end).abs().max() <= 2.0 ** -20


def test_scan_empty():
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    h0 = rnd(gen(1), 3, 4)
    h, last = nn.gated_scan(z(3, 0, 4), z(3, 0, 4), h0)
    assert h.shape == (3, 0, 4) and torch.equal(last, h0)
    assert not nn.gated_scan(z(3, 0, 4), z(3, 0, 4))[1].any()
    assert nn.gated_scan(z(0, 5, 4), z(0, 5, 4))[0].shape == (0, 5, 4)
    assert nn.gated_scan(z(3, 5, 0), z(3, 5, 0))[1].shape == (3, 0)
    dl = rnd(gen(2), 3, 4)
    assert torch.equal(nn.gated_scan_backward(z(3, 0, 4), z(3, 0, 4), z(3, 0, 4), z(3, 0, 4), h0, None, dl)[2], dl)


def test_scan_past_32_bit_offsets():
    stride = (1 << 30) + 16
    store = torch.empty(stride * 4 + 64, dtype=torch.bfloat16, device="cuda")
    x, gate, out = (store.as_strided((1, 5, 16), (0, stride, 1), o) for o in (0, 16, 32))
    vx, vg, h0, _ = scan_inputs(torch.bfloat16, 1, 5, 16, "rows", None)
    x.copy_(vx)
    gate.copy_(vg)
    h, last = nn.gated_scan(x, gate, h0, out=out)
    want, end = nn.gated_scan(vx, vg, h0)
    assert torch.equal(h, want) and torch.equal(last, end)


def check_scan_grad(dt, b, t, c, how="rows", resets=None, h0=True, dlast=True, seed=0):
    x, gate, s0, reset = scan_inputs(dt, b, t, c, how, resets, seed)
    s0 = s0 if h0 else None
    g = gen(seed + 50)
    dh = seq(rnd(g, b, t, c, dt=dt), how)
    dl = rnd(g, b, c) if dlast else None
    r = full(reset, x.shape)
    h = seq(scan64(x, gate, s0, r)[0].to(dt), how)
    dx, dg, dh0 = nn.gated_scan_backward(dh, x, gate, h, s0, reset, dl)
    assert dx.dtype == dt and dg.dtype == dt and dh0.dtype == torch.float32
    a = torch.sigmoid(gate.double())
    keep = a if r is None else torch.where(r != 0, torch.zeros_like(a), a)
    before = torch.cat([(torch.zeros(b, 1, c, device="cuda", dtype=torch.float64) if s0 is None else s0.double()[:, None]),
                        h.double()[:, :-1]], 1)
    if r is not None:
        before = torch.where(r != 0, torch.zeros_like(before), before)
    d = torch.zeros(b, c, dtype=torch.float64, device="cuda") if dl is None else dl.double()
    want_x, want_g = torch.empty_like(a), torch.empty_like(a)
    big = 0.0
    for k in range(t - 1, -1, -1):
        d = d + dh[:, k].double()
        big = max(big, float(d.abs().max()))
        want_x[:, k] = (1 - a[:, k]) * d
        want_g[:, k] = a[:, k] * (1 - a[:, k]) * (before[:, k] - x[:, k].double()) * d
        d = keep[:, k] * d
    e = scan_err(t) * (big + 1)
    within(dx, want_x, e + U[dt] * want_x.abs())
    within(dg, want_g, e * (1 + (before - x.double()).abs()) + U[dt] * want_g.abs())
    within(dh0, d, e)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("b,t,c", [(1, 1, 1), (4, 1, 33), (1, 2, 8), (2, 3, 5), (3, 17, 64), (1, 1000, 3),
                                   (2, 1025, 72), (1, 4099, 256), (5, 64, 1000), (300, 5, 7), (1, 20000, 16)])
def test_scan_backward_sizes(dt, b, t, c):
    check_scan_grad(dt, b, t, c)
    check_scan_grad(dt, b, t, c, resets="rows", h0=False, dlast=False)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("how", ["history", "time inside", "halves", "odd"])
@pytest.mark.parametrize("resets", ["rows", "each", "inside"])
@pytest.mark.parametrize("b,t,c", [(3, 70, 40), (2, 3000, 24)])
def test_scan_backward_layouts_and_resets(dt, how, resets, b, t, c):
    check_scan_grad(dt, b, t, c, how, resets)


@pytest.mark.parametrize("t", [7, 2500])
def test_scan_gradient_against_differences(t):
    """Central differences of L = sum(r * h) + sum(q * last) in f32, along random unit directions: noise of the loss's
    roundings over 2 eps, and eps^2 of the third derivatives."""
    b, c, eps = 2, 12, 2.0 ** -5
    x, gate, h0, reset = scan_inputs(torch.float32, b, t, c, "rows", "rows", mean=0.0)
    g = gen(31)
    r, q = rnd(g, b, t, c), rnd(g, b, c)

    def loss(x, gate, h0):
        h, last = nn.gated_scan(x, gate, h0, reset)
        return (h.double() * r.double()).sum() + (last.double() * q.double()).sum()

    h, _ = nn.gated_scan(x, gate, h0, reset)
    grads = nn.gated_scan_backward(r, x, gate, h, h0, reset, q)
    for i, v in enumerate((x, gate, h0)):
        d = rnd(g, *v.shape)
        d = d / d.norm()
        up, down = [x, gate, h0], [x, gate, h0]
        up[i], down[i] = v + eps * d, v - eps * d
        num = (loss(*up) - loss(*down)) / (2 * eps)
        want = (grads[i].double() * d.double()).sum()
        noise = math.sqrt(b * t * c) * 2.0 ** -20 / eps
        assert abs(num - want) <= noise + 4 * eps * eps * float(r.abs().max()) * float(x.abs().max())


# ── Muon ──────────────────────────────────────────────────────────────────

def ns64(u, steps=5):
    x = u.double()
    x = x / (x.flatten(1).norm(dim=1)[:, None, None] + 1e-7)
    tall = x.shape[1] > x.shape[2]
    x = x.mT if tall else x
    for _ in range(steps):
        g = x @ x.mT
        x = 3.4445 * x + (-4.7750 * g + 2.0315 * g @ g) @ x
    return x.mT if tall else x


# An iteration's slope is at most 3.4445, so a relative error e of the first products grows at most 3.4445^5 = 485
# fold; f32-class products are 2^-22 off, a few of them to an iteration.
NS_TOL = 485 * 4 * 2.0 ** -22


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("b,r,c", [(1, 1, 1), (1, 1, 40), (2, 8, 8), (3, 12, 64), (3, 64, 12), (1, 128, 30), (2, 65, 129),
                                   (1, 128, 128), (2, 128, 256), (1, 200, 333), (1, 515, 258), (2, 640, 512)])
def test_orthogonalize(dt, b, r, c):
    x = rnd(gen(11), b, r, c, dt=dt, std=0.01)
    got = nn.orthogonalize(x)
    want = ns64(x)
    assert got.dtype == dt and got.shape == x.shape
    assert (got.double() - want).norm() <= (NS_TOL + U[dt]) * want.norm()
    assert torch.equal(nn.orthogonalize(x[0]), got[0])
    t = nn.orthogonalize(x.transpose(1, 2))
    assert (t.transpose(1, 2).double() - want).norm() <= (NS_TOL + U[dt]) * want.norm()


@pytest.mark.parametrize("r,c", [(128, 128), (100, 256), (300, 300), (515, 1030), (1024, 512)])
def test_orthogonalize_is_as_near_as_f32_products(r, c):
    """The header's claim: the error against 64 bits is that of the same iteration in f32 products, give or take the
    chance in both (a factor of two) and a floor of 2^-20."""
    x = rnd(gen(20), 1, r, c)
    want, y = ns64(x), x / x.norm()
    y = y.mT if r > c else y
    for _ in range(5):
        g = y @ y.mT
        y = 3.4445 * y + (-4.7750 * g + 2.0315 * g @ g) @ y
    y = y.mT if r > c else y
    got, plain = ((v.double() - want).norm() / want.norm() for v in (nn.orthogonalize(x), y))
    assert got <= 2 * plain + 2.0 ** -20


@pytest.mark.parametrize("m,k,n", [(1000, 512, 512), (700, 2040, 1000)])
def test_linear_f32_is_as_near_as_f32_products(m, k, n):
    g = gen(21)
    x, w = rnd(g, m, k), rnd(g, n, k, std=1 / math.sqrt(k))
    want = x.double() @ w.double().t()
    got, plain = ((v.double() - want).norm() / want.norm() for v in (nn.linear(x, w), x @ w.t()))
    assert got <= 2 * plain


@pytest.mark.parametrize("steps", [1, 2, 8])
@pytest.mark.parametrize("r,c", [(48, 96), (300, 200)])
def test_orthogonalize_steps(steps, r, c):
    x = rnd(gen(12), 1, r, c)
    want = ns64(x, steps)
    assert (nn.orthogonalize(x, steps=steps).double() - want).norm() <= 3.4445 ** max(steps - 5, 0) * NS_TOL * want.norm()


@pytest.mark.parametrize("r,c", [(40, 40), (40, 300), (256, 300)])
def test_orthogonalize_scales_and_zeros(r, c):
    """Scale does not matter down to tiny gradients; a zero matrix stays zero beside others; a NaN stays in its own."""
    x = rnd(gen(13), 1, r, c).expand(5, r, c) * torch.tensor([1.0, 1e-4, 1e6, 0.0, float("nan")], device="cuda")[:, None, None]
    got = nn.orthogonalize(x)
    want = ns64(x[:3])
    assert (got[:3].double() - want).norm() <= NS_TOL * want.norm()
    assert not got[3].any() and got[4].isnan().all()


def test_orthogonalize_low_rank():
    """Rank 2 of 64: the zero directions stay zero (up to the products' roundings)."""
    g = gen(14)
    x = (rnd(g, 64, 2) @ rnd(g, 2, 100))[None]
    s = torch.linalg.svdvals(nn.orthogonalize(x)[0].double())
    assert s[:2].min() > 0.6 and s[:2].max() < 1.3 and s[2:].max() < 0.05


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("b,r,c", [(1, 16, 16), (3, 128, 128), (2, 64, 300), (2, 300, 64), (1, 520, 260)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_update(dt, b, r, c, nesterov):
    g = gen(15)
    w, m, gr = rnd(g, b, r, c, std=0.1), rnd(g, b, r, c, std=0.01), rnd(g, b, r, c, dt=dt, std=0.01)
    w0, m0 = w.double(), m.double()
    copy = torch.empty(b, r, c, dtype=torch.bfloat16, device="cuda")
    nn.muon_update(w, gr, m, lr=0.02, mu=0.9, nesterov=nesterov, weight_decay=0.1, copy=copy)
    m1 = 0.9 * m0 + gr.double()
    within(m, m1, 2.0 ** -22 * (m0.abs() + gr.double().abs()))
    o = ns64(gr.double() + 0.9 * m1 if nesterov else m1)
    step = 0.02 * math.sqrt(max(1.0, r / c)) * o
    want = (1 - 0.02 * 0.1) * w0 - step
    assert (w.double() - want).norm() <= NS_TOL * step.norm() + 2.0 ** -22 * want.norm()
    assert torch.equal(copy, w.to(torch.bfloat16))


def test_muon_update_strides():
    g = gen(16)
    big = [rnd(g, 2, 96, 80) for _ in range(3)]
    w, gr, m = (v[:, 3:67, 1:41] for v in big)
    rest = [v.clone() for v in big]
    ww, gg, mm = (v[:, 3:67, 1:41].contiguous() for v in big)
    nn.muon_update(w, gr, m, lr=0.1)
    nn.muon_update(ww, gg, mm, lr=0.1)
    assert torch.equal(w, ww) and torch.equal(m, mm)
    for v, old, changed in zip(big, rest, (True, False, True)):
        old[:, 3:67, 1:41] = v[:, 3:67, 1:41]
        assert torch.equal(v, old)  # nothing outside the views


def test_muon_single_matrix_and_empty_batch():
    g = gen(17)
    w, gr, m = rnd(g, 32, 48), rnd(g, 32, 48), torch.zeros(32, 48, device="cuda")
    w3, m3 = w[None].clone(), m[None].clone()
    nn.muon_update(w, gr, m, lr=0.1)
    nn.muon_update(w3, gr[None], m3, lr=0.1)
    assert torch.equal(w, w3[0]) and torch.equal(m, m3[0])
    e = torch.zeros(0, 4, 4, device="cuda")
    nn.muon_update(e, e, e, lr=0.1)
    assert nn.orthogonalize(e).shape == (0, 4, 4)


# ── streams ───────────────────────────────────────────────────────────────

def test_operators_run_on_the_current_stream():
    """Work queued before and after on a side stream is ordered with the operators, which wait for nothing else."""
    g = gen(18)
    n = 512
    x, w = rnd(g, 4096, n, dt=torch.bfloat16), rnd(g, n, n, dt=torch.bfloat16, std=0.05)
    want = nn.linear(x, w, activation="tanh")
    hw, lw = nn.gated_scan(want[None], want[None])
    ow = nn.orthogonalize(hw[:, :n].float())
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        late = torch.zeros_like(x)
        torch.cuda._sleep(20_000_000)
        late.copy_(x)
        y = nn.linear(late, w, activation="tanh")
        h, last = nn.gated_scan(y[None], y[None])
        o = nn.orthogonalize(h[:, :n].float())
        total = o.sum()
    s.synchronize()
    assert torch.equal(y, want) and torch.equal(h, hw) and torch.equal(last, lw) and torch.equal(o, ow)
    assert torch.equal(total, ow.sum())


def test_operators_capture_into_a_graph():
    """One control step of a block, captured and replayed on new inputs."""
    g = gen(19)
    x, w1 = rnd(g, 64, 32, dt=torch.bfloat16), rnd(g, 128, 32, dt=torch.bfloat16, std=0.2)
    w2, state = rnd(g, 32, 64, dt=torch.bfloat16, std=0.2), torch.zeros(64, 64, device="cuda")

    def step(x, state):
        z = nn.linear(x, w1)
        h, state = nn.gated_scan(z[:, None, :64], z[:, None, 64:], state)
        return nn.linear(h[:, 0], w2, residual=x, activation="silu"), state

    want = step(x, state)
    static_x, static_s = torch.zeros_like(x), torch.zeros_like(state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static_x, static_s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, s1 = step(static_x, static_s)
    static_x.copy_(x)
    static_s.copy_(state)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want[0]) and torch.equal(s1, want[1])
