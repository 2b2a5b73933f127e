"""The recurrent-block operators (phyz_b200.nn) at the edges of their ranges, against their definitions in 64 bits.

Tolerances come from the arithmetic: u is the unit roundoff of an array's type (2^-24, 2^-8, 2^-11), results are
rounded to it once, in f16 with an absolute 2^-25 below its normal range. Weights are the identity, so that a product
moves each value as it is and elements are compared one by one.
"""
import pytest
import torch

from phyz_b200 import nn

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = list(U)
ACTS = ["none", "relu", "tanh", "silu", "gelu"]


def rnd(seed, *shape, dt=torch.float32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)


def act64(z, act):
    return {"none": lambda v: v * 1.0, "relu": torch.relu, "tanh": torch.tanh, "silu": torch.nn.functional.silu,
            "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[act](z)


def layout(t, how):
    """t's values by rows, by features, or either from an odd offset (which no wide access can take)."""
    order, odd = how.split()[0], how.endswith("odd")
    v = t if order == "rows" else t.t()
    flat = torch.empty(v.numel() + 1, dtype=t.dtype, device=t.device)
    flat = flat[1:] if odd else flat[:-1]
    out = flat.view(v.shape)
    out.copy_(v)
    return out if order == "rows" else out.t()


def outliers(dt, sizes, m, n):
    """N(0, 1), with every second value of the first half of the rows one of `sizes`: beside a small one along either
    side, in a pair or a vector of any width. In the second half every value of a row is."""
    z = rnd(1, m, n)
    sizes = torch.tensor([v for v in sizes if abs(v) < (6.5e4 if dt is torch.float16 else 3e38)], device="cuda")
    pick = sizes[torch.arange(m * n, device="cuda").view(m, n) * 7 % len(sizes)]
    odd = (torch.arange(m, device="cuda")[:, None] + torch.arange(n, device="cuda")) % 2 == 1
    odd |= torch.arange(m, device="cuda")[:, None] >= m // 2
    return torch.where(odd, pick, z).to(dt)


LARGE = [5.0, 10.0, 20.0, 30.0, 50.0, 100.0, 300.0, 1000.0, 6e4, 1e6, 1e13, 1e20, 1e30]
ORDERS = [("rows", "rows"), ("rows odd", "rows"), ("features", "features"), ("features odd", "features"),
          ("rows", "features"), ("features", "rows")]  # of dy and of pre


# A slope is s + z s (1 - s) w(z) with s a sigmoid of a few f32 roundings, whose exponential's argument x is off by
# some 2^-23 |x|. s (1 - s) decays with e^-|x|, faster than anything it is multiplied by, so the products stay under 2
# and the slope's error under 32 roundings wherever z is: the tolerance does not grow with |z|.
def check_slopes(dt, act, dy_how, pre_how, m, n, sizes):
    pre, dy = layout(outliers(dt, sizes, m, n), pre_how), layout(rnd(2, m, n, dt=dt), dy_how)
    x, w = layout(rnd(3, m, n, dt=dt), dy_how.split()[0]), torch.eye(n, device="cuda", dtype=dt)
    dx, _, db = nn.linear_backward(dy, x, w, pre, activation=act)
    z = pre.double().requires_grad_()
    slope, = torch.autograd.grad(act64(z, act).sum(), z)
    want = dy.double() * slope
    err = dy.double().abs() * 32 * 2.0 ** -23
    off = (dx.double() - want).abs()
    assert torch.isfinite(dx.double()).all()
    assert (off <= err + 2 * U[dt] * (want.abs() + err) + 2.0 ** -24).all(), float((off / (dy.double().abs() + 1e-3)).max())
    tol = (err + (m + 8) * 2.0 ** -23 * want.abs()).sum(0)
    assert ((db.double() - want.sum(0)).abs() <= tol).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dy_how,pre_how", ORDERS)
def test_slopes_of_large_values(dt, act, dy_how, pre_how):
    check_slopes(dt, act, dy_how, pre_how, 600, 64, LARGE)
    check_slopes(dt, act, dy_how, pre_how, 4096, 512, LARGE)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dy_how,pre_how", ORDERS)
def test_slopes_of_large_negative_values(dt, act, dy_how, pre_how):
    sizes = [-v for v in LARGE] + LARGE[::3]
    check_slopes(dt, act, dy_how, pre_how, 600, 64, sizes)
    check_slopes(dt, act, dy_how, pre_how, 4096, 512, sizes)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n", [(1, 40), (7, 64), (600, 64), (4096, 512)])
@pytest.mark.parametrize("how", ["rows", "features"])
def test_activations_of_large_values(dt, act, m, n, how):
    """z s is off by some roundings of itself (s by 2^-23 |z| of itself where it is small: then z^2 s is under 1), and
    nothing of z is left where s has vanished."""
    x = layout(outliers(dt, LARGE + [-v for v in LARGE], m, n), how)
    y = nn.linear(x, torch.eye(n, device="cuda", dtype=dt), activation=act)
    want = act64(x.double(), act)
    err = 16 * 2.0 ** -23 * (1 + want.abs())
    assert torch.isfinite(y.double()).all()
    assert ((y.double() - want).abs() <= err + U[dt] * (want.abs() + err) + 2.0 ** -25).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ["tanh", "silu", "gelu"])
def test_slopes_of_infinities_and_nan(dt, act):
    """A layer of one feature, so that no product mixes elements: the slope's limits at the infinities, and a NaN stays
    one, alone."""
    pre = rnd(4, 256, 1, dt=dt)
    dy, one = rnd(5, 256, 1, dt=dt), torch.ones(1, 1, device="cuda", dtype=dt)
    clean = nn.linear_backward(dy, pre, one, pre, activation=act)[0]
    pre[3], pre[64], pre[65] = float("nan"), float("inf"), float("-inf")
    dx = nn.linear_backward(dy, pre, one, pre, activation=act)[0]
    assert dx[3].isnan() and not dx[65].any()
    assert dx[64].abs() <= 2.0 ** -20 if act == "tanh" else (dx[64] - dy[64]).abs() <= dy[64].abs() * 4 * U[dt]
    keep = torch.ones(256, dtype=torch.bool, device="cuda")
    keep[[3, 64, 65]] = False
    assert torch.equal(dx[keep], clean[keep])


# ── gated scan: gates that are nearly shut ────────────────────────────────

# 1 - a is e a with e = 2^-x, x the gate over log 2: x is off by some 2^-24 of itself (29 at a gate of 20), the
# exponential, the reciprocal and the products by a few roundings, so 1 - a is within 32 roundings of itself however
# small it is. Every sum here is of values of one sign, so what t steps add is t roundings more, and the relative
# tolerance holds for each element by itself.
def near_each(got, want, t, dt):
    tol = (64 + 4 * t) * 2.0 ** -23 + U[dt]
    small = 2.0 ** -25 if dt is torch.float16 else 2.0 ** -126
    assert ((got.double() - want).abs() <= tol * want.abs() + small).all(), \
        f"relative error {float(((got.double() - want) / want).abs().max()):.3g}"


SHUT = [(1, 1, 64), (3, 1, 7), (3, 40, 64), (5, 40, 7), (1, 3000, 64), (1, 3000, 3)]  # one step, tiles, plain, both cut


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,c", SHUT)
@pytest.mark.parametrize("resets", [False, True])
def test_scan_inputs_through_shut_gates(dt, b, t, c, resets):
    gate = (8 + 12 * torch.rand(b, t, c, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))).to(dt)
    x = (rnd(7, b, t, c).abs() + 0.5).to(dt)
    reset = (torch.arange(t, device="cuda") % 16 == 5).to(torch.uint8).expand(b, t) if resets else None
    h, last = nn.gated_scan(x, gate, None, reset)
    state, want = torch.zeros(b, c, device="cuda", dtype=torch.float64), torch.empty_like(x, dtype=torch.float64)
    a, shut = torch.sigmoid(gate.double()), torch.sigmoid(-gate.double())
    for k in range(t):
        if resets and k % 16 == 5:
            state = torch.zeros_like(state)
        state = a[:, k] * state + shut[:, k] * x[:, k].double()
        want[:, k] = state
    near_each(h, want, t, dt)
    near_each(last, state, t, torch.float32)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,c", SHUT)
@pytest.mark.parametrize("resets", [False, True])
def test_scan_gradients_through_shut_gates(dt, b, t, c, resets):
    gate = (8 + 12 * torch.rand(b, t, c, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8))).to(dt)
    x, h, dh = ((rnd(s, b, t, c).abs() + 0.5).to(dt) for s in (9, 10, 11))
    x = -x  # (so that h - x does not cancel either)
    h0, dl = rnd(12, b, c).abs() + 0.5, rnd(13, b, c).abs()
    reset = (torch.arange(t, device="cuda") % 16 == 5).to(torch.uint8).expand(b, t) if resets else None
    dx, dg, dh0 = nn.gated_scan_backward(dh, x, gate, h, h0, reset, dl)
    a, shut = torch.sigmoid(gate.double()), torch.sigmoid(-gate.double())
    before = torch.cat([h0.double()[:, None], h.double()[:, :-1]], 1)
    want_x, want_g, d = torch.empty_like(a), torch.empty_like(a), dl.double()
    for k in range(t - 1, -1, -1):
        drop = resets and k % 16 == 5
        d = d + dh[:, k].double()
        want_x[:, k] = shut[:, k] * d
        want_g[:, k] = a[:, k] * shut[:, k] * ((0 if drop else before[:, k]) - x[:, k].double()) * d
        d = torch.zeros_like(d) if drop else a[:, k] * d
    near_each(dx, want_x, t, dt)
    near_each(dg, want_g, t, dt)
    near_each(dh0, d, t, torch.float32)


@pytest.mark.parametrize("t,c", [(1, 64), (1, 7), (40, 64), (40, 7)])
def test_scan_of_extreme_gates(t, c):
    """Open and shut to the end of the range, and a NaN, which stays in its chain and is not taken for a gate."""
    x, h0 = rnd(14, 4, t, c), rnd(15, 4, c)
    for value in (200.0, 3e38, float("inf")):
        h, last = nn.gated_scan(x, torch.full_like(x, value), h0)
        assert torch.equal(h, h0[:, None].expand_as(h)) and torch.equal(last, h0)
        h, last = nn.gated_scan(x, torch.full_like(x, -value), h0)
        assert torch.equal(h, x) and torch.equal(last, x[:, -1])
        dx, dg, dh0 = nn.gated_scan_backward(x, x, torch.full_like(x, -value), x, h0)
        assert torch.equal(dx, x) and dg.abs().max() <= 2.0 ** -80 and dh0.abs().max() <= 2.0 ** -80
    gate = torch.zeros_like(x)
    want, _ = nn.gated_scan(x, gate, h0)
    gate[1, 0, 2] = float("nan")
    reset = torch.zeros(4, t, dtype=torch.uint8, device="cuda")
    reset[:, 0] = 1  # (the state is dropped, the gate still weighs x)
    h, _ = nn.gated_scan(x, gate, h0)
    hr, _ = nn.gated_scan(x, gate, h0, reset)
    dx, _, _ = nn.gated_scan_backward(x, x, gate, x, h0, reset)
    assert h[1, :, 2].isnan().all() and hr[1, :, 2].isnan().all() and dx[1, 0, 2].isnan()
    h[1, :, 2] = want[1, :, 2]
    assert torch.equal(h, want)


# ── small f32 layers: the order of a gradient's result ────────────────────

def best_us(f):
    """Device time of one of ten calls captured in a graph, the best of twelve replays."""
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(10):
            f()
    best = 1e9
    for _ in range(12):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 100)
    return best


@pytest.mark.parametrize("order", ["rows", "features"])
def test_small_gradient_is_written_along_its_order(order):
    """dx = dy w of an 8 to 128 layer's mirror image is the product that its forward makes, and takes as long (within
    half; stored against its order it took 28 us where it takes 13)."""
    x, wide, w = layout(rnd(20, 65536, 8), order), layout(rnd(21, 65536, 128), order), rnd(22, 128, 8)
    narrow = w.t().contiguous()  # the layer 128 -> 8
    forward = best_us(lambda: nn.linear(x, w))
    dx = best_us(lambda: nn.linear_backward(x, wide, narrow, bias=False, need_dw=False))
    assert dx <= 1.5 * forward, (dx, forward)


@pytest.mark.parametrize("m,k,n", [(40, 30, 70), (3000, 30, 64), (65536, 24, 12)])
def test_small_gradients_in_either_order(m, k, n):
    """dw and dx where the caller keeps them the other way round: the same values."""
    x, w, dy = rnd(23, m, k), rnd(24, n, k), rnd(25, m, n)
    dx, dw, _ = nn.linear_backward(dy, x, w, bias=False)
    tx, tw = torch.full((k, m), float("nan"), device="cuda"), torch.full((k, n), float("nan"), device="cuda")
    args = nn._LINEAR_GRAD.pack(0, 0, 0, m, k, n, dy.data_ptr(), n, 1, 0, 0, 0, x.data_ptr(), k, 1, w.data_ptr(), k, 1,
                                tx.data_ptr(), 1, m, tw.data_ptr(), 1, n, 0)
    nn._linear_grad(args, 0)
    assert torch.equal(tx.t(), dx) and torch.equal(tw.t(), dw)


# ── waits ─────────────────────────────────────────────────────────────────

def test_status_waits_for_every_stream():
    """What it reports is of all calls so far: work on a side stream (which does not wait for the default one, nor the
    other way round) has finished when it returns."""
    x, w = rnd(26, 512, 64, dt=torch.bfloat16), rnd(27, 64, 64, dt=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        nn.linear(x, w)  # (so that nothing is set up or allocated below)
    nn.status()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # a tenth of a second
        y = nn.linear(x, w)
        done = side.record_event()
    assert not done.query()
    nn.status()
    assert done.query()
    assert torch.equal(y, nn.linear(x, w))


# ── more features than a launch has blocks along its second side ──────────

@pytest.mark.parametrize("order", ["rows", "features"])
def test_small_layers_of_millions_of_features(order):
    """Small whole numbers, which f32 sums hold exactly in every order."""
    n = 4_200_000
    x = layout((torch.arange(9, device="cuda") + 1.0)[:, None], order)
    w = (torch.arange(n, device="cuda") % 97).float()[:, None]
    y = nn.linear(x, w)
    assert torch.equal(y, x * w.t())
    few = nn.linear(x[:4], w.expand(n, 2)[:, ::2])
    assert torch.equal(few, y[:4])
    # as the inputs' side: dx [9][n], dw [3][n]
    dy, v = layout(x.repeat(1, 3), order), torch.ones(3, 1, device="cuda") * w.t()
    dx, dw, _ = nn.linear_backward(dy, y, v, bias=False)
    assert torch.equal(dx, 3 * x * w.t())
    assert torch.equal(dw, (x * x).sum() * w.t().expand(3, n))
