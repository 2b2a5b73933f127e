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
