"""The recurrent-block operators' argument checks, through the C ABI and through phyz_b200.nn, without a device: a
refused call returns its status and message before it touches the device or any address it was given."""
import ctypes as C

import pytest
import torch

from phyz_b200 import _lib, nn

P = 1 << 12  # a stand-in address, aligned, never read


def linear_args(dtype=1, act=0, dev=0, m=4, k=8, n=16, x=P, xs=(8, 1), w=P, ws=(8, 1), b=0, r=0, rs=(0, 0), y=P,
                ys=(16, 1), p=0, ps=(0, 0)):
    return nn._LINEAR.pack(dtype, act, dev, m, k, n, x, *xs, w, *ws, b, r, *rs, y, *ys, p, *ps)


def grad_args(dtype=1, act=0, dev=0, m=4, k=8, n=16, dy=P, dys=(16, 1), p=0, ps=(0, 0), x=P, xs=(8, 1), w=P,
              ws=(8, 1), dx=P, dxs=(8, 1), dw=P, dws=(8, 1), db=0):
    return nn._LINEAR_GRAD.pack(dtype, act, dev, m, k, n, dy, *dys, p, *ps, x, *xs, w, *ws, dx, *dxs, dw, *dws, db)


def scan_args(dtype=0, dev=0, b=2, t=3, c=4, x=P, xs=(12, 4, 1), g=P, gs=(12, 4, 1), h0=0, h0s=(0, 0), r=0,
              rs=(0, 0, 0), h=P, hs=(12, 4, 1), last=0):
    return nn._SCAN.pack(dtype, dev, b, t, c, x, *xs, g, *gs, h0, *h0s, r, *rs, h, *hs, last)


def scan_grad_args(dtype=0, dev=0, b=2, t=3, c=4, dh=P, x=P, g=P, h=P, s=(12, 4, 1), h0=0, h0s=(0, 0), r=0,
                   rs=(0, 0, 0), dl=0, dls=(0, 0), dx=P, dxs=(12, 4, 1), dg=P, dh0=0):
    return nn._SCAN_GRAD.pack(dtype, dev, b, t, c, dh, *s, x, *s, g, *s, h, *s, h0, *h0s, r, *rs, dl, *dls, dx, *dxs,
                              dg, *s, dh0)


def muon_args(dtype=0, dev=0, steps=5, b=1, r=4, c=8, g=P, m=P, w=P, s=(32, 8, 1), cdt=0, copy=0, lr=0.1):
    return nn._MUON.pack(dtype, dev, 1, steps, b, r, c, g, *s, m, *s, w, *s, cdt, 0, copy, *s, lr, 0.9, 0.0, 1.0)


def orth_args(dtype=0, dev=0, steps=5, b=1, r=4, c=8, x=P, xs=(32, 8, 1), o=P, os=(32, 8, 1)):
    return nn._ORTH.pack(dtype, dev, steps, 0, b, r, c, x, *xs, o, *os)


CASES = [
    ("linear", linear_args(dtype=3), "dtype"), ("linear", linear_args(dtype=-1), "dtype"),
    ("linear", linear_args(act=5), "activation"), ("linear", linear_args(k=0), "k = 0"),
    ("linear", linear_args(n=0), "n = 0"), ("linear", linear_args(m=-1), "m = -1"),
    ("linear", linear_args(m=1 << 31), "m = "), ("linear", linear_args(x=0), "x is null"),
    ("linear", linear_args(w=0), "w is null"), ("linear", linear_args(y=0), "y is null"),
    ("linear", linear_args(x=P + 1), "aligned"), ("linear", linear_args(b=P + 2), "bias"),
    ("linear", linear_args(xs=(-8, 1)), "negative"), ("linear", linear_args(ys=(0, 1)), "stride of 0"),
    ("linear", linear_args(xs=(1 << 46, 1)), "2^46"), ("linear", linear_args(r=P + 1, rs=(16, 1)), "residual"),
    ("linear", linear_args(p=P, ps=(16, 0)), "pre"),
    ("linear_grad", grad_args(dtype=7), "dtype"), ("linear_grad", grad_args(act=2), "pre is null"),
    ("linear_grad", grad_args(dy=0), "dy is null"), ("linear_grad", grad_args(dxs=(0, 1)), "dx"),
    ("linear_grad", grad_args(dws=(8, 0)), "dw"), ("linear_grad", grad_args(db=P + 1), "dbias"),
    ("gated_scan", scan_args(dtype=9), "dtype"), ("gated_scan", scan_args(t=-1), "t = -1"),
    ("gated_scan", scan_args(b=1 << 30, c=1 << 30), "chains"), ("gated_scan", scan_args(x=0), "x is null"),
    ("gated_scan", scan_args(g=P + 2), "gate"), ("gated_scan", scan_args(hs=(12, 0, 1)), "h is written"),
    ("gated_scan", scan_args(h0=P + 1), "h0"), ("gated_scan", scan_args(last=P + 3), "h_last"),
    ("gated_scan", scan_args(r=P, rs=(-1, 0, 0)), "reset"),
    ("gated_scan_grad", scan_grad_args(dh=0), "dh is null"), ("gated_scan_grad", scan_grad_args(h=0), "h is null"),
    ("gated_scan_grad", scan_grad_args(dxs=(0, 4, 1)), "dx"), ("gated_scan_grad", scan_grad_args(dl=P + 1), "dh_last"),
    ("muon_update", muon_args(steps=0), "steps"), ("muon_update", muon_args(steps=17), "steps"),
    ("muon_update", muon_args(r=0), "rows"), ("muon_update", muon_args(b=70000), "batch"),
    ("muon_update", muon_args(g=0), "grad is null"), ("muon_update", muon_args(lr=float("nan")), "finite"),
    ("muon_update", muon_args(copy=P, cdt=0), "copy_dtype"), ("muon_update", muon_args(s=(32, 0, 1)), "momentum"),
    ("orthogonalize", orth_args(steps=-3), "steps"), ("orthogonalize", orth_args(x=0), "x is null"),
    ("orthogonalize", orth_args(os=(32, 8, 0)), "out"),
]


@pytest.mark.parametrize("op,args,word", CASES)
def test_refused_with_a_message(op, args, word):
    lib = _lib.load()
    assert getattr(lib, f"phyzb_{op}")(args, C.c_void_p(256), 1 << 62, None) == _lib.ERR_INVALID
    assert word in lib.phyzb_last_error().decode()


def test_sides_past_the_limit_are_too_large():
    lib = _lib.load()
    n = _lib.MUON_MAX_SIDE + 1
    assert lib.phyzb_orthogonalize(orth_args(r=n, xs=(n * 8, 8, 1), os=(n * 8, 8, 1)), None, 0, None) == \
        _lib.ERR_TOO_LARGE
    assert str(n) in lib.phyzb_last_error().decode()


def test_null_arguments_and_small_workspaces():
    lib = _lib.load()
    for op in _lib.NN_OPS:
        assert getattr(lib, f"phyzb_{op}")(None, None, 0, None) == _lib.ERR_INVALID
    need = C.c_int64(-1)
    big = muon_args(r=300, c=400, s=(120000, 400, 1))  # (small matrices need no workspace)
    assert lib.phyzb_muon_workspace(big, None) == _lib.ERR_INVALID
    assert lib.phyzb_muon_workspace(big, C.byref(need)) == 0 and need.value > 0
    assert lib.phyzb_muon_update(big, C.c_void_p(256), need.value - 1, None) == _lib.ERR_INVALID
    assert "smaller" in lib.phyzb_last_error().decode()
    assert lib.phyzb_muon_update(big, None, need.value, None) == _lib.ERR_INVALID
    assert lib.phyzb_muon_update(big, C.c_void_p(16), need.value, None) == _lib.ERR_INVALID
    assert "256" in lib.phyzb_last_error().decode()


def test_no_device_is_an_error():
    lib = _lib.load()
    if lib.phyzb_device_count() > 0:
        pytest.skip("a device is present")
    ws = C.c_void_p(256)
    for op, args in (("linear", linear_args()), ("linear_grad", grad_args()), ("gated_scan", scan_args()),
                     ("gated_scan_grad", scan_grad_args()), ("muon_update", muon_args()),
                     ("orthogonalize", orth_args())):
        assert getattr(lib, f"phyzb_{op}")(args, ws, 1 << 62, None) == _lib.ERR_NO_DEVICE


def test_packed_structs_have_the_header_sizes(tmp_path):
    import subprocess
    from pathlib import Path

    inc = Path(__file__).resolve().parents[1] / "include"
    names = {"linear": nn._LINEAR, "linear_grad": nn._LINEAR_GRAD, "scan": nn._SCAN, "scan_grad": nn._SCAN_GRAD,
             "muon": nn._MUON, "orthogonalize": nn._ORTH}
    body = "".join(f'printf("%zu\\n", sizeof(phyzb_{n}_args));' for n in names)
    (tmp_path / "s.c").write_text('#include <stdio.h>\n#include "phyzb.h"\nint main(void){' + body + "return 0;}\n")
    subprocess.run(["gcc", "-I", str(inc), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    sizes = subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()
    for (n, st), size in zip(names.items(), sizes):
        assert st.size == int(size), n


def test_python_checks():
    x, w = torch.zeros(4, 8), torch.zeros(16, 8)
    with pytest.raises(ValueError, match="CUDA"):
        nn.linear(x, w)
    with pytest.raises(ValueError, match="float64"):
        nn.linear(x.double(), w.double())
    with pytest.raises(ValueError, match="matrices"):
        nn.linear(x[0], w)
    with pytest.raises(ValueError, match="b, t, c"):
        nn.gated_scan(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        nn.gated_scan(x[None], x[None])
    with pytest.raises(ValueError, match="momentum|CUDA|wanted"):
        nn.muon_update(w, w, x, lr=0.1)
    with pytest.raises(ValueError, match="rows"):
        nn.orthogonalize(x[0])


@pytest.mark.gpu
def test_python_checks_on_a_device():
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(16, 8, device="cuda")
    g = torch.zeros(2, 3, 4, device="cuda")
    for call, word in ((lambda: nn.linear(x, w[:, :7]), "weight"), (lambda: nn.linear(x, w.half()), "weight"),
                       (lambda: nn.linear(x, w, torch.zeros(15, device="cuda")), "bias"),
                       (lambda: nn.linear(x, w, torch.zeros(16)), "bias"),
                       (lambda: nn.linear(x, w, activation="softplus"), "softplus"),
                       (lambda: nn.linear(x, w, residual=x), "residual"),
                       (lambda: nn.linear_backward(torch.zeros(4, 16, device="cuda"), x, w, activation="tanh"), "pre"),
                       (lambda: nn.gated_scan(g, g[:, :2]), "gate"),
                       (lambda: nn.gated_scan(g, g, reset=torch.zeros(2, 3, device="cuda")), "reset"),
                       (lambda: nn.gated_scan_backward(g[:1], g, g, g), "dh"),
                       (lambda: nn.muon_update(w, w.cpu(), w, lr=0.1), "grad"),
                       (lambda: nn.muon_update(w, w, w.half(), lr=0.1), "momentum"),
                       (lambda: nn.muon_update(w, w, w.clone(), lr=0.1, copy=w.clone()), "copy")):
        with pytest.raises(ValueError, match=word):
            call()
