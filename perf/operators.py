"""The recurrent block's operators as a user calls them, and the same in plain torch.

Three operators of phyz_b200.nn: the linear layer with its epilogue (forward and
backward), the gated scan over time (forward, backward, one step), and the Muon
update with its orthogonalisation. `run` calls the framework's where `own` is
true, and else computes the same in 32 bits from elementary torch operations.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315
NS_STEPS = 5
NS_EPS = 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
GELU_C, GELU_K = math.sqrt(2.0 / math.pi), 0.044715

# What a drawn case may cost at most: the largest listed one of its operator.
LINEAR_MOST = 262144 * 1024 * 1024  # rows * in * out
SCAN_MOST = 64 * 1024 * 1024        # values of x
MUON_MOST = 2 * 2048 ** 3           # matrices * short^2 * long


def listed():
    return [
        # one world's policy step while it is being served: a hidden layer of one row
        {"name": "linear step", "op": "linear", "dir": "fwd", "type": "bf16", "m": 1, "k": 512, "n": 1024,
         "act": "silu", "bias": True, "residual": False, "order": "rows", "train": False},
        # the quadruped's 30 observations in the policy history's order, [feature][world], first layer, training form
        {"name": "linear history f32", "op": "linear", "dir": "fwd", "type": "f32", "m": 65536, "k": 30, "n": 64,
         "act": "tanh", "bias": True, "residual": False, "order": "features", "train": True},
        # a hidden layer over every world of the quadruped batch, with the block's skip connection: the largest forward
        {"name": "linear batch", "op": "linear", "dir": "fwd", "type": "bf16", "m": 262144, "k": 1024, "n": 1024,
         "act": "silu", "bias": True, "residual": True, "order": "rows", "train": False},
        # the training step's backward pass over a minibatch of 65536 rows
        {"name": "linear backward", "op": "linear", "dir": "bwd", "type": "bf16", "m": 65536, "k": 1024, "n": 1024,
         "act": "gelu", "bias": True, "residual": False, "order": "rows", "train": True},
        # odd widths, rows that are no multiple of anything, f16
        {"name": "linear backward ragged", "op": "linear", "dir": "bwd", "type": "f16", "m": 1537, "k": 515, "n": 129,
         "act": "tanh", "bias": True, "residual": False, "order": "rows", "train": True},
        # one control step of 4096 worlds: the state is read, advanced and written
        {"name": "scan step", "op": "scan", "dir": "fwd", "type": "f32", "b": 4096, "t": 1, "c": 256, "order": "rows",
         "reset": 0.005},
        # few long recordings: parallel only over 2 x 512 channels unless the time axis is split
        {"name": "scan long", "op": "scan", "dir": "fwd", "type": "bf16", "b": 2, "t": 32769, "c": 512, "order": "rows",
         "reset": 0.0},
        # a rollout of 64 control steps in the history's order, [step][feature][world], with episode ends
        {"name": "scan history", "op": "scan", "dir": "fwd", "type": "f32", "b": 64, "t": 64, "c": 16384,
         "order": "history", "reset": 0.01},
        # the training step's backward pass through time
        {"name": "scan backward", "op": "scan", "dir": "bwd", "type": "bf16", "b": 64, "t": 1024, "c": 1024,
         "order": "rows", "reset": 0.002},
        # the hidden matrices of a small policy and its critic, stacked: where latency counts
        {"name": "muon small", "op": "muon", "type": "f32", "b": 8, "rows": 128, "cols": 128},
        # the orthogonalised direction alone, odd sizes
        {"name": "orthogonalize ragged", "op": "orth", "type": "f32", "b": 3, "rows": 515, "cols": 1030},
        # wide layers, gradients in bf16 as a mixed-precision step leaves them
        {"name": "muon large", "op": "muon", "type": "bf16", "b": 2, "rows": 2048, "cols": 2048},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "scan", "scan", "muon"])
    if op == "linear":
        while True:
            case = {"op": "linear", "dir": rng.choice(["fwd", "bwd"]), "type": rng.choice(["f32", "bf16", "bf16", "f16"]),
                    "m": _log(rng, 1, 262144), "k": _log(rng, 8, 2048), "n": _log(rng, 8, 2048),
                    "act": rng.choice(["none", "relu", "tanh", "silu", "gelu"]), "bias": rng.random() < 0.8,
                    "residual": rng.random() < 0.5, "order": rng.choice(["rows", "rows", "features"])}
            if rng.random() < 0.5:  # widths of real layers are often round
                case["k"], case["n"] = max(8, case["k"] // 8 * 8), max(8, case["n"] // 8 * 8)
            if case["dir"] == "bwd":
                case["residual"] = False
            case["train"] = case["dir"] == "bwd" or rng.random() < 0.5
            passes = 2 if case["dir"] == "bwd" else 1
            if passes * case["m"] * case["k"] * case["n"] <= LINEAR_MOST and case["m"] * max(case["k"], case["n"]) <= 2 ** 28:
                return case
    if op == "scan":
        while True:
            case = {"op": "scan", "dir": rng.choice(["fwd", "bwd"]), "type": rng.choice(["f32", "bf16", "f16"]),
                    "b": _log(rng, 1, 4096), "t": _log(rng, 1, 40000), "c": _log(rng, 8, 16384),
                    "order": rng.choice(["rows", "history"]), "reset": rng.choice([0.0, 0.002, 0.05])}
            if case["b"] * case["t"] * case["c"] <= SCAN_MOST:
                return case
    while True:
        case = {"op": rng.choice(["muon", "orth"]), "type": rng.choice(["f32", "bf16"]), "b": _log(rng, 1, 16),
                "rows": _log(rng, 8, 2048), "cols": _log(rng, 8, 2048)}
        s, l = sorted((case["rows"], case["cols"]))
        if case["b"] * s * s * l <= MUON_MOST:
            return case


# ── plain forms ───────────────────────────────────────────────────────────

def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "tanh":
        return torch.tanh(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.tanh(GELU_C * (z + GELU_K * z * z * z)))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "tanh":
        t = torch.tanh(z)
        return 1.0 - t * t
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        t = torch.tanh(GELU_C * (z + GELU_K * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * GELU_C * (1.0 + 3.0 * GELU_K * z * z)
    return torch.ones_like(z)


def _shift(v, d):
    """v one step of `d` later along time, and what stands before the first."""
    return torch.cat([torch.zeros_like(v[:, :d]), v[:, :-d]], 1)


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from h = 0, in log2(T) passes of doubling spans."""
    d = 1
    while d < a.shape[1]:
        b = b + a * _shift(b, d)
        a = a * _shift(a, d)
        d *= 2
    return b


def _plain_scan(x, g, h0, reset):
    x, g = x.float(), g.float()
    a = torch.sigmoid(g)
    b = (1.0 - a) * x
    if reset is not None:
        a = torch.where(reset != 0, torch.zeros_like(a), a)
    first = b[:, :1] + a[:, :1] * h0[:, None]
    return _scan(a, torch.cat([first, b[:, 1:]], 1))


def _plain_scan_backward(s):
    x, g, h, dh = (s[k].float() for k in ("x", "g", "h", "dh"))
    a = torch.sigmoid(g)
    keep = a if s["reset"] is None else torch.where(s["reset"] != 0, torch.zeros_like(a), a)
    prev = torch.cat([s["h0"][:, None], h[:, :-1]], 1)
    if s["reset"] is not None:
        prev = torch.where(s["reset"] != 0, torch.zeros_like(prev), prev)
    dh = torch.cat([dh[:, :-1], dh[:, -1:] + s["dh_last"][:, None]], 1)
    carry = torch.cat([keep[:, 1:], torch.zeros_like(keep[:, :1])], 1)
    d = _scan(carry.flip(1), dh.flip(1)).flip(1)
    dx = (1.0 - a) * d
    dg = dx * a * (prev - x)
    return dx.to(s["x"].dtype), dg.to(s["x"].dtype), keep[:, 0] * d[:, 0]


def _plain_ns(x):
    x = x / (torch.sqrt((x * x).sum((1, 2), keepdim=True)) + NS_EPS)
    wide = x.shape[1] <= x.shape[2]
    x = x if wide else x.transpose(1, 2)
    for _ in range(NS_STEPS):
        g = x @ x.transpose(1, 2)
        x = NS_A * x + (NS_B * g + NS_C * (g @ g)) @ x
    return x if wide else x.transpose(1, 2)


def _plain(s):
    case = s["case"]
    op, typ = case["op"], TYPES[case["type"]]
    if op == "linear" and case["dir"] == "fwd":
        z = s["x"].float() @ s["w"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"]
        y = _act(z, case["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return (y.to(typ), z.to(typ)) if case["train"] else y.to(typ)
    if op == "linear":
        dz = s["dy"].float() * _act_grad(s["z"].float(), case["act"])
        grads = {"dx": (dz @ s["w"].float()).to(typ), "dw": (dz.t() @ s["x"].float()).to(typ)}
        if case["bias"]:
            grads["db"] = dz.sum(0)
        return grads
    if op == "scan" and case["dir"] == "fwd":
        h = _plain_scan(s["x"], s["g"], s["h0"], s["reset"])
        return h.to(typ), h[:, -1].contiguous()
    if op == "scan":
        return _plain_scan_backward(s)
    if op == "orth":
        return _plain_ns(s["g"].float()).to(typ)
    w, m, g = s["w"], s["m"], s["g"].float()
    m.mul_(MOMENTUM).add_(g)
    scale = math.sqrt(max(1.0, case["rows"] / case["cols"]))
    w.mul_(1.0 - LR * DECAY).sub_(_plain_ns(g + MOMENTUM * m), alpha=LR * scale)
    return w, m


# ── the framework's operators ─────────────────────────────────────────────

def _own(s):
    from phyz_b200 import nn

    case = s["case"]
    op = case["op"]
    if op == "linear" and case["dir"] == "fwd":
        return nn.linear(s["x"], s["w"], s["bias"], activation=case["act"], residual=s["residual"],
                         save_pre=case["train"])
    if op == "linear":
        dx, dw, db = nn.linear_backward(s["dy"], s["x"], s["w"], s["z"], activation=case["act"], bias=case["bias"])
        return {"dx": dx, "dw": dw, "db": db} if case["bias"] else {"dx": dx, "dw": dw}
    if op == "scan" and case["dir"] == "fwd":
        return nn.gated_scan(s["x"], s["g"], s["h0"], s["reset"])
    if op == "scan":
        return nn.gated_scan_backward(s["dh"], s["x"], s["g"], s["h"], s["h0"], s["reset"], s["dh_last"])
    if op == "orth":
        return nn.orthogonalize(s["g"])
    nn.muon_update(s["w"], s["g"], s["m"], lr=LR, mu=MOMENTUM, weight_decay=DECAY)
    return s["w"], s["m"]


def run(state):
    return _own(state) if own else _plain(state)


# ── inputs ────────────────────────────────────────────────────────────────

def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, typ=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(std).add_(mean).to(typ)

    op, typ = case["op"], TYPES[case["type"]]
    s = {"case": case}
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]

        def rows(r, f, std=1.0):  # [r, f] in the case's order: by rows, or each feature's rows together
            return normal(r, f, std=std, typ=typ) if case["order"] == "rows" else normal(f, r, std=std, typ=typ).t()

        s["x"] = rows(m, k)
        s["w"] = normal(n, k, std=1.0 / math.sqrt(k), typ=typ)
        s["bias"] = normal(n, std=0.1) if case["bias"] else None
        if case["dir"] == "fwd":
            s["residual"] = rows(m, n) if case["residual"] else None
        else:
            # the pre-activations that the forward pass left; gradients of a mean over the rows, scaled for f16
            z = s["x"].float() @ s["w"].float().t() + (s["bias"] if case["bias"] else 0.0)
            s["z"] = z.to(typ)
            s["dy"] = rows(m, n, std=0.1)
    elif op == "scan":
        b, t, c = case["b"], case["t"], case["c"]

        def seq(std=1.0, mean=0.0):  # [b, t, c], or the view of a history [t][b][c]
            v = normal(b, t, c, std=std, mean=mean, typ=typ) if case["order"] == "rows" else \
                normal(t, b, c, std=std, mean=mean, typ=typ).transpose(0, 1)
            return v

        s["x"], s["g"] = seq(), seq(std=1.5, mean=2.0)
        s["h0"] = normal(b, c, std=0.5)
        s["reset"] = None
        if case["reset"] > 0:
            # an episode ends for a whole sequence (rows), or for one world at all its features (history: worlds inside)
            shape = (b, t, 1) if case["order"] == "rows" else (1, t, c)
            hit = torch.rand(*shape, generator=gen, device="cuda") < case["reset"]
            s["reset"] = hit.to(torch.uint8).expand(b, t, c)
        if case["dir"] == "bwd":
            s["h"] = _plain_scan(s["x"], s["g"], s["h0"], s["reset"]).to(typ)
            if case["order"] == "history":
                s["h"] = s["h"].transpose(0, 1).contiguous().transpose(0, 1)
            s["dh"] = seq(std=0.1)
            s["dh_last"] = normal(b, c, std=0.1)
    else:
        b, r, c = case["b"], case["rows"], case["cols"]
        s["g"] = normal(b, r, c, std=1e-3, typ=typ)
        if op == "muon":
            s["w"] = normal(b, r, c, std=1.0 / math.sqrt(c))
            s["m"] = normal(b, r, c, std=3e-3)
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ── cost and definition ───────────────────────────────────────────────────

def work(case):
    op = case["op"]
    e = {"f32": 4, "bf16": 2, "f16": 2}[case["type"]]
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        if case["dir"] == "fwd":
            outs = 1 + int(case["train"]) + int(case["residual"])
            return {"bytes": e * (m * k + n * k + outs * m * n) + 4 * n * int(case["bias"]), "flops": 2 * m * n * k}
        reads = m * n * (1 if case["act"] == "none" else 2) + m * k + n * k
        return {"bytes": e * (reads + m * k + n * k) + 4 * n * int(case["bias"]), "flops": 4 * m * n * k}
    if op == "scan":
        b, t, c = case["b"], case["t"], case["c"]
        flags = 0 if case["reset"] == 0 else t * (b if case["order"] == "rows" else c)
        if case["dir"] == "fwd":
            return {"bytes": 3 * e * b * t * c + 8 * b * c + flags, "flops": 4 * b * t * c}
        return {"bytes": 6 * e * b * t * c + 12 * b * c + flags, "flops": 9 * b * t * c}
    b, r, c = case["b"], case["rows"], case["cols"]
    s, l = min(r, c), max(r, c)
    # X X^T and its square are symmetric: half of each is enough
    flops = b * NS_STEPS * (s * s * l + s * s * s + 2 * s * s * l)
    return {"bytes": b * r * c * (2 * e if op == "orth" else e + 16), "flops": flops}


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    d = lambda v: None if v is None else v.double()  # noqa: E731
    if op == "linear":
        x, w = d(s["x"]), d(s["w"])
        if case["dir"] == "fwd":
            z = torch.matmul(x, w.T)
            if case["bias"]:
                z += d(s["bias"])
            y = {"none": lambda v: v.clone(), "relu": torch.relu, "tanh": torch.tanh,
                 "silu": torch.nn.functional.silu,
                 "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["act"]](z)
            if s["residual"] is not None:
                y += d(s["residual"])
            return (y, z) if case["train"] else y
        z = d(s["z"]).requires_grad_()
        y = {"none": lambda v: v * 1.0, "relu": torch.relu, "tanh": torch.tanh, "silu": torch.nn.functional.silu,
             "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["act"]](z)
        (dz,) = torch.autograd.grad(y, z, d(s["dy"]))
        grads = {"dx": torch.matmul(dz, w), "dw": torch.matmul(dz.T, x)}
        if case["bias"]:
            grads["db"] = torch.sum(dz, 0)
        return grads
    if op == "scan":
        # step by step along time
        x, g, h0 = d(s["x"]), d(s["g"]), d(s["h0"])
        T = x.shape[1]
        keep = torch.ones_like(x) if s["reset"] is None else 1.0 - d(s["reset"])
        a = 1.0 / (1.0 + torch.exp(-g))
        if case["dir"] == "fwd":
            out, h = torch.empty_like(x), h0
            for t in range(T):
                h = a[:, t] * keep[:, t] * h + (1.0 - a[:, t]) * x[:, t]
                out[:, t] = h
            return out, h
        h, dh = d(s["h"]), d(s["dh"])
        dx, dg, carry = torch.empty_like(x), torch.empty_like(x), d(s["dh_last"])
        for t in range(T - 1, -1, -1):
            total = dh[:, t] + carry
            before = (h[:, t - 1] if t else h0) * keep[:, t]
            dx[:, t] = total * (1.0 - a[:, t])
            dg[:, t] = total * (before - x[:, t]) * a[:, t] * (1.0 - a[:, t])
            carry = total * a[:, t] * keep[:, t]
        return dx, dg, carry
    u = d(s["g"])
    if op == "muon":
        m = MOMENTUM * d(s["m"]) + u
        u = u + MOMENTUM * m
    norm = torch.linalg.matrix_norm(u)[:, None, None] + NS_EPS
    x = u / norm
    tall = x.shape[1] > x.shape[2]
    for _ in range(NS_STEPS):  # by the right for tall matrices: X (X^T X)
        gram = torch.matmul(x.mT, x) if tall else torch.matmul(x, x.mT)
        poly = NS_B * gram + NS_C * torch.matmul(gram, gram)
        x = NS_A * x + (torch.matmul(x, poly) if tall else torch.matmul(poly, x))
    if op == "orth":
        return x
    scale = math.sqrt(max(1.0, case["rows"] / case["cols"]))
    return d(s["w"]) * (1.0 - LR * DECAY) - LR * scale * x, m
