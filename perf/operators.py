"""Cases and plain forms of the training operators: layer norm (forward; forward and backward) and the orthogonalised
update (Newton-Schulz alone; a whole Muon step over the matrices of a net).

`own` says which side `run` computes: the plain torch form (False) or the framework's entry points (True)."""
import math

import torch

own = False

EPS_LN = 1e-5
EPS_NS = 1e-7
COEFFS = (3.4445, -4.7750, 2.0315)
STEPS = 5
LR, MU, WD, RMS = 0.02, 0.95, 0.01, 0.2

# the matrices (count x rows x columns) of the nets of exps/nnyu.yaml: conv weights flattened to (out, in * taps)
GEN = "28x256x2304,4x256x1152,4x128x576,2x64x49"
DIS = "1x2048x9216,1x1024x4608,1x512x2304,1x256x1152,2x128x576,2x64x49,1x20x8192"
VAE = "1x50x108,2x20x50,1x50x20,1x108x50"

LN_MOST = 131072 * 256          # elements of the largest layer-norm case
NS_MOST = 2.9e11                # operations of the largest update, counted as `_ns_flops` does


def _ln(name, op, dtype, rows, cols):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "cols": cols}


def listed():
    return [
        # hidden layer of the pose VAE at its batch size of 64: launch latency
        _ln("ln_fwd_pose_hidden", "ln_fwd", "float32", 64, 50),
        # every pixel's 256 channels of the 32x32 latent maps of 128 samples, bf16 activations
        _ln("ln_fwd_pixels_bf16", "ln_fwd", "bfloat16", 131072, 256),
        # a few samples' pooled features, one-row-sized work with odd columns
        _ln("ln_train_few_odd", "ln_train", "float32", 7, 1023),
        # the same latent maps in f32, training: the largest ordinary call
        _ln("ln_train_pixels", "ln_train", "float32", 131072, 256),
        # ragged rows of an odd width in bf16
        _ln("ln_train_ragged_bf16", "ln_train", "bfloat16", 8191, 2049),
        # a whole [256, 32, 32] map normalised at once (batch 32): rows far longer than a workgroup holds
        _ln("ln_train_maps", "ln_train", "float32", 32, 262144),
        # one matrix of the pose VAE
        {"name": "ns_pose", "op": "ns", "dtype": "float32", "count": 1, "rows": 108, "cols": 50},
        # odd sizes, tall, bf16
        {"name": "ns_tall_odd_bf16", "op": "ns", "dtype": "bfloat16", "count": 3, "rows": 1021, "cols": 333},
        # the residual blocks' 3x3 convs of the generator
        {"name": "ns_res_blocks", "op": "ns", "dtype": "float32", "count": 28, "rows": 256, "cols": 2304},
        # optimiser steps over all matrices of a net
        {"name": "muon_vae", "op": "muon", "shapes": VAE},
        {"name": "muon_gen", "op": "muon", "shapes": GEN},
        {"name": "muon_dis", "op": "muon", "shapes": DIS},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("ln_fwd", "ln_train", "ln_train", "ns", "muon"))
    if op in ("ln_fwd", "ln_train"):
        cols = _log(rng, 5, 262144)     # (below that a row has hardly a direction left that layer norm does not remove)
        return {"op": op, "dtype": rng.choice(("float32", "bfloat16")), "rows": _log(rng, 1, max(1, min(131072, LN_MOST // cols))), "cols": cols}
    if op == "ns":
        while True:
            c = {"op": op, "dtype": rng.choice(("float32", "bfloat16")), "count": _log(rng, 1, 32), "rows": _log(rng, 1, 4096),
                 "cols": _log(rng, 1, 9216)}
            if work(c)["flops"] <= NS_MOST and c["count"] * c["rows"] * c["cols"] <= 1 << 25:
                return c
    while True:
        parts = ["%dx%dx%d" % (_log(rng, 1, 12), _log(rng, 2, 2048), _log(rng, 2, 9216)) for _ in range(rng.randint(1, 6))]
        c = {"op": op, "shapes": ",".join(parts)}
        if work(c)["flops"] <= NS_MOST and sum(n * r * k for n, r, k in _groups(c["shapes"])) <= 1 << 25:
            return c


def _groups(text):
    return [tuple(int(v) for v in part.split("x")) for part in text.split(",")]


def _gradients(count, rows, cols, gen):
    """Gradient-like matrices: a decaying low-rank part under noise, of a size that differs from matrix to matrix."""
    dev = gen.device
    rank = max(1, min(rows, cols) // 8)
    left = torch.randn(count, rows, rank, generator=gen, device=dev)
    right = torch.randn(count, rank, cols, generator=gen, device=dev)
    decay = torch.arange(1, rank + 1, device=dev, dtype=torch.float32).rsqrt()
    g = torch.matmul(left * decay, right) / math.sqrt(rank) + torch.randn(count, rows, cols, generator=gen, device=dev)
    return g * (1e-3 * torch.exp(torch.randn(count, 1, 1, generator=gen, device=dev)))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    s = dict(case)
    if case["op"] in ("ln_fwd", "ln_train"):
        rows, cols, dtype = case["rows"], case["cols"], getattr(torch, case["dtype"])
        size = torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device=dev))
        x = torch.randn(rows, cols, generator=gen, device=dev) * size + torch.randn(rows, 1, generator=gen, device=dev)
        s["x"] = x.to(dtype)
        s["w"] = 1.0 + 0.2 * torch.randn(cols, generator=gen, device=dev)
        s["b"] = 0.2 * torch.randn(cols, generator=gen, device=dev)
        if case["op"] == "ln_train":
            s["dy"] = torch.randn(rows, cols, generator=gen, device=dev).to(dtype)
            for k in ("x", "w", "b"):
                s[k].requires_grad_(True)
        return s
    if case["op"] == "ns":
        s["g"] = _gradients(case["count"], case["rows"], case["cols"], gen).to(getattr(torch, case["dtype"]))
        return s
    # one flat buffer each of weights, gradients and momenta, as the framework's arena keeps them, and a view per matrix
    total = sum(n * r * k for n, r, k in _groups(case["shapes"]))
    s["p"] = torch.empty(total, device=dev)
    s["g"] = torch.empty(total, device=dev)
    s["m"] = torch.empty(total, device=dev)
    s["views"], at = [], 0
    for n, r, k in _groups(case["shapes"]):
        e = at + n * r * k
        s["p"][at:e] = torch.randn(e - at, generator=gen, device=dev) * 0.02
        s["g"][at:e] = _gradients(n, r, k, gen).reshape(-1)
        s["m"][at:e] = 4.0 * _gradients(n, r, k, gen).reshape(-1)
        s["views"] += [tuple(s[b][at + i * r * k:at + (i + 1) * r * k].view(r, k) for b in ("p", "g", "m")) for i in range(n)]
        at = e
    return s


def _orthogonal(g):
    """Plain Newton-Schulz of a stack of matrices [count, rows, columns] in f32."""
    x = g if g.shape[1] <= g.shape[2] else g.transpose(1, 2).contiguous()
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPS_NS)
    a, b, c = COEFFS
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x if g.shape[1] <= g.shape[2] else x.transpose(1, 2).contiguous()


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        if state["op"] in ("ln_fwd", "ln_train"):
            x, w, b = state["x"].float(), state["w"], state["b"]
            xc = x - x.mean(1, keepdim=True)
            r = (xc.square().mean(1, keepdim=True) + EPS_LN).rsqrt()
            xh = xc * r
            y = (xh * w + b).to(state["x"].dtype)
            if state["op"] == "ln_fwd":
                return y
            dy = state["dy"].float()
            g = dy * w
            dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
            return {"y": y, "dx": dx.to(state["x"].dtype), "dw": (dy * xh).sum(0), "db": dy.sum(0)}
        if state["op"] == "ns":
            return _orthogonal(state["g"].float()).to(state["g"].dtype)
        at = 0
        for n, r, k in _groups(state["shapes"]):
            e = at + n * r * k
            p, g, m = (state[b][at:e].view(n, r, k) for b in ("p", "g", "m"))
            m.mul_(MU).add_(g)
            o = _orthogonal(g + MU * m)
            p.mul_(1.0 - LR * WD).sub_(o, alpha=LR * RMS * math.sqrt(max(r, k)))
            at = e
        return {"p": state["p"], "m": state["m"]}


def _run_own(state):
    from lsps_amd import ops
    if state["op"] == "ln_fwd":
        return ops.layer_norm(state["x"], (state["cols"],), state["w"], state["b"], EPS_LN)
    if state["op"] == "ln_train":
        x, w, b = state["x"], state["w"], state["b"]
        y = ops.layer_norm(x, (state["cols"],), w, b, EPS_LN)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), state["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if state["op"] == "ns":
        return ops.newton_schulz(state["g"], STEPS, COEFFS, EPS_NS)
    p, g, m = zip(*state["views"])
    ops.muon_step_(p, g, m, lr=LR, momentum=MU, nesterov=True, weight_decay=WD, rms=RMS, steps=STEPS, coeffs=COEFFS, eps=EPS_NS)
    return {"p": state["p"], "m": state["m"]}


def _ns_flops(rows, cols):
    """Products on the shorter side's Gram matrix; a product whose result is symmetric counts half."""
    m, n = min(rows, cols), max(rows, cols)
    return 3.0 * m * m * n + (4 * STEPS - 3) * float(m) ** 3


def work(case):
    if case["op"] in ("ln_fwd", "ln_train"):
        size = 4 if case["dtype"] == "float32" else 2
        n = case["rows"] * case["cols"]
        train = case["op"] == "ln_train"      # forward: x in, y out; backward: x and dy in, dx out
        return {"bytes": n * size * (5 if train else 2) + case["cols"] * 4 * (5 if train else 2), "flops": n * (20 if train else 8)}
    if case["op"] == "ns":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": 2 * size * case["count"] * case["rows"] * case["cols"], "flops": case["count"] * _ns_flops(case["rows"], case["cols"])}
    groups = _groups(case["shapes"])          # g in; m and p in and out
    return {"bytes": sum(20 * n * r * k for n, r, k in groups), "flops": sum(n * _ns_flops(r, k) for n, r, k in groups)}


def _poly64(g):
    """X f(X^T X) in 64 bits on the right-hand Gram matrix when that is the smaller one, else on the left-hand one."""
    x = g / (torch.linalg.matrix_norm(g, keepdim=True) + EPS_NS)
    right = x.shape[-1] < x.shape[-2]
    eye = torch.eye(min(x.shape[-2:]), dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        k = torch.matmul(x.mT.contiguous(), x) if right else torch.matmul(x, x.mT.contiguous())
        f = COEFFS[0] * eye + torch.matmul(COEFFS[1] * eye + COEFFS[2] * k, k)
        x = torch.matmul(x, f) if right else torch.matmul(f, x)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("ln_fwd", "ln_train"):
            x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
            n = float(case["cols"])
            mean = x.sum(-1, keepdim=True) / n
            std = torch.sqrt(((x - mean) ** 2).sum(-1, keepdim=True) / n + EPS_LN)
            y = (x - mean) / std * w + b
            if case["op"] == "ln_fwd":
                return y
            dy = s["dy"].double()
            z = (x - mean) / std
            dz = dy * w
            dx = (dz - (dz.sum(-1, keepdim=True) + z * (dz * z).sum(-1, keepdim=True)) / n) / std
            return {"y": y, "dx": dx, "dw": (dy * z).sum(0), "db": dy.sum(0)}
        if case["op"] == "ns":
            return _poly64(s["g"].double())
        p, m = s["p"].double(), s["m"].double() * MU + s["g"].double()
        u = s["g"].double() + MU * m
        at = 0
        for n, r, k in _groups(case["shapes"]):
            e = at + n * r * k
            p[at:e] -= LR * (WD * p[at:e] + RMS * math.sqrt(max(r, k)) * _poly64(u[at:e].view(n, r, k)).reshape(-1))
            at = e
        return {"p": p, "m": m}
