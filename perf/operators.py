"""What is timed of the dense operators on device tensors (`sclens_amd.dense`), with their plain forms.

    linear           y = act(x w' + b) + r            x [M, K], w [N, K], b [N], r and y [M, N]
    linear_backward  dz = dy * act'(z),  dx = dz w,  dw = dz' x,  db = column sums of dz   (z = x w' + b as the forward saved it)
    orthogonalize    x0 = g / (|g|_F + eps);  per step (a, b, c):  A = x x',  x <- a x + (b A + c A A) x   (x with rows <= columns,
                     transposed before and after if it has more rows): all singular values are driven towards 1

`own = False` computes them from elementary torch operations in 32 bits, rounded once at the end; `own = True` makes the calls of a
user of `sclens_amd.dense`. `exact` states the definitions again in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-7
UPDATE_STEP = (3.4445, -4.7750, 2.0315)  # the steep quintic of an optimiser's update: singular values end near 1
POLAR_STEP = (1.875, -1.25, 0.375)       # p(1) = 1, p'(1) = p''(1) = 0: cubic convergence to exactly 1


def _schedule(kind):
    return [UPDATE_STEP] * 5 if kind == "update" else [UPDATE_STEP] * 5 + [POLAR_STEP] * 3


# ------------------------------------------------------------------------------------------------------------------ cases
def _lin(name, M, K, N, dtype, act, bias, residual):
    return {"name": name, "op": "linear", "M": M, "K": K, "N": N, "dtype": dtype, "act": act, "bias": bias, "residual": residual}


def _bwd(name, M, K, N, dtype, act, bias):
    return {"name": name, "op": "linear_backward", "M": M, "K": K, "N": N, "dtype": dtype, "act": act, "bias": bias}


def _ort(name, batch, rows, cols, dtype, schedule, spectrum):
    return {"name": name, "op": "orthogonalize", "batch": batch, "rows": rows, "cols": cols, "dtype": dtype, "schedule": schedule,
            "spectrum": spectrum}


def listed():
    return [
        # one row through a square layer: what serving one cell / one token at a time costs (weights streamed once)
        _lin("linear_one_row_bf16", 1, 4096, 4096, "bf16", "silu", True, False),
        # sizes nothing divides: cells and genes after quality control are whatever is left
        _lin("linear_ragged_fp16", 777, 1001, 515, "fp16", "gelu", True, True),
        # scores of cells that were not in the decomposition: scaled genes onto 40 signals, the centring as the bias
        _lin("linear_project_cells_fp32", 20000, 10000, 40, "fp32", "none", True, False),
        # the widening layer of a block at an ordinary batch
        _lin("linear_block_bf16", 2048, 2048, 8192, "bf16", "gelu", True, False),
        # the largest: a long batch, with the skip connection added in the same pass
        _lin("linear_large_bf16", 8192, 8192, 8192, "bf16", "silu", True, True),
        # gradients of a small head on 93 robust signals: latency
        _bwd("backward_head_fp32", 200, 93, 50, "fp32", "relu", True),
        # gradients of the widening layer at an ordinary batch
        _bwd("backward_block_bf16", 2048, 1024, 4096, "bf16", "gelu", True),
        # gradients at a long batch
        _bwd("backward_large_bf16", 8192, 4096, 8192, "bf16", "silu", True),
        # rotations that align the 40 signals of every pair of 20 ensemble members (190 pairs), to full convergence
        _ort("orthogonalize_pairs_fp32", 190, 40, 40, "fp32", "polar", "rotation"),
        # nearest orthonormal basis of the ensemble's averaged signal vectors: 100 000 cells x 40 signals
        _ort("orthogonalize_basis_fp32", 1, 100000, 40, "fp32", "polar", "basis"),
        # an optimiser's update of four wide weight matrices
        _ort("orthogonalize_wide_bf16", 4, 1024, 4096, "bf16", "update", "gradient"),
        # and of the largest square one
        _ort("orthogonalize_square_bf16", 1, 4096, 4096, "bf16", "update", "gradient"),
    ]


def _log_size(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    # a third each: any integer, a multiple of 8, a multiple of 64
    unit = rng.choice((1, 8, 64))
    return max(lo, min(hi, max(1, v // unit) * unit))


def _fits(case):
    """no drawn case costs more than the largest listed one: 2 x 8192^3 flops (fp32 throughout in the plain form), 1.7 GB"""
    w = work(case)
    limit = 2.0 * 8192 ** 3
    plain = w["flops"]
    if case["op"] == "orthogonalize":
        m, n = sorted((case["rows"], case["cols"]))
        plain = case["batch"] * len(_schedule(case["schedule"])) * (4.0 * m * m * n + 2.0 * m * m * m)
    return plain <= limit and w["bytes"] <= 1.7e9


def _draw_once(rng):
    op = rng.choice(("linear", "linear", "linear_backward", "orthogonalize"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    act = rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh"))
    bias = rng.random() < 0.7
    if op == "linear":
        kind = rng.choice(("rows", "block", "block", "project", "reconstruct"))
        if kind == "rows":
            M, K, N = _log_size(rng, 1, 64), _log_size(rng, 64, 16384), _log_size(rng, 16, 16384)
        elif kind == "block":
            M, K, N = _log_size(rng, 65, 8192), _log_size(rng, 64, 8192), _log_size(rng, 64, 8192)
        elif kind == "project":
            M, K, N = _log_size(rng, 1000, 20000), _log_size(rng, 1000, 30000), _log_size(rng, 8, 128)
        else:
            M, K, N = _log_size(rng, 100, 8192), _log_size(rng, 8, 128), _log_size(rng, 1000, 30000)
        return _lin(None, M, K, N, dtype, act, bias, rng.random() < 0.4)
    if op == "linear_backward":
        return _bwd(None, _log_size(rng, 1, 8192), _log_size(rng, 16, 8192), _log_size(rng, 16, 8192), dtype, act, bias)
    kind = rng.choice(("pairs", "basis", "matrix", "matrix"))
    if kind == "pairs":
        m = _log_size(rng, 4, 128)
        return _ort(None, _log_size(rng, 1, 256), m, m, dtype, "polar", "rotation")
    if kind == "basis":
        return _ort(None, 1, _log_size(rng, 2000, 100000), _log_size(rng, 4, 128), dtype, "polar", "basis")
    rows, cols = _log_size(rng, 64, 4096), _log_size(rng, 64, 8192)
    return _ort(None, rng.choice((1, 1, 2, 5)), rows, cols, dtype, "update", "gradient")


def draw(rng):
    while True:
        case = _draw_once(rng)
        if _fits(case):
            del case["name"]
            return case


# ----------------------------------------------------------------------------------------------------------------- inputs
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _matrices(case, gen):
    """matrices to orthogonalise, as their users hold them"""
    B, r, c = case["batch"], case["rows"], case["cols"]
    if case["spectrum"] == "rotation":  # products v1' v2 of two members' unit vectors: a rotation with noise, shrunk a little
        x = 0.25 / math.sqrt(c) * _randn(gen, B, r, c)
        x += 0.8 * torch.eye(r, c, device="cuda")
    elif case["spectrum"] == "basis":  # an average of nearly aligned unit vectors
        x = _randn(gen, B, r, c)
        x = x + 0.3 * x.roll(1, dims=-1)
        x /= x.norm(dim=-2, keepdim=True)
        x *= 0.7 + 0.3 * torch.rand(c, generator=gen, device="cuda")
    else:  # momentum of a weight's gradient: a few strong directions over a broad floor
        k = max(1, min(r, c) // 16)
        scale = torch.logspace(0, -1.5, k, device="cuda")
        x = torch.matmul(_randn(gen, B, r, k) * scale, _randn(gen, B, k, c)) * (1e-3 / math.sqrt(k))
        x += 1e-3 * _randn(gen, B, r, c)
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 2654435761 % (2 ** 31) + 17)
    dt = DTYPES[case["dtype"]]
    st = {"case": dict(case)}
    if case["op"] == "orthogonalize":
        st["x"] = _matrices(case, gen).to(dt)
        st["schedule"] = _schedule(case["schedule"])
        return st
    M, K, N = case["M"], case["K"], case["N"]
    st["x"] = _randn(gen, M, K).to(dt)
    st["w"] = (_randn(gen, N, K) / math.sqrt(K)).to(dt)
    st["b"] = (0.5 * _randn(gen, N)).to(dt) if case["bias"] else None
    if case["op"] == "linear":
        st["r"] = _randn(gen, M, N).to(dt) if case["residual"] else None
    else:
        z = torch.matmul(st["x"].float(), st["w"].float().t())
        if case["bias"]:
            z = z + st["b"].float()
        st["z"] = z.to(dt)  # saved by the forward pass
        st["dy"] = _randn(gen, M, N).to(dt)
    return st


# ------------------------------------------------------------------------------------------------------------ plain forms
def _act(z, kind):
    if kind == "none":
        return z
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    u = math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)
    return 0.5 * z * (1 + torch.tanh(u))


def _act_grad(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _plain(st):
    case = st["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "linear":
        z = torch.matmul(st["x"].float(), st["w"].float().t())
        if st["b"] is not None:
            z = z + st["b"].float()
        y = _act(z, case["act"])
        if st["r"] is not None:
            y = y + st["r"].float()
        return y.to(dt)
    if case["op"] == "linear_backward":
        dz = st["dy"].float()
        if case["act"] != "none":
            dz = dz * _act_grad(st["z"].float(), case["act"])
        out = {"dx": torch.matmul(dz, st["w"].float()).to(dt), "dw": torch.matmul(dz.t(), st["x"].float()).to(dt)}
        if case["bias"]:
            out["db"] = dz.sum(dim=0).to(dt)
        return out
    x = st["x"].float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-1, -2).contiguous()
    x = x / (torch.sqrt((x * x).sum(dim=(-2, -1), keepdim=True)) + EPS)
    for a, b, c in st["schedule"]:
        A = torch.matmul(x, x.transpose(-1, -2).contiguous())
        x = a * x + torch.matmul(b * A + c * torch.matmul(A, A), x)
    if tall:
        x = x.transpose(-1, -2).contiguous()
    return x.to(dt)


def _kernels(st):
    from sclens_amd import dense

    case = st["case"]
    if case["op"] == "linear":
        return dense.linear(st["x"], st["w"], bias=st["b"], residual=st["r"], activation=case["act"])
    if case["op"] == "linear_backward":
        dx, dw, db = dense.linear_backward(st["dy"], st["x"], st["w"], preact=st["z"], activation=case["act"], need_bias=case["bias"])
        out = {"dx": dx, "dw": dw}
        if case["bias"]:
            out["db"] = db
        return out
    return dense.orthogonalize(st["x"], coefficients=st["schedule"], eps=EPS)


def run(state):
    return _kernels(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------- what it takes
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "orthogonalize":
        m, n = sorted((case["rows"], case["cols"]))
        steps = len(_schedule(case["schedule"]))
        # Symmetric products count once per pair. Step by step: x x' (m^2 n), A A (m^3), the product with x (2 m^2 n). Or all steps on
        # the m x m side: x x' once, per step A A, the next A (two symmetric products) and the running product, then 2 m^2 n.
        direct = steps * (3.0 * m * m * n + 1.0 * m ** 3)
        small = 3.0 * m * m * n + steps * 4.0 * m ** 3
        return {"bytes": 2 * case["batch"] * m * n * size, "flops": case["batch"] * min(direct, small)}
    M, K, N = case["M"], case["K"], case["N"]
    if case["op"] == "linear":
        elems = M * K + N * K + M * N + (N if case["bias"] else 0) + (M * N if case["residual"] else 0)
        return {"bytes": elems * size, "flops": 2.0 * M * N * K}
    elems = 2 * (M * K + N * K) + M * N * (1 if case["act"] == "none" else 2) + (N if case["bias"] else 0)
    return {"bytes": elems * size, "flops": 4.0 * M * N * K}


# ------------------------------------------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    d = torch.float64
    if case["op"] == "orthogonalize":
        g = st["x"].to(d)
        out = []
        for x in g.unbind(0):
            # the definition on whichever side is small: x p(x'x) = p(x x') x, so tall matrices need no transposition here
            tall = x.size(0) > x.size(1)
            x = x / (torch.linalg.vector_norm(x) + EPS)
            eye = torch.eye(min(x.shape), dtype=d, device=x.device)
            for a, b, c in st["schedule"]:
                A = x.t() @ x if tall else x @ x.t()
                P = a * eye + b * A + c * (A @ A)
                x = x @ P if tall else P @ x
            out.append(x)
        return torch.stack(out)
    x, w = st["x"].to(d), st["w"].to(d)
    if case["op"] == "linear":
        z = x @ w.t()
        if st["b"] is not None:
            z += st["b"].to(d)
        kind = case["act"]
        if kind == "relu":
            z = z.clamp(min=0)
        elif kind == "silu":
            z = z * torch.sigmoid(z)
        elif kind == "gelu":
            z = z * torch.special.ndtr(z)
        elif kind == "gelu_tanh":
            z = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return z if st["r"] is None else z + st["r"].to(d)
    z, g = st["z"].to(d), st["dy"].to(d)
    kind = case["act"]
    if kind == "relu":
        g = torch.where(z > 0, g, torch.zeros_like(g))
    elif kind == "silu":
        s = torch.sigmoid(z)
        g = g * (s + z * s * (1 - s))
    elif kind == "gelu":
        g = g * (torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
    elif kind == "gelu_tanh":
        k2 = 2 * math.sqrt(2 / math.pi)
        s = torch.sigmoid(k2 * (z + 0.044715 * z ** 3))
        g = g * (s + z * s * (1 - s) * k2 * (1 + 0.134145 * z * z))
    out = {"dx": g @ w, "dw": g.t().contiguous() @ x}
    if case["bias"]:
        out["db"] = g.sum(0)
    return out
