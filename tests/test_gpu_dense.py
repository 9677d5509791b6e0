"""MI355X: the dense operators on device tensors (sclens_amd.dense) against their definitions in 64 bits.

Two kinds of cases. Whole numbers: every product and partial sum is exact in fp32 (below 2^24), so the result has to be the rounded exact
one, bit for bit, whatever the order of the sums -- a dropped, doubled or misplaced term cannot hide. Real numbers: bounds from the
roundings that the operator is documented to make, u = eps / 2 of the type for each.
"""
import math
import zlib

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF16, F16, F32]
U = {t: torch.finfo(t).eps / 2 for t in TYPES}  # half a step, relative: 2^-8 (eight significant bits), 2^-11, 2^-24
UPDATE = [(3.4445, -4.7750, 2.0315)] * 5
POLAR = UPDATE + [(1.875, -1.25, 0.375)] * 3


@pytest.fixture(scope="module")
def dense():
    from sclens_amd import dense as d

    return d


def ints(gen, shape, dtype, top=4):
    return torch.randint(-top, top + 1, shape, generator=gen, device="cuda").to(dtype)


def gen_for(*key):
    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(repr(key).encode()) % (2 ** 31))
    return g


def padded(t, extra, offset=0):
    """the same rows with a longer leading dimension, starting `offset` elements into the storage"""
    buf = torch.full((t.size(0) * (t.size(1) + extra) + offset + 8,), 77.0, dtype=t.dtype, device=t.device)
    v = buf[offset: offset + t.size(0) * (t.size(1) + extra)].view(t.size(0), t.size(1) + extra)[:, : t.size(1)]
    v.copy_(t)
    return v


def act64(z, kind):
    if kind == "relu":
        return z.clamp(min=0)
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return z * torch.special.ndtr(z)
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def act_grad64(z, kind):
    z = z.detach().clone().requires_grad_(True)
    act64(z, kind).sum().backward()
    return z.grad


# sizes around the tiles (64, 128, 256), the stages (64 columns), the chunks (8 columns), one, and nothing
SHAPES = [(1, 1, 1), (1, 4096, 4096), (1, 100, 33), (2, 64, 64), (3, 8, 65), (5, 7, 9), (16, 4104, 200), (17, 999, 130), (33, 72, 500),
          (64, 64, 64), (65, 63, 66), (100, 1001, 515), (127, 128, 129), (200, 93, 50), (256, 256, 256), (257, 520, 255), (300, 40, 1500),
          (513, 1100, 770), (1000, 2000, 40), (2049, 129, 8), (1030, 1032, 1028), (2048, 520, 2056), (700, 3, 900), (4, 20000, 24),
          (1500, 8, 3), (40, 16000, 40)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_whole_numbers_are_exact(dense, M, K, N, dtype):
    g = gen_for("lin", M, K, N)
    top = 4 if dtype != BF16 else 2
    x, w, b, r = ints(g, (M, K), dtype, top), ints(g, (N, K), dtype, top), ints(g, (N,), dtype, 9), ints(g, (M, N), dtype, 9)
    z = x.double() @ w.double().t() + b.double()
    assert z.abs().max() < 2 ** 24
    y, pre = dense.linear(x, w, bias=b, residual=r, activation="relu", save_preact=True)
    assert torch.equal(pre, z.to(dtype))
    assert torch.equal(y, (z.clamp(min=0) + r.double()).float().to(dtype))
    assert torch.equal(dense.linear(x, w), (x.double() @ w.double().t()).float().to(dtype))


# sizes that reach every tile (256, 192, 128 with two and four stages, 64), split contractions with few results, planes of fp32 (the
# second and third), rows that do not start on 16 bytes, streams past a short side
LARGE = [(4096, 72, 4096), (4096, 1024, 4096), (4100, 1030, 4090), (2900, 200, 2950), (8192, 136, 1024), (2048, 1032, 2048), (1024, 264, 1040),
         (300, 8200, 300), (130, 4104, 4096), (3000, 1000, 100), (60, 2001, 3000), (5000, 640, 128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", LARGE)
def test_linear_whole_numbers_large(dense, M, K, N, dtype):
    g = gen_for("large", M, K, N)
    x, w, b, r = ints(g, (M, K), dtype, 1), ints(g, (N, K), dtype, 1), ints(g, (N,), dtype, 9), ints(g, (M, N), dtype, 9)
    z = x.double() @ w.double().t() + b.double()
    y, pre = dense.linear(x, w, bias=b, residual=r, activation="relu", save_preact=True)
    assert torch.equal(pre, z.float().to(dtype))
    assert torch.equal(y, (z.clamp(min=0) + r.double()).float().to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(4096, 4096, 4096), (2048, 1032, 1030), (1000, 2001, 1500), (4100, 520, 3000), (64, 4096, 2048)])
def test_backward_whole_numbers_large(dense, M, K, N, dtype):
    g = gen_for("blarge", M, K, N)
    x, w, dy, z = ints(g, (M, K), dtype, 1), ints(g, (N, K), dtype, 1), ints(g, (M, N), dtype, 1), ints(g, (M, N), dtype, 3)
    dz = dy.double() * (z.double() > 0)
    dx, dw, db = dense.linear_backward(dy, x, w, preact=z, activation="relu")
    assert torch.equal(dx, (dz @ w.double()).float().to(dtype))
    assert torch.equal(dw, (dz.t().contiguous() @ x.double()).float().to(dtype))
    assert torch.equal(db, dz.sum(0).float().to(dtype))
    # parts of it give the same bits
    assert torch.equal(dense.linear_backward(dy, None, w, preact=z, activation="relu", need_weight=False, need_bias=False)[0].float(), dx.float())
    assert torch.equal(dense.linear_backward(dy, x, None, preact=z, activation="relu", need_x=False)[1].float(), dw.float())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (2, 64, 64), (5, 7, 9), (65, 63, 66), (127, 128, 129), (200, 93, 50), (257, 520, 255),
                                   (513, 1100, 770), (1030, 1032, 1028), (2049, 129, 8), (8, 2000, 700), (1, 513, 514), (3000, 16, 1)])
@pytest.mark.parametrize("act", ["none", "relu"])
def test_backward_whole_numbers_are_exact(dense, M, K, N, act, dtype):
    g = gen_for("bwd", M, K, N)
    x, w, dy, z = ints(g, (M, K), dtype, 2), ints(g, (N, K), dtype, 2), ints(g, (M, N), dtype, 2), ints(g, (M, N), dtype, 3)
    dz = dy.double() if act == "none" else dy.double() * (z.double() > 0)
    dx, dw, db = dense.linear_backward(dy, x, w, preact=z if act != "none" else None, activation=act)
    assert torch.equal(dx, (dz @ w.double()).float().to(dtype))
    assert torch.equal(dw, (dz.t() @ x.double()).float().to(dtype))
    assert torch.equal(db, dz.sum(0).float().to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("extra,offset", [(0, 0), (8, 0), (8, 8), (3, 0), (1, 1), (0, 3), (16, 5)])
def test_strides_and_addresses(dense, dtype, extra, offset):
    g = gen_for("strides", extra, offset)
    M, K, N = 130, 200, 136
    x, w = ints(g, (M, K), dtype, 2), ints(g, (N, K), dtype, 2)
    b, r, dy, z = ints(g, (N,), dtype, 9), ints(g, (M, N), dtype, 9), ints(g, (M, N), dtype, 2), ints(g, (M, N), dtype, 3)
    xs, ws, rs = padded(x, extra, offset), padded(w, extra, offset), padded(r, extra, offset)
    bs = torch.cat([b.new_zeros(offset + 1), b])[offset + 1:]
    want = (x.double() @ w.double().t() + b.double() + r.double()).float().to(dtype)
    assert torch.equal(dense.linear(xs, ws, bias=bs, residual=rs), want)
    dz = dy.double() * (z.double() > 0)
    dx, dw, db = dense.linear_backward(padded(dy, extra, offset), xs, ws, preact=padded(z, extra, offset), activation="relu")
    assert torch.equal(dx, (dz @ w.double()).float().to(dtype))
    assert torch.equal(dw, (dz.t() @ x.double()).float().to(dtype))
    assert torch.equal(db, dz.sum(0).float().to(dtype))
    o = torch.randn(60, 90, generator=g, device="cuda").to(dtype)
    assert torch.equal(dense.orthogonalize(padded(o, extra, offset)), dense.orthogonalize(o))
    # leading axes, and rows taken out of a wider tensor
    x3 = torch.zeros(2, 65, K + 24, dtype=dtype, device="cuda")[:, :, 8: 8 + K]
    x3.copy_(x.view(2, 65, K))
    assert torch.equal(dense.linear(x3, w, bias=b, residual=r.view(2, 65, N)), want.view(2, 65, N))
    assert torch.equal(dense.linear(x[3], w, bias=b, residual=r[3]), want[3])


def linear_bound(x, w, b, r, act, dtype):
    """z is a sum of K products held in fp32: at most K + 2 roundings of at most the sum of the terms' magnitudes (twice, for sums that
    cut instead of rounding); the fp32 pieces leave out at most 2^-23 of a term. |act'| <= 1.13; an activation's own evaluation: a few units of
    |z| + 1 in fp32 (expf, erff, tanhf are below 4). One rounding to the type at the end."""
    S = x.double().abs() @ w.double().abs().t() + (b.double().abs() if b is not None else 0)
    z = x.double() @ w.double().t() + (b.double() if b is not None else 0)
    y = act64(z, act) + (r.double() if r is not None else 0)
    err = 1.13 * 2 * (x.size(-1) + 3) * 2.0 ** -24 * S + 16 * 2.0 ** -24 * (z.abs() + 1) + 2.0 ** -23 * y.abs()
    tiny = {BF16: 2.0 ** -133, F16: 2.0 ** -24, F32: 2.0 ** -149}[dtype]
    return z, y, err * 1.01 + U[dtype] * 1.01 * (y.abs() + err) + tiny


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M,K,N", [(1, 600, 700), (9, 130, 64), (150, 93, 300), (520, 256, 264)])
def test_linear_real_numbers(dense, M, K, N, act, dtype):
    g = gen_for("real", M, K, N)
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    w = (torch.randn(N, K, generator=g, device="cuda") * 3 / math.sqrt(K)).to(dtype)
    b, r = torch.randn(N, generator=g, device="cuda").to(dtype), torch.randn(M, N, generator=g, device="cuda").to(dtype)
    for bias, res in ((None, None), (b, r)):
        _, want, tol = linear_bound(x, w, bias, res, act, dtype)
        got = dense.linear(x, w, bias=bias, residual=res, activation=act).double()
        assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M,K,N", [(1, 60, 70), (150, 93, 300), (520, 256, 264)])
def test_backward_real_numbers(dense, M, K, N, act, dtype):
    """against the formula: dz is computed in fp32 (act' to 32 units of 2^-24 (1 + |z|)) and rounded once to the type, then the products"""
    g = gen_for("breal", M, K, N)
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    w = (torch.randn(N, K, generator=g, device="cuda") / math.sqrt(K)).to(dtype)
    z, dy = (torch.randn(M, N, generator=g, device="cuda") * 2).to(dtype), torch.randn(M, N, generator=g, device="cuda").to(dtype)
    dz = dy.double() * act_grad64(z.double(), act)
    ddz = dy.double().abs() * 32 * 2.0 ** -24 * (1 + z.double().abs())
    if dtype != F32:
        ddz = ddz + U[dtype] * 1.01 * (dz.abs() + ddz) + (2.0 ** -25 if dtype == F16 else 0)
    got = dense.linear_backward(dy, x, w, preact=z, activation=act)
    want = (dz @ w.double(), dz.t() @ x.double(), dz.sum(0))
    acc = (dz.abs() @ w.double().abs() * (2 * (N + 3)), dz.abs().t() @ x.double().abs() * (2 * (M + 3)), dz.abs().sum(0) * (M + 3))
    prop = (ddz @ w.double().abs(), ddz.t() @ x.double().abs(), ddz.sum(0))
    for a, b, c, d in zip(got, want, acc, prop):
        tol = (2.0 ** -24 * c + d) * 1.02
        tol = tol + U[dtype] * 1.01 * (b.abs() + tol) + (2.0 ** -24 if dtype == F16 else 2.0 ** -140)
        assert ((a.double() - b).abs() <= tol).all(), ((a.double() - b).abs() / tol).max()


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_gradient_against_differences(dense, act):
    """directional derivatives of the forward call itself, fp32: central differences of step h have an error of order h^2 (third
    derivatives below 4) and of the forward's rounding / h"""
    g = gen_for("diff", act)
    M, K, N = 37, 50, 45
    x, w = torch.randn(M, K, generator=g, device="cuda"), torch.randn(N, K, generator=g, device="cuda") / math.sqrt(K)
    b, dy = torch.randn(N, generator=g, device="cuda"), torch.randn(M, N, generator=g, device="cuda")
    _, z = dense.linear(x, w, bias=b, activation=act, save_preact=True)
    if act == "relu":  # away from the kink
        dy = torch.where(z.abs() > 0.05, dy, torch.zeros_like(dy))
    dx, dw, db = dense.linear_backward(dy, x, w, preact=z, activation=act)
    h = 2.0 ** -8
    for name, t, d in (("x", x, dx), ("w", w, dw), ("b", b, db)):
        v = torch.randn(t.shape, generator=g, device="cuda")
        v /= v.norm()
        f = {}
        for s in (1, -1):
            a = {"x": x, "w": w, "b": b}
            a[name] = t + s * h * v
            f[s] = dense.linear(a["x"], a["w"], bias=a["b"], activation=act).double()
        num = ((f[1] - f[-1]) * dy.double()).sum() / (2 * h)
        ana = (d.double() * v.double()).sum()
        zv = x.double().norm() + w.double().norm() * math.sqrt(M) + math.sqrt(M)  # no direction moves z by more, in norm
        tol = dy.double().abs().max() * (4 * h * h * zv + 2.0 ** -20 / h * math.sqrt(M * N))
        assert (num - ana).abs() <= tol, (name, num, ana, tol)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_extremes(dense, dtype):
    """infinities, NaN and the type's largest values reach exactly the results that contain them"""
    g = gen_for("extreme")
    for M, K, N in ((70, 96, 90), (1, 96, 90), (300, 300, 300), (2048, 264, 2048), (3000, 520, 40), (40, 520, 3000), (4096, 1024, 4096)):
        x, w = ints(g, (M, K), dtype, 3), ints(g, (N, K), dtype, 3)
        w[5] = 1
        w[6] = 0
        x[0, 3] = math.inf
        if M > 40:
            x[33, 7] = math.nan
            x[34, 2], x[34, 9] = math.inf, -math.inf
        y = dense.linear(x, w).double()
        want = x.double() @ w.double().t()
        assert torch.equal(torch.isnan(y), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(y, nan=0.0, posinf=1e300, neginf=-1e300), torch.nan_to_num(want.to(dtype).double(), nan=0.0, posinf=1e300, neginf=-1e300))
    # the largest value survives a product with one; twice it overflows
    big = torch.finfo(dtype).max
    x, w = torch.zeros(3, 16, device="cuda", dtype=dtype), torch.eye(16, device="cuda", dtype=dtype)
    x[0, 0], x[1, 1], x[2, 2] = big, -big, torch.finfo(dtype).tiny
    assert torch.equal(dense.linear(x, w), x)
    assert torch.isinf(dense.linear(x, 2 * w)[0, 0])


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_to_do(dense, dtype):
    e = lambda *s: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    assert dense.linear(e(0, 5), e(4, 5)).shape == (0, 4)
    assert dense.linear(e(3, 5), e(0, 5)).shape == (3, 0)
    b = torch.arange(4, device="cuda").to(dtype)
    assert torch.equal(dense.linear(e(3, 0), e(4, 0), bias=b, residual=e(3, 4) + 1), (b + 1).expand(3, 4))
    dx, dw, db = dense.linear_backward(e(0, 4), e(0, 5), e(4, 5))
    assert dx.shape == (0, 5) and torch.equal(dw, e(4, 5)) and torch.equal(db, e(4))
    dx, dw, db = dense.linear_backward(e(3, 0), e(3, 5), e(0, 5))
    assert torch.equal(dx, e(3, 5)) and dw.shape == (0, 5) and db.shape == (0,)
    dx, dw, db = dense.linear_backward(e(3, 4) + 1, e(3, 0), e(4, 0))
    assert dx.shape == (3, 0) and dw.shape == (4, 0) and torch.equal(db, e(4) + 3)
    assert dense.orthogonalize(e(0, 5, 6)).shape == (0, 5, 6) and dense.orthogonalize(e(5, 0)).shape == (5, 0)
    assert torch.equal(dense.orthogonalize(e(2, 5, 6)), e(2, 5, 6)) and torch.equal(dense.orthogonalize(e(100, 120)), e(100, 120))
    assert [t is None for t in dense.linear_backward(e(3, 4), e(3, 5), None, need_x=False, need_bias=False)] == [True, False, True]


def test_rows_behind_the_result_are_left_alone(dense):
    """the C entry writes into the caller's matrices: nothing outside their rows and columns"""
    import ctypes as C

    from sclens_amd._lib import Context

    ctx = Context(0)
    try:
        for dtype, code in ((BF16, 1), (F16, 2), (F32, 0)):
            for M, K, N in ((1, 64, 70), (5, 7, 9), (130, 72, 135), (300, 264, 520)):
                g = gen_for("behind", M)
                x, w = ints(g, (M, K), dtype, 2), ints(g, (N, K), dtype, 2)
                y = torch.full((M + 3, N + 5), -7.0, dtype=dtype, device="cuda")
                ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
                n = C.c_int64(ws.numel())
                stream = torch.cuda.current_stream().cuda_stream
                ctx.check(ctx.lib.sclens_hip_linear(ctx.h, stream, code, M, N, K, x.data_ptr(), K, w.data_ptr(), K, None, None, 0, 0,
                                                    y.data_ptr(), N + 5, None, 0, ws.data_ptr(), C.byref(n)))
                assert torch.equal(y[:M, :N], (x.double() @ w.double().t()).float().to(dtype))
                assert (y[M:] == -7).all() and (y[:, N:] == -7).all()
                for rows, cols in ((M, N), (N, M)):
                    o = torch.randn(2, rows, cols, generator=g, device="cuda").to(dtype)
                    out = torch.full((2, rows + 2, cols + 3), -7.0, dtype=dtype, device="cuda")
                    coef = (C.c_double * 15)(*[v for t in UPDATE for v in t])
                    n = C.c_int64(ws.numel())
                    ctx.check(ctx.lib.sclens_hip_orthogonalize(ctx.h, stream, code, 2, rows, cols, o.data_ptr(), rows * cols, cols, out.data_ptr(),
                                                               (rows + 2) * (cols + 3), cols + 3, 5, coef, 1e-7, ws.data_ptr(), C.byref(n)))
                    assert torch.equal(out[:, :rows, :cols], dense.orthogonalize(o))
                    assert (out[:, rows:] == -7).all() and (out[:, :, cols:] == -7).all()
    finally:
        torch.cuda.synchronize()
        ctx.close()


# ---------------------------------------------------------------------------------------------------------- orthogonalize
def orth64(x, schedule, eps=1e-7):
    x = x.double()
    x = x / (x.flatten(-2).norm(dim=-1)[..., None, None] + eps)
    tall = x.size(-2) > x.size(-1)
    if tall:
        x = x.transpose(-1, -2).contiguous()
    for a, b, c in schedule:
        A = x @ x.transpose(-1, -2).contiguous()
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.transpose(-1, -2).contiguous() if tall else x


def orth_bound(x, schedule, dtype):
    """Frobenius distance that the roundings of the steps can cause, per matrix. With u the unit of what is kept between the products
    (fp16 for the 16-bit types, the fp32 sums otherwise), step t starts from an x off by e_t: the step's map has derivatives of at most
    L_t = max(|p'|, |p(s) / s|) over the singular values that occur, so e_{t+1} <= L_t e_t + what the step rounds: A and A A by u and the
    sum's 2 (k + 3) 2^-24 of |x| |x|', P by u, the result by u, each times the norms it meets."""
    u = 2.0 ** -11 if dtype != F32 else 2.0 ** -23
    X = x.double()
    X = X / (X.flatten(-2).norm(dim=-1)[..., None, None] + 1e-7)
    m, n = min(X.shape[-2:]), max(X.shape[-2:])
    s = torch.linalg.svdvals(X.cpu())
    acc = 2 * (math.sqrt(n) + 3) * 2.0 ** -24  # statistically independent roundings of a sum of n terms (worst case n: not met)
    e = u * s.norm(dim=-1)
    for a, b, c in schedule:
        top = s.max(dim=-1).values
        grid = torch.linspace(0, 1, 513, dtype=torch.float64) * 1.02 * top[..., None]
        L = torch.maximum((a + 3 * b * grid ** 2 + 5 * c * grid ** 4).abs().max(-1).values, (a + b * grid ** 2 + c * grid ** 4).abs().max(-1).values)
        lam = s ** 2
        dA = (2 * u + acc) * lam.norm(dim=-1)
        dP = (abs(b) + 2 * abs(c) * top ** 2) * dA + (2 * u + acc) * (abs(b) * lam.norm(dim=-1) + abs(c) * (lam ** 2).norm(dim=-1))
        p = (a * s + b * s ** 3 + c * s ** 5).abs()
        e = L * e + dP * top + (2 * u + acc) * (abs(a) * s.norm(dim=-1) + p.norm(dim=-1))
        s = p
    return e + U[dtype] * s.norm(dim=-1)


ORTH = [(1, 1, 1), (1, 1, 50), (1, 50, 1), (3, 4, 4), (20, 40, 40), (2, 33, 64), (1, 64, 65), (1, 66, 63), (4, 93, 93), (2, 128, 100), (1, 5, 3000),
        (1, 3001, 40), (1, 5000, 64), (1, 2000, 100), (1, 130, 700), (1, 700, 130), (2, 256, 512), (1, 515, 300), (1, 1024, 520), (1, 65, 4100), (1, 2048, 1100)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,rows,cols", ORTH)
def test_orthogonalize_update(dense, batch, rows, cols, dtype):
    g = gen_for("orth", batch, rows, cols)
    x = torch.randn(batch, rows, cols, generator=g, device="cuda")
    x[:, :, 0] *= 5
    x = x.to(dtype)
    got, want = dense.orthogonalize(x, coefficients=UPDATE).double(), orth64(x, UPDATE)
    off = (got - want).flatten(1).norm(dim=1).cpu()
    tol = orth_bound(x, UPDATE, dtype)
    assert (off <= tol).all(), (off / tol).max()
    assert torch.equal(dense.orthogonalize(x), dense.orthogonalize(x, coefficients=UPDATE))  # the default, and the same bits again


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,rows,cols", [(190, 40, 40), (3, 64, 64), (7, 93, 93), (1, 4000, 40), (1, 40, 900), (2, 150, 150), (1, 600, 200)])
def test_orthogonalize_converges_to_the_orthogonal_factor(dense, batch, rows, cols, dtype):
    """a well conditioned x: the factor of its singular value decomposition. The last steps contract what came before in the singular
    values, so what is left is of the order of the last roundings (kept values u, sums) times the norm, plus the turn of the basis by
    the first roundings over the smallest singular value: constants of 8 and 4 cover the three products of a step and five steps."""
    g = gen_for("polar", batch, rows, cols)
    k = min(rows, cols)
    q = torch.linalg.qr(torch.randn(batch, max(rows, cols), k, generator=g, device="cuda").double().cpu())[0]
    v = torch.linalg.qr(torch.randn(batch, k, k, generator=g, device="cuda").double().cpu())[0]
    s = torch.linspace(0.5, 1.0, k, dtype=torch.float64)
    x = (q * s) @ v
    x = (x.transpose(-1, -2) if rows < cols else x).contiguous().cuda().to(dtype)
    uu, _, vv = torch.linalg.svd(x.double().cpu(), full_matrices=False)
    want = (uu @ vv).cuda()
    got = dense.orthogonalize(x, coefficients=POLAR).double()
    u = 2.0 ** -11 if dtype != F32 else 2.0 ** -23
    tol = ((8 + 4 / 0.5 * 5) * (u + math.sqrt(max(rows, cols)) * 2.0 ** -24) + U[dtype]) * math.sqrt(k)
    off = (got - want).flatten(1).norm(dim=1)
    assert (off <= tol).all(), (off.max(), tol)


@pytest.mark.parametrize("dtype", TYPES)
def test_orthogonalize_keeps_matrices_apart(dense, dtype):
    g = gen_for("apart")
    for rows, cols in ((30, 40), (100, 150), (300, 64), (900, 30)):
        x = torch.randn(4, rows, cols, generator=g, device="cuda").to(dtype)
        clean = dense.orthogonalize(x)
        one = torch.stack([dense.orthogonalize(x[i]) for i in range(4)])
        x[1, 3, 5] = math.nan
        x[2] = 0
        y = dense.orthogonalize(x)
        assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3])
        assert torch.isnan(y[1]).all() and (y[2] == 0).all()
        tol = orth_bound(one, UPDATE, dtype)  # other launches for one matrix than for four: the same within the roundings
        assert ((one.double() - clean.double()).flatten(1).norm(dim=1).cpu() <= 2 * tol).all()
        x[1, 3, 5] = math.inf
        assert torch.equal(dense.orthogonalize(x)[0], clean[0])


@pytest.mark.parametrize("dtype,scale", [(BF16, 1e30), (BF16, 1e-20), (F16, 3e4), (F32, 1e30), (F32, 1e-18)])
def test_orthogonalize_large_and_small_entries(dense, dtype, scale):
    g = gen_for("scale")
    for rows, cols in ((40, 40), (200, 130), (3000, 20)):
        x = (torch.rand(rows, cols, generator=g, device="cuda") * 2 - 1)
        x = (x * scale).to(dtype)
        got, want = dense.orthogonalize(x, coefficients=UPDATE, eps=0.0).double(), orth64(x, UPDATE, 0.0)
        assert (got - want).norm().cpu() <= orth_bound(x.double() / scale, UPDATE, dtype)


# ---------------------------------------------------------------------------------------------- together, streams, graphs
def test_a_run_of_them_together(dense):
    """a two-layer head on scores: forward, gradients, orthogonalised update; then the bases of two runs turned onto each other"""
    from sclens_amd import api

    g = gen_for("together")
    x = torch.randn(300, 93, generator=g, device="cuda")
    w1, w2 = torch.randn(256, 93, generator=g, device="cuda") / 9.6, torch.randn(10, 256, generator=g, device="cuda") / 16
    b1, b2, t = torch.zeros(256, device="cuda"), torch.zeros(10, device="cuda"), torch.randn(300, 10, generator=g, device="cuda")
    h, z = dense.linear(x, w1, bias=b1, activation="silu", save_preact=True)
    y = dense.linear(h, w2, bias=b2, residual=-t)  # the residual of a least-squares fit
    dh, dw2, db2 = dense.linear_backward(y, h, w2)
    _, dw1, db1 = dense.linear_backward(dh, x, w1, preact=z, activation="silu", need_x=False)
    step = dense.orthogonalize(dw1)
    p = [v.double().cpu().requires_grad_(True) for v in (w1, b1, w2, b2)]
    zz = x.double().cpu() @ p[0].t() + p[1]
    loss = 0.5 * ((zz * torch.sigmoid(zz)) @ p[2].t() + p[3] - t.double().cpu()).square().sum()
    loss.backward()
    for got, ref in zip((dw1, db1, dw2, db2), p):
        # fp32 throughout: sums of at most 300 terms, three in a row, relative to the gradient's own largest entry and the terms' size
        assert (got.double().cpu() - ref.grad).abs().max() <= 2 * 3 * 303 * 2.0 ** -24 * 16 * ref.grad.abs().max()
    off = (step.double() - orth64(dw1, UPDATE)).norm().cpu()
    assert off <= orth_bound(dw1, UPDATE, F32)
    # alignment: rotation of one run's vectors onto the other's
    v1 = torch.linalg.qr(torch.randn(500, 12, generator=g, device="cuda").cpu())[0]
    rot = torch.linalg.qr(torch.randn(12, 12, generator=g, device="cuda").cpu())[0]
    r = dense.orthogonalize(torch.from_numpy(api.corr_mat((v1 @ rot).numpy(), v1.numpy())).contiguous().cuda(), coefficients=POLAR)
    back = dense.linear((v1 @ rot).cuda(), r.t().contiguous())
    # singular values 1 +- roundings: the factor is off by a few units per step, eight steps
    assert (back.cpu() - v1).abs().max() < 8 * 16 * 2.0 ** -23


def test_other_streams_and_repetition(dense):
    g = gen_for("streams")
    x, w = torch.randn(700, 520, generator=g, device="cuda").to(BF16), torch.randn(640, 520, generator=g, device="cuda").to(BF16)
    dy, o = torch.randn(700, 640, generator=g, device="cuda").to(BF16), torch.randn(2, 200, 300, generator=g, device="cuda").to(BF16)
    ref = (dense.linear(x, w), *dense.linear_backward(dy, x, w), dense.orthogonalize(o))
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    out = []
    for _ in range(3):
        for s in side:  # both streams are busy at once: each call has its own scratch
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                out.append((dense.linear(x, w), *dense.linear_backward(dy, x, w), dense.orthogonalize(o)))
    torch.cuda.synchronize()
    for got in out:
        for a, b in zip(got, ref):
            assert torch.equal(a, b)


def test_captured_and_replayed(dense):
    g = gen_for("graph")
    x, w = torch.randn(300, 200, generator=g, device="cuda").to(BF16), torch.randn(310, 200, generator=g, device="cuda").to(BF16)
    xf = torch.randn(65, 33, generator=g, device="cuda")
    dy, o = torch.randn(300, 310, generator=g, device="cuda").to(BF16), torch.randn(130, 100, generator=g, device="cuda").to(BF16)
    of = torch.randn(3, 40, 40, generator=g, device="cuda")

    def work():
        return (dense.linear(x, w, activation="gelu"), dense.linear(xf, xf), *dense.linear_backward(dy, x, w), dense.orthogonalize(o),
                dense.orthogonalize(of), dense.linear(x[:1], w))

    work()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs alive at once: their scratch must not be shared with each other's results
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = work()
        graphs.append((gr, res))
    for rep in range(4):
        for t in (x, w, dy, o, xf, of):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda").to(t.dtype))
        eager = [t.clone() for t in work()]
        for gr, res in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for gr, res in graphs:
            for a, b in zip(res, eager):
                assert torch.equal(a, b), rep


def test_orthogonalize_in_planes(dense):
    """fp32 of the size that is taken apart into three planes"""
    g = gen_for("planes")
    for rows, cols in ((2100, 2304), (2304, 2100)):
        x = torch.randn(rows, cols, generator=g, device="cuda")
        off = (dense.orthogonalize(x).double() - orth64(x, UPDATE)).norm().cpu()
        # the bound of orth_bound without the singular values of 2100 x 2304: x0 has norm 1 and singular values below
        # (sqrt(rows) + sqrt(cols)) 1.05 / |x|_F; per step L <= 3.4445, at most (2 u + acc) of norms below sqrt(2100) 1.21
        u, acc = 2.0 ** -23, 2 * (math.sqrt(2304) + 3) * 2.0 ** -24
        e = u
        for _ in range(5):
            e = 3.4445 * e + (2 * u + acc) * (3.4445 + 2 * (4.775 + 2.0315 * 2)) * 1.21 * math.sqrt(2100)
        assert off <= e, (off, e)


def test_two_threads_at_once(dense):
    import threading

    g = gen_for("threads")
    x, w = torch.randn(257, 100, generator=g, device="cuda"), torch.randn(130, 100, generator=g, device="cuda")
    ref = dense.linear(x, w), dense.orthogonalize(x)
    torch.cuda.synchronize()
    bad = []

    def job():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(10):
                y, o = dense.linear(x, w), dense.orthogonalize(x)
                s.synchronize()
                if not (torch.equal(y, ref[0]) and torch.equal(o, ref[1])):
                    bad.append(1)

    ts = [threading.Thread(target=job) for _ in range(3)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_offsets_behind_32_bits(dense):
    """operands and results of more than 2^31 elements: the last rows are right"""
    M, K, N = 300000, 8, 7700
    x = torch.zeros(M, K, dtype=BF16, device="cuda")
    x[:, 0] = 1
    x[-3:, 1] = 2
    w = torch.zeros(N, K, dtype=BF16, device="cuda")
    w[:, 0], w[:, 1] = 1, 3
    w[-1] = 5
    y = dense.linear(x, w)
    assert y.numel() > 2 ** 31 and (y[:-3, :-1] == 1).all() and (y[-3:, :-1] == 7).all() and (y[:-3, -1] == 5).all() and (y[-3:, -1] == 15).all()


def test_device_refusals_leave_no_error_behind(dense):
    x = torch.ones(4, 4, device="cuda")
    with pytest.raises(Exception):
        dense.orthogonalize(x, coefficients=[(50.0, 0.0, 0.0)] * 20)
    assert torch.equal(dense.linear(x, x), torch.full((4, 4), 4.0, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S", [24, 40, 120])
@pytest.mark.parametrize("K", [257, 321, 415, 449, 1025, 2047])
def test_stream_whose_last_stage_is_short(dense, K, S, dtype):
    """one short side, rows off 16 bytes: the last stage of the contraction holds 1, 31, 63 or 2 x 32 - 1 columns"""
    g = gen_for("stream tail", K, S)
    R = 1 + 2 ** 27 // (K * S)
    x, w = ints(g, (R, K), dtype, 1), ints(g, (S, K), dtype, 1)
    ref = x.double() @ w.double().t()
    for _ in range(2):
        assert torch.equal(dense.linear(x, w), ref.float().to(dtype))
        assert torch.equal(dense.linear(w, x), ref.t().float().to(dtype))


def test_long_contractions(dense):
    """rows of more than 2^24 elements, fp32 and 16 bits: the last columns of the last rows are read"""
    K = 2 ** 24 + 72
    for dtype, M in ((F32, 70), (BF16, 80)):
        x = torch.zeros(M, K, dtype=dtype, device="cuda")
        x[:, 5], x[:, -1] = 1, 2
        x[-1, -2] = 3
        w = torch.zeros(M - 2, K, dtype=dtype, device="cuda")
        w[:, 5], w[:, -1] = torch.arange(M - 2).to("cuda", dtype), 4
        w[-1, -2] = 7
        ref = (torch.arange(M - 2, dtype=torch.float64) + 8).repeat(M, 1)
        ref[-1, -1] += 21
        assert torch.equal(dense.linear(x, w).cpu(), ref.to(dtype))
        del x, w


def test_rows_too_long_are_refused_before_anything_runs(dense):
    """size queries of the C entries: no memory is named, nothing is launched"""
    import ctypes as C

    ctx = dense.Context(0)
    lib, n, some = ctx.lib, C.c_int64(0), 1 << 20  # (an address that is never read)
    long = 2 ** 25 + 64
    assert lib.sclens_hip_linear(ctx.h, None, 1, 200, 200, long, some, long, some, long, None, None, 200, 0, some, 200, None, 200, None, n) == 1
    assert lib.sclens_hip_linear(ctx.h, None, 1, 200, 200, long - 64, some, long, some, long, None, None, 200, 0, some, 200, None, 200, None, n) == 8
    assert n.value > 0
    for dtype, N, rc in ((1, long, 1), (1, 2 ** 25, 8), (0, 2 ** 24 + 64, 1), (0, 2 ** 24, 8)):
        n.value = 0
        assert lib.sclens_hip_linear_backward(ctx.h, None, dtype, 400, N, 500, some, N, some, 500, some, 500, None, N, 0, some, 500, some, 500,
                                              some, None, n) == rc
    coef = (C.c_double * 3)(1.5, -0.5, 0.0)
    n.value = 0
    assert lib.sclens_hip_orthogonalize(ctx.h, None, 1, 1, 200, long, some, 0, long, some, 0, long, 1, coef, 1e-7, None, n) == 1
    assert "more than" in lib.sclens_hip_last_error(ctx.h).decode()


def test_workspace_of_many_matrices_is_asked_for_before_the_first_is_written(dense):
    """32 769 matrices: the last one alone takes another path than the runs of 32 768, and needs scratch that they do not"""
    import ctypes as C

    g = gen_for("many")
    B, rows, cols = 32769, 3, 1100
    x = torch.randn(B, rows, cols, generator=g, device="cuda").to(F16)
    y = torch.full_like(x, 7.0)
    ctx = dense.Context(0)
    coef, n = (C.c_double * 15)(*[v for t in UPDATE for v in t]), C.c_int64(0)

    def call(ws):
        return ctx.lib.sclens_hip_orthogonalize(ctx.h, torch.cuda.current_stream().cuda_stream, 2, B, rows, cols, x.data_ptr(), rows * cols, cols,
                                                y.data_ptr(), rows * cols, cols, 5, coef, 1e-7, ws, n)

    assert call(None) == 8 and n.value > 0
    torch.cuda.synchronize()
    assert (y == 7).all()
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    assert call(ws.data_ptr()) == 0
    got = dense.orthogonalize(x)
    assert torch.equal(got, y)
    assert torch.equal(y[32768], dense.orthogonalize(x[32768]))
    for i in (0, 1, 32766, 32767):  # alone they take the last one's path: sums in another order in fp64, one step of fp16 below 2
        assert (y[i] - dense.orthogonalize(x[i])).abs().max() <= 2.0 ** -10


def test_many_steps(dense):
    """more steps than the single-launch kernels carry along: the tiled products take them"""
    g = gen_for("many steps")
    q = torch.linalg.qr(torch.randn(90, 40, generator=g, device="cuda").double().cpu())[0]
    for dtype in TYPES:
        x = (q * torch.linspace(1, 2, 40)).to("cuda", dtype).contiguous()
        y = dense.orthogonalize(x, coefficients=UPDATE[:3] + [(1.875, -1.25, 0.375)] * 40)
        off = (y.double().t() @ y.double() - torch.eye(40, device="cuda", dtype=torch.float64)).norm().item()
        # Converged: the last step's x = a x + P x has the roundings of its 40 x 40 products (fp16 for 16-bit types) and of the result on
        # it, each at most half a step of entries whose norm is sqrt(40): x' x is off by twice their sum, a = 1.875 and |P| <= 1.875
        u = U[F32] if dtype is F32 else U[F16]
        acc = 0 if dtype is not F32 else 2 * 40 * U[F32]
        assert off <= 2 * math.sqrt(40) * (U[dtype] + 1.875 * 4 * (u + acc)), (dtype, off)


def test_coefficients_that_grow(dense):
    g = gen_for("growth")
    x = torch.randn(2, 200, 150, generator=g, device="cuda")
    for dtype in TYPES:
        y = dense.orthogonalize(x.to(dtype), coefficients=[(1.0, 0.0, 1e4), (1e-4, 0.0, 0.0)] if dtype is F32 else [(1.0, 0.0, 0.0)])
        assert torch.isfinite(y).all()
    with pytest.raises(Exception, match="grow"):
        dense.orthogonalize(x, coefficients=[(1e10, 0.0, 0.0)])
    with pytest.raises(Exception, match="grow"):
        dense.orthogonalize(x, coefficients=[(float("nan"), 0.0, 0.0)])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("R,S,K", [(20000, 40, 1001), (20000, 16, 3001), (20000, 93, 2111), (20000, 128, 1983), (30000, 60, 1023)])
def test_long_streams(dense, R, S, K, dtype):
    """long enough that a short side is streamed past, in contractions that end inside a stage and inside a chunk"""
    g = gen_for("long stream", R, S, K)
    x, w = ints(g, (R, K), dtype, 1), ints(g, (S, K), dtype, 1)
    ref = x.double() @ w.double().t()
    assert torch.equal(dense.linear(x, w), ref.float().to(dtype))
    assert torch.equal(dense.linear(w, x), ref.t().float().to(dtype))
