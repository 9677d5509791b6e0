"""MI355X: the dense operators on device tensors where their ranges end -- long schedules on low-rank matrices, magnitudes near the types'
limits, addresses off 16 bytes in the tiled kernels, parts of a gradient -- against their definitions in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

from test_gpu_dense import BF16, F16, F32, POLAR, TYPES, U, UPDATE, gen_for, ints, orth64, orth_bound, padded  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dense():
    from sclens_amd import dense as d

    return d


# ---------------------------------------------------------------------------------------------------------- orthogonalize
LOW_RANK = [(40, 2000, 20), (2000, 40, 20), (64, 1500, 8), (30, 1200, 29), (64, 4096, 32)]


def low_rank(g, rows, cols, rank, dtype):
    """whole numbers that every type holds: the singular values behind `rank` are exactly zero"""
    x = ints(g, (rows, rank), F32, 1).double() @ ints(g, (rank, cols), F32, 1).double()
    assert x.abs().max() <= 256 if dtype is BF16 else 2048
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,rank", LOW_RANK)
@pytest.mark.parametrize("steps", [8, 11, 12, 17, 18, 20, 24])
def test_orthogonalize_low_rank_many_steps(dense, steps, rows, cols, rank, dtype):
    """A step takes every singular value of 0 .. 1.2024 into 0 .. 1.2024 (the largest value of p there). Roundings fill the empty directions and
    grow like any small singular value, so the bound holds for them too, but for those of the last steps: a step rounds x, A and P by u
    and its sums by 2 (sqrt(n) + 3) 2^-24, three times, each a matrix of norm below u |x|_F <= u 1.21 sqrt(m) times |P| <= 3.4445, and the
    result by u of its type. |p'| <= 3.4445 lifts what one step leaves over the bound by that much in the next, where p itself
    (p' < 0 at 1.2024 down to 0.7, p(1.2024) < 1) brings it back: twice the rounding of a step is allowed."""
    g = gen_for("low rank", rows, cols, rank)
    x = low_rank(g, rows, cols, rank, dtype)
    y = dense.orthogonalize(x, coefficients=[UPDATE[0]] * steps)
    assert torch.isfinite(y).all()
    u = 2.0 ** -11 if dtype is not F32 else 2.0 ** -23
    m, n = min(rows, cols), max(rows, cols)
    per_step = 3 * (u + 2 * (math.sqrt(n) + 3) * 2.0 ** -24) * 3.4445 * 1.21 * math.sqrt(m)
    top = torch.linalg.svdvals(y.double().cpu()).max().item()
    assert top <= 1.2024 + 2 * 3.4445 * per_step + U[dtype] * 1.21 * math.sqrt(m), top
    if steps <= 11:  # few enough that the roundings in the empty directions have not grown to one
        off = (y.double() - orth64(x, [UPDATE[0]] * steps)).norm().cpu()
        assert off <= orth_bound(x, [UPDATE[0]] * steps, dtype), off


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,rows,cols", [(1, 1, 3000), (2, 3000, 1), (3, 9, 500), (2, 500, 17), (130, 40, 200)])
def test_orthogonalize_many_steps_of_short_sides(dense, batch, rows, cols, dtype):
    """full rank, a schedule that converges: whichever path takes it, x' x is the identity up to the last step's roundings"""
    g = gen_for("many short", batch, rows, cols)
    k = min(rows, cols)
    q = torch.linalg.qr(torch.randn(batch, max(rows, cols), k, generator=g, device="cuda").double().cpu())[0]
    x = q * torch.linspace(1, 2, k, dtype=torch.float64)
    x = (x.transpose(-1, -2) if rows < cols else x).contiguous().to("cuda", dtype)
    y = dense.orthogonalize(x, coefficients=UPDATE[:3] + [POLAR[-1]] * 20).double()
    gram = y @ y.transpose(-1, -2).contiguous() if rows < cols else y.transpose(-1, -2).contiguous() @ y
    off = (gram - torch.eye(k, device="cuda", dtype=torch.float64)).flatten(1).norm(dim=1).max().item()
    # x = a x + P x: the roundings of its products (fp16 for 16-bit types, sums of max(rows, cols) terms) and of the result, each at most half a
    # step of entries whose norm is sqrt(k); a = 1.875, |P| <= 1.875, and x' x is off by twice their sum
    u = U[F32] if dtype is F32 else U[F16]
    acc = 2 * (math.sqrt(max(rows, cols)) + 3) * 2.0 ** -24
    assert off <= 2 * math.sqrt(k) * (U[dtype] + 1.875 * 4 * (u + acc)), off


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,rank", LOW_RANK)
@pytest.mark.parametrize("steps", [5, 8, 9, 10, 11])
def test_orthogonalize_low_rank_short_side(dense, steps, rows, cols, rank, dtype):
    """The m x m side in fp64: A_0 is off by at most m 2^-53, which grows by at most a^2 in a step, 1.1 times that in sum; P is off by (|b| + 2 |c| |A|)
    times it, |A| <= 1.45 (10.7), on an x of norm at most 1.21. The result is rounded to fp32 and to its type."""
    x = low_rank(gen_for("low rank", rows, cols, rank), rows, cols, rank, dtype)
    y, want = dense.orthogonalize(x, coefficients=[UPDATE[0]] * steps).double(), orth64(x, [UPDATE[0]] * steps)
    tol = 1.01 * (U[dtype] + 2.0 ** -24) * want.norm() + 1.1 * 1.21 * 10.7 * min(rows, cols) * 2.0 ** -53 * 3.4445 ** (2 * (steps - 1))
    if dtype is F16:  # (entries below its normal numbers)
        tol = tol + 2.0 ** -25 * math.sqrt(rows * cols)
    assert (y - want).norm() <= tol, ((y - want).norm().item(), tol.item())


# ---------------------------------------------------------------------------------------------------------- beside other libraries
def test_an_error_that_somebody_else_has_left_stays_theirs(dense):
    """the runtime keeps one last error per thread: a call of this library neither reports it as its own nor takes it away"""
    lib = dense.Context(0).lib
    for name in ("hipSetDevice", "hipPeekAtLastError", "hipGetLastError"):
        getattr(lib, name).restype = int
    g = gen_for("pending")
    small, big = ints(g, (40, 40), F32, 2), ints(g, (600, 1040), BF16, 1)
    grad = ints(g, (600, 600), BF16, 1)

    def calls():
        return (dense.linear(small, small), dense.linear(small[:3], small), dense.linear(big, big), *dense.linear_backward(grad, big, big),
                *dense.linear_backward(small, small, small), dense.orthogonalize(small), dense.orthogonalize(big), dense.orthogonalize(big[:40]))

    want = calls()
    torch.cuda.synchronize()
    lib.hipGetLastError()
    assert lib.hipSetDevice(9999) == 101  # refused by the runtime on the host; nothing has happened on the device
    got = []
    try:
        got = calls()
        pending = lib.hipPeekAtLastError()
    finally:
        lib.hipGetLastError()
    assert pending == 101
    for a, b in zip(got, want):
        assert torch.equal(a, b)


GROWING = [[(16.0, 0.0, 0.0), (1.5, -0.5, 0.0)], [(1.0, 0.0, 1e3), (1.0, 0.0, 0.0)], [(4.0, 0.0, 0.0), (1.5, -0.5, 0.0), (1.0, 0.0, 0.0)],
           [(12.0, -30.0, 19.0)] * 2, [(0.01, 0.0, 0.0), (100.0, 0.0, 0.0)], [(5e3, 0.0, 0.0), (1.0, 0.0, 0.0)], [(1.0, 1e5, 0.0)]]


def step_bounds(schedule):
    """the largest singular value that could be there before each step"""
    b = [1.0]
    for a1, a3, a5 in schedule:
        s = torch.linspace(0, b[-1], 20001, dtype=torch.float64)
        b.append((a1 * s + a3 * s ** 3 + a5 * s ** 5).abs().max().item() * 1.001)
    return b


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("schedule", GROWING)
@pytest.mark.parametrize("rows,cols", [(200, 150), (130, 700), (600, 300)])
def test_schedules_whose_bound_grows(dense, rows, cols, schedule, dtype):
    """the scales of 16-bit x, A and P come from the bound: besides orth_bound's relative roundings, entries are rounded to steps of
    2^-24 / scale, scale >= 2^13 / bound of what is held, half a step each: (sqrt(m) + sqrt(n)) 2^-38 bound in norm for x, and for A and P
    2 sqrt(m) 2^-38 of theirs times what the step makes of them; what a step leaves grows by the following steps' |p'|"""
    g = gen_for("growing", rows, cols)
    x = torch.randn(rows, cols, generator=g, device="cuda").to(dtype)
    got, want = dense.orthogonalize(x, coefficients=schedule).double(), orth64(x, schedule)
    tol = orth_bound(x, schedule, dtype)
    if dtype is not F32:
        m, n = min(rows, cols), max(rows, cols)
        s = torch.linalg.svdvals((x.double() / (x.double().norm() + 1e-7)).cpu())
        e = 0.0
        for (a, b, c), B in zip(schedule, step_bounds(schedule)):
            top = s.max().item()
            q = torch.linspace(0, 1.02 * top, 513, dtype=torch.float64)
            L = max((a + 3 * b * q ** 2 + 5 * c * q ** 4).abs().max().item(), (a + b * q ** 2 + c * q ** 4).abs().max().item())
            P = abs(b) * B ** 2 + abs(c) * B ** 4
            e = L * (e + math.sqrt(m * n) * 2.0 ** -38 * B) + top * m * 2.0 ** -38 * ((abs(b) + 2 * abs(c) * top ** 2) * B ** 2 + P)
            s = (a * s + b * s ** 3 + c * s ** 5).abs()
        tol = tol + e
    assert (got - want).norm().cpu() <= tol, ((got - want).norm().item(), tol)


def test_16_bits_that_do_not_suffice_are_refused(dense):
    x = torch.ones(200, 150, device="cuda")
    for schedule in ([(1.0, 0.0, 60.0), (0.0, 0.0, 1.0)], [(1.0, 0.0, 900.0), (0.0, 1.0, 0.0)], [(1.0, 0.0, 3e8), (1.0, 0.0, 0.0)]):
        assert torch.isfinite(dense.orthogonalize(x, coefficients=schedule)).all()
        small = dense.orthogonalize(x[:100, :100].to(F16).contiguous(), coefficients=schedule)  # one launch, in fp32
        assert small.shape == (100, 100)
        for dtype in (BF16, F16):
            with pytest.raises(Exception, match="16 bits"):
                dense.orthogonalize(x.to(dtype), coefficients=schedule)
    assert torch.equal(dense.orthogonalize(x.to(F16)), dense.orthogonalize(x.to(F16)))


# ---------------------------------------------------------------------------------------------------------------- activations
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


def ends_of(dtype):
    """infinities, NaN, the type's largest and smallest values, the places where exponentials leave fp32 and where clamps begin"""
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    v = [0.0, tiny, 1e-3, 0.5, 1.0, 3.0, 5.5, 9.0, 9.9, 11.5, 12.5, 13.9, 14.1, 15.0, 40.0, 86.0, 88.5, 89.0, 103.0, 105.0, 200.0, 1e4, 6e4, 1e6,
         1e12, 1.5e13, 1e18, 1.7e19, 2e19, 1e30, 1e38, big, math.inf]
    z = torch.tensor([s * t for t in v for s in (1, -1)] + [math.nan], dtype=torch.float64).to(dtype)
    return z.cuda()


def normal_cdf(z):
    """(torch.special.ndtr is 1 + erf, zero from -8.3 on)"""
    return 0.5 * torch.special.erfc(-z * math.sqrt(0.5))


def act_limits(z, kind):
    """in 64 bits, the limits at infinities"""
    if kind == "none":
        return z
    if kind == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    c = z.clamp(-1e150, 1e150)  # (infinities too; NaN stays)
    if kind == "gelu":
        s = normal_cdf(c)
    else:
        s = torch.sigmoid(c if kind == "silu" else 2 * math.sqrt(2 / math.pi) * (c + 0.044715 * c.clamp(-1e3, 1e3) ** 3))
    return torch.where(z == math.inf, z, c * s)


def act_grad_limits(z, kind):
    c = z.clamp(-1e3, 1e3)  # every derivative is 0 or 1 to the last bit there
    if kind == "relu":
        return torch.where(z.isnan(), z, (z > 0).double())
    if kind == "silu":
        s = torch.sigmoid(c)
        return s * (1 + c * (1 - s))
    if kind == "gelu":
        return normal_cdf(c) + c * torch.exp(-0.5 * c * c) / math.sqrt(2 * math.pi)
    k2 = 2 * math.sqrt(2 / math.pi)
    s = torch.sigmoid(k2 * (c + 0.044715 * c ** 3))
    return s + c * s * (1 - s) * k2 * (1 + 0.134145 * c * c)


def assert_close_or_same(got, want, tol, dtype):
    """non-finite results are the ones that the rounded exact result has; finite ones are within tol"""
    rounded = want.to(dtype).double()
    assert torch.equal(got.isnan(), rounded.isnan()), (got, rounded)
    inf = rounded.isinf() | got.isinf()
    assert torch.equal(got[inf], rounded[inf])
    ok = ((got - want).abs() <= tol) | inf | rounded.isnan()
    assert ok.all(), (got[~ok], want[~ok])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,K,N", [(8, 8, 64), (40, 8, 64), (520, 1040, 264), (70, 3, 90)])
def test_activations_at_their_ends(dense, M, K, N, act, dtype):
    """x w' = z exactly (one column of x times one; the others zero), past few rows, in tiles, in one launch"""
    z = ends_of(dtype)
    col = z.repeat(M // z.numel() + 1)[:M] if M >= z.numel() else None
    for first in range(0, z.numel(), M) if col is None else (0,):
        c = (z[first: first + M] if col is None else col)
        x = torch.zeros(c.numel(), K, dtype=dtype, device="cuda")
        x[:, K // 2] = c
        w = torch.zeros(N, K, dtype=dtype, device="cuda")
        w[:, K // 2] = 1
        got = dense.linear(x, w, activation=act).double()
        zz = c.double()[:, None].expand(-1, N)
        want = act_limits(zz, act)
        # the activation in fp32: sigmoid and tail from exp2 of a rounded product, relative 2^-23 per unit of the exponent (at most 104 before
        # the result is zero) and 16 roundings; absolute: below the smallest normal numbers of fp32, and what |z| times those is
        rel = 2.0 ** -24 * (16 + 2 * 104)
        e = want.abs() * rel + 2.0 ** -126 * (2 + zz.abs().clamp(max=200))
        assert_close_or_same(got, want, e + U[dtype] * 1.01 * (want.abs() + e) + (2.0 ** -25 if dtype is F16 else 2.0 ** -126), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS[1:])
@pytest.mark.parametrize("N", [67, 400])
def test_derivatives_at_their_ends(dense, N, act, dtype):
    """one row of gradients: dbias is dz"""
    z = ends_of(dtype).repeat(N // 60 + 1)[:N][None].contiguous()
    dy = torch.full_like(z, 0.75)
    x, w = torch.ones(1, 8, dtype=dtype, device="cuda"), torch.ones(N, 8, dtype=dtype, device="cuda")
    _, _, db = dense.linear_backward(dy, x, w, preact=z, activation=act)
    d = act_grad_limits(z.double(), act)[0]
    # derivative in fp32: sigmoid to 2^-24 (16 + 2 |exponent|) of itself, times 1 + |z| terms that cancel: absolute, 32 units of (1 + |z|) where it
    # has not reached 0 or 1 (|z| <= 110 for SiLU)
    tol = 0.75 * 32 * 2.0 ** -24 * (1 + z.double()[0].abs().clamp(max=110))
    assert_close_or_same(db.double(), 0.75 * d, tol + U[dtype] * 1.01 * (0.75 * d.abs() + tol) + (2.0 ** -25 if dtype is F16 else 0), dtype)


# ------------------------------------------------------------------------------------------------------------------ gradients
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(300, 40, 64), (700, 93, 510), (2304, 2176, 2048), (4096, 1024, 1000)])
def test_parts_of_a_gradient_have_the_bits_of_the_whole(dense, M, K, N, dtype):
    """one launch, tiles as the matrices lie, and (fp32) three planes"""
    g = gen_for("parts", M, K, N)
    x, w, dy, z = (torch.randn(*s, generator=g, device="cuda").to(dtype) for s in ((M, K), (N, K), (M, N), (M, N)))
    dx, dw, db = dense.linear_backward(dy, x, w, preact=z, activation="silu")
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1)):
        got = dense.linear_backward(dy, x if need[1] else None, w if need[0] else None, preact=z, activation="silu", need_x=bool(need[0]),
                                    need_weight=bool(need[1]), need_bias=bool(need[2])) if need[0] or need[1] else \
            dense.linear_backward(dy, x, w, preact=z, activation="silu", need_x=False, need_weight=False)
        for part, whole, wanted in zip(got, (dx, dw, db), need):
            assert part is None if not wanted else torch.equal(part, whole), need


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M,K,N", [(520, 1040, 648), (1000, 77, 450), (60, 600, 4000)])
@pytest.mark.parametrize("top", [1e-6, 3e-3, 6e4])
def test_fp16_gradients_of_any_size_keep_their_bits(dense, top, M, K, N, act):
    """dz is held in fp16 under a scale that brings the largest |dy| to 2^14 or more: half a step of dz is 2^-11 of it or, below 2^-14 of the scaled
    numbers, 2^-25 / scale <= 2^-39 of the largest |dy|. Nothing overflows: |dz| <= 1.13 |dy|. Derivatives and sums as in test_gpu_dense."""
    g = gen_for("fp16 scale", M, K, N, act)
    z = (torch.randn(M, N, generator=g, device="cuda") * 2).to(F16)
    dy = (torch.randn(M, N, generator=g, device="cuda") * top / 8).clamp(-top, top).to(F16)
    dy[M // 2, N // 3] = top
    z[M // 2, N // 3] = 1.5  # where GELU's derivative is above 1.12: dz = 67 000
    # results of ordinary size whatever the gradients' is
    x = (torch.randn(M, K, generator=g, device="cuda") * min(1e3, 1 / top / 100)).to(F16)
    w = (torch.randn(N, K, generator=g, device="cuda") * min(1e3, 1 / top / 100)).to(F16)
    d = dy.double().abs().max().item()
    dz = dy.double() * act_grad_limits(z.double(), act)
    ddz = dy.double().abs() * 32 * 2.0 ** -24 * (1 + z.double().abs())
    ddz = ddz + U[F16] * 1.01 * (dz.abs() + ddz) + 2.0 ** -39 * d
    dx, dw, db = dense.linear_backward(dy, x, w, preact=z, activation=act)
    for got, want, terms, prop in ((dx, dz @ w.double(), dz.abs() @ w.double().abs() * (2 * (N + 3)), ddz @ w.double().abs()),
                                   (dw, dz.t().contiguous() @ x.double(), dz.abs().t().contiguous() @ x.double().abs() * (2 * (M + 3)),
                                    ddz.t().contiguous() @ x.double().abs()),
                                   (db, dz.sum(0), dz.abs().sum(0) * (M + 3), (dy.double().abs() * 32 * 2.0 ** -24 * (1 + z.double().abs())).sum(0))):
        tol = (2.0 ** -24 * terms + prop) * 1.02
        assert_close_or_same(got.double(), want, tol + U[F16] * 1.01 * (want.abs() + tol) + 2.0 ** -25, F16)
    # rows of zeros, all zeros, and what is not finite beside what is
    dy2 = dy.clone()
    dy2[0], dy2[1, 5], dy2[2, 7] = 0, math.inf, math.nan
    dx2, dw2, db2 = dense.linear_backward(dy2, x, w, preact=z, activation=act)
    assert torch.equal(dx2[3:], dx[3:]) and (dx2[0] == 0).all() and not torch.isfinite(dx2[1:3]).any()
    want = (dy2.double() * act_grad_limits(z.double(), act)).sum(0).to(F16)  # (sums of gradients next to 65504 may pass it)
    assert torch.equal(torch.isfinite(db2), torch.isfinite(want)) and not torch.isfinite(db2[[5, 7]]).any()
    z0 = dense.linear_backward(torch.zeros_like(dy), x, w, preact=z, activation=act)
    assert all((t == 0).all() for t in z0)


# -------------------------------------------------------------------------------------------------------------------- sizes
def test_few_rows_past_very_many_weights(dense):
    """more groups of 16 weights than one side of a grid holds"""
    N, K = 2 ** 27 + 21, 8
    w = torch.ones(N, K, dtype=BF16, device="cuda")
    w[-1, 3] = 5
    w[2 ** 26 + 3, 0] = -1
    x = torch.ones(2, K, dtype=BF16, device="cuda")
    x[1] = 2
    y = dense.linear(x, w)
    want = torch.full((N,), 8.0, dtype=BF16, device="cuda")
    want[-1], want[2 ** 26 + 3] = 12, 6
    assert torch.equal(y[0], want) and torch.equal(y[1], 2 * want)


def test_more_rows_than_a_grid_holds_are_refused(dense):
    """size queries: no memory is named, nothing is launched"""
    import ctypes as C

    ctx = dense.Context(0)
    lib, n, some = ctx.lib, C.c_int64(0), 1 << 20  # (an address that is never read)
    for M, N, rc in ((2 ** 30, 24, 1), (24, 2 ** 30, 1), (2 ** 30 - 64, 24, 8)):
        n.value = 0
        assert lib.sclens_hip_linear(ctx.h, None, 1, M, N, 2049, some, 2049, some, 2049, None, None, N, 0, some, N, None, N, None, n) == rc
        assert rc == 8 or "rows" in lib.sclens_hip_last_error(ctx.h).decode()
    for M, rc in ((2 ** 30, 1), (2 ** 30 - 64, 8)):
        n.value = 0
        assert lib.sclens_hip_linear_backward(ctx.h, None, 1, M, 24, 24, some, 24, some, 24, some, 24, None, 24, 0, some, 24, some, 24, some, None, n) == rc


# --------------------------------------------------------------------------------------------- addresses in the larger kernels
ADDRESSES = [(0, 0), (8, 0), (8, 8), (8, 4), (16, 5), (3, 0), (1, 1), (0, 3)]


def spread(t, extra, offset):
    """rows `extra` apart in a buffer of NaN, which no result may see, `offset` elements into the storage"""
    buf = torch.full((t.size(0) * (t.size(1) + extra) + offset + 8,), math.nan, dtype=t.dtype, device=t.device)
    v = buf[offset: offset + t.size(0) * (t.size(1) + extra)].view(t.size(0), t.size(1) + extra)[:, : t.size(1)]
    v.copy_(t)
    return v


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("extra,offset", ADDRESSES)
@pytest.mark.parametrize("M,K,N", [(520, 1032, 648), (515, 1030, 641), (20000, 1001, 40), (30, 2056, 3000), (2304, 1024, 1100)])
def test_strides_and_addresses_in_tiles_and_streams(dense, M, K, N, extra, offset, dtype):
    """past the sizes of the one-launch kernels: every operand with its own stride and address, what lies between the rows is NaN"""
    g = gen_for("tile strides", M, K, N)
    x, w = ints(g, (M, K), dtype, 1), ints(g, (N, K), dtype, 1)
    b, r, dy, z = ints(g, (N,), dtype, 9), ints(g, (M, N), dtype, 9), ints(g, (M, N), dtype, 1), ints(g, (M, N), dtype, 3)
    xs, ws, rs = spread(x, extra, offset), spread(w, 2 * extra, 0), spread(r, extra // 2, offset)
    bs = torch.cat([b.new_full((offset + 1,), math.nan), b])[offset + 1:]
    zz = x.double() @ w.double().t() + b.double()
    y, pre = dense.linear(xs, ws, bias=bs, residual=rs, activation="relu", save_preact=True)
    assert torch.equal(pre, zz.float().to(dtype))
    assert torch.equal(y, (zz.clamp(min=0) + r.double()).float().to(dtype))
    assert torch.equal(dense.linear(x, spread(w, extra, offset)), (zz - b.double()).float().to(dtype))
    dys, zs = spread(dy, extra, 0), spread(z, 3 * extra, offset)
    for act, pre_in, dz in (("relu", zs, dy.double() * (z.double() > 0)), ("none", None, dy.double())):
        dx, dw, db = dense.linear_backward(dys, xs, ws, preact=pre_in, activation=act)
        assert torch.equal(dx, (dz @ w.double()).float().to(dtype))
        assert torch.equal(dw, (dz.t().contiguous() @ x.double()).float().to(dtype))
        assert torch.equal(db, dz.sum(0).float().to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("extra,offset", ADDRESSES)
@pytest.mark.parametrize("rows,cols", [(200, 304), (201, 303), (304, 200), (3000, 40), (40, 3000), (41, 700)])
def test_strides_and_addresses_of_larger_orthogonalizations(dense, rows, cols, extra, offset, dtype):
    g = gen_for("orth strides", rows, cols)
    x = torch.randn(3, rows, cols, generator=g, device="cuda").to(dtype)
    want = dense.orthogonalize(x[1].contiguous())
    assert torch.equal(dense.orthogonalize(spread(x[1], extra, offset)), want)
    # a batch whose matrices lie apart, each with longer rows
    buf = torch.full((3, rows + 2, cols + extra), math.nan, dtype=dtype, device="cuda")
    v = buf[:, 1: 1 + rows, :cols]
    v.copy_(x)
    assert torch.equal(dense.orthogonalize(v), dense.orthogonalize(x))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(5, 7, 9), (130, 200, 136), (520, 1032, 648), (515, 1030, 641), (2304, 1024, 1100)])
def test_results_with_longer_rows(dense, M, K, N, dtype):
    """the C entries write results whose rows lie apart, on any element: nothing between the rows, before or behind them"""
    import ctypes as C

    ctx = dense.Context(0)
    lib, code = ctx.lib, dense.DTYPES[dtype]
    g = gen_for("long results", M, K, N)
    x, w, b = ints(g, (M, K), dtype, 1), ints(g, (N, K), dtype, 1), ints(g, (N,), dtype, 9)
    r, dy, z = ints(g, (M, N), dtype, 9), ints(g, (M, N), dtype, 1), ints(g, (M, N), dtype, 3)
    ws = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream

    def result(rows, cols, extra, offset):
        buf = torch.full((rows * (cols + extra) + offset + 64,), -7.0, dtype=dtype, device="cuda")
        return buf, buf[offset: offset + rows * (cols + extra)].view(rows, cols + extra)

    def untouched(buf, v, cols, offset):
        assert (v[:, cols:] == -7).all() and (buf[:offset] == -7).all() and (buf[offset + v.numel():] == -7).all()

    for extra, offset in ((8, 0), (8, 8), (3, 0), (5, 1), (16, 4)):
        (yb, y), (pb, p) = result(M, N, extra, offset), result(M, N, 2 * extra, 0)
        n = C.c_int64(ws.numel())
        ctx.check(lib.sclens_hip_linear(ctx.h, stream, code, M, N, K, x.data_ptr(), K, w.data_ptr(), K, b.data_ptr(), r.data_ptr(), N, 1,
                                        y.data_ptr(), N + extra, p.data_ptr(), N + 2 * extra, ws.data_ptr(), C.byref(n)))
        zz = x.double() @ w.double().t() + b.double()
        assert torch.equal(p[:, :N], zz.float().to(dtype)) and torch.equal(y[:, :N], (zz.clamp(min=0) + r.double()).float().to(dtype))
        untouched(yb, y, N, offset)
        untouched(pb, p, N, 0)
        (xb, dx), (wb, dw), (bb, db) = result(M, K, extra, offset), result(N, K, 2 * extra, 0), result(1, N, 0, offset)
        n = C.c_int64(ws.numel())
        ctx.check(lib.sclens_hip_linear_backward(ctx.h, stream, code, M, N, K, dy.data_ptr(), N, x.data_ptr(), K, w.data_ptr(), K, z.data_ptr(), N, 1,
                                                 dx.data_ptr(), K + extra, dw.data_ptr(), K + 2 * extra, db.data_ptr(), ws.data_ptr(), C.byref(n)))
        dz = dy.double() * (z.double() > 0)
        assert torch.equal(dx[:, :K], (dz @ w.double()).float().to(dtype))
        assert torch.equal(dw[:, :K], (dz.t().contiguous() @ x.double()).float().to(dtype))
        assert torch.equal(db[0], dz.sum(0).float().to(dtype))
        untouched(xb, dx, K, offset)
        untouched(wb, dw, K, 0)
        untouched(bb, db, N, offset)
    torch.cuda.synchronize()
    ctx.close()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("M,K,N", [(200, 93, 50), (520, 1032, 648), (515, 1030, 641), (2304, 2176, 2048)])
def test_gradients_of_infinities(dense, M, K, N, act, dtype):
    """infinities and NaN of every operand reach exactly the results that contain them, whole numbers elsewhere"""
    g = gen_for("grad extremes", M, K, N)
    x, w, dy, z = ints(g, (M, K), dtype, 1), ints(g, (N, K), dtype, 1), ints(g, (M, N), dtype, 1), ints(g, (M, N), dtype, 3)
    dy[3, 5], dy[7, 9], dy[8, 1], dy[8, 2] = math.inf, math.nan, math.inf, -math.inf
    x[11, 13], x[12, 2] = -math.inf, math.nan
    w[17, 19], w[18, 7] = math.inf, math.nan
    dz = dy.double() * ((z.double() > 0) if act == "relu" else 1)
    dx, dw, db = dense.linear_backward(dy, x, w, preact=z if act == "relu" else None, activation=act)
    for got, want in ((dx, dz @ w.double()), (dw, dz.t().contiguous() @ x.double()), (db, dz.sum(0))):
        want = want.float().to(dtype).double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fix = dict(nan=0.0, posinf=1e300, neginf=-1e300)
        assert torch.equal(torch.nan_to_num(got.double(), **fix), torch.nan_to_num(want, **fix))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(5, 100000), (100000, 5)])
def test_orthogonalize_many_steps_of_a_long_side(dense, rows, cols, dtype):
    g = gen_for("long side")
    x = torch.randn(rows, cols, generator=g, device="cuda").to(dtype)
    y = dense.orthogonalize(x, coefficients=UPDATE[:3] + [POLAR[-1]] * 20).double()
    gram = y @ y.t() if rows < cols else y.t().contiguous() @ y
    u = U[F32] if dtype is F32 else U[F16]
    off = (gram - torch.eye(5, device="cuda", dtype=torch.float64)).norm().item()
    assert off <= 2 * math.sqrt(5) * (U[dtype] + 1.875 * 4 * (u + 2 * (math.sqrt(1e5) + 3) * 2.0 ** -24)), off


def test_scaled_gradients_captured_and_replayed(dense):
    """the scale of fp16 gradients is found on the device: a replay uses that of its own inputs, and two graphs share nothing"""
    g = gen_for("scaled graph")
    M, K, N = 520, 200, 648
    x, w = torch.randn(M, K, generator=g, device="cuda").to(F16), torch.randn(N, K, generator=g, device="cuda").to(F16)
    z, dy = torch.randn(M, N, generator=g, device="cuda").to(F16), torch.randn(M, N, generator=g, device="cuda").to(F16)
    o = torch.randn(40, 300, generator=g, device="cuda").to(F16)

    def work():
        return (*dense.linear_backward(dy, x, w, preact=z, activation="gelu"), dense.orthogonalize(o, coefficients=UPDATE + UPDATE + UPDATE))

    work()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = work()
        graphs.append((gr, res))
    for scale in (1.0, 1e-6, 3e3, 0.0, 1e-3):
        dy.copy_(torch.randn(M, N, generator=g, device="cuda") * scale)
        eager = [t.clone() for t in work()]
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            for a, b in zip(res, eager):
                assert torch.equal(a, b), scale


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,rank", LOW_RANK + [(60, 90, 10), (3, 128, 2)])
@pytest.mark.parametrize("steps", [12, 14, 16, 30])
def test_orthogonalize_low_rank_in_runs(dense, steps, rows, cols, rank, dtype):
    """Between two runs of the m x m side (eleven steps, at most 24) x is rounded to fp32, 2^-24 of a norm of at most 1.21 sqrt(m) counted once
    too often, which no step makes more than 4 times as large (|p'| <= 3.97 up to 1.2024); likewise what the fp64 of the definition here rounds.
    From 22 steps on both have grown to one in the empty directions: what remains is that nothing leaves 0 .. 1.2024."""
    x = low_rank(gen_for("low rank", rows, cols, rank), rows, cols, rank, dtype)
    y = dense.orthogonalize(x, coefficients=[UPDATE[0]] * steps).double()
    assert torch.isfinite(y).all()
    m, n = min(rows, cols), max(rows, cols)
    top = torch.linalg.svdvals(y.cpu()).max().item()
    assert top <= 1.2024 + (U[dtype] + 8 * (math.sqrt(n) + 3) * 2.0 ** -24) * 1.21 * math.sqrt(m), top
    if steps <= 16:
        want = orth64(x, [UPDATE[0]] * steps)
        tol = 1.01 * (U[dtype] + 2.0 ** -24) * want.norm() + 1.21 * math.sqrt(m) * (1.1 * 2.0 ** -24 * 4.0 ** (steps - 11) +
                                                                                   2 * (math.sqrt(n) + 3) * 2.0 ** -53 * 4.0 ** steps)
        if dtype is F16:
            tol = tol + 2.0 ** -25 * math.sqrt(rows * cols)
        if n > 128 or steps > 24:
            assert (y - want).norm() <= tol, ((y - want).norm().item(), tol.item())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(40, 900), (3000, 12)])
def test_short_side_schedules_that_shrink_and_grow_back(dense, rows, cols, dtype):
    """one run of the m x m side in fp64, however small x is in between: 24 factors and their product, the norm, the result's rounding"""
    x = torch.randn(rows, cols, generator=gen_for("shrink", rows, cols), device="cuda").to(dtype)
    y = dense.orthogonalize(x, coefficients=[(1e-4, 0.0, 0.0)] * 12 + [(1e4, 0.0, 0.0)] * 12).double()
    want = x.double() / (x.double().norm() + 1e-7)
    assert ((y - want).abs() <= (U[dtype] + 2.0 ** -24) * 1.01 * want.abs() + (2.0 ** -25 if dtype is F16 else 0)).all()
