"""The layer operators on the GPU against their formulas in 64 bits.

Tolerances are error bounds worked out per element from the formulas: a float32 sum of n terms is off by
at most (n + 4) 2^-24 of the sum of their magnitudes (two spare roundings for the terms themselves, two for what
surrounds the sum), a function of an inexact argument by its slope, a rounded output by half a step.
"""
import math
from fractions import Fraction

import pytest

pytestmark = pytest.mark.gpu

import torch

import alphazero_amd as mctx
from alphazero_amd import _native as nat

U = 2.0 ** -24
# half a step relative to the value: p significant bits give steps of 2^(1-p) of the value's power of two, and the
# value is at least that power (float32: p = 24, bfloat16: 8, float16: 11)
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}   # least spacing
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def close(got, want, bound, dtype, what):
    """|got - want| <= bound + the rounding of the output to its type."""
    assert got.dtype == dtype and got.shape == want.shape, what
    want = want.cpu()
    tol = bound.cpu() + HALF[dtype] * (want.abs() + bound.cpu()) + TINY[dtype]
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), f"{what}: off by {float((off / tol).max()):.3g} times the bound"


def act64(z, act):
    """(value, slope, largest curvature)."""
    if act is None:
        return z, torch.ones_like(z), 0.0
    if act == "relu":
        return z.clamp(min=0), (z > 0).double(), 0.0
    if act == "swish":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p)), 0.5
    c = torch.special.ndtr(z)
    return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 0.8


def check_dense(x, w, b, r, dy, act, y, grads):
    """Every output of dense against its formula; grads: (dx, dw, db, dr) or None."""
    T = x.dtype
    # (64-bit products on the CPU)
    x, w, dy = (None if v is None else v.detach().double().cpu() for v in (x, w, dy))
    b = torch.zeros(w.shape[1], dtype=torch.float64) if b is None else b.detach().double().cpu()
    M, K = x.shape
    N = w.shape[1]
    z = x @ w + b
    size = x.abs() @ w.abs() + b.abs()
    ez = (K + 4) * U * size
    value, slope, curve = act64(z, act)
    want = value if r is None else value + r.detach().double().cpu()
    close(y, want, 1.2 * ez + 8 * U * (value.abs() + want.abs()), T, "y")
    if grads is None:
        return
    kept = ez + (2.0 ** -11 * z.abs() + 2.0 ** -25 if T != torch.float32 else 0)
    eslope = curve * kept + 16 * U
    if act == "relu":
        eslope = (z.abs() <= kept).double()
    dz = dy * slope
    edz32 = dy.abs() * eslope + 2 * U * dz.abs()
    edz = edz32 if act is None and T != torch.float32 else edz32 + HALF[T] * (dz.abs() + edz32) + TINY[T]
    dx, dw, db, dr = grads
    close(dx, dz @ w.t(), edz @ w.abs().t() + (N + 4) * U * (dz.abs() + edz) @ w.abs().t(), T, "dx")
    close(dw, x.t() @ dz, x.abs().t() @ edz + (M + 4) * U * x.abs().t() @ (dz.abs() + edz), T, "dw")
    if db is not None:
        close(db, dz.sum(0), edz32.sum(0) + (M + 4) * U * (dz.abs() + edz32).sum(0), T, "db")
    if dr is not None:
        assert torch.equal(dr.double().cpu(), dy)


SIZES = [(1, 1, 1), (1, 64, 64), (2, 3, 5), (17, 33, 65), (64, 256, 256), (63, 100, 36), (65, 128, 129),
         (130, 72, 200), (257, 64, 8), (300, 520, 264), (1, 1000, 7), (5, 2048, 3), (1025, 40, 24), (256, 256, 256),
         (512, 320, 384), (700, 192, 256), (1100, 72, 300), (1027, 131, 517), (600, 1500, 700), (500, 1001, 600),
         (5000, 20, 100), (3, 5000, 40), (40, 3, 5000)]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("T", TYPES, ids=str)
def test_dense_and_gradients(T, M, K, N):
    for i, (act, bias, res) in enumerate([(None, False, False), ("relu", True, True), ("swish", True, False),
                                          ("gelu", False, True), (None, True, True), ("swish", False, True)]):
        x = rand((M, K), T, 10 * i + 1).requires_grad_()
        w = rand((K, N), T, 10 * i + 2, K ** -0.5).requires_grad_()
        b = rand((N,), T, 10 * i + 3).requires_grad_() if bias else None
        r = rand((M, N), T, 10 * i + 4).requires_grad_() if res else None
        dy = rand((M, N), T, 10 * i + 5)
        y = mctx.dense(x, w, b, act, r)
        leaves = [t for t in (x, w, b, r) if t is not None]
        g = list(torch.autograd.grad(y, leaves, dy))
        dx, dw = g[:2]
        db = g[2] if bias else None
        dr = g[-1] if res else None
        check_dense(x, w, b, r, dy, act, y.detach(), (dx, dw, db, dr))
        with torch.no_grad():
            assert torch.equal(mctx.dense(x, w, b, act, r), y)


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("M,K,N", [(2048, 512, 1024), (1000, 1024, 768), (4100, 256, 328), (2049, 1000, 1032),
                                   (256, 4096, 512)])
def test_dense_large(T, M, K, N):
    x, w = rand((M, K), T, 1).requires_grad_(), rand((K, N), T, 2, K ** -0.5).requires_grad_()
    b, r = rand((N,), T, 3).requires_grad_(), rand((M, N), T, 4).requires_grad_()
    dy = rand((M, N), T, 5)
    y = mctx.dense(x, w, b, "swish", r)
    check_dense(x, w, b, r, dy, "swish", y.detach(), torch.autograd.grad(y, (x, w, b, r), dy))


@pytest.mark.parametrize("T", TYPES, ids=str)
def test_dense_some_gradients_only(T):
    x, w, b = rand((70, 48), T, 1), rand((48, 36), T, 2, 0.15), rand((36,), T, 3)
    dy = rand((70, 36), T, 4)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    full = torch.autograd.grad(mctx.dense(*leaves, "gelu"), leaves, dy)
    for i in range(3):
        args = [x, w, b]
        args[i] = args[i].clone().requires_grad_()
        (one,) = torch.autograd.grad(mctx.dense(*args, "gelu"), args[i], dy)
        assert torch.equal(one, full[i])


def test_dense_gradient_against_differences():
    """d(sum(y c)) / d(leaf) along random directions, float32, central differences in 64 bits of the definition."""
    x, w, b = rand((9, 14), torch.float32, 1), rand((14, 11), torch.float32, 2, 0.3), rand((11,), torch.float32, 3)
    c = rand((9, 11), torch.float32, 4)
    for act in ("swish", "gelu"):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        grads = torch.autograd.grad(mctx.dense(*leaves, act), leaves, c)
        for k in range(3):
            v = rand(leaves[k].shape, torch.float32, 50 + k).double()

            def value(h):
                p = [t.double() for t in (x, w, b)]
                p[k] = p[k] + h * v
                return (act64(p[0] @ p[1] + p[2], act)[0] * c.double()).sum()
            slope = float((value(1e-4) - value(-1e-4)) / 2e-4)
            got = float((grads[k].double() * v).sum())
            # differences: h^2 f''' / 6 ~ 1e-8 a term; float32 gradient: sums of up to 14 terms of size ~ 1
            size = float((grads[k].double() * v).abs().sum()) + 1
            assert abs(got - slope) <= (64 * U + 1e-6) * size


@pytest.mark.parametrize("T", TYPES, ids=str)
def test_dense_shapes_strides_and_streams(T):
    base = rand((6, 4, 2 * 40 + 1), T, 1)
    x = base[..., 1::2]                      # strided, offset
    w = rand((24, 40), T, 2, 0.2).t()        # transposed
    b = rand((48,), T, 3)[::2]
    r = rand((4, 6, 24), T, 4).transpose(0, 1)
    plain = mctx.dense(x.contiguous().view(24, 40), w.contiguous(), b.contiguous(), "swish", r.reshape(24, 24))
    y = mctx.dense(x, w, b, "swish", r)
    assert y.shape == (6, 4, 24) and torch.equal(y.view(24, 24), plain)
    # one row without batch axes, no rows
    assert torch.equal(mctx.dense(x[2, 3], w, b, "swish", r[2, 3]), y[2, 3]) or T == torch.float32
    assert mctx.dense(x[:0], w, b).shape == (0, 4, 24)
    e = x[:0].contiguous().requires_grad_()
    wl = w.contiguous().requires_grad_()
    dx, dw = torch.autograd.grad(mctx.dense(e, wl), (e, wl), torch.zeros((0, 4, 24), dtype=T, device="cuda"))
    assert dx.shape == e.shape and bool((dw == 0).all())
    # a contiguous view that is not 16-byte aligned, with its gradients
    flat = rand((1 + 65 * 64,), T, 5)
    u = flat[1:].view(65, 64).detach().requires_grad_()
    v = rand((64, 64), T, 6, 0.1).requires_grad_()
    dy = rand((65 * 64 + 1,), T, 7)[1:].view(65, 64)
    yy = mctx.dense(u, v, None, "relu")
    dx, dw = torch.autograd.grad(yy, (u, v), dy)
    check_dense(u, v, None, None, dy, "relu", yy.detach(), (dx, dw, None, None))
    # an expanded output gradient, another stream
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = mctx.dense(u, v, None, "relu")
        g1 = torch.autograd.grad(z.sum(), v)[0]
    torch.cuda.current_stream().wait_stream(s)
    g2 = torch.autograd.grad(mctx.dense(u, v, None, "relu"), v, torch.ones((65, 64), dtype=T, device="cuda"))[0]
    assert torch.equal(g1, g2)


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("M,K,N", [(70, 96, 80), (600, 512, 576), (1300, 1304, 1300)])
def test_dense_non_finite_values_stay_in_their_rows(T, M, K, N):
    """An infinity or NaN of x reaches its own row of y and nothing else, one of the kernel its column."""
    x, w = rand((M, K), T, 1), rand((K, N), T, 2, 0.1)
    plain = mctx.dense(x, w)
    x2 = x.clone()
    x2[3, 5], x2[M - 1, K - 1] = math.inf, math.nan
    y = mctx.dense(x2, w)
    rows = [i for i in range(M) if i not in (3, M - 1)]
    assert torch.equal(y[rows], plain[rows])
    want = torch.where(w[5].float() > 0, math.inf, -math.inf)
    assert torch.equal(y[3].float(), want)      # (no weight is zero)
    assert bool(torch.isnan(y[M - 1]).all())
    w2 = w.clone()
    w2[K - 1, 7] = -math.inf
    y = mctx.dense(x, w2)
    cols = [j for j in range(N) if j != 7]
    assert torch.equal(y[:, cols], plain[:, cols])
    assert torch.equal(y[:, 7].float(), torch.where(x[:, K - 1].float() > 0, -math.inf, math.inf))
    # the same in the gradients: a non-finite dy
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    dy = rand((M, N), T, 3)
    clean = torch.autograd.grad(mctx.dense(xl, wl), (xl, wl), dy)
    dy[3, 7] = math.inf
    dx, dw = torch.autograd.grad(mctx.dense(xl, wl), (xl, wl), dy)
    assert torch.equal(dx[[i for i in range(M) if i != 3]], clean[0][[i for i in range(M) if i != 3]])
    assert torch.equal(dx[3].float(), torch.where(w[:, 7].float() > 0, math.inf, -math.inf))
    assert torch.equal(dw[:, cols], clean[1][:, cols])
    assert torch.equal(dw[:, 7].float(), torch.where(x[3].float() > 0, math.inf, -math.inf))


@pytest.mark.parametrize("M,K,N", [(70, 96, 80), (600, 512, 576), (1300, 1304, 1300)])
def test_dense_float32_extremes(M, K, N):
    """float32 keeps its range and its precision on values far apart: exact where the sum has one term."""
    x = torch.zeros((M, K), device="cuda")
    w = torch.zeros((K, N), device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    cols = torch.arange(M, device="cuda") % K
    x[torch.arange(M, device="cuda"), cols] = torch.randn(M, generator=g, device="cuda") * \
        10.0 ** (torch.rand(M, generator=g, device="cuda") * 60 - 30)
    w[:] = torch.randn((K, N), generator=g, device="cuda")
    want = (x[torch.arange(M, device="cuda"), cols].double().unsqueeze(1) * w[cols].double())
    got = mctx.dense(x, w).double()
    assert bool(((got - want).abs() <= 8 * U * want.abs()).all())
    big = torch.full((M, K), 3e38, device="cuda")
    one = torch.zeros((K, N), device="cuda")
    one[0] = 1.0
    assert torch.equal(mctx.dense(big, one), torch.full((M, N), 3e38, device="cuda"))
    largest = torch.finfo(torch.float32).max
    assert torch.equal(mctx.dense(torch.full_like(big, largest), one), torch.full((M, N), largest, device="cuda"))


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float16], ids=str)
def test_dense_slope_beyond_the_kept_range(T):
    """The 16-bit layers keep z as float16: the slopes of pre-activations beyond its range and below its spacing."""
    big = 60000.0 if T == torch.float16 else 1e30
    x = torch.tensor([[1.0], [-1.0], [1e-7]], device="cuda", dtype=T).requires_grad_()
    w = torch.tensor([[big, 2.0 ** -14]], device="cuda", dtype=T)
    for act, far in (("relu", (1.0, 0.0)), ("swish", (1.0, 0.0)), ("gelu", (1.0, 0.0))):
        b = torch.zeros(2, device="cuda", dtype=T).requires_grad_()
        (db,) = torch.autograd.grad(mctx.dense(x[:1], w, b, act)[:, 0].sum(), b)
        assert float(db[0]) == far[0]
        (db,) = torch.autograd.grad(mctx.dense(x[1:2], w, b, act)[:, 0].sum(), b)
        assert float(db[0]) == far[1]
    b = torch.zeros(2, device="cuda", dtype=T).requires_grad_()
    (db,) = torch.autograd.grad(mctx.dense(x[2:], w, b, "relu")[:, 1].sum(), b)
    assert float(db[1]) == 1.0               # z = 1e-7 * 2^-14, positive


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("M,K,N", [(20, 48, 40), (1100, 72, 300), (600, 1500, 700), (1024, 512, 1024)])
def test_dense_writes_over_its_residual(T, M, K, N):
    """C ABI: y may be the residual itself, in every form of the product."""
    x, w, r = rand((M, K), T, 1), rand((K, N), T, 2, K ** -0.5), rand((M, N), T, 3)
    want = mctx.dense(x, w, None, "swish", r)
    lib, code = nat.lib(), {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[T]
    n = lib.az_dense_workspace_bytes(code, M, K, N, 0)
    ws = torch.empty(n + 16, dtype=torch.uint8, device="cuda")
    nat.check(lib.az_dense_forward(code, nat.ACT_SWISH, M, K, N, nat.ptr(x), nat.ptr(w), None, nat.ptr(r), nat.ptr(r), None,
                                   nat.ptr(ws), n, nat.stream_ptr()))
    torch.cuda.synchronize()
    assert torch.equal(r, want)


def test_second_derivatives_are_refused():
    x, w = rand((5, 6), torch.float32, 1).requires_grad_(), rand((6, 7), torch.float32, 2).requires_grad_()
    for y in (mctx.dense(x, w, None, "swish"), mctx.layer_norm(x)):
        (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


# ---------------------------------------------------------------- layer norm
def check_norm(x, scale, bias, eps, dy, y, grads):
    T = x.dtype
    P = (scale if scale is not None else bias).dtype if scale is not None or bias is not None else T
    x = x.detach().double()
    M, D = x.shape
    g = torch.ones(D, dtype=torch.float64, device="cuda") if scale is None else scale.detach().double()
    b = torch.zeros(D, dtype=torch.float64, device="cuda") if bias is None else bias.detach().double()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = d * rstd
    n = (D + 4) * U
    emean = n * x.abs().mean(1, keepdim=True)
    ed = emean + U * (d.abs() + emean)
    # relative error of rstd: half of that of var + eps
    evar = 0.5 * (2 * (ed * d.abs()).mean(1, keepdim=True) + (ed * ed).mean(1, keepdim=True) + n * var) / (var + eps) + 4 * U
    ex = rstd * ed + (xhat.abs() + rstd * ed) * (evar + 2 * U)
    want = xhat * g + b
    close(y, want, ex * g.abs() + 4 * U * (xhat * g).abs() + 2 * U * want.abs(), T, "y")
    if grads is None:
        return
    dy = dy.double()
    h = dy * g
    m1, m2 = h.mean(1, keepdim=True), (h * xhat).mean(1, keepdim=True)
    em1 = n * h.abs().mean(1, keepdim=True)
    em2 = n * (h * xhat).abs().mean(1, keepdim=True) + 1.01 * (h.abs() * ex).mean(1, keepdim=True)
    inner = h - m1 - xhat * m2
    size = h.abs() + m1.abs() + (xhat * m2).abs()
    bound = rstd * (U * h.abs() + em1 + (xhat.abs() + ex) * em2 + ex * m2.abs() + 4 * U * size) + \
        (rstd * inner).abs() * (evar + 4 * U)
    dx, dg, db = grads
    close(dx, rstd * inner, bound, T, "dx")
    nm = (M + 4) * U
    if dg is not None:
        close(dg, (dy * xhat).sum(0), (dy.abs() * ex).sum(0) + nm * (dy.abs() * (xhat.abs() + ex)).sum(0), P, "dscale")
    if db is not None:
        close(db, dy.sum(0), nm * dy.abs().sum(0), P, "dbias")


@pytest.mark.parametrize("M,D", [(1, 1), (3, 2), (1, 8), (5, 7), (130, 64), (64, 256), (33, 255), (9, 257), (1000, 129),
                                 (17, 1024), (6, 1025), (11, 2047), (700, 2048), (5, 4096), (4, 4097), (3, 8200),
                                 (2, 16384), (3, 16385), (2, 20001)])
@pytest.mark.parametrize("T", TYPES, ids=str)
def test_layer_norm_and_gradients(T, M, D):
    for i, (P, has) in enumerate([(T, "sb"), (torch.float32, "sb"), (T, "s"), (T, "b"), (T, "")]):
        x = (rand((M, D), torch.float32, 10 * i + 1) * 2 + rand((M, 1), torch.float32, 10 * i + 2)).to(T).requires_grad_()
        s = (1 + rand((D,), torch.float32, 10 * i + 3, 0.2)).to(P).requires_grad_() if "s" in has else None
        b = rand((D,), P, 10 * i + 4).requires_grad_() if "b" in has else None
        dy = rand((M, D), T, 10 * i + 5)
        y = mctx.layer_norm(x, s, b)
        g = dict(zip("x" + has, torch.autograd.grad(y, [t for t in (x, s, b) if t is not None], dy)))
        check_norm(x, s, b, 1e-6, dy, y.detach(), (g["x"], g.get("s"), g.get("b")))
        with torch.no_grad():
            assert torch.equal(mctx.layer_norm(x, s, b), y)


@pytest.mark.parametrize("T", TYPES, ids=str)
def test_layer_norm_many_rows(T):
    """More rows than the backward pass has workgroups, a ragged last one."""
    for M, D in ((5003, 96), (2501, 1200), (777, 5000), (300, 17000)):
        x, s, b = rand((M, D), T, 1).requires_grad_(), rand((D,), T, 2).requires_grad_(), rand((D,), T, 3).requires_grad_()
        dy = rand((M, D), T, 4)
        y = mctx.layer_norm(x, s, b, eps=1e-3)
        check_norm(x, s, b, 1e-3, dy, y.detach(), torch.autograd.grad(y, (x, s, b), dy))


def test_layer_norm_far_from_zero_and_strided():
    # a mean a thousand times the deviation: no cancellation in the variance
    x = 1000 + rand((50, 300), torch.float32, 1)
    check_norm(x, None, None, 1e-6, None, mctx.layer_norm(x), None)
    z = rand((4, 600, 5), torch.bfloat16, 2).transpose(1, 2)[..., ::2]
    s = rand((600,), torch.bfloat16, 3)[::2]
    y = mctx.layer_norm(z, s)
    assert y.shape == (4, 5, 300)
    assert torch.equal(y.view(20, 300), mctx.layer_norm(z.contiguous().view(20, 300), s.contiguous()))
    u = rand((1 + 40 * 64,), torch.float16, 4)[1:].view(40, 64)
    check_norm(u, None, None, 1e-6, None, mctx.layer_norm(u), None)
    assert mctx.layer_norm(z[:0]).shape == (0, 5, 300)
    e, sl = z[:0].contiguous().requires_grad_(), s.contiguous().requires_grad_()
    dx, ds = torch.autograd.grad(mctx.layer_norm(e, sl), (e, sl), torch.zeros((0, 5, 300), dtype=e.dtype, device="cuda"))
    assert dx.shape == e.shape and bool((ds == 0).all())
    # a constant row: variance 0
    c = torch.full((3, 70), 5.0, device="cuda")
    assert bool((mctx.layer_norm(c) == 0).all())
    # a NaN stays in its row
    c[1, 3] = math.nan
    y = mctx.layer_norm(c)
    assert bool(torch.isnan(y[1]).all()) and bool((y[[0, 2]] == 0).all())


def test_layer_norm_gradient_against_differences():
    x, s = rand((7, 24), torch.float32, 1), rand((24,), torch.float32, 2)
    c = rand((7, 24), torch.float32, 3)
    leaves = [x.clone().requires_grad_(), s.clone().requires_grad_()]
    grads = torch.autograd.grad(mctx.layer_norm(*leaves), leaves, c)
    for k in range(2):
        v = rand(leaves[k].shape, torch.float32, 9 + k).double()

        def value(h):
            p = [x.double(), s.double()]
            p[k] = p[k] + h * v
            d = p[0] - p[0].mean(1, keepdim=True)
            return (d / ((d * d).mean(1, keepdim=True) + 1e-6).sqrt() * p[1] * c.double()).sum()
        slope = float((value(1e-4) - value(-1e-4)) / 2e-4)
        got = (grads[k].double() * v)
        assert abs(float(got.sum()) - slope) <= (64 * U + 1e-6) * (float(got.abs().sum()) + 1)


# ---------------------------------------------------------------- sampling
LEAST = 2.0 ** -40


def sample64(logits, u, temperature, top_k, top_p, min_p, invalid):
    """One row by the definition: (action, log_prob).  The float64 weights are added and compared as whole
    multiples of 2^-100 (exact for weights of at least 2^-47), so that sums that meet a border exactly do."""
    legal = [i for i, l in enumerate(logits) if not math.isnan(l) and l > -math.inf and not (invalid and invalid[i])]
    if not legal:
        return 0, -math.inf
    top = max(logits[i] for i in legal)
    if top == math.inf:
        legal = [i for i in legal if logits[i] == math.inf]
        logits = {i: 0.0 for i in legal}
        top = 0.0
    if not temperature > 0:
        temperature, top_k = 1.0, 1
    order = sorted(legal, key=lambda i: (-logits[i], i))
    if top_k > 0:
        order = order[:top_k]
    w = {i: math.exp((logits[i] - top) / temperature) for i in order}
    parts = {i: int(math.ldexp(w[i], 100)) for i in order}
    if top_p < 1.0:
        goal, cum, keep = Fraction(top_p) * sum(parts.values()), 0, []
        for i in order:
            if keep and not cum < goal:
                break
            keep.append(i)
            cum += parts[i]
        order = keep
    order = sorted(i for i in order if w[i] >= max(min(min_p, 1.0), LEAST))
    total = sum(parts[i] for i in order)
    goal, cum = Fraction(u) * total, 0
    for i in order:
        cum += parts[i]
        if cum > goal:
            break
    return i, math.log(w[i]) - math.log(total / (1 << 100))


def check_sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, invalid=None):
    action, lp = mctx.sample_actions(logits, u, temperature, top_k, top_p, min_p, invalid)
    assert action.dtype == torch.int32 and lp.dtype == torch.float32
    B = logits.shape[0]
    rows = [v.tolist() if torch.is_tensor(v) else [v] * B for v in (temperature, top_k, top_p, min_p)]
    ls, us = logits.double().tolist(), u.double().tolist()
    inv = None if invalid is None else (invalid != 0).tolist()
    for b in range(B):
        want = sample64(ls[b], us[b], *(r[b] for r in rows), inv and inv[b])
        what = f"row {b}: {int(action[b])} {float(lp[b])}, want {want}"
        assert int(action[b]) == want[0], what
        if want[1] == -math.inf:
            assert float(lp[b]) == -math.inf, what
        else:   # a float32 of a 64-bit log; the total is a sum of integers at least 2^-41 fine
            assert abs(float(lp[b]) - want[1]) <= U * abs(want[1]) + 1e-9, what


def uniforms(B, seed):
    return torch.rand((B,), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


OPTIONS = [dict(), dict(top_k=1), dict(top_k=5), dict(top_p=0.9), dict(top_p=0.3, temperature=0.7), dict(min_p=0.1),
           dict(top_k=40, top_p=0.8, min_p=0.01, temperature=1.3), dict(temperature=0.0), dict(top_k=3, top_p=0.5),
           dict(top_k=300, temperature=2.0), dict(top_p=0.0), dict(min_p=1.0), dict(temperature=50.0, top_p=0.99)]


@pytest.mark.parametrize("A", [1, 2, 3, 18, 64, 65, 255, 256, 257, 362, 511, 513, 1000, 2048, 2049, 5000])
@pytest.mark.parametrize("T", TYPES, ids=str)
def test_sample_actions(T, A):
    B = 37 if A <= 513 else 5
    for i, kw in enumerate(OPTIONS):
        logits = rand((B, A), T, 100 + i, 2.5)
        inv = None if i % 2 else torch.rand((B, A), generator=torch.Generator(device="cuda").manual_seed(i), device="cuda") < 0.4
        check_sample(logits, uniforms(B, i), invalid=inv, **kw)


@pytest.mark.parametrize("A", [8192, 8193, 16384, 20000, 32768, 32769, 70001])
def test_sample_actions_large(A):
    for i, kw in enumerate(OPTIONS):
        logits = rand((2, A), TYPES[i % 3], 7 + i, 3.0)
        check_sample(logits, uniforms(2, i), invalid=None if i % 2 else logits > 4, **kw)


@pytest.mark.parametrize("A", [5, 300, 1500, 9000, 40000])
def test_sample_actions_ties(A):
    """Equal logits by index, at every truncation: one value, two values, both zeros, logits a step apart."""
    B = 6
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.999, 0.9999999], device="cuda")
    same = torch.zeros((B, A), device="cuda")
    two = torch.zeros((B, A), device="cuda")
    two[:, ::3] = 1.0
    zeros = same.clone()
    zeros[:, ::2] = -0.0
    step = 5.0 + torch.arange(A, device="cuda").remainder(7).float() * 2.0 ** -21
    for logits in (same, two, zeros, step.expand(B, A), same - 1e30):
        for kw in (dict(), dict(top_k=3), dict(top_k=A // 2 + 1), dict(top_p=0.5), dict(top_p=0.75, top_k=A // 2 + 1),
                   dict(top_k=2, top_p=0.6), dict(min_p=0.5), dict(temperature=0.0)):
            check_sample(logits, u, **kw)


@pytest.mark.parametrize("A", [7, 300, 1500, 9000, 40000])
def test_sample_actions_special_values(A):
    B = 8
    logits = rand((B, A), torch.float32, 3, 2.0)
    logits[0] = -math.inf                                   # nothing legal
    logits[1, :] = math.nan
    logits[1, A - 1] = -3e38                                # one legal action, far down
    logits[2, 1], logits[2, A - 2] = math.inf, math.inf     # shared by two
    logits[3, ::2] = -math.inf
    logits[4, 0] = 3e38                                     # the rest is never drawn
    logits[5, 2] = math.nan
    inv = torch.zeros((B, A), device="cuda")
    inv[6] = 1                                              # nothing legal by the mask
    inv[7, : A - 1] = 2.5                                   # float masks
    for kw in (dict(), dict(top_k=2), dict(top_p=0.4), dict(min_p=0.2), dict(temperature=0.0),
               dict(top_k=4, top_p=0.9, temperature=0.6)):
        for mask in (inv, inv != 0, (inv != 0).to(torch.uint8)):
            check_sample(logits, uniforms(B, 5), invalid=mask, **kw)


def test_sample_actions_parameters_by_row_and_extremes():
    B, A = 12, 400
    logits = rand((B, A), torch.float32, 1, 2.5)
    dev = "cuda"
    temperature = torch.tensor([1.0, 0.0, 0.5, 2.0, 1e-3, 30.0, 1.0, 1.0, 0.8, 1.2, -1.0, math.nan], device=dev)
    top_k = torch.tensor([0, 5, 1, 400, 1000, 3, -2, 50, 0, 7, 0, 0], device=dev)
    top_p = torch.tensor([1.0, 1.0, 0.5, 0.25, 0.9, 1.0, 0.125, 1.5, -0.5, 1.0, 0.5, 1.0], device=dev)
    min_p = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0, 0.5, 0.0, 0.0625, 0.0, 2.0, 0.0, -1.0], device=dev)
    for seed in range(4):
        check_sample(logits, uniforms(B, seed), temperature, top_k, top_p, min_p)
    check_sample(logits, uniforms(B, 9), temperature=1e-310)
    check_sample(logits, uniforms(B, 9), temperature=1e-290)
    check_sample(logits, uniforms(B, 9), temperature=1e-30, top_p=0.5)
    check_sample(logits, uniforms(B, 9), temperature=1e300, top_p=0.5, top_k=300)
    # uniforms outside [0, 1) take the nearest end
    u = torch.tensor([-1.0, math.nan, 1.0, 2.0], device=dev)
    a, lp = mctx.sample_actions(logits[:4], u, top_k=1)
    assert torch.equal(a.long(), logits[:4].argmax(1)) and bool((lp == 0).all())
    # strides, no rows, one result whatever the call
    wide = rand((20, 2 * 90), torch.bfloat16, 2, 2.0)
    v = wide[:, ::2]
    a1, l1 = mctx.sample_actions(v, uniforms(20, 1), top_p=0.9)
    a2, l2 = mctx.sample_actions(v.contiguous(), uniforms(20, 1), top_p=0.9)
    assert torch.equal(a1, a2) and torch.equal(l1, l2)
    odd = rand((1 + 20 * 90,), torch.bfloat16, 2, 2.0)[1:].view(20, 90)
    check_sample(odd, uniforms(20, 1), top_p=0.9)
    a, lp = mctx.sample_actions(v[:0], uniforms(0, 1))
    assert a.shape == (0,) and lp.shape == (0,)


@pytest.mark.parametrize("A", [18, 400, 1500, 9000, 40000])
def test_sample_actions_wide_counts_and_endless_temperatures(A):
    """64-bit counts beyond 32 bits mean all actions; an infinite temperature makes the legal actions equal."""
    logits = rand((4, A), torch.float32, 2, 2.5)
    counts = torch.tensor([2 ** 32 + 1, 2 ** 63 - 1, 1, -2 ** 40], device="cuda")
    check_sample(logits, uniforms(4, 3), top_k=counts)
    check_sample(logits, uniforms(4, 4), top_k=torch.tensor([0, 1, 2, 255], dtype=torch.uint8, device="cuda"))
    endless = torch.tensor([math.inf, 1.0, math.inf, 3e38], device="cuda")
    for kw in (dict(), dict(top_k=3), dict(top_p=0.5), dict(min_p=0.5)):
        check_sample(logits, uniforms(4, 5), temperature=endless, **kw)


def test_sample_actions_follow_the_distribution():
    """2^16 evenly spread uniforms: counts of each action off by at most one from its probability's share."""
    n = 1 << 16
    u = (torch.arange(n, device="cuda", dtype=torch.float32)) / n
    logits = rand((1, 40), torch.float32, 3, 1.5)
    a, _ = mctx.sample_actions(logits.expand(n, 40), u, temperature=0.9, top_k=20)
    p = logits[0].double() / 0.9
    p[p < p.sort(descending=True).values[19]] = -math.inf
    p = torch.softmax(p, 0) * n
    assert bool(((torch.bincount(a.long(), minlength=40).double() - p).abs() <= 1.001).all())


# ---------------------------------------------------------------- captured and concurrent calls
@pytest.mark.parametrize("T", TYPES, ids=str)
def test_layers_in_a_captured_graph(T):
    """A block's forward and backward pass and a draw, captured once and replayed on new inputs, with eager work
    between the replays."""
    M, D = 96, 128
    w, b = rand((D, D), T, 1, 0.1).requires_grad_(), rand((D,), T, 2).requires_grad_()
    s = rand((D,), T, 3).requires_grad_()
    x = rand((M, D), T, 4).requires_grad_()
    dy = rand((M, D), T, 5)
    u = uniforms(M, 6)

    def body(x, dy, u):
        h = mctx.layer_norm(x, s, b)
        y = mctx.dense(h, w, b, "swish", x)
        g = torch.autograd.grad(y, (x, w, b, s), dy)
        a, lp = mctx.sample_actions(y.detach(), u, top_k=10, top_p=0.9)
        return (y.detach(), a, lp) + g

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body(x, dy, u)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body(x, dy, u)
    for seed in range(4):
        with torch.no_grad():
            x.copy_(rand((M, D), T, 20 + seed))
        dy.copy_(rand((M, D), T, 30 + seed))
        u.copy_(uniforms(M, 40 + seed))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = body(x, dy, u)
        for g_, w_ in zip(got, want):
            assert torch.equal(g_, w_)


def test_two_calls_at_once_on_two_streams():
    T = torch.float32
    x, w = rand((512, 384), T, 1).requires_grad_(), rand((384, 256), T, 2, 0.1).requires_grad_()
    dy = rand((512, 256), T, 3)
    want = torch.autograd.grad(mctx.dense(x, w, None, "gelu"), (x, w), dy)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(torch.autograd.grad(mctx.dense(x, w, None, "gelu"), (x, w), dy))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


# ---------------------------------------------------------------- the operators together, as the package uses them
def plain_forward(nets, obs, mean=None, std=None):
    """ResidualNetworks.forward in the leaves' type, by elementary operations."""
    def norm(h, s, b):
        d = h - h.mean(1, keepdim=True)
        return d / ((d * d).mean(1, keepdim=True) + 1e-6).sqrt() * s + b
    it = iter(nets)
    obs = obs if mean is None else (obs - mean) / std
    h = obs @ next(it) + next(it)
    for _ in range((len(nets) - 8) // 6):
        u = norm(h, next(it), next(it)) @ next(it) + next(it)
        h = h + (u * torch.sigmoid(u)) @ next(it) + next(it)
    h = norm(h, next(it), next(it))
    return h @ next(it) + next(it), h @ next(it) + next(it)


@pytest.mark.parametrize("T,tol", [(torch.float32, 2e-5), (torch.bfloat16, 0.06), (torch.float16, 0.008)], ids=str)
def test_residual_networks_and_gradients(T, tol):
    """Forward and gradients of a whole network against 64 bits.  Tolerances (of the tensors' norms): the network is
    eleven layers deep and normalised, and an error travels on by the residual path unchanged; each layer adds some
    half steps of its type (float32: sums of up to 400 terms), 11 layers x 2 directions x half a step, some
    of them doubled by a slope: 22 x 2^-24 x 8, 22 x 2^-8 x 0.7, 22 x 2^-11 x 0.7."""
    g = torch.Generator(device="cuda").manual_seed(5)
    nets = mctx.ResidualNetworks(400, 3, num_atoms=5, width=192, blocks=3, generator=g, dtype=T)
    leaves = [p.requires_grad_() for p in nets.leaves()]
    obs = rand((130, 10, 10, 4), torch.float32, 1)
    cl, cv = rand((130, 3), torch.float32, 2), rand((130, 5), torch.float32, 3)
    logits, value = nets.forward(obs)
    assert logits.dtype == value.dtype == torch.float32 and logits.shape == (130, 3) and value.shape == (130, 5)
    grads = torch.autograd.grad((logits * cl).sum() + (value * cv).sum(), leaves)
    ref = [p.detach().double().cpu().requires_grad_() for p in leaves]
    rl, rv = plain_forward(ref, obs.to(T).double().cpu().reshape(130, 400))
    rgrads = torch.autograd.grad((rl * cl.double().cpu()).sum() + (rv * cv.double().cpu()).sum(), ref)
    for got, want in zip((logits, value) + grads, (rl, rv) + rgrads):
        want = want.detach()
        off = torch.linalg.vector_norm(got.detach().double().cpu() - want) / torch.linalg.vector_norm(want)
        assert float(off) <= tol, (tuple(want.shape), float(off))


def test_native_learner_step_against_library_calls():
    """One minibatch update of the MLP learner with layers.dense and with library calls: the same losses and, up to
    float32 sums in another order, the same gradients; the default is the library's."""
    from alphazero_amd import learner as L
    from alphazero_amd import networks
    g = torch.Generator(device="cuda").manual_seed(3)
    N, obs, A, K = 257, 6, 3, 4
    layout = L.row_layout(obs, A, K)
    rows = torch.rand((N, layout["_width"]), generator=g, device="cuda")
    rows[:, layout["raw_action"][0]] = 1
    data = L.unpack_rows(layout, rows)
    mean, std = torch.zeros(obs, device="cuda"), torch.ones(obs, device="cuda")
    pol = networks.init_mlp((obs, 64, 64, A), g)
    val = networks.init_mlp((obs, 256, 256, 256, K), g)
    leaves = [p.requires_grad_() for p in L.flat_leaves(pol, val)]
    out = {}
    for native in (False, True):
        total, metrics = L.compute_muzero_loss(pol, val, mean, std, data, K, native_dense=native)
        out[native] = (total, torch.autograd.grad(total, leaves))
    # a loss is a mean of sums through 4 layers of up to 256 terms: 4 x 256 roundings at the very most
    assert abs(float(out[True][0] - out[False][0])) <= 1024 * U * abs(float(out[False][0]))
    for a, b in zip(out[True][1], out[False][1]):
        # both sides' sums of up to 257 rows x 256 terms; 2e-5 of the norm is 300 half steps
        assert float(torch.linalg.vector_norm(a - b)) <= 2e-5 * float(torch.linalg.vector_norm(b)) + 1e-9


def test_prior_policy():
    B, A = 64, 18
    logits = rand((B, A), torch.float32, 1, 2.0)
    inv = (torch.rand((B, A), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < 0.3).float()
    inv[5] = 1
    root = mctx.RootFnOutput(prior_logits=logits, value=torch.zeros(B, device="cuda"), embedding=None)
    out = mctx.prior_policy((), 7, root, invalid_actions=inv, temperature=0.0)
    assert out.search_tree is None and out.action.dtype == torch.int32
    masked = logits.masked_fill(inv != 0, -math.inf)
    want = masked.argmax(1)
    want[5] = 0
    assert torch.equal(out.action.long(), want)
    p = torch.nan_to_num(torch.softmax(masked.double(), 1))
    assert bool(((out.action_weights.double() - p).abs() <= 64 * U * p + 1e-12).all()) and bool((p[5] == 0).all())
    # the same key, the same draw; the random numbers are jax.random.uniform's
    from alphazero_amd import prng
    a, b = (mctx.prior_policy((), 7, root, top_p=0.9) for _ in range(2))
    u = torch.from_numpy((prng.random_bits32(prng.as_key(7), B) >> 9).astype("float32")).cuda() * 2.0 ** -23
    assert torch.equal(a.action, b.action)
    assert torch.equal(a.action, mctx.sample_actions(logits, u, top_p=0.9)[0])


def test_prior_policy_of_special_logits():
    """The weights follow the draw: NaN and -inf are illegal, +inf logits share the row."""
    nan, inf = math.nan, math.inf
    logits = torch.tensor([[0.0, nan, 0.0, -inf], [inf, 1.0, nan, inf], [nan] * 4, [-inf] * 4, [3.0, 3.0, 3.0, 3.0],
                           [0.0, nan, 0.0, 5.0]], device="cuda")
    inv = torch.zeros_like(logits)
    inv[5, 3] = 1
    root = mctx.RootFnOutput(prior_logits=logits, value=torch.zeros(6, device="cuda"), embedding=None)
    out = mctx.prior_policy((), 3, root, invalid_actions=inv)
    want = torch.tensor([[0.5, 0, 0.5, 0], [0.5, 0, 0, 0.5], [0] * 4, [0] * 4, [0.25] * 4, [0.5, 0, 0.5, 0]], device="cuda")
    assert torch.equal(out.action_weights, want)      # (powers of two: exact)
    drawn = out.action_weights.gather(1, out.action.long()[:, None])[:, 0]
    assert bool(((drawn > 0) == (want.sum(1) > 0)).all())


@pytest.mark.parametrize("kw", [dict(env_id="CartPole-v1", native_dense=True),
                                dict(env_id="Breakout-MinAtar", torso="residual", residual_width=64)],
                         ids=["native_dense", "residual_torso"])
@pytest.mark.parametrize("graph", [True, False], ids=["graph", "eager"])
def test_trainer_runs_on_the_operators(kw, graph):
    from alphazero_amd.trainer import Config, Trainer
    cfg = Config(num_envs=32, unroll_length=4, num_simulations=8, policy="gumbel", use_gae=False, max_replay_size=512,
                 min_replay_size=0, replay_buffer_batch_size=32, num_minibatches=4, value_hidden=(64, 64),
                 policy_hidden=(32, 32), graph_sgd=graph, **kw)
    tr = Trainer(cfg, device="cuda")
    before = [p.clone() for p in tr.optimizer.params]
    m = tr.train(3)
    assert all(math.isfinite(v) for v in m.values()), m
    assert (tr._graphed is not None) == graph
    assert all(not torch.equal(a, b) for a, b in zip(before, tr.optimizer.params))
    for search in (True, False):
        ev = tr.evaluate(num_eval_envs=8, episode_length=6, search=search)
        assert math.isfinite(ev["eval/episode_reward"]) and ev["eval/avg_episode_length"] > 0


def test_graphed_learner_equals_the_eager_one():
    """Captured minibatch updates on the operators, replayed, against eager ones on the same rows: bit by bit."""
    from alphazero_amd import learner as L
    obs, A, K, n = 400, 3, 1, 96
    layout = L.row_layout(obs, A, K)
    results = []
    for graphed in (False, True):
        g = torch.Generator(device="cuda").manual_seed(3)
        nets = mctx.ResidualNetworks(obs, A, K, width=64, blocks=2, generator=g)
        opt = L.ClipAdam(L.flat_leaves(nets, None), 1e-3, total_timesteps=100)
        mean, std = torch.zeros(obs, device="cuda"), torch.ones(obs, device="cuda")
        step = L.GraphedMinibatchStep(nets, None, opt, layout, n, K, "cuda") if graphed else None
        losses = []
        for i in range(5):
            rows = torch.rand((n, layout["_width"]), generator=g, device="cuda")
            rows[:, layout["raw_action"][0]] = 1
            if graphed:
                m = step(rows, mean, std)
            else:
                m = L.minibatch_step(nets, None, mean, std, L.unpack_rows(layout, rows), opt, K)
            losses.append(float(m["total_loss"]))
        results.append((losses, [p.detach().clone() for p in opt.params]))
    # (the learning rate comes from the device in the graph: a float32 of the same double expression)
    assert results[0][0] == pytest.approx(results[1][0], rel=1e-5)
    for a, b in zip(results[0][1], results[1][1]):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)


def test_dense_split_large_tiles():
    """A long reduction over few outputs in float32: 256 x 256 tiles, the reduction split (dkernel), and the forms
    beside it; against 64-bit products on the GPU."""
    M, K, N = 12288, 1000, 1024
    x, w = rand((M, K), torch.float32, 1).requires_grad_(), rand((K, N), torch.float32, 2, K ** -0.5).requires_grad_()
    dy = rand((M, N), torch.float32, 3)
    y = mctx.dense(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    xd, wd, g = x.detach().double(), w.detach().double(), dy.double()
    close(y.detach(), xd @ wd, (K + 4) * U * (xd.abs() @ wd.abs()), torch.float32, "y")
    close(dx, g @ wd.t().contiguous(), (N + 4) * U * (g.abs() @ wd.abs().t().contiguous()), torch.float32, "dx")
    xt = xd.t().contiguous()
    close(dw, xt @ g, (M + 4) * U * (xt.abs() @ g.abs()), torch.float32, "dw")


def test_dense_of_nothing_but_nan():
    """A diverged float32 layer: every output of the large products is worked out again, in the time of some steps."""
    M, K, N = 4096, 1024, 1024
    x, w = torch.full((M, K), math.nan, device="cuda").requires_grad_(), rand((K, N), torch.float32, 1).requires_grad_()
    dy = rand((M, N), torch.float32, 2)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    y = mctx.dense(x, w, None, "swish")
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    end.record()
    torch.cuda.synchronize()
    assert bool(torch.isnan(y).all()) and bool(torch.isnan(dx).all()) and bool(torch.isnan(dw).all())
    # three products of 4.3e9 multiply-adds: milliseconds; a term-by-term fallback would take tens of seconds
    assert start.elapsed_time(end) < 1000


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("M,K,N", [(64, 256, 256), (300, 520, 264), (1003, 401, 517), (700, 2048, 40), (1024, 1024, 1024),
                                   (1100, 1032, 1100), (4100, 1032, 4104), (64, 4096, 4096)])
@pytest.mark.parametrize("act", ["swish", "gelu"])
def test_dense_gradients_of_16_bits_are_as_exact_as_their_rounding(T, M, K, N, act):
    """The gradients' errors against those of their last rounding alone, by their norms.  What is added before it: z
    is kept in float16, off by half a step (at most 2^-11 |z|, of which the root mean square is 0.58 or less, as of any value spread
    evenly over a step), which moves dz by |dy z act''(z)| as much; dz is kept to 2^-16 of itself at least; float32 sums
    of n terms are off by less than n 2^-24 of their norm, here 2^-12 of 16-bit steps.  Errors of separate terms have
    signs of their own, so their squares add up.  1.02 for the scatter of the norms themselves: each has 10^4
    values or more, whose squares' mean scatters by 1 percent."""
    x, w = rand((M, K), T, 1).requires_grad_(), rand((K, N), T, 2, K ** -0.5).requires_grad_()
    b, dy = rand((N,), T, 3), rand((M, N), T, 4)
    dx, dw = torch.autograd.grad(mctx.dense(x, w, b, act), (x, w), dy)
    x, w, dy = x.detach().double(), w.detach().double(), dy.double()
    z = x @ w + b.double()
    slope = act64(z, act)[1]
    if act == "swish":
        p = torch.sigmoid(z)
        bend = p * (1 - p) * (2 + z * (1 - 2 * p))
    else:
        bend = (2 - z * z) * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    dz = dy * slope
    off = 0.58 * 2.0 ** -11 * (dy * z * bend).abs() + 2.0 ** -16 * dz.abs()
    sq = off * off
    for got, want, added in ((dx, dz @ w.t().contiguous(), sq.sum(0) @ (w * w).t().contiguous().sum(1)),
                             (dw, x.t().contiguous() @ dz, (x * x).sum(1) @ sq.sum(1))):
        rounding = (want.to(T).double() - want).square().sum()
        err = (got.double() - want).square().sum()
        if float(rounding) == 0:
            continue
        assert float(err.sqrt()) <= 1.02 * float((rounding + added).sqrt()), (float(err.sqrt()), float(rounding.sqrt()))


@pytest.mark.parametrize("M,N", [(2900, 3000), (4096, 4096)], ids=["tiles of 128", "tiles of 256"])
def test_dense_float32_planes_are_added_the_small_ones_first(M, N):
    """Large float32 products on planes of 8 bits, x = x0 + x1 + x2: one term of 2^12, all others +-(1 + 2^-9) + 2^-18,
    whose first two planes cancel in pairs, times 1.  The third planes' 2046 x 2^-18 are 16 steps of the sum: added up before
    the first planes they are exact (11 bits) and the sum is rounded once; an accumulator of 2^12 (steps of 2^-11)
    would swallow 32 x 2^-18 at a time."""
    K = 2048
    terms = torch.empty(K, device="cuda")
    terms[0::2], terms[1::2] = 1 + 2.0 ** -9 + 2.0 ** -18, -(1 + 2.0 ** -9) + 2.0 ** -18
    terms[0], terms[1] = 2.0 ** 12, 0.0
    want = 2.0 ** 12 + (K - 2) * 2.0 ** -18
    one = torch.ones((), device="cuda")
    a = terms.expand(M, K).contiguous()
    y = mctx.dense(a, one.expand(K, N).contiguous())
    assert float((y.double() - want).abs().max()) <= 2.0 ** -11
    y = mctx.dense(one.expand(M, K).contiguous(), terms.unsqueeze(1).expand(K, N).contiguous())
    assert float((y.double() - want).abs().max()) <= 2.0 ** -11
    # the gradients' products: dx of [M, N] over K, dkernel of [M, N] over K
    x = torch.zeros((M, N), device="cuda", requires_grad=True)
    (dx,) = torch.autograd.grad(mctx.dense(x, one.expand(N, K).contiguous()), x, a)
    assert float((dx.double() - want).abs().max()) <= 2.0 ** -11
    w = torch.zeros((M, N), device="cuda", requires_grad=True)
    (dw,) = torch.autograd.grad(mctx.dense(a.t().contiguous(), w), w, one.expand(K, N).contiguous())
    assert float((dw.double() - want).abs().max()) <= 2.0 ** -11


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("act,least", [("gelu", -9.0), ("swish", -80.0)])
def test_dense_activation_tails(T, act, least):
    """Value and slope keep their relative precision far down the negative side.  One input a row and a kernel of 1, so
    that z is x itself.  In steps of U: gelu's argument z / sqrt 2 is off by two, which its integral magnifies (z^2 + 1) times;
    erfc, exp and a reciprocal are off by less than five each, what surrounds them by less than six.  exp(-z^2 / 2) of the
    slope: an argument of two roundings, z^2 steps.  swish: its exponent is held to less than a step of its result."""
    x = torch.linspace(least, 0.0, 1009, device="cuda").to(T)
    z = x.double()
    xl = x.unsqueeze(1).contiguous().requires_grad_()
    y = mctx.dense(xl, torch.ones((1, 1), dtype=T, device="cuda"), None, act)
    (dx,) = torch.autograd.grad(y, xl, torch.ones_like(y))
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        density = z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        want, slope, size, grown = z * cdf, cdf + density, cdf + density.abs(), 2 * z * z
    else:
        p = 1 / (1 + torch.exp(-z))
        want, slope, size, grown = z * p, p * (1 + z * (1 - p)), p * (1 + z.abs()), 0.0
    close(y.detach()[:, 0], want, (grown + 16) * U * want.abs(), T, "y")
    # (a 16-bit layer keeps z as float16, which holds x of either type here but for bfloat16's smallest)
    close(dx[:, 0], slope, (grown + 24) * U * size + (2.0 ** -16 * slope.abs() + 2.0 ** -24 if T != torch.float32 else 0), T, "dx")


@pytest.mark.parametrize("A", [200, 300, 1000, 1500, 9000, 40000])
def test_sample_actions_share_of_a_top_k_that_ends_far_down(A):
    """top_p is a share of the top_k's probability also where the top_k ends 32 temperatures below the largest logit,
    among actions that are never drawn.  They hold f = e^-32 = 1.27e-14 each, and n of them are in the top_k: a share
    p = 1/2 - d keeps one of the two equal actions in front of them where p (2 + n f) <= 1, and a share of all A - 2 would keep
    both where p (2 + (A - 2) f) > 1.  Weights are whole multiples of 2^-51 (above 1024 actions up to 2^-46), f of 28.5
    (0.89, rounded to 1): sums of n of them are off by at most n / 2, so a border has to be that far away.  n = 1 and d = (A - 2) f / 8: 7
    (0.2) times A - 2 to either side.  n = A / 2 - 2 and d = 3 A f / 16: 3.6 (0.08) times A below, the rounding being
    in the share's favour by 0.05 A of it, 3.6 (0.16) times A above."""
    far = math.exp(-32.0)
    logits = torch.full((2, A), -32.0, device="cuda")
    logits[:, 3], logits[:, A - 5] = 0.0, 0.0
    u = torch.tensor([0.75, 0.25], device="cuda")
    p = 0.5 - (A - 2) * far / 8
    for T in (torch.float32, torch.float16):
        check_sample(logits.to(T), u, top_k=3, top_p=p)
        check_sample(logits.to(T), u, top_k=A // 2, top_p=0.5 - 3 * A * far / 16)
        check_sample(logits.to(T), u, top_k=0, top_p=p)
    if A == 40000:
        # a row whose candidates are more than the list holds, 5000 equal ones: 2500 hold p (5000 + n f) for n = 1 (7000 units
        # to spare) and do not for n = 35000 (8600, the rounding adding 1900 to them); 20000 would leave 350, less than the rounding
        logits[:, :] = -32.0
        logits[:, 100:5100] = 0.0
        u = torch.tensor([0.9999, 0.5], device="cuda")
        for k in (5001, 0):
            check_sample(logits, u, top_k=k, top_p=0.5 - 2e-14)


@pytest.mark.parametrize("A", [18, 300, 1000, 1500, 9000, 40000])
def test_sample_actions_logits_further_apart_than_a_float32(A):
    """Logits whose difference is beyond float32, at temperatures of that size: far apart as numbers, near as weights."""
    logits = rand((4, A), torch.float32, 1, 1e38).clamp(-3.4e38, 3.4e38)
    logits[:, 1], logits[:, A - 2] = -3.4e38, 3.4e38
    temperature = torch.tensor([math.inf, 3e38, 1e38, 2e37], device="cuda")
    for i, kw in enumerate((dict(), dict(top_k=5), dict(top_k=A - 1), dict(top_p=0.5), dict(top_p=0.99, top_k=A - 2),
                            dict(min_p=0.1), dict(top_k=A // 2 + 1, top_p=0.9))):
        check_sample(logits, uniforms(4, 3 + i), temperature=temperature, **kw)


# ---------------------------------------------------------------- the forms of large layers
def check_dense_large(x, w, b, r, dy, act, y, grads):
    """check_dense with 64-bit products on the GPU, and with dz as the kernels keep it: to 2^-16 of itself in a 16-bit layer."""
    T = x.dtype
    x, w, dy = (v.detach().double() for v in (x, w, dy))
    b = torch.zeros(w.shape[1], dtype=torch.float64, device="cuda") if b is None else b.detach().double()
    (M, K), N = x.shape, w.shape[1]
    wt, xt = w.t().contiguous(), x.t().contiguous()
    z = x @ w + b
    ez = (K + 4) * U * (x.abs() @ w.abs() + b.abs())
    value, slope, curve = act64(z, act)
    want = value if r is None else value + r.detach().double()
    close(y, want, 1.2 * ez + 8 * U * (value.abs() + want.abs()), T, "y")
    kept = ez + (2.0 ** -11 * z.abs() + 2.0 ** -25 if T != torch.float32 else 0)
    eslope = (z.abs() <= kept).double() if act == "relu" else curve * kept + 16 * U
    dz = dy * slope
    exact = dy.abs() * eslope + 2 * U * dz.abs()
    edz = exact if act in (None, "relu") or T == torch.float32 else exact + 2.0 ** -16 * (dz.abs() + exact) + TINY[T]
    dx, dw, db, dr = grads
    close(dx, dz @ wt, edz @ wt.abs() + (N + 4) * U * (dz.abs() + edz) @ wt.abs(), T, "dx")
    close(dw, xt @ dz, xt.abs() @ edz + (M + 4) * U * xt.abs() @ (dz.abs() + edz), T, "dw")
    if db is not None:
        close(db, dz.sum(0), exact.sum(0) + (M + 4) * U * (dz.abs() + exact).sum(0), T, "db")
    if dr is not None:
        assert torch.equal(dr.double(), dy)


def step_and_check(T, M, K, N, act, bias=True, res=True, offset=0):
    """One training step of a layer whose tensors begin `offset` elements behind an aligned address."""
    def tensor(shape, seed, scale=1.0):
        n = math.prod(shape)
        return rand((n + offset,), T, seed, scale)[offset:].view(shape)
    x, w = tensor((M, K), 1).requires_grad_(), tensor((K, N), 2, K ** -0.5).requires_grad_()
    b = tensor((N,), 3).requires_grad_() if bias else None
    r = tensor((M, N), 4).requires_grad_() if res else None
    dy = tensor((M, N), 5)
    y = mctx.dense(x, w, b, act, r)
    g = torch.autograd.grad(y, [t for t in (x, w, b, r) if t is not None], dy)
    check_dense_large(x, w, b, r, dy, act, y.detach(), (g[0], g[1], g[2] if bias else None, g[-1] if res else None))


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("M,K,N,act", [
    (4200, 328, 4100, "swish"),     # y in tiles of 256 with every edge ragged, operands copied
    (4200, 320, 4104, "gelu"),      # y in tiles of 256, operands in place
    (4100, 256, 4104, None),
    (4200, 4100, 328, "swish"),     # dx
    (4200, 4104, 320, "relu"),      # dx over one plane of dz
    (328, 4100, 4200, "swish"),     # dkernel
    (320, 4104, 4160, None),
    (16400, 2040, 2000, "gelu"),    # dkernel with its reduction split
    (16400, 2040, 2000, None),
])
def test_dense_of_16_bits_in_large_tiles(T, M, K, N, act):
    step_and_check(T, M, K, N, act)


@pytest.mark.parametrize("M,K,N,act", [(2100, 1032, 1100, "swish"), (2101, 1033, 1101, "gelu"), (2100, 1032, 1100, "relu"),
                                       (4100, 264, 4104, "swish"), (4104, 4100, 260, "gelu"), (12288, 1000, 1024, "swish")])
def test_dense_of_float32_planes_with_activations(M, K, N, act):
    """The large float32 products' epilogue, dz as planes behind a slope, rows of dz padded to whole steps."""
    step_and_check(torch.float32, M, K, N, act)


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("M,K,N,act", [(1000, 1024, 768, "swish"), (2100, 1088, 1152, "relu"), (4200, 320, 4160, None),
                                       (700, 392, 904, "gelu")])
def test_dense_large_and_not_aligned(T, M, K, N, act):
    """Sizes whose operands the wide kernel would read in place, one element off."""
    step_and_check(T, M, K, N, act, offset=1)


def test_dense_one_row_is_a_row_of_many():
    """Another form may serve one row than many: the same sums in another order."""
    for T in TYPES:
        x, w, b, r = rand((24, 40), T, 1), rand((40, 24), T, 2, 0.2), rand((24,), T, 3), rand((24, 24), T, 4)
        many, one = mctx.dense(x, w, b, "swish", r), mctx.dense(x[15], w, b, "swish", r[15])
        size = x[15].abs().double() @ w.abs().double() + b.abs().double() + r[15].abs().double()
        # (a slope of swish is at most 1.1; the rounding of either side)
        close(one, many[15].double(), 2 * 1.2 * 44 * U * size + 8 * U * size + HALF[T] * many[15].double().abs(), T, "row")


@pytest.mark.parametrize("B", [2049, 4100, 8195])
def test_sample_actions_many_rows_left_to_the_second_kernel(B):
    """Rows that one kernel leaves to the other, of which a workgroup takes several: rows without a cut by their parameters,
    and equal logits, in turn with rows that are not left; against the same rows in calls of few, and some by the definition."""
    A = 4500
    logits = rand((B, A), torch.float32, 1, 2.5)
    logits[::3] = 1.5
    u = uniforms(B, 2)
    at = torch.arange(B, device="cuda")
    top_p = torch.where(at % 2 == 0, 0.9, 1.0).float()
    top_k = torch.where(at % 5 == 0, 7, 0).int()
    logits[B - 2] = -math.inf
    for kw in (dict(top_p=top_p, top_k=top_k), dict(top_p=0.5), dict(temperature=torch.full((B,), 0.8, device="cuda"))):
        action, lp = mctx.sample_actions(logits, u, **kw)
        for first in range(0, B, 500):
            part = slice(first, first + 500)
            few = {k: v[part] if torch.is_tensor(v) else v for k, v in kw.items()}
            a, l = mctx.sample_actions(logits[part], u[part], **few)
            assert torch.equal(a, action[part]) and torch.equal(l, lp[part])
        rows = torch.cat([at[:8], at[-8:]])
        check_sample(logits[rows], u[rows], **{k: v[rows] if torch.is_tensor(v) else v for k, v in kw.items()})


@pytest.mark.parametrize("T", TYPES, ids=str)
@pytest.mark.parametrize("M,K,N", [(70, 96, 80), (300, 520, 264), (901, 901, 450), (1300, 1304, 1300)])
def test_dense_gradients_of_infinite_operands(T, M, K, N):
    """C ABI: an infinity of x reaches its row of dkernel and one of the kernel its column of dx, as infinities, over either
    plane of dz too; nothing else changes."""
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[T]
    x, w, dy = rand((M, K), T, 1), rand((K, N), T, 2, K ** -0.5), rand((M, N), T, 3)
    z = rand((M, N), torch.float32 if T == torch.float32 else torch.float16, 4)
    lib = nat.lib()
    n = lib.az_dense_workspace_bytes(code, M, K, N, 1)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")

    def gradients(x, w):
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        nat.check(lib.az_dense_backward(code, nat.ACT_SWISH, M, K, N, nat.ptr(x), nat.ptr(w), nat.ptr(z), nat.ptr(dy), nat.ptr(dx),
                                        nat.ptr(dw), None, nat.ptr(ws), n, nat.stream_ptr()))
        return dx, dw
    dx, dw = gradients(x, w)
    x2, w2 = x.clone(), w.clone()
    x2[3, 5], w2[7, 9] = math.inf, -math.inf
    dx2, dw2 = gradients(x2, w2)
    # (a slope's sign: swish falls below z = -1.278; values around it and of dy around 0 are left out)
    dz = dy.double() * act64(z.double(), "swish")[1]
    clear = dz.abs() > 1e-3
    rows, cols = [i for i in range(K) if i != 5], [i for i in range(K) if i != 7]
    assert torch.equal(dw2[rows], dw[rows]) and torch.equal(dx2[:, cols], dx[:, cols])
    assert torch.equal(dw2[5].double()[clear[3]], (dz[3] * math.inf)[clear[3]])
    assert torch.equal(dx2[:, 7].double()[clear[:, 9]], (dz[:, 9] * -math.inf)[clear[:, 9]])
