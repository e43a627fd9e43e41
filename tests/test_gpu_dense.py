"""The dense operators (dgprf.linear, dgprf.dropout) against their definition in float64: sizes from
one row to many tiles, odd sizes, strides, masks, every type and activation, gradients, streams and
captured graphs."""
import numpy as np
import pytest
import torch

import dgprf
from dgprf import _native as N
from dense_reference import ACTS, TYPES, Linear, check, keep_mask, scale_of

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(g, *shape, t=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(t)


def grid(g, *shape, t=torch.float32, top=2):
    """Small whole numbers: their products and sums are exact in 32 bits, in any order."""
    return torch.randint(-top, top + 1, shape, generator=g).to(t)


def run(x, w, b=None, act="none", r=None, p=0.0, seed=0, sub=0, dy=None, **kw):
    """Result and gradients of CPU arguments, on the GPU."""
    leaf = [None if v is None else v.to(DEV).requires_grad_(dy is not None) for v in (x, w, b, r)]
    y = dgprf.linear(leaf[0], leaf[1], leaf[2], act, leaf[3], p, seed, sub, **kw)
    if dy is None:
        return (y,)
    asked = [v for v in leaf if v is not None]
    got = iter(torch.autograd.grad(y, asked, dy.to(DEV)))
    return (y, *(None if v is None else next(got) for v in leaf))


# one row, two, rows of the 32-row tile and of larger ones; K and N below, at and above a 16-byte piece, a
# fragment, a stage and a tile; one and many parts of K
SIZES = [(1, 1, 1), (1, 64, 64), (1, 2048, 512), (2, 37, 131), (3, 1030, 200), (5, 8, 4096), (8, 1500, 129),
         (9, 1, 7), (9, 64, 128), (17, 515, 33), (32, 4096, 256), (33, 33, 65), (64, 128, 8), (100, 200, 300),
         (128, 64, 128), (129, 1025, 257), (255, 72, 1001), (256, 2048, 256), (700, 9, 700), (1000, 333, 5)]
BIG = [(4096, 72, 2560), (2561, 40, 4097), (4100, 136, 2600)]


@pytest.mark.parametrize("tname", TYPES)
@pytest.mark.parametrize("size", SIZES + BIG, ids=str)
def test_products_exact(size, tname):
    """Whole numbers: the sums have no rounding, so results and gradients are the exact ones, rounded
    to the type once."""
    m, k, n = size
    t, g = TYPES[tname], _gen(m * 7 + k * 3 + n)
    x, w, b, r, dy = grid(g, m, k, t=t), grid(g, k, n, t=t), grid(g, n, t=t), grid(g, m, n, t=t), grid(g, m, n, t=t)
    if m * k * n > 1e8:  # the reference of the large ones in float32 on the GPU is exact, too
        d = lambda v: v.to(DEV).float()  # noqa: E731
    else:
        d = lambda v: v.double()  # noqa: E731
    y, dx, dw, db, dr = run(x, w, b, r=r, dy=dy)
    for name, got, want in (("y", y, d(x) @ d(w) + d(b) + d(r)), ("dx", dx, d(dy) @ d(w).t().contiguous()),
                            ("dw", dw, d(x).t().contiguous() @ d(dy)), ("db", db, d(dy).sum(0)), ("dr", dr, d(dy))):
        assert got.dtype == t and torch.equal(got.cpu(), want.to(t).cpu()), name


@pytest.mark.parametrize("tname", ["fp16", "bf16"])
@pytest.mark.parametrize("size", [(2000, 1030, 1999), (1777, 1008, 2056), (2048, 8192, 1024), (2040, 2050, 4000),
                                  (2500, 1999, 2500)], ids=str)
def test_products_of_one_tile_a_cu(size, tname):
    """Results of up to 256 tiles and longer K, whole and in parts: whole numbers again, with a bias, a
    residual, relu and a mask in the epilogue."""
    m, k, n = size
    t, g = TYPES[tname], _gen(m + k + n)
    x, w, b, r, dy = grid(g, m, k, t=t), grid(g, k, n, t=t), grid(g, n, t=t), grid(g, m, n, t=t), grid(g, m, n, t=t)
    keep = 2 * keep_mask(m, n, 32768, 7, 8).to(DEV).float()
    d = lambda v: v.to(DEV).float()  # noqa: E731
    z = d(x) @ d(w) + d(b)
    dz = d(dy) * keep * (z > 0)
    y, dx, dw, db, dr = run(x, w, b, "relu", r, 0.5, 7, 8, dy)
    for name, got, want in (("y", y, keep * z.clamp(min=0) + d(r)), ("dx", dx, dz @ d(w).t().contiguous()),
                            ("dw", dw, d(x).t().contiguous() @ dz), ("db", db, dz.sum(0)), ("dr", dr, d(dy))):
        assert got.dtype == t and torch.equal(got, want.to(t)), name


@pytest.mark.parametrize("tname", ["fp16", "bf16"])
@pytest.mark.parametrize("size", [(783, 5958, 268), (1227, 4998, 785), (1570, 14992, 2436), (2306, 15230, 1788)], ids=str)
def test_large_tiles_in_parts_of_k(size, tname):
    """Long sums of results with few large tiles: whole numbers again, a mask after the join."""
    m, k, n = size
    g = torch.Generator(device=DEV)
    g.manual_seed(m)
    draw = lambda *s: torch.randint(-2, 3, s, generator=g, device=DEV).to(TYPES[tname])  # noqa: E731
    x, w, b, r = draw(m, k), draw(k, n), draw(n), draw(m, n)
    want = 2 * keep_mask(m, n, 32768, 7, 8).to(DEV) * (x.float() @ w.float() + b.float()).clamp(min=0) + r.float()
    assert torch.equal(dgprf.linear(x, w, b, "relu", r, 0.5, 7, 8), want.to(x.dtype))


# 16-bit products that, by the rule of sizes, run: x W as 256 x 256 tiles, dz W^T as 128 x 128 in parts;
# x W as 256 x 128, x^T dz as 128 x 128 in parts; x W as 256 x 128 with two groups; dz W^T as 256 x 256;
# x^T dz as 256 x 256, and x W as 128 x 128 with two groups; that in parts; x^T dz as 256 x 128 with two groups,
# in parts; as 256 x 256 in parts; as 128 x 128 in parts; dz W^T as 256 x 128; and some of them with odd sizes
TILED = [(1500, 776, 8200), (33000, 520, 264), (16400, 72, 136), (8200, 1544, 776), (777, 3000, 4104), (250, 4088, 4104),
         (16400, 3000, 136), (16400, 4088, 1032), (8200, 776, 264), (33000, 264, 520), (1499, 775, 8199),
         (32999, 519, 263), (16399, 71, 135), (8199, 1543, 775), (16399, 2999, 135)]


@pytest.mark.parametrize("tname", TYPES)
@pytest.mark.parametrize("size", TILED, ids=str)
def test_epilogues_of_large_tiles(size, tname):
    """Bias, relu, mask and residual at once, and all gradients: whole numbers, whose sums are exact."""
    m, k, n = size
    t, g = TYPES[tname], torch.Generator(device=DEV)
    g.manual_seed(m + k + n)
    draw = lambda *s: torch.randint(-2, 3, s, generator=g, device=DEV).to(t)  # noqa: E731
    leaf, dy = [v.requires_grad_() for v in (draw(m, k), draw(k, n), draw(n), draw(m, n))], draw(m, n)
    keep = dgprf.dropout(torch.ones(m, n, device=DEV), 0.5, seed=7, sub=8)  # 0 or 2
    y = dgprf.linear(*leaf[:3], "relu", leaf[3], 0.5, 7, 8)
    got = torch.autograd.grad(y, leaf, dy)
    x, w, b, r = (v.detach().float() for v in leaf)
    z = x @ w + b
    dz = dy.float() * keep * (z > 0)
    want = (keep * z.clamp(min=0) + r, dz @ w.t().contiguous(), x.t().contiguous() @ dz, dz.sum(0), dy)
    for name, u, v in zip(("y", "dx", "dw", "db", "dr"), (y, *got), want):
        assert torch.equal(u, v.to(t)), name


@pytest.mark.parametrize("tname", TYPES)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("size", [(1500, 776, 8200), (33000, 519, 264), (16400, 72, 136), (500, 1000, 2056), (250, 4088, 4104)],
                         ids=str)
def test_activations_of_large_tiles(size, act, tname):
    m, k, n = size
    t, g = TYPES[tname], torch.Generator(device=DEV)
    g.manual_seed(m + k + n)
    draw = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device=DEV) * scale).to(t)  # noqa: E731
    x, w, b, r, dy = draw(m, k), draw(k, n, scale=k ** -0.5), draw(n), draw(m, n), draw(m, n)
    ref = Linear(x, w, b, act, r, dy=dy)
    leaf = [v.requires_grad_() for v in (x, w, b)]
    y = dgprf.linear(*leaf, act, r)
    dx, dw, db = torch.autograd.grad(y, leaf, dy)
    for name, u, v, tol in (("y", y, ref.y, ref.y_tol), ("dx", dx, ref.dx, ref.dx_tol), ("dw", dw, ref.dw, ref.dw_tol),
                            ("db", db, ref.db, ref.db_tol)):
        check(u, v.cpu(), tol.cpu(), name)


@pytest.mark.parametrize("tname", TYPES)
@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
@pytest.mark.parametrize("size", [(1, 2049, 300), (1, 5000, 1031), (2, 2052, 1000), (2, 4099, 333), (1, 2048, 1031), (2, 2048, 520)],
                         ids=str)
def test_one_and_two_rows(size, act, tname):
    """Long sums of one row and two, with everything in the epilogue."""
    m, k, n = size
    t, g = TYPES[tname], _gen(m + k + n)
    x, w, b, r = normal(g, m, k, t=t), normal(g, k, n, t=t, scale=k ** -0.5), normal(g, n, t=t), normal(g, m, n, t=t)
    dy = normal(g, m, n, t=t)
    ref = Linear(x, w, b, act, r, int(0.3 * 65536 + 0.5), 3, 4, dy)
    y, dx, dw, db, dr = run(x, w, b, act, r, 0.3, 3, 4, dy)
    for name, u, v, tol in (("y", y, ref.y, ref.y_tol), ("dx", dx, ref.dx, ref.dx_tol), ("dw", dw, ref.dw, ref.dw_tol),
                            ("db", db, ref.db, ref.db_tol)):
        check(u, v, tol, name)
    assert torch.equal(dr.cpu(), dy)


@pytest.mark.parametrize("tname", TYPES)
@pytest.mark.parametrize("m, k", [(1, 72), (1, 2100), (2, 72), (2, 2100)])
def test_strides_of_one_and_two_rows(m, k, tname):
    """Weights, inputs and residuals inside larger tensors, at any offset, and transposed ones: the results
    of contiguous copies."""
    t, g, n = TYPES[tname], _gen(m + k), 104
    base, wide = grid(g, m, k + 24, t=t).to(DEV), grid(g, k + 2, n + 9, t=t).to(DEV)
    res, row = grid(g, m, n + 9, t=t).to(DEV), grid(g, 1, n, t=t).to(DEV)
    bias = grid(g, n + 9, t=t).to(DEV)
    for off in (0, 1, 8):
        for x, w, r in ((base[:, off:off + k], wide[1:k + 1, off:off + n], res[:, off:off + n]),
                        (base[:, :k], wide[off % 2:k + off % 2, :n], row.expand(m, n)),
                        (base[:, :k].t().contiguous().t(), wide[:k, :n].t().contiguous().t(), res[:, off:off + n])):
            b = bias[off:off + n]
            y = dgprf.linear(x, w, b, "relu", r, 0.25, 5, 6)
            c = [v.clone(memory_format=torch.contiguous_format) for v in (x, w, b, r)]
            assert torch.equal(y, dgprf.linear(*c[:3], "relu", c[3], 0.25, 5, 6))
            keep = 4 / 3 * keep_mask(m, n, 16384, 5, 6).float().to(DEV)
            z = (x.double() @ w.double() + b.double()).clamp(min=0)
            want = z * keep + r.double()
            tol = torch.finfo(t).eps / 2 * want.abs() + 2.0 ** -22 * (want.abs() + z * keep)
            check(y, want.cpu(), tol.cpu(), off)


@pytest.mark.parametrize("tname", TYPES)
def test_relative_precision_of_activations(tname):
    """Down their negative side, as far as the results are normal numbers.  The normal tail is a fit of 4e-7
    (8.4e-6 for 16 bits, up to 6.5); an exponential's relative error is its exponent's absolute one, so it
    grows with the exponent: z^2 / 2 has two roundings and a constant's (2.5 2^-24 of it), z log2 e one and a
    constant's, and gelu_tanh's argument at most six more; 1 ulp for each of v_exp and v_rcp, 2^-24 for each of
    up to four sums and products."""
    t, few = TYPES[tname], 2 * 2.0 ** -23 + 4 * 2.0 ** -24
    from dense_reference import act as f
    one = torch.ones(1, 1, dtype=t, device=DEV)
    for act, low in (("gelu", -12.0 if t == torch.float32 else -6.5), ("gelu_tanh", -9.0), ("silu", -80.0)):
        x = torch.linspace(low, 0, 40001, dtype=torch.float64).to(t)[:, None]
        z = x.double()
        arg = {"gelu": 2.5 * z * z / 2, "silu": 1.5 * z.abs(),
               "gelu_tanh": 8 * 2 * (2 / np.pi) ** 0.5 * (z.abs() + 0.044715 * z.abs() ** 3)}[act]
        rel = few + 2.0 ** -24 * arg + (0 if act != "gelu" else 4e-7 if t == torch.float32 else 8.4e-6)
        want = f(z, act)
        tol = rel * want.abs()
        tol = tol + torch.finfo(t).eps / 2 * (want.abs() + tol) + torch.finfo(t).smallest_normal * torch.finfo(t).eps
        check(dgprf.linear(x.to(DEV), one, activation=act), want, tol, act)


@pytest.mark.parametrize("tname", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("size", [(1, 300, 200), (6, 65, 77), (40, 256, 136), (200, 784, 300), (130, 515, 261)], ids=str)
def test_linear_and_gradients(size, act, tname):
    m, k, n = size
    t, g = TYPES[tname], _gen(m + k + n)
    make = grid if act == "relu" else normal  # relu's slope jumps at 0: z without rounding
    x, w = make(g, m, k, t=t), make(g, k, n, t=t) if act == "relu" else normal(g, k, n, t=t, scale=k ** -0.5)
    b, r, dy = make(g, n, t=t), normal(g, m, n, t=t), normal(g, m, n, t=t)
    p, seed, sub = 0.3, 0x1234567890ABCDEF, (1 << 33) + 5
    thr = int(p * 65536 + 0.5)
    ref = Linear(x, w, b, act, r, thr, seed, sub, dy)
    y, dx, dw, db, dr = run(x, w, b, act, r, p, seed, sub, dy)
    check(y, ref.y, ref.y_tol, "y")
    check(dx, ref.dx, ref.dx_tol, "dx")
    check(dw, ref.dw, ref.dw_tol, "dw")
    check(db, ref.db, ref.db_tol, "db")
    assert torch.equal(dr.cpu(), dy)
    again = run(x, w, b, act, r, p, seed, sub, dy)
    assert all(torch.equal(u, v) for u, v in zip((y, dx, dw, db), again)), "not the same twice"
    # without gradients: the same kernel without what backward needs
    assert torch.equal(run(x, w, b, act, r, p, seed, sub)[0], y)
    ref = Linear(x, w, None, act)
    check(run(x, w, None, act)[0], ref.y, ref.y_tol, "y without bias, dropout, residual")


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_gradient_against_differences(act):
    """d/dh of sum(dy y) along a direction of x, w and b, by the central difference of the float64
    definition at h = 2^-10 (third derivatives below 4: off by less than 4 h^2 sum|dy| |dz|^3 / 6)."""
    g = _gen(3)
    m, k, n, h = 12, 24, 40, 2.0 ** -10
    x, w, b, dy = normal(g, m, k), normal(g, k, n, scale=k ** -0.5), normal(g, n, scale=0.1), normal(g, m, n)
    vx, vw, vb = normal(g, m, k, scale=0.1), normal(g, k, n, scale=0.1 * k ** -0.5), normal(g, n, scale=0.1)
    thr, seed, sub = 16384, 99, 7
    from dense_reference import act as f
    keep = keep_mask(m, n, thr, seed, sub).double() * scale_of(thr)

    def loss(e):
        z = (x.double() + e * vx.double()) @ (w.double() + e * vw.double()) + b.double() + e * vb.double()
        return float((dy.double() * keep * f(z, act)).sum())

    want = (loss(h) - loss(-h)) / (2 * h)
    _, dx, dw, db, _ = run(x, w, b, act, None, 0.25, seed, sub, dy)
    got = sum(float((d.double().cpu() * v.double()).sum()) for d, v in ((dx, vx), (dw, vw), (db, vb)))
    ref = Linear(x, w, b, act, None, thr, seed, sub, dy)
    tol = sum(float((e * v.double().abs()).sum()) for e, v in ((ref.dx_tol, vx), (ref.dw_tol, vw), (ref.db_tol, vb)))
    dz = vx.double() @ w.double() + x.double() @ vw.double() + vb.double()
    tol += float(4 * h * h / 6 * (dy.double().abs() * keep * (dz.abs() + 0.1) ** 3).sum()) * 4
    assert abs(got - want) < tol, (got, want, tol)


@pytest.mark.parametrize("tname", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (1, 1024), (5, 24), (200, 1024), (17, 1001), (4, 3, 40), (9,)], ids=str)
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(shape, p, tname):
    t, g = TYPES[tname], _gen(len(shape) * 100 + shape[-1])
    x, r, dy = normal(g, *shape, t=t), normal(g, *shape, t=t), normal(g, *shape, t=t)
    seed, sub, n = 2 ** 63 + 12345, 2 ** 40 + 3, shape[-1]
    thr = int(p * 65536 + 0.5)
    keep = keep_mask(x.numel() // n, n, thr, seed, sub).reshape(shape).double()
    s = np.float32(65536.0 / (65536 - thr)) if thr < 65536 else np.float32(0)
    # in 32 bits: one product, one sum, one rounding to the type
    drop = lambda v: torch.where(keep > 0, v.float() * float(s), torch.zeros(()))  # noqa: E731
    xd, rd = x.to(DEV).requires_grad_(), r.to(DEV).requires_grad_()
    y = dgprf.dropout(xd, p, residual=rd, seed=seed, sub=sub)
    dx, dr = torch.autograd.grad(y, (xd, rd), dy.to(DEV))
    # v_mul then v_add, or one fma: half a step of 32 bits apart, which may change the type's rounding
    want = drop(x) + r.float()
    tol = torch.finfo(t).eps / 2 * want.abs().double() + 2.0 ** -23 * (want.abs() + drop(x).abs()).double() + 1e-30
    if t == torch.float16:
        tol = tol + 2.0 ** -25
    check(y, want.double(), tol, "y")
    assert torch.equal(dx.cpu(), drop(dy).to(t)) and torch.equal(dr.cpu(), dy)
    assert torch.equal(dgprf.dropout(x.to(DEV), p, seed=seed, sub=sub).cpu(), drop(x).to(t))


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("size", [(40, 24, 56), (400, 72, 520)], ids=str)
def test_gradients_where_scaled_ones_overflow(size, act):
    """fp16: s dy is above the type's largest value, dx and dW are not."""
    t, g = torch.float16, _gen(13)
    m, k, n = size
    for p, top in ((0.75, 30000), (65535 / 65536, 1)):
        x, w = normal(g, m, k, t=t, scale=2.0 ** -9), normal(g, k, n, t=t, scale=2.0 ** -10)
        dy = (torch.randint(0, 2, (m, n), generator=g) * 2 - 1).to(t) * top
        thr = int(p * 65536 + 0.5)
        ref = Linear(x, w, None, act, None, thr, 1, 2, dy)
        assert float(ref.dx.abs().max()) < 60000 and float(ref.dw.abs().max()) < 60000 < scale_of(thr) * top
        assert n < 100 or bool(ref.dx.any())
        _, dx, dw, _, _ = run(x, w, None, act, None, p, 1, 2, dy)
        # dz / s is stored, so its smallest step counts s times
        more = scale_of(thr) * torch.finfo(t).smallest_normal * torch.finfo(t).eps
        check(dx, ref.dx, ref.dx_tol + more * w.double().abs().sum(1), "dx")
        check(dw, ref.dw, ref.dw_tol + more * x.double().abs().sum(0)[:, None], "dw")


def test_linear_takes_dropouts_mask():
    """The mask depends on (seed, sub, row, column, n) alone: every path of linear has the one of dropout."""
    for m, n in ((1, 40), (7, 136), (20, 264), (150, 100), (513, 130), (4096, 2560)):
        one, w, b = torch.ones(m, 8, device=DEV), torch.zeros(8, n, device=DEV), torch.ones(n, device=DEV)
        want = dgprf.dropout(torch.ones(m, n, device=DEV), 0.4, seed=5, sub=6)
        assert torch.equal(dgprf.linear(one, w, b, dropout=0.4, seed=5, sub=6), want), (m, n)
        assert 0 < int((want == 0).sum()) < m * n
        assert not torch.equal(dgprf.linear(one, w, b, dropout=0.4, seed=5, sub=7), want)


def test_dropped_elements_are_zero_whatever_they_hold():
    x = torch.full((64, 256), float("nan"), device=DEV)
    x[::2] = float("inf")
    keep = keep_mask(64, 256, 32768, 1, 2).to(DEV)
    y = dgprf.dropout(x, 0.5, seed=1, sub=2)
    assert bool((y[~keep] == 0).all()) and not bool(torch.isfinite(y[keep]).any())
    assert bool((dgprf.dropout(x, 1.0, seed=1, sub=2) == 0).all())
    # a gradient that is not finite where the mask dropped does not get through
    v = torch.ones(64, 32, device=DEV, requires_grad=True)
    w = torch.ones(32, 256, device=DEV, requires_grad=True)
    y = dgprf.linear(v, w, activation="gelu", dropout=0.5, seed=1, sub=2)
    dy = torch.where(keep, torch.ones_like(y), torch.full_like(y, float("nan")))
    assert all(bool(torch.isfinite(d).all()) for d in torch.autograd.grad(y, (v, w), dy))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("tname", TYPES)
def test_not_finite_values(tname, act):
    """An infinite or NaN input reaches its own row of the result and no other; slopes at infinity are
    the limits 0 or 1."""
    t, g = TYPES[tname], _gen(1)
    for m in (4, 70):
        x, w = normal(g, m, 64, t=t).abs() + 0.5, normal(g, 64, 96, t=t).abs() + 0.5
        x, w = x.to(DEV), w.to(DEV)
        clean = dgprf.linear(x, w, activation=act)
        for bad in (float("inf"), float("nan")):
            x2 = x.clone()
            x2[2, 5] = bad
            x2.requires_grad_()
            y = dgprf.linear(x2, w, activation=act)
            assert torch.equal(y[torch.arange(m) != 2], clean[torch.arange(m) != 2])
            assert bool((torch.isinf(y[2]) if bad == float("inf") else torch.isnan(y[2])).all())
            dx, = torch.autograd.grad(y, x2, torch.ones_like(y))
            if bad == float("inf"):
                assert bool(torch.isfinite(dx).all())
            else:
                assert bool(torch.isfinite(dx[torch.arange(m) != 2]).all())


@pytest.mark.parametrize("tname", TYPES)
@pytest.mark.parametrize("m", [3, 24, 150])
def test_strides(m, tname):
    """Rows apart, columns of a larger tensor, transposed operands, a residual row for all, odd
    offsets: the same results as of contiguous copies, and nothing outside is touched."""
    t, g, k, n = TYPES[tname], _gen(m), 72, 104
    base = grid(g, m, k + 24, t=t).to(DEV)
    wide = grid(g, k + 2, n + 8, t=t).to(DEV)
    bias = grid(g, n, t=t).to(DEV)
    row = grid(g, 1, n, t=t).to(DEV)
    dy = grid(g, m, n, t=t).to(DEV)

    def both(x, w, r, dy):
        out = []
        for c in (False, True):
            leaf = [(v.contiguous() if c else v).detach() for v in (x, w, r)]
            leaf[2] = leaf[2].clone() if c else leaf[2]
            for v in leaf:
                v.requires_grad_()
            y = dgprf.linear(leaf[0], leaf[1], bias, "none", leaf[2])
            out.append((y, *torch.autograd.grad(y, leaf, dy.contiguous() if c else dy)))
        for u, v in zip(*out):
            assert torch.equal(u, v)

    for off in (0, 1, 8):
        both(base[:, off:off + k], wide[1:k + 1, off:off + n], row.expand(m, n), dy)
    both(base[:, :k], wide[:k, :n], dy, row.expand(m, n))
    xt, wt = grid(g, k, m, t=t).to(DEV).t(), grid(g, n, k, t=t).to(DEV).t()
    both(xt, wt, grid(g, n, m, t=t).to(DEV).t(), grid(g, n, m, t=t).to(DEV).t())
    both(base[::2, :k], wide[:k, :n], dy[::2], dy[::2])
    both(base[:, 3:3 + k], wide[:k, 5:5 + n], dy, dy)


def test_negated_views():
    """The imaginary part of a conjugate is a view of the other sign's memory: its values count."""
    g = _gen(14)
    ones = [torch.complex(normal(g, *s), normal(g, *s)).to(DEV).conj().imag for s in ((6, 1), (1, 9), (9,), (6, 9), (6, 9))]
    ones += [torch._neg_view(normal(g, *s).to(DEV)) for s in ((6, 8), (8, 9), (9,), (6, 9), (6, 9))]
    for views in (ones[:5], ones[5:]):
        assert all(v.is_neg() for v in views)
        for args in (views, [v.clone() for v in views]):
            leaf = [v.detach().requires_grad_() for v in args[:4]]
            y = dgprf.linear(*leaf[:3], "silu", leaf[3], 0.25, 1, 2)
            z = dgprf.dropout(args[0], 0.25, residual=args[0], seed=1, sub=2)
            got = (y, z, *torch.autograd.grad(y, leaf, args[4]))
            want = got if args is views else want
            assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_leading_dimensions_and_no_rows():
    g = _gen(4)
    x, w = normal(g, 3, 5, 16).to(DEV).requires_grad_(), normal(g, 16, 24).to(DEV).requires_grad_()
    b = normal(g, 24).to(DEV).requires_grad_()
    y = dgprf.linear(x, w, b, "silu")
    assert y.shape == (3, 5, 24)
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    flat = x.detach().reshape(15, 16).requires_grad_()
    y2 = dgprf.linear(flat, w, b, "silu")
    dx2, dw2 = torch.autograd.grad(y2, (flat, w), torch.ones_like(y2))
    assert torch.equal(y.reshape(15, 24), y2) and torch.equal(dx.reshape(15, 16), dx2) and torch.equal(dw, dw2)
    v = x[0, 0].detach()
    assert torch.equal(dgprf.linear(v, w.detach(), b.detach(), "silu"), y2[0].detach()) or \
        torch.allclose(dgprf.linear(v, w.detach(), b.detach(), "silu"), y2[0].detach(), rtol=1e-5, atol=1e-5)
    for t in TYPES.values():
        x0 = torch.empty(0, 16, device=DEV, dtype=t, requires_grad=True)
        w0, b0 = w.detach().to(t).requires_grad_(), b.detach().to(t).requires_grad_()
        y0 = dgprf.linear(x0, w0, b0, "gelu", dropout=0.5)
        assert y0.shape == (0, 24)
        dx0, dw0, db0 = torch.autograd.grad(y0, (x0, w0, b0), torch.empty_like(y0))
        assert dx0.shape == (0, 16) and not dw0.any() and not db0.any()
        assert dgprf.dropout(torch.empty(3, 0, device=DEV, dtype=t), 0.5).shape == (3, 0)


def test_gradients_asked_for_alone():
    g = _gen(5)
    x, w, b, r = normal(g, 40, 24), normal(g, 24, 56), normal(g, 56), normal(g, 40, 56)
    dy = normal(g, 40, 56).to(DEV)
    full = run(x, w, b, "gelu", r, 0.2, 3, 4, dy.cpu())
    for i in range(4):
        leaf = [v.to(DEV) for v in (x, w, b, r)]
        leaf[i].requires_grad_()
        y = dgprf.linear(*leaf[:3], "gelu", leaf[3], 0.2, 3, 4)
        got, = torch.autograd.grad(y, leaf[i], dy)
        assert torch.equal(got, full[1 + i])
    # one tensor in two places: the sum of its gradients
    s = normal(g, 24, 24).to(DEV).requires_grad_()
    y = dgprf.linear(s, s, residual=s)
    d = torch.ones_like(y)
    got, = torch.autograd.grad(y, s, d)
    c = s.detach().double()
    want = d.double() @ c.t() + c.t() @ d.double() + d.double()
    assert (got.double() - want).abs().max() < 60 * 2.0 ** -23 * (1 + 2 * c.abs().sum(0).max() + 2 * c.abs().sum(1).max())
    with pytest.raises(RuntimeError):
        y = dgprf.linear(s, s, activation="gelu")
        first, = torch.autograd.grad(y.sum(), s, create_graph=True)
        torch.autograd.grad(first.sum(), s)


def test_masks_come_from_the_global_generator():
    x = torch.ones(64, 64, device=DEV)
    dgprf.set_seed(11)
    a, b = dgprf.dropout(x, 0.5), dgprf.dropout(x, 0.5)
    assert not torch.equal(a, b)
    dgprf.set_seed(11)
    assert torch.equal(a, dgprf.dropout(x, 0.5)) and torch.equal(b, dgprf.dropout(x, 0.5))
    step = torch.tensor([5], device=DEV)
    assert torch.equal(dgprf.dropout(x, 0.5, seed=1, sub=2, step=step), dgprf.dropout(x, 0.5, seed=1, sub=7))


def test_steps_of_calls_do_not_meet():
    """With a step and the default numbers, no mask of one call comes up in another, whatever the steps."""
    x, masks = torch.ones(64, 64, device=DEV), []
    dgprf.set_seed(11)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    for i in range(4):
        dgprf.set_seed(11)
        step.fill_(i)
        masks += [dgprf.dropout(x, 0.5, step=step), dgprf.linear(x, torch.eye(64, device=DEV), dropout=0.5, step=step)]
        masks += [dgprf.dropout(x, 0.5)] if i == 0 else []
    assert len({m.cpu().numpy().tobytes() for m in masks}) == len(masks)


def _block(x, w1, b1, w2, b2, step=None):
    """The operators as a network uses them: up-projection, dropout, down-projection onto the residual."""
    h = dgprf.linear(x, w1, b1, "gelu", dropout=0.2, seed=8, sub=0, step=step)
    y = dgprf.linear(h, w2, b2, residual=x, dropout=0.1, seed=8, sub=1 << 32, step=step)
    return dgprf.dropout(y, 0.1, seed=8, sub=1 << 33, step=step)


@pytest.mark.parametrize("tname", TYPES)
def test_block(tname):
    """A run of the operators against the same in float64 where every operator's result is rounded to
    the type, as it is when handed on: an error of half a step goes through each later operator."""
    t, g = TYPES[tname], _gen(6)
    m, d, f = 96, 64, 200
    x, w1, b1 = normal(g, m, d, t=t), normal(g, d, f, t=t, scale=d ** -0.5), normal(g, f, t=t, scale=0.1)
    w2, b2, dy = normal(g, f, d, t=t, scale=f ** -0.5), normal(g, d, t=t, scale=0.1), normal(g, m, d, t=t)
    leaf = [v.to(DEV).requires_grad_() for v in (x, w1, b1, w2, b2)]
    y = _block(*leaf)
    got = torch.autograd.grad(y, leaf, dy.to(DEV))
    # operator by operator, on what the one before gave
    h = dgprf.linear(*leaf[:3], "gelu", dropout=0.2, seed=8, sub=0).detach().cpu()
    r1 = Linear(x, w1, b1, "gelu", None, int(0.2 * 65536 + 0.5), 8, 0)
    check(h, r1.y, r1.y_tol, "h")
    thr = int(0.1 * 65536 + 0.5)
    dy2 = dgprf.dropout(dy.to(DEV), 0.1, seed=8, sub=1 << 33).cpu()
    r2 = Linear(h, w2, b2, "none", x, thr, 8, 1 << 32, dy2)
    y2 = dgprf.linear(h.to(DEV), leaf[3].detach(), leaf[4].detach(), residual=leaf[0].detach(), dropout=0.1,
                      seed=8, sub=1 << 32)
    check(y2, r2.y, r2.y_tol, "y before the last dropout")
    assert torch.equal(y, dgprf.dropout(y2, 0.1, seed=8, sub=1 << 33))
    check(got[3], r2.dw, r2.dw_tol, "dw2")
    check(got[4], r2.db, r2.db_tol, "db2")
    hl = h.to(DEV).requires_grad_()
    dh, = torch.autograd.grad(dgprf.linear(hl, leaf[3], leaf[4], dropout=0.1, seed=8, sub=1 << 32), hl, dy2.to(DEV))
    r3 = Linear(x, w1, b1, "gelu", None, int(0.2 * 65536 + 0.5), 8, 0, dh.cpu())
    check(got[1], r3.dw, r3.dw_tol, "dw1")
    check(got[2], r3.db, r3.db_tol, "db1")
    eps = torch.finfo(t).eps
    check(got[0], r3.dx + dy2.double(), r3.dx_tol + eps * (r3.dx.abs() + dy2.double().abs()), "dx")


def test_captured_training_step():
    """Forward and backward captured once and replayed, with eager work between the replays: the
    device counter gives every replay the mask of the eager call with that number."""
    g = _gen(7)
    leaf = [v.to(DEV).requires_grad_() for v in (normal(g, 300, 64), normal(g, 64, 96, scale=0.1), normal(g, 96),
                                                 normal(g, 96, 64, scale=0.1), normal(g, 64))]
    dy = normal(g, 300, 64).to(DEV)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = _block(*leaf, step=step)
        torch.autograd.grad(y, leaf, dy)
    torch.cuda.current_stream().wait_stream(side)
    del y
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _block(*leaf, step=step)
        got = torch.autograd.grad(y, leaf, dy)
        step += 1
    step.zero_()
    for i in range(4):
        at = torch.full((1,), i, dtype=torch.int64, device=DEV)
        y2 = _block(*leaf, step=at)
        want = torch.autograd.grad(y2, leaf, dy)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, y2) and all(torch.equal(u, v) for u, v in zip(got, want)), i
        assert int(step) == i + 1


def test_capture_beside_an_eager_graph():
    """A backward pass captured while an eager graph of the same leaves lives is refused, before anything
    is enqueued; once that graph is gone, the same capture works."""
    x, w = torch.ones(4, 8, device=DEV, requires_grad=True), torch.ones(8, 16, device=DEV, requires_grad=True)
    dy = torch.ones(4, 16, device=DEV)
    for op in (lambda: dgprf.linear(x, w, activation="relu"), lambda: dgprf.dropout(dgprf.linear(x, w), 0.0),
               lambda: dgprf.linear(dgprf.dropout(x, 0.0), w),
               lambda: dgprf.dropout(dgprf.linear(x, w).detach(), 0.0, residual=dgprf.linear(x, w))):
        held = op()
        with pytest.raises(RuntimeError, match="being captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                y = op()
                torch.autograd.grad(y, (x, w), dy)
        assert torch.equal(torch.autograd.grad(held, w, dy)[0], torch.full_like(w, 4))
        del held, y
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = op()
            dx, dw = torch.autograd.grad(y, (x, w), dy)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert bool((dx == 16).all()) and bool((dw == 4).all())
        del y


def test_capture_beside_an_eager_graph_of_a_viewed_leaf():
    """The same refusal where a leaf stands behind a view, a copy or other operations, whose nodes are new
    while the leaf's is the living graph's."""
    x, w = torch.ones(2, 3, 8, device=DEV, requires_grad=True), torch.ones(8, 8, device=DEV, requires_grad=True)
    b = torch.ones(16, device=DEV, requires_grad=True)
    dy = torch.ones(2, 3, 8, device=DEV)
    x0, w0 = x.detach(), w.detach()
    for op, of in ((lambda: dgprf.linear(x, w0), x), (lambda: dgprf.linear(x0, w.t()), w),
                   (lambda: dgprf.linear(x0, w0, b[::2]), b), (lambda: dgprf.dropout(2 * x, 0.0), x),
                   (lambda: dgprf.linear(x0, w0, residual=x * x), x),
                   (lambda: dgprf.linear(dgprf.dropout(x, 0.0), w0), x)):
        held = op()
        with pytest.raises(RuntimeError, match="being captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                y = op()
                torch.autograd.grad(y, of, dy)
        want = torch.autograd.grad(held, of, dy)[0]
        del held, y
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = op()
            got, = torch.autograd.grad(y, of, dy)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        del y


def test_graphed_module():
    """Forward and backward captured apart by torch.cuda.make_graphed_callables, inputs and weights behind
    views: every replay has the eager results."""
    g = _gen(15)

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = torch.nn.Parameter(normal(g, 56, 24, scale=0.2))
            self.b = torch.nn.Parameter(normal(g, 56))

        def forward(self, x):
            return dgprf.linear(x, self.w.t(), self.b, "silu", dropout=0.2, seed=1, sub=2)

    block, sample = Block().to(DEV), normal(g, 2, 5, 24).to(DEV).requires_grad_()
    cases = []
    for _ in range(3):
        x, dy = normal(g, 2, 5, 24).to(DEV).requires_grad_(), normal(g, 2, 5, 56).to(DEV)
        y = block(x)
        cases.append((x, dy, y.detach(), torch.autograd.grad(y, (x, *block.parameters()), dy)))
        del y
    graphed = torch.cuda.make_graphed_callables(block, (sample,))
    for x, dy, y, want in cases:
        z = graphed(x)
        got = torch.autograd.grad(z, (x, *block.parameters()), dy)
        assert torch.equal(z, y) and all(torch.equal(u, v) for u, v in zip(got, want))


def test_two_graphs_and_streams():
    """Two captured calls do not share scratch, and a call on another stream is ordered there."""
    g = _gen(8)
    xs = [normal(g, 20, 2048).to(DEV) for _ in range(2)]
    w = normal(g, 2048, 512, scale=0.02).to(DEV)
    want = [dgprf.linear(x, w, activation="gelu") for x in xs]
    graphs, outs = [], []
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(dgprf.linear(x, w, activation="gelu"))
        graphs.append(gr)
    for _ in range(3):
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, gr in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                gr.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(outs, want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = dgprf.linear(xs[0], w, activation="gelu")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want[0])


def test_rows_around_are_left_alone():
    """The C entry points write the m rows of y and nothing behind them."""
    import ctypes
    m, k, n = 21, 40, 30
    x, w = torch.ones(m, k, device=DEV), torch.ones(k, n, device=DEV)
    y = torch.full((m + 2, n), 7.0, device=DEV)
    a = N.Linear(dtype=N.F32, act=0, m=m, k=k, n=n, ldx=k, ldw=n, ldr=0, x=x.data_ptr(), w=w.data_ptr(),
                 y=y.data_ptr())
    need = ctypes.c_int64()
    N.call("dgprf_linear_scratch", ctypes.byref(a), ctypes.byref(need))
    scratch = torch.empty(max(16, need.value), dtype=torch.uint8, device=DEV)
    N.call("dgprf_linear_forward", ctypes.byref(a), ctypes.c_void_p(scratch.data_ptr()), need.value,
           ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert bool((y[:m] == k).all()) and bool((y[m:] == 7).all())


def test_gradients_that_share_rows():
    """The gradient of a sum over rows is one row for all: its products and sums, an infinite element
    among them where the products have no other."""
    g = _gen(9)
    for m, act, p in ((5, "none", 0.0), (70, "none", 0.0), (200, "gelu", 0.3)):
        x, w, b = (grid(g, *s).to(DEV).requires_grad_() for s in ((m, 40), (40, 56), (56,)))
        y = dgprf.linear(x, w, b, act, dropout=p, seed=1, sub=2)
        row = grid(g, 1, 56).to(DEV)
        got = torch.autograd.grad(y, (x, w, b), row.expand(m, 56), retain_graph=True)
        want = torch.autograd.grad(y, (x, w, b), row.expand(m, 56).contiguous(), retain_graph=True)
        assert all(torch.equal(u, v) for u, v in zip(got, want))
        one = torch.autograd.grad(y.sum(), (x, w, b), retain_graph=True)
        want = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        assert all(torch.equal(u, v) for u, v in zip(one, want))
    x = torch.ones(70, 40, device=DEV)
    w = torch.ones(40, 56, device=DEV, requires_grad=True)
    row = torch.ones(1, 56, device=DEV)
    row[0, 3] = float("inf")
    dw, = torch.autograd.grad(dgprf.linear(x, w), w, row.expand(70, 56))
    assert bool(torch.isinf(dw[:, 3]).all()) and bool((dw[:, :3] == 70).all()) and bool((dw[:, 4:] == 70).all())


def test_refusals():
    x, w = torch.zeros(4, 8, device=DEV), torch.zeros(8, 16, device=DEV)
    for bad in (lambda: dgprf.linear(x, w.half()), lambda: dgprf.linear(x.double(), w.double()),
                lambda: dgprf.linear(x, w, torch.zeros(16, device=DEV).bfloat16()),
                lambda: dgprf.linear(x, w, residual=torch.zeros(4, 16, device=DEV).half()),
                lambda: dgprf.dropout(x, 0.5, residual=x.half()), lambda: dgprf.dropout(x.long(), 0.5)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: dgprf.linear(x, w[:7]), lambda: dgprf.linear(x, w[0]), lambda: dgprf.linear(x, w, x[0]),
                lambda: dgprf.linear(x, w, residual=x), lambda: dgprf.linear(x, w[:, :0]),
                lambda: dgprf.linear(x[:, :0], w[:0]), lambda: dgprf.linear(x, w.cpu()),
                lambda: dgprf.linear(x, w, activation="tanh"), lambda: dgprf.linear(x, w, dropout=1.5),
                lambda: dgprf.linear(x, w, residual=torch.zeros(1, 16, device=DEV)),
                lambda: dgprf.linear(x, w, dropout=0.5, step=torch.zeros(1, device=DEV)),
                lambda: dgprf.linear(x, w, dropout=0.5, step=torch.zeros(1, dtype=torch.int64)),
                lambda: dgprf.dropout(x, -0.1), lambda: dgprf.dropout(x, 0.5, residual=x[:2]),
                lambda: dgprf.linear(torch.zeros(2, (1 << 20) + 8, device=DEV)[:, :8].as_strided((2, 8), ((1 << 20) + 8, 1)), w)):
        with pytest.raises(ValueError):
            bad()
    # what backward needs was changed in between
    wg = w.clone().requires_grad_()
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    y = dgprf.linear(x, wg, dropout=0.5, seed=1, sub=1, step=step)
    step += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), wg)


def test_forward_mode_refused():
    """A tangent of any argument, and of the gradient that a backward pass gets, is an error."""
    import torch.autograd.forward_ad as fw
    args = [torch.ones(s, device=DEV) for s in ((4, 8), (8, 16), (16,), (4, 16))]
    for which in range(4):
        for asks in (False, True):  # another argument asks for a gradient, or none does
            with fw.dual_level():
                a = [v.clone().requires_grad_(asks) for v in args]
                a[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    dgprf.linear(*a[:3], residual=a[3])
    for op, leaf in ((lambda v: dgprf.linear(v, args[1]), (4, 8)), (lambda v: dgprf.dropout(v, 0.5), (4, 16))):
        v = torch.ones(leaf, device=DEV, requires_grad=True)
        y = op(v)
        with fw.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, v, fw.make_dual(args[3], torch.ones_like(y)))


def test_captured_masks_are_drawn_on_each_replay():
    """Captured with neither sub nor step, a call is refused; with a step every replay has a mask of its
    own, with sub alone all have the mask of sub."""
    from layers import DenseLayer
    x, w = torch.ones(16, 64, device=DEV), torch.eye(64, device=DEV)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    layer = DenseLayer(64, 64, dropout=0.5)
    layer.set_training(True)
    for op in (lambda: dgprf.dropout(x, 0.5), lambda: dgprf.linear(x, w, dropout=0.5, seed=4), lambda: layer(x)):
        op()
        with pytest.raises(RuntimeError, match="needs step"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                x + 1
                op()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, z, u = dgprf.dropout(x, 0.5, step=step), dgprf.dropout(x, 0.5, sub=9), dgprf.dropout(x, 1.0)
        step += 1
    masks = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        masks.append(y.clone())
        assert torch.equal(z, dgprf.dropout(x, 0.5, sub=9)) and not bool(u.any())
    assert not any(torch.equal(masks[i], masks[j]) for i, j in ((0, 1), (0, 2), (1, 2)))


def test_second_derivatives_refused():
    """A gradient made with create_graph carries the error, with a residual and without, so a penalty on it
    does not lose its gradient silently; the gradient itself is the ordinary one."""
    x, w = torch.ones(8, 8, device=DEV, requires_grad=True), torch.ones(8, 8, device=DEV, requires_grad=True)
    b = torch.ones(8, device=DEV, requires_grad=True)
    for op, leaf in ((lambda: dgprf.linear(x, w, b, "gelu"), x), (lambda: dgprf.linear(x, w, b), w),
                     (lambda: dgprf.linear(x, w, b, "silu"), b), (lambda: dgprf.linear(x, w, residual=x), x),
                     (lambda: dgprf.dropout(x, 0.5, seed=1, sub=2), x), (lambda: dgprf.dropout(w, 0.5, residual=x), w)):
        y = op()
        for top in (y.sum(), y.square().sum()):
            want, = torch.autograd.grad(top, leaf, retain_graph=True)
            g, = torch.autograd.grad(top, leaf, create_graph=True)
            assert g.requires_grad and torch.equal(g, want)
            with pytest.raises(RuntimeError, match="no second derivative"):
                torch.autograd.grad(g.square().sum() + leaf.sum(), leaf)
    # the residual's gradient is the incoming one, with its own derivative
    g, = torch.autograd.grad(dgprf.dropout(w, 0.5, residual=x).square().sum(), x, create_graph=True)
    assert bool((torch.autograd.grad(g.sum(), x)[0] == 2).all())


@pytest.mark.parametrize("reentrant", [False, True])
def test_activation_checkpointing(reentrant):
    """A recomputed forward pass makes the masks that are given, and the same gradients; it does not draw
    the generator's next ones."""
    from torch.utils.checkpoint import checkpoint
    g = _gen(12)
    x, w = normal(g, 40, 24).to(DEV).requires_grad_(), normal(g, 24, 56, scale=0.2).to(DEV).requires_grad_()
    dy = normal(g, 40, 56).to(DEV)

    def run(wrap, sub):
        # (a dropout at the end would not be run again: it saves nothing)
        f = lambda v: dgprf.linear(dgprf.dropout(v, 0.4, sub=sub[0]), w, activation="gelu", dropout=0.3, sub=sub[1])  # noqa: E731
        y = checkpoint(f, x, use_reentrant=reentrant) if wrap else f(x)
        x.grad = w.grad = None
        y.backward(dy)
        return y.detach(), x.grad, w.grad

    assert all(torch.equal(u, v) for u, v in zip(run(True, (5, 6)), run(False, (5, 6))))
    for sub in ((5, None), (None, 6), (None, None)):
        run(False, sub)
        with pytest.raises(RuntimeError, match="needs sub"):
            run(True, sub)
    torch.cuda.synchronize()


def test_offsets_past_32_bits():
    """65,600 rows of 32,768 elements: the last rows of a result, and gradients over all of them."""
    m, k, n, t = 65600, 16, 32768, torch.bfloat16
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    x = torch.randint(-2, 3, (m, k), generator=g, device=DEV).to(t).requires_grad_()
    w = torch.randint(-2, 3, (k, n), generator=g, device=DEV).to(t).requires_grad_()
    y = dgprf.linear(x, w, dropout=0.5, seed=3, sub=4)
    tail = slice(m - 300, m)
    part = keep_rows(m - 300, 300, n, 32768, 3, 4).to(DEV)
    want = torch.where(part, 2 * (x[tail].float() @ w.float()), torch.zeros((), device=DEV)).to(t)
    assert torch.equal(y[tail], want)
    assert torch.equal(dgprf.dropout(torch.ones_like(y), 0.5, seed=3, sub=4)[tail] != 0, part)
    # a gradient of the tail alone, so that the sums are exact
    dy = torch.zeros_like(y)
    dy[tail] = 1
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    dz = 2 * part.float()
    assert not bool(dx[: m - 300].any()) and torch.equal(dx[tail], (dz @ w.float().t().contiguous()).to(t))
    assert torch.equal(dw, (x[tail].float().t().contiguous() @ dz).to(t))


def test_most_rows():
    """As many rows as are allowed, and more groups than a launch has threads in a dimension."""
    m, t = 2 ** 31 - 512, torch.float16
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GB")
    x = torch.zeros(m, 1, dtype=t, device=DEV)
    for first in (0, 2 ** 30 - 100, m - 200):
        x[first:first + 200] = torch.arange(1, 201, dtype=t, device=DEV)[:, None]
    w = torch.full((1, 1), 2.0, dtype=t, device=DEV, requires_grad=True)
    y = dgprf.linear(x, w, residual=x)
    assert torch.equal(y.detach()[m - 200:], 3 * x[m - 200:]) and torch.equal(y.detach()[2 ** 30 - 100:2 ** 30 + 100], 3 * x[:200])
    assert not bool(y.detach()[200:2 ** 30 - 100].any()) and not bool(y.detach()[2 ** 30 + 100:m - 200].any())
    dy = torch.zeros_like(x)
    dy[m - 200:] = 0.5
    dw, = torch.autograd.grad(y, w, dy)
    assert float(dw) == float(torch.tensor(0.5 * 200 * 201 / 2).to(t))  # 10050: fp16's steps there are 8
    del x, y, dy
    rows = 2 ** 32 + 300
    y = dgprf.dropout(torch.ones(1, 1, dtype=t, device=DEV).expand(rows, 1), 0.5, seed=3, sub=4)
    for first in (0, 2 ** 30 - 100, 2 ** 32 - 100, rows - 200):
        assert torch.equal(y[first:first + 200].cpu() != 0, keep_rows(first, 200, 1, 32768, 3, 4)), first


@pytest.mark.parametrize("tname", TYPES)
@pytest.mark.parametrize("size", [(1, 2 ** 20, 16), (2, 2 ** 20, 9), (3, 2 ** 20 - 1, 8), (40, 2 ** 20, 8), (1, 8, 2 ** 20),
                                  (16, 24, 2 ** 20), (300, 3, 2 ** 20 - 1)], ids=str)
def test_widest(size, tname):
    """The longest sums and rows that are allowed: whole numbers, whose sums here stay below 2^22."""
    m, k, n = size
    t, g = TYPES[tname], _gen(m + k + n)
    x, w, b, dy = grid(g, m, k, t=t), grid(g, k, n, t=t), grid(g, n, t=t), grid(g, m, n, t=t)
    y, dx, dw, db, _ = run(x, w, b, dy=dy)
    d = lambda v: v.to(DEV).float()  # noqa: E731
    for name, got, want in (("y", y, d(x) @ d(w) + d(b)), ("dx", dx, d(dy) @ d(w).t().contiguous()),
                            ("dw", dw, d(x).t().contiguous() @ d(dy)), ("db", db, d(dy).sum(0))):
        assert got.dtype == t and torch.equal(got, want.to(t)), name


def test_relu_passes_a_nan_on():
    """z = NaN: the result is NaN, and the gradient goes through as for z > 0."""
    for t in TYPES.values():
        x, w = torch.ones(6, 8, dtype=t, device=DEV), torch.ones(8, 16, dtype=t, device=DEV)
        x[2, 3] = float("nan")
        x.requires_grad_()
        y = dgprf.linear(x, w, activation="relu")
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert bool(torch.isnan(y[2]).all()) and bool((dx == 16).all())


def test_gradient_of_rows_far_apart():
    x, w = torch.ones(3, 8, device=DEV, requires_grad=True), torch.ones(8, 16, device=DEV, requires_grad=True)
    dy = torch.ones(3, (1 << 20) + 16, device=DEV)[:, :16]
    dx, dw = torch.autograd.grad(dgprf.linear(x, w), (x, w), dy)
    assert bool((dx == 16).all()) and bool((dw == 3).all())


def keep_rows(first, rows, n, thr, seed, sub):
    """keep_mask's rows first .. first + rows - 1 (groups numbered from row 0)."""
    from oracle import rng
    groups = -(-n // 8)
    ctr = np.zeros((rows * groups, 4), dtype=np.uint64)
    q = np.arange(first * groups, (first + rows) * groups, dtype=np.uint64)
    ctr[:, 0], ctr[:, 1], ctr[:, 2] = q & np.uint64(0xFFFFFFFF), sub & 0xFFFFFFFF, sub >> 32
    ctr[:, 3] = (q >> np.uint64(32)) + np.uint64(8 << 24)
    h = np.ascontiguousarray(rng.philox4x32_10(ctr, (seed & 0xFFFFFFFF, seed >> 32))).view(np.uint16)
    return torch.from_numpy(np.ascontiguousarray(h.reshape(rows, groups * 8)[:, :n] >= thr))


def test_layers():
    """DenseLayer / DropoutLayer: the functions' results and gradients, inside a stack with the
    random-feature layers, and an optimizer's step by its formula."""
    from experiments.optimizers import Adam
    from kernels import RBFKernel
    from layers import DenseLayer, DropoutLayer, GPLayer, RBFLayer
    from utils import BNN_from_list
    dgprf.set_seed(5)
    up, down, drop = DenseLayer(6, 40, "silu", dropout=0.2), DenseLayer(40, 6, bias=False), DropoutLayer(0.5)
    assert [tuple(v.shape) for v in up.trainable_variables] == [(6, 40), (40,)]
    assert len(down.trainable_variables) == 1 and drop.trainable_variables == ()
    X = np.random.default_rng(0).standard_normal((50, 6))
    x = torch.as_tensor(X, dtype=torch.float32).to(DEV)
    assert torch.equal(up(X), dgprf.linear(x, up.W, up.b, "silu")) and drop(x) is x
    up.set_training(True)
    drop.set_training(True)
    h = up(X, seed=1, sub=2)
    assert torch.equal(h, dgprf.linear(x, up.W, up.b, "silu", dropout=0.2, seed=1, sub=2))
    y = drop(down(h, residual=x), seed=1, sub=3)
    variables = up.trainable_variables + down.trainable_variables
    grads = torch.autograd.grad(y.square().sum(), variables)
    y2 = dgprf.dropout(dgprf.linear(h.detach(), down.W, residual=x), 0.5, seed=1, sub=3)
    dw, = torch.autograd.grad(y2.square().sum(), down.W)
    assert torch.equal(grads[2], dw)
    before = [v.detach().clone() for v in variables]
    Adam(learning_rate=0.01).apply_gradients(zip(grads, variables))
    for v, b, gr in zip(variables, before, grads):  # the first step: m / sqrt(v) is the gradient's sign
        assert torch.allclose(v.detach(), b - 0.01 * gr / (gr.abs() + 1e-7 / 0.001 ** 0.5), rtol=1e-5, atol=2e-7)
    net = BNN_from_list([DenseLayer(6, 16, "gelu"), DenseLayer(16, 3), RBFLayer(RBFKernel(3, is_ard=True), 20),
                         GPLayer(40, 2)])
    assert net(X).shape == (50, 2) and bool(torch.isfinite(net(X)).all())
    half = DenseLayer(6, 8, dtype=torch.bfloat16)
    assert half(X).dtype == torch.bfloat16
    with pytest.raises(ValueError):
        half(X[:, :5])
