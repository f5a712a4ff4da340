"""LayerNorm with weight and bias against fp64.

Bounds, per element, from the arithmetic (u = 2^-24, the most an fp32 rounding is off relative to the value;
r = the storage type's: u, or 2^-8 for bf16, counted once for each rounding to it):
- a sum of n terms in which no term passes through more than k additions is off by at
  most k u sum|terms|; rows are summed by at least 64 lanes' worth of parallel sums or in
  registers, so k = cols / 64 + 32 covers every kernel;
- xhat = (x - mean) rstd is off by E = (k + 10) u (rstd (mean|x| + |x|) + |xhat|), from the
  mean's error, the differences' roundings and rstd's;
- the rest follows term by term (below).
"""
import pytest

torch = pytest.importorskip("torch")

import cgadimpl_amd as agk  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
R = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
EPS = 1e-5


def reference(x, gamma, beta, dy, eps=EPS):
    """(y, dx, dgamma, dbeta) in fp64 and the bound of each."""
    r = R[x.dtype]
    rows, cols = x.shape
    k = cols / 64 + 32
    x, dy = x.double(), dy.double()
    g = gamma.double() if gamma is not None else torch.ones(cols, device=x.device).double()
    b = beta.double() if beta is not None else torch.zeros(cols, device=x.device).double()
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = (x - mean) * rstd
    ab = torch.abs
    E = (k + 10) * U * (rstd * (ab(x).mean(1, keepdim=True) + ab(x)) + ab(xhat))
    y = xhat * g + b
    ey = r * ab(y) + ab(g) * E + 4 * U * (ab(xhat * g) + ab(b))
    h = dy * g
    mh, mhx = h.mean(1, keepdim=True), (h * xhat).mean(1, keepdim=True)
    dx = rstd * (h - mh - xhat * mhx)
    emh = k * U * ab(h).mean(1, keepdim=True)
    emhx = k * U * ab(h * xhat).mean(1, keepdim=True) + (ab(h) * E).mean(1, keepdim=True)
    edx = r * ab(dx) + rstd * (8 * U * (ab(h) + ab(mh) + ab(xhat * mhx)) + emh + E * ab(mhx) +
                               ab(xhat) * emhx) + (k + 8) * U * ab(dx)
    # rows: at most ceil(rows / 256) terms in a lane, then the rows a workgroup holds side by side
    n = rows / 256 + min(rows, 1024) + 8
    dg, db = (dy * xhat).sum(0), dy.sum(0)
    edg = n * U * ab(dy * xhat).sum(0) + (ab(dy) * E).sum(0) + U * ab(dg)
    edb = n * U * ab(dy).sum(0) + U * ab(db)
    return (y, dx, dg, db), (ey, edx, edg, edb)


def check(got, ref, bound, what):
    d = (got.double() - ref).abs()
    bad = ~(d <= bound + 1e-300)
    assert not bad.any(), (what, int(bad.sum()), float((d / (bound + 1e-300)).max()))


def inputs(rows, cols, dtype, seed=0, mean=0.25, offset=0):
    """offset: elements by which every tensor starts off its (256-byte aligned) allocation."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + rows * 31 + cols)

    def place(t):
        t = t.to(dtype)
        buf = torch.empty(t.numel() + offset, dtype=dtype, device="cuda")
        v = buf[offset:].view(t.shape)
        v.copy_(t)
        return v
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    return (place(rn(rows, cols) + mean), place(torch.rand(cols, generator=gen, device="cuda") + 0.5),
            place(0.1 * rn(cols)), place(rn(rows, cols)))


# a column count per kernel shape of either type, its edges, and the looped kernel's
COLS = [1, 2, 3, 4, 7, 8, 9, 16, 31, 64, 100, 128, 250, 256, 512, 520, 1000, 1024, 1030, 2048, 4096,
        4097, 5120, 8192, 8195, 13824, 16384, 16388, 20001]
ROWS = [1, 5, 255, 300]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", COLS)
def test_against_fp64(cuda, dtype, cols):
    for rows in ROWS if cols <= 8195 else [1, 37]:
        x, g, b, dy = inputs(rows, cols, dtype)
        y, mean, rstd = agk.layernorm_affine_fwd(x, g, b, EPS)
        dx, dg, db = agk.layernorm_affine_bwd(x, g, mean, rstd, dy)
        assert dg.dtype == db.dtype == torch.float32 and mean.shape == rstd.shape == (rows, 1)
        ref, bound = reference(x, g, b, dy)
        for got, want, tol, what in zip((y, dx, dg, db), ref, bound, ("y", "dx", "dgamma", "dbeta")):
            check(got, want, tol, (what, rows, cols))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(70000, 24), (20000, 72), (3000, 1030), (1031, 4096), (4100, 2052)])
def test_many_rows(cuda, dtype, rows, cols):
    x, g, b, dy = inputs(rows, cols, dtype)
    y, mean, rstd = agk.layernorm_affine_fwd(x, g, b, EPS)
    dx, dg, db = agk.layernorm_affine_bwd(x, g, mean, rstd, dy)
    ref, bound = reference(x, g, b, dy)
    for got, want, tol, what in zip((y, dx, dg, db), ref, bound, ("y", "dx", "dgamma", "dbeta")):
        check(got, want, tol, what)
    again = agk.layernorm_affine_bwd(x, g, mean, rstd, dy)
    assert all(torch.equal(p, q) for p, q in zip((dx, dg, db), again))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [8, 64, 1024, 4096, 16400])
@pytest.mark.parametrize("offset", [1, 3])
def test_unaligned(cuda, dtype, cols, offset):
    x, g, b, dy = inputs(67, cols, dtype, offset=offset)
    assert x.data_ptr() % 16 != 0
    y, mean, rstd = agk.layernorm_affine_fwd(x, g, b, EPS)
    dx, dg, db = agk.layernorm_affine_bwd(x, g, mean, rstd, dy, dx=dy.clone())
    ref, bound = reference(x, g, b, dy)
    for got, want, tol, what in zip((y, dx, dg, db), ref, bound, ("y", "dx", "dgamma", "dbeta")):
        check(got, want, tol, what)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(9, 1030), (300, 72), (40, 4096), (3, 7), (5, 20001)])
def test_optional_parts_and_accumulation(cuda, dtype, rows, cols):
    x, g, b, dy = inputs(rows, cols, dtype)
    _, mean, rstd = agk.layernorm_affine_fwd(x, g, b, EPS)
    dx, dg, db = agk.layernorm_affine_bwd(x, g, mean, rstd, dy)
    # each output alone has the same bits
    for want in ((True, False, False), (False, True, False), (False, False, True)):
        got = agk.layernorm_affine_bwd(x, g, mean, rstd, dy, want_dx=want[0], want_dgamma=want[1],
                                       want_dbeta=want[2])
        for have, full, w in zip(got, (dx, dg, db), want):
            assert (have is not None) == w and (not w or torch.equal(have, full))
    # added into what was there, each by its own bit; the gradient is rounded... in fp32 first
    odx, odg, odb = torch.randn_like(x), torch.randn_like(dg), torch.randn_like(db)
    ref, bound = reference(x, g, b, dy)
    for bits in (1, 2, 4, 7):
        p, q, s = odx.clone(), odg.clone(), odb.clone()
        agk.layernorm_affine_bwd(x, g, mean, rstd, dy, dx=p, dgamma=q, dbeta=s, accumulate=bits)
        if bits & 1:
            want = odx.double() + ref[1]
            check(p, want, bound[1] + 2 * R[dtype] * want.abs() + U * ref[1].abs(), "dx")
        else:
            assert torch.equal(p, dx)
        assert torch.equal(q, odg + dg if bits & 2 else dg)
        assert torch.equal(s, odb + db if bits & 4 else db)
    # without weight, bias or either
    for gamma, beta in ((None, b), (g, None), (None, None)):
        y, m2, r2 = agk.layernorm_affine_fwd(x, gamma, beta, EPS)
        got = agk.layernorm_affine_bwd(x, gamma, m2, r2, dy)
        ref2, bound2 = reference(x, gamma, beta, dy)
        for have, want, tol in zip((y,) + got, ref2, bound2):
            check(have, want, tol, "optional")
    y0, _, _ = agk.layernorm_fwd(x, EPS)
    assert torch.equal(agk.layernorm_affine_fwd(x, None, None, EPS)[0], y0)
    # in place: y over x, dx over dy
    y, _, _ = agk.layernorm_affine_fwd(x, g, b, EPS)
    xc, dyc = x.clone(), dy.clone()
    agk.layernorm_affine_fwd(xc, g, b, EPS, y=xc)
    assert torch.equal(xc, y)
    agk.layernorm_affine_bwd(x, g, mean, rstd, dyc, dx=dyc)
    assert torch.equal(dyc, dx)


def test_special_rows(cuda):
    """Constant rows (var = 0: xhat = 0, y = beta), a large common offset, and a NaN or an
    infinity in one row, which stays in that row's y and dx."""
    for dtype in (torch.float32, torch.bfloat16):
        x, g, b, dy = inputs(20, 1030, dtype)
        x[3] = 2.5
        x[4] = 0.0
        x[5] += 300.0
        clean = x.clone()
        y, mean, rstd = agk.layernorm_affine_fwd(x, g, b, EPS)
        dx, dg, db = agk.layernorm_affine_bwd(x, g, mean, rstd, dy)
        ref, bound = reference(x, g, b, dy)
        for got, want, tol, what in zip((y, dx, dg, db), ref, bound, ("y", "dx", "dg", "db")):
            check(got, want, tol, what)
        assert torch.equal(y[3], b) and torch.equal(y[4], b)
        x[7, 11] = float("nan")
        x[9, 1029] = float("inf")
        y2, m2, r2 = agk.layernorm_affine_fwd(x, g, b, EPS)
        dx2, dg2, db2 = agk.layernorm_affine_bwd(x, g, m2, r2, dy)
        keep = torch.tensor([i not in (7, 9) for i in range(20)], device="cuda")
        assert torch.equal(y2[keep], y[keep]) and torch.equal(dx2[keep], dx[keep])
        assert y2[7].isnan().all() and dx2[7].isnan().all() and y2[9, 1029].isnan()
        assert torch.equal(db2, db)
        assert dg2.isnan().all() and not clean.isnan().any()


def test_empty_calls(cuda):
    x = torch.empty(0, 40, device="cuda")
    g = torch.ones(40, device="cuda")
    y, mean, rstd = agk.layernorm_affine_fwd(x, g, g)
    dg, db = torch.full((40,), 3.0, device="cuda"), torch.full((40,), 4.0, device="cuda")
    agk.layernorm_affine_bwd(x, g, mean, rstd, x, dgamma=dg, dbeta=db, accumulate=2)
    assert y.shape == (0, 40) and (dg == 3).all() and (db == 0).all()


def test_refusals(cuda):
    x, g, b, dy = inputs(6, 64, torch.float32)
    _, mean, rstd = agk.layernorm_affine_fwd(x, g, b)
    with pytest.raises(TypeError):
        agk.layernorm_affine_fwd(x, g.bfloat16(), b)
    with pytest.raises(ValueError):
        agk.layernorm_affine_fwd(x, g[:63], b)
    with pytest.raises(ValueError):
        agk.layernorm_affine_fwd(x.t(), None, None)
    with pytest.raises(TypeError):
        agk.layernorm_affine_fwd(x.half(), None, None)
    with pytest.raises(ValueError):
        agk.layernorm_affine_bwd(x, g, mean[:5], rstd, dy)
    with pytest.raises(TypeError):
        agk.layernorm_affine_bwd(x, g, mean, rstd, dy.bfloat16())
    with pytest.raises(agk.AgkError):
        agk.layernorm_affine_bwd(x, g, mean, rstd, dy,
                                 workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))


def test_graph_and_streams(cuda):
    """Captured and replayed with eager calls of the same tensors between, and on a side stream."""
    x, g, b, dy = inputs(300, 1030, torch.bfloat16)

    def step():
        y, mean, rstd = agk.layernorm_affine_fwd(x, g, b)
        return (y,) + agk.layernorm_affine_bwd(x, g, mean, rstd, dy)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        nx, _, _, ndy = inputs(300, 1030, torch.bfloat16, seed=seed + 1)
        x.copy_(nx)
        dy.copy_(ndy)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_gradients_against_differences(cuda):
    """Central differences of sum(dy * y) in fp64 along random directions of x, gamma, beta."""
    x, g, b, dy = inputs(6, 72, torch.float32)
    _, mean, rstd = agk.layernorm_affine_fwd(x, g, b)
    dx, dg, db = agk.layernorm_affine_bwd(x, g, mean, rstd, dy)

    def f(x, g, b):
        m = x.mean(1, keepdim=True)
        v = ((x - m) ** 2).mean(1, keepdim=True)
        return (dy.double() * ((x - m) / torch.sqrt(v + EPS) * g + b)).sum()
    args = [t.double() for t in (x, g, b)]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    for i, grad in enumerate((dx, dg, db)):
        d = torch.randn(args[i].shape, generator=gen, device="cuda").double()
        h = 1e-4  # error of order h^2 times third derivatives of size 1: 1e-8
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + h * d, args[i] - h * d
        want = (f(*hi) - f(*lo)) / (2 * h)
        got = (grad.double() * d).sum()
        # 1e-6 of the terms' magnitude: 32 u and the differences' own error
        assert abs(got - want) <= 1e-6 * (grad.double() * d).abs().sum(), (i, got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(700, 16384), (600, 9000), (530, 8193), (520, 12001),
                                       (1030, 5001), (300, 16383), (900, 6144), (257, 10240)])
def test_wide_rows_several_to_a_workgroup(cuda, dtype, rows, cols):
    x, g, b, dy = inputs(rows, cols, dtype, seed=7)
    y, mean, rstd = agk.layernorm_affine_fwd(x, g, b, EPS)
    dx, dg, db = agk.layernorm_affine_bwd(x, g, mean, rstd, dy)
    ref, bound = reference(x, g, b, dy)
    for got, want, tol, what in zip((y, dx, dg, db), ref, bound, ("y", "dx", "dgamma", "dbeta")):
        check(got, want, tol, what)
    # into what is there: each output's own addition, one rounding more
    old = [torch.randn_like(v) for v in (dx, dg, db)]
    into = [v.clone() for v in old]
    agk.layernorm_affine_bwd(x, g, mean, rstd, dy, dx=into[0], dgamma=into[1], dbeta=into[2],
                             accumulate=True)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    for got, base, want, tol, r in zip(into, old, ref[1:], bound[1:], (half, 2.0 ** -24, 2.0 ** -24)):
        total = base.double() + want
        check(got, total, tol + 2 * r * (total.abs() + tol), "accumulated")
    only = agk.layernorm_affine_bwd(x, g, mean, rstd, dy, want_dx=False)
    assert only[0] is None and torch.equal(only[1], dg) and torch.equal(only[2], db)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(300, 16383), (4100, 2052), (600, 8193), (20, 9001)])
def test_wide_rows_in_place(cuda, dtype, rows, cols):
    x, g, b, dy = inputs(rows, cols, dtype, seed=8)
    y, mean, rstd = agk.layernorm_affine_fwd(x, g, b, EPS)
    dx, dg, db = agk.layernorm_affine_bwd(x, g, mean, rstd, dy)
    xc, dyc = x.clone(), dy.clone()
    _, m2, r2 = agk.layernorm_affine_fwd(xc, g, b, EPS, y=xc)
    assert torch.equal(xc, y) and torch.equal(m2, mean) and torch.equal(r2, rstd)
    _, dg2, db2 = agk.layernorm_affine_bwd(x, g, mean, rstd, dyc, dx=dyc)
    assert torch.equal(dyc, dx) and torch.equal(dg2, dg) and torch.equal(db2, db)
