"""The vocabulary head's cross entropy against fp64.

Bounds, per element (u = 2^-24: the most an fp32 rounding is off relative to the value; r: the
storage type's, u or 2^-8 for bf16):
- a logit, a sum of D products in fp32, is off by dz <= (D + 2) u sum|x w| + the products' own
  error: none for bf16 (exact in fp32); for fp32, whose operands go in as two fp16 halves a + b,
  scaled so that the largest value is below 2^15: |x - a| <= 2^-11 |x|, |x - a - b| <= 2^-22 |x|, so the
  two remainders and b b', which are left out, are at most 3 * 2^-22 = 12 u of a product; and where a half
  is below fp16's normal range its error is 2^-25 of a unit, 2^-39 of the scaled maximum's 2^14,
  for either operand (two halves: 2^-38), against the other one's value;
- a sum of exponentials of logits: each term relative to itself by dz + 8 u (its argument's
  rounding, the exponential's last places; |arg| exp(arg) <= 0.4 for the argument's scale) and
  the adding by the depth of the sums, at most 128 in a block, then the blocks in turn
  (vocab / 32 of them in 64 or more lanes) and a tree: k = 160 + vocab / 2048;
- so the loss is off by 2 max dz + (k + 8) u + 4 u (|m| + |l| + |loss|);
- a probability p by p (2 max dz + (k + 16) u + 2 u (|z - m| + |l|)), G = w (p - [label]) by that
  and, for bf16, one rounding;
- dx and dw: those errors through |w| and |x|, the fp32 sums ((n + 8) u of the terms'
  magnitude), and one rounding to storage.
"""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import cgadimpl_amd as agk  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
R = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
BF, F = torch.bfloat16, torch.float32


def products(a, b, dt):
    """The error of a sum of products a @ b in fp32 (without the sum's own)."""
    a, b = a.abs(), b.abs()
    if dt == BF:
        return 0.0
    low = 2.0 ** -38 * (a.max() * b.sum(0, keepdim=True) + a.sum(1, keepdim=True) * b.max())
    return 12 * U * (a @ b) + low


def reference(x, w, labels, dloss, dw_dtype=None):
    """((loss, dx, dw), bounds) in fp64; dloss None: the loss alone."""
    dt = x.dtype
    D, V, N = x.shape[1], w.shape[0], x.shape[0]
    keep = labels >= 0
    x, w = x.double(), w.double()
    if dloss is not None:
        keep_g = keep & (dloss != 0)
    x0 = torch.where(keep[:, None], x, 0.0)
    z = x0 @ w.T
    dz = (D + 2) * U * (x0.abs() @ w.abs().T) + products(x0, w.T, dt)
    m = z.amax(1, keepdim=True)
    l = torch.log(torch.exp(z - m).sum(1, keepdim=True))
    at = labels.clamp(min=0)[:, None]
    loss = ((m + l) - z.gather(1, at))[:, 0]
    k = 160 + V / 2048
    worst = dz.amax(1)
    eloss = 2 * worst + (k + 8) * U + 4 * U * (m.abs()[:, 0] + l.abs()[:, 0] + loss.abs())
    loss, eloss = torch.where(keep, loss, 0.0), torch.where(keep, eloss, 0.0)
    if dloss is None:
        return (loss,), (eloss,)
    wt = torch.where(keep_g, dloss.double(), 0.0)[:, None]
    x1 = torch.where(keep_g[:, None], x0, 0.0)
    p = torch.exp(z - m - l)
    one = torch.zeros_like(p).scatter_(1, at, 1.0)
    G = wt * (p - one)
    rel = 2 * worst[:, None] + (k + 16) * U + 2 * U * ((z - m).abs() + l.abs())
    eG = wt.abs() * p * rel + 4 * U * G.abs() + (2.0 ** -8 * G.abs() if dt == BF else 0.0)
    dx, dw = G @ w, G.T @ x1
    pieces = 8
    edx = eG @ w.abs() + (V + pieces + 8) * U * (G.abs() @ w.abs()) + products(G, w, dt) + \
        (R[dt] + 2 * U) * dx.abs()
    edw = eG.T @ x1.abs() + (N + 8) * U * (G.abs().T @ x1.abs()) + products(G.T, x1, dt) + \
        (R[dw_dtype or F] + 2 * U) * dw.abs()
    return (loss, dx, dw), (eloss, edx, edw)


def check(got, ref, bound, what):
    d = (got.double() - ref).abs()
    bad = ~(d <= bound + 1e-35)
    assert not bad.any(), (what, int(bad.sum()), float((d / (bound + 1e-35)).max()))


def inputs(N, V, D, dtype, seed=0, ignored=0.25, equal=False):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + N * 101 + V * 13 + D)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, w = rn(N, D).to(dtype), (rn(V, D) * (2.0 / D ** 0.5)).to(dtype)
    labels = torch.randint(V, (N,), generator=gen, device="cuda")
    labels = torch.where(torch.rand(N, generator=gen, device="cuda") < ignored, -100, labels)
    dloss = torch.full((N,), 1.0 / N, device="cuda") if equal else rn(N)
    return x, w, labels, dloss


SIZES = [  # tokens, vocabulary, width
    (1, 1, 8), (1, 1000, 64), (2, 31, 16), (7, 257, 64), (8, 64, 40), (16, 5003, 128), (33, 96, 24),
    (64, 4096, 192), (65, 8191, 64), (129, 1003, 72), (130, 63, 8), (300, 4099, 136), (520, 2500, 56),
    (1031, 511, 128), (2049, 3001, 64),
]


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("N,V,D", SIZES)
def test_against_fp64(cuda, dtype, N, V, D):
    if dtype == F:
        D -= 3 if D > 8 else 5  # any width
    x, w, labels, dloss = inputs(N, V, D, dtype)
    loss, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    assert loss.shape == (N,) and stats.shape == (N, 2) and loss.dtype == F
    for dw_dtype in ([F, BF] if dtype == BF else [F]):
        dx, dw = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, dw_dtype=dw_dtype)
        assert dx.dtype == dtype and dw.dtype == dw_dtype
        ref, bound = reference(x, w, labels, dloss, dw_dtype)
        for got, want, tol, what in zip((loss, dx, dw), ref, bound, ("loss", "dx", "dw")):
            check(got, want, tol, (what, N, V, D))


@pytest.mark.parametrize("N,V,D", [(2048, 20011, 64), (4099, 9000, 72), (1024, 40000, 128)])
def test_large_tiles(cuda, N, V, D):
    """Enough tiles for the 256 x 256 kernel in every product, with and without edges."""
    x, w, labels, dloss = inputs(N, V, D, BF, equal=True)
    loss, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    dx, dw = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, dw_dtype=BF)
    ref, bound = reference(x, w, labels, dloss, BF)
    for got, want, tol, what in zip((loss, dx, dw), ref, bound, ("loss", "dx", "dw")):
        check(got, want, tol, what)
    again = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, dw_dtype=BF)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
    l2, s2 = agk.linear_cross_entropy_fwd(x, w, labels)
    assert torch.equal(l2, loss) and torch.equal(s2, stats)


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("N,V,D", [(5, 3001, 64), (300, 2500, 72), (1031, 1100, 128)])
def test_pieces(cuda, dtype, N, V, D):
    """Pieces of the vocabulary: dw has the same bits, dx is summed in another order."""
    x, w, labels, dloss = inputs(N, V, D, dtype)
    _, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    whole = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss)
    ref, bound = reference(x, w, labels, dloss)
    for piece in (1, 256, 300, 1024, V, 10 * V):
        dx, dw = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, piece=piece)
        check(dx, ref[1], bound[1], ("dx", piece))
        check(dw, ref[2], bound[2], ("dw", piece))
        if piece >= V:
            assert torch.equal(dx, whole[0]) and torch.equal(dw, whole[1])


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("N,V,D", [(9, 700, 64), (300, 1100, 40)])
def test_outputs_and_accumulation(cuda, dtype, N, V, D):
    x, w, labels, dloss = inputs(N, V, D, dtype)
    _, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    dx, dw = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss)
    a, b = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, want_dw=False)
    assert b is None and torch.equal(a, dx)
    a, b = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, want_dx=False)
    assert a is None and torch.equal(b, dw)
    assert agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, want_dx=False,
                                        want_dw=False) == (None, None)
    ref, bound = reference(x, w, labels, dloss)
    for piece in (0, 256):
        for bits in (1, 2, 3):
            odx, odw = torch.randn_like(x), torch.randn_like(dw)
            p, q = odx.clone(), odw.clone()
            agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, dx=p, dw=q, accumulate=bits,
                                         piece=piece)
            want = odx.double() * (bits & 1) + ref[1]
            check(p, want, bound[1] + (2 * R[dtype] + 8 * U) * (want.abs() + odx.double().abs()),
                  "dx")
            want = odw.double() * (bits >> 1) + ref[2]
            check(q, want, bound[2] + 4 * U * (want.abs() + odw.double().abs()), "dw")
    # leading axes
    if N % 3 == 0:
        l3, s3 = agk.linear_cross_entropy_fwd(x.view(3, N // 3, D), w, labels.view(3, -1))
        assert l3.shape == (3, N // 3) and s3.shape == (3, N // 3, 2)
        assert torch.equal(s3.view(N, 2), stats)


@pytest.mark.parametrize("dtype", [F, BF])
def test_tokens_left_out(cuda, dtype):
    """Negative labels and zero weights: no loss, no gradient, whatever x holds there."""
    N, V, D = 70, 999, 64
    x, w, labels, dloss = inputs(N, V, D, dtype, ignored=0.0)
    labels[5:30] = -1
    labels[40] = -(1 << 62)
    dloss[50] = 0.0
    clean_loss, clean_stats = agk.linear_cross_entropy_fwd(x, w, labels)
    clean = agk.linear_cross_entropy_bwd(x, w, labels, clean_stats, dloss)
    ref, bound = reference(x, w, labels, dloss)
    for got, want, tol, what in zip((clean_loss,) + clean, ref, bound, ("loss", "dx", "dw")):
        check(got, want, tol, what)
    x[6], x[7], x[40], x[50] = float("nan"), float("inf"), float("-inf"), float("nan")
    dloss[8] = float("nan")
    loss, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    dx, dw = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss)
    assert (loss[5:30] == 0).all() and loss[40] == 0 and loss[50].isnan()
    assert (dx[5:30] == 0).all() and (dx[40] == 0).all() and (dx[50] == 0).all()
    assert torch.equal(dx, clean[0]) and torch.equal(dw, clean[1])
    # all of them
    labels[:] = -100
    loss, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    dx, dw = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss)
    assert (loss == 0).all() and (dx == 0).all() and (dw == 0).all()
    dx, dw = torch.ones_like(x), torch.ones(V, D, device="cuda")
    agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, dx=dx, dw=dw, accumulate=True)
    assert (dx == 1).all() and (dw == 1).all()


@pytest.mark.parametrize("dtype", [F, BF])
def test_labels_past_the_vocabulary_and_special_values(cuda, dtype):
    N, V, D = 33, 300, 64
    x, w, labels, dloss = inputs(N, V, D, dtype, ignored=0.0)
    labels[0], labels[1] = 0, V - 1
    good = agk.linear_cross_entropy_fwd(x, w, labels)
    gx, _ = agk.linear_cross_entropy_bwd(x, w, labels, good[1], dloss)
    labels[4], labels[20] = V, 1 << 62
    loss, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    assert loss[4].isnan() and loss[20].isnan()
    keep = torch.ones(N, dtype=torch.bool, device="cuda")
    keep[4] = keep[20] = False
    assert torch.equal(loss[keep], good[0][keep])
    dx, dw = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss)
    assert dx[4].isnan().all() and dx[20].isnan().all() and torch.equal(dx[keep], gx[keep])
    assert dw.isnan().all()
    # logits hundreds apart: nothing overflows, and a NaN stays in its row's loss and dx
    x, w, labels, dloss = inputs(N, V, D, dtype, ignored=0.0)
    x *= 300
    ref, bound = reference(x, w, labels, dloss)
    loss, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    dx, dw = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss)
    for got, want, tol, what in zip((loss, dx, dw), ref, bound, ("loss", "dx", "dw")):
        check(got, want, tol, what)
    x[9, 3] = float("nan")
    l2, _ = agk.linear_cross_entropy_fwd(x, w, labels)
    assert l2[9].isnan() and torch.equal(l2[:9], loss[:9]) and torch.equal(l2[10:], loss[10:])
    # equal weights of any size: the same dx up to the factor
    dloss[:] = 1.0
    a, _ = agk.linear_cross_entropy_bwd(x[:9], w, labels[:9], stats[:9], dloss[:9])
    dloss[:] = 2.0 ** -20
    b, _ = agk.linear_cross_entropy_bwd(x[:9], w, labels[:9], stats[:9], dloss[:9])
    assert torch.equal(a.float() * 2.0 ** -20, b.float())


def test_leading_dimensions(cuda):
    """x and w as columns of wider matrices (the C ABI's ldx and ldw)."""
    N, V, D, LX, LW = 37, 500, 64, 80, 96
    for dtype, code in ((BF, agk.AGK_BF16), (F, agk.AGK_F32)):
        x, w, labels, dloss = inputs(N, V, D, dtype)
        xw, ww = torch.full((N, LX), 9.0, device="cuda", dtype=dtype), \
            torch.full((V, LW), 9.0, device="cuda", dtype=dtype)
        xw[:, :D], ww[:, :D] = x, w
        loss, stats = agk.linear_cross_entropy_fwd(x, w, labels)
        dx, dw = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss)
        lib = agk.lib()
        need = max(lib.agk_linear_xent_fwd_workspace_bytes(N, V, D, code),
                   lib.agk_linear_xent_bwd_workspace_bytes(N, V, D, code, 256))
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        l2, s2 = torch.empty_like(loss), torch.empty_like(stats)
        dx2, dw2 = torch.empty_like(dx), torch.empty_like(dw)
        st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.agk_linear_xent_fwd(xw.data_ptr(), LX, ww.data_ptr(), LW, labels.data_ptr(),
                                       l2.data_ptr(), s2.data_ptr(), ws.data_ptr(), need, N, V, D,
                                       code, st) == 0
        assert lib.agk_linear_xent_bwd(xw.data_ptr(), LX, ww.data_ptr(), LW, labels.data_ptr(),
                                       s2.data_ptr(), dloss.data_ptr(), dx2.data_ptr(),
                                       dw2.data_ptr(), agk.AGK_F32, ws.data_ptr(), need, N, V, D,
                                       256, code, 0, st) == 0
        torch.cuda.synchronize()
        assert torch.equal(l2, loss) and torch.equal(s2, stats) and torch.equal(dw2, dw)
        ref, bound = reference(x, w, labels, dloss)
        check(dx2, ref[1], bound[1], "dx")


def test_empty_and_refusals(cuda):
    x, w = torch.empty(0, 64, device="cuda", dtype=BF), torch.ones(10, 64, device="cuda", dtype=BF)
    labels = torch.empty(0, dtype=torch.int64, device="cuda")
    loss, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    dx, dw = agk.linear_cross_entropy_bwd(x, w, labels, stats, loss)
    assert loss.numel() == 0 and (dw == 0).all() and dx.shape == x.shape
    dw = torch.ones(10, 64, device="cuda", dtype=BF)
    agk.linear_cross_entropy_bwd(x, w, labels, stats, loss, dw=dw, accumulate=True)
    assert (dw == 1).all()
    agk.linear_cross_entropy_bwd(x, w, labels, stats, loss, dw=dw)
    assert (dw == 0).all()

    x, w, labels, dloss = inputs(4, 10, 64, BF)
    _, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    with pytest.raises(TypeError):
        agk.linear_cross_entropy_fwd(x, w.float(), labels)
    with pytest.raises(TypeError):
        agk.linear_cross_entropy_fwd(x, w, labels.int())
    with pytest.raises(ValueError):
        agk.linear_cross_entropy_fwd(x, w, labels[:3])
    with pytest.raises(ValueError):
        agk.linear_cross_entropy_fwd(x[:, :56], w, labels)
    with pytest.raises(ValueError):
        agk.linear_cross_entropy_fwd(x.t().contiguous().t(), w, labels)
    with pytest.raises(agk.AgkError):
        agk.linear_cross_entropy_fwd(x[:, :60].contiguous(), w[:, :60].contiguous(), labels)
    with pytest.raises(TypeError):
        agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss.double())
    with pytest.raises(ValueError):
        agk.linear_cross_entropy_bwd(x, w, labels, stats[:3], dloss)
    with pytest.raises(agk.AgkError):
        agk.linear_cross_entropy_bwd(x.float(), w.float(), labels, stats, dloss, dw_dtype=BF)
    with pytest.raises(agk.AgkError):
        agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss,
                                     workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("dtype", [F, BF])
def test_graph_and_streams(cuda, dtype):
    N, V, D = 300, 1500, 64
    x, w, labels, dloss = inputs(N, V, D, dtype)

    def step():
        loss, stats = agk.linear_cross_entropy_fwd(x, w, labels)
        return (loss,) + agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, piece=512)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        nx, nw, nl, nd = inputs(N, V, D, dtype, seed=seed + 1)
        for t, n in ((x, nx), (w, nw), (labels, nl), (dloss, nd)):
            t.copy_(n)
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
    """Central differences of sum(dloss * loss) in fp64 along random directions of x and w."""
    x, w, labels, dloss = inputs(12, 150, 24, F)
    _, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    grads = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss)
    keep = labels >= 0

    def f(x, w):
        logp = torch.log_softmax(x @ w.T, 1)
        return -(dloss.double() * logp.gather(1, labels.clamp(min=0)[:, None])[:, 0])[keep].sum()
    args = [x.double(), w.double()]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    for i in range(2):
        d = torch.randn(args[i].shape, generator=gen, device="cuda").double()
        h = 1e-5  # the differences' own error: h^2 times third derivatives of some hundreds
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + h * d, args[i] - h * d
        want = (f(*hi) - f(*lo)) / (2 * h)
        terms = grads[i].double() * d
        assert abs(terms.sum() - want) <= 1e-5 * terms.abs().sum(), (i, terms.sum(), want)


@pytest.mark.parametrize("N", [70, 170])
def test_left_out_rows_do_not_set_the_scale(cuda, N):
    # the fp32 operands are scaled by their matrix's largest value: rows without a loss have no part
    x, w, labels, dloss = inputs(N, 300, 33, F, seed=21)
    labels[::7] = -1
    dirty = torch.where((labels < 0)[:, None], 1e30, x)
    out = agk.linear_cross_entropy_fwd(dirty, w, labels)
    (loss,), (bound,) = reference(x, w, labels, None)
    check(out[0], loss, bound, "loss")
    clean = agk.linear_cross_entropy_fwd(x, w, labels)
    keep = labels >= 0
    assert torch.equal(out[0], clean[0]) and torch.equal(out[1][keep], clean[1][keep])
    for a, b in zip(agk.linear_cross_entropy_bwd(dirty, w, labels, out[1], dloss),
                    agk.linear_cross_entropy_bwd(x, w, labels, clean[1], dloss)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("N", [40, 150])
@pytest.mark.parametrize("ex,ew", [(0, -101), (0, -99), (-101, 0), (-60, -60), (30, -101), (60, -60)])
def test_scales_of_any_size(cuda, N, ex, ew):
    x, w, labels, dloss = inputs(N, 200, 29, F, seed=22)
    x, w = x * 2.0 ** ex, w * 2.0 ** ew
    loss, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    dx, dw = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss)
    ref, bound = reference(x, w, labels, dloss)
    for got, want, tol, what in zip((loss, dx, dw), ref, bound, ("loss", "dx", "dw")):
        check(got, want, tol, what)
        assert got.abs().max() > 0


@pytest.mark.parametrize("N,V,D,pitch", [
    (1, 12289, 64, 64), (33, 13001, 192, 192), (64, 33001, 128, 128), (20, 32900, 64, 64),
    (7, 20011, 200, 256), (64, 33003, 72, 128), (65, 25000, 192, 192), (100, 30011, 136, 192),
    (3, 33001, 72, 72), (20, 20011, 40, 64), (64, 40003, 8, 64)])
def test_few_tokens_of_many_words(cuda, N, V, D, pitch):
    # one column of tiles whose workgroups start their walks of K at different tiles
    x, w, labels, dloss = inputs(N, V, D, BF, seed=23)
    wide = torch.full((V, pitch), float("nan"), device="cuda", dtype=BF)
    wide[:, :D] = w
    lib = agk.lib()
    P = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    loss, stats = torch.empty(N, device="cuda"), torch.empty(N, 2, device="cuda")
    dx, dw = torch.empty_like(x), torch.empty(V, D, device="cuda")
    nf = lib.agk_linear_xent_fwd_workspace_bytes(N, V, D, agk.AGK_BF16)
    nb = lib.agk_linear_xent_bwd_workspace_bytes(N, V, D, agk.AGK_BF16, 0)
    ws = torch.empty(max(nf, nb), dtype=torch.uint8, device="cuda")
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.agk_linear_xent_fwd(P(x), D, P(wide), pitch, P(labels), P(loss), P(stats), P(ws), nf,
                                   N, V, D, agk.AGK_BF16, st) == 0
    assert lib.agk_linear_xent_bwd(P(x), D, P(wide), pitch, P(labels), P(stats), P(dloss), P(dx),
                                   P(dw), agk.AGK_F32, P(ws), nb, N, V, D, 0, agk.AGK_BF16, 0,
                                   st) == 0
    ref, bound = reference(x, w, labels, dloss)
    for got, want, tol, what in zip((loss, dx, dw), ref, bound, ("loss", "dx", "dw")):
        check(got, want, tol, (what, N, V, D))


def test_rows_of_unlike_sizes(cuda):
    # fp32 forward: each row and each word has a scale of its own, so large ones cost others nothing
    x, w, labels, _ = inputs(150, 900, 61, F, seed=24, ignored=0.0)
    x, w = x.clone(), w.clone()
    x[::5] *= 2.0 ** -30
    w[::7] *= 2.0 ** 20
    x[:, 0] = 0.0                      # words of 2^20 meet tokens of 2^-30 in most columns
    x[1::2] *= 2.0 ** -22
    (want,), (bound,) = reference(x, w, labels, None)
    # the products' own error, by rows instead of by matrices
    a, b = x.double().abs(), w.double().abs()
    low = 2.0 ** -38 * (a.amax(1, keepdim=True) * b.sum(1) + a.sum(1, keepdim=True) * b.amax(1))
    z = a @ b.T
    dz = ((x.shape[1] + 2 + 12) * U * z + low).amax(1)
    zz = x.double() @ w.double().T
    m = zz.amax(1)
    l = torch.logsumexp(zz, 1) - m
    tight = 2 * dz + (168 + 900 / 2048) * U + 4 * U * (m.abs() + l.abs() + want.abs())
    got = agk.linear_cross_entropy_fwd(x, w, labels)[0]
    check(got, want, tight, "loss")


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("N", [1, 31, 33, 128, 129])
@pytest.mark.parametrize("piece", [1, 512, 0])
def test_few_tokens_in_pieces(cuda, dtype, N, piece):
    V, D = 1700, 72 if dtype == BF else 71
    x, w, labels, dloss = inputs(N, V, D, dtype, seed=25)
    loss, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    dx0 = torch.randn(N, D, device="cuda").to(dtype)
    dw0 = torch.randn(V, D, device="cuda")
    dx, dw = dx0.clone(), dw0.clone()
    agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, dx=dx, dw=dw, accumulate=True,
                                 piece=piece)
    new = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, piece=piece)
    ref, bound = reference(x, w, labels, dloss)
    for got, added, base, want, tol, what in zip(new, (dx, dw), (dx0, dw0), ref[1:], bound[1:],
                                                 ("dx", "dw")):
        check(got, want, tol, what)
        r = R[got.dtype]
        check(added, base.double() + want, tol + r * (base.double() + want).abs() + 2 * r * tol, what)


@pytest.mark.parametrize("piece", [0, 1024])
@pytest.mark.parametrize("N", [4097, 4103, 4160])
def test_a_few_tokens_past_whole_tiles(cuda, N, piece):
    # their dx is a product of its own
    V, D = 3000, 2048
    x, w, labels, dloss = inputs(N, V, D, BF, seed=26)
    loss, stats = agk.linear_cross_entropy_fwd(x, w, labels)
    dx0 = torch.randn(N, D, device="cuda").to(BF)
    into = dx0.clone()
    dx, dw = agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, piece=piece)
    agk.linear_cross_entropy_bwd(x, w, labels, stats, dloss, dx=into, want_dw=False, piece=piece,
                                 accumulate=True)
    ref, bound = reference(x, w, labels, dloss)
    for got, want, tol, what in zip((loss, dx, dw), ref, bound, ("loss", "dx", "dw")):
        check(got, want, tol, what)
    total = dx0.double() + ref[1]
    check(into, total, bound[1] + 2.0 ** -8 * total.abs() + 2.0 ** -7 * bound[1], "dx added")
