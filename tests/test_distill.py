"""Distillation from a teacher's top logits against fp64.

Bounds, per element (u = 2^-24 and r as the storage type's half step, 2^-8 for bf16):
- the teacher's p, a softmax of k entries in fp32: relative e_p = (k / 64 + 24 + 4 |t - max| / T) u;
- the student's sum of exponentials: relative (cols / 256 + 40) u with the arguments' and the
  exponentials' roundings (|arg| exp(arg) <= 0.4);
- log q by that, 4 u |z - m| / T and 4 u l; the loss by T^2 sum p (those + |log p - log q| (e_p + k / 64 u));
- q relative by the same, dz = c (q - p) by |c| (q, p times theirs) and one rounding to storage.
"""
import pytest

torch = pytest.importorskip("torch")

import cgadimpl_amd as agk  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
R = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float64: 0.0}
BF, F = torch.bfloat16, torch.float32
NEG = float("-inf")


def reference(z, index, t, dloss, T):
    dt = z.dtype
    rows, cols = z.shape
    k = index.shape[1]
    z, t = z.double() / T, t.double() / T
    has = (index >= 0) & (t > NEG)
    some = has.any(1)
    t = torch.where(has, t, NEG)
    top = torch.where(some, t.amax(1) if k else torch.zeros(rows, device=z.device).double(),
                      0.0)[:, None] if k else torch.zeros(rows, 1, device=z.device).double()
    e = torch.exp(t - top)
    p = e / torch.where(some, e.sum(1), 1.0)[:, None]
    ep = (k / 64 + 24 + 4 * torch.where(has, (t - top).abs(), 0.0)) * U
    m = z.amax(1, keepdim=True)
    l = torch.log(torch.exp(z - m).sum(1, keepdim=True))
    logq = z - m - l
    elogq = (cols / 256 + 40) * U + 4 * U * ((z - m).abs() + l.abs())
    at = index.clamp(min=0)
    lq = logq.gather(1, at)
    logp = torch.log(torch.where(p > 0, p, 1.0))
    # a p that fp32 rounds to 0 (2^-126 and below) adds nothing either way
    d = torch.where(p > 0, logp - lq, 0.0)
    loss = T * T * (p * d).sum(1)
    eloss = T * T * (p * (torch.where(p > 0, elogq.gather(1, at), 0.0) +
                          d.abs() * (ep + (k / 64 + 8) * U) + ep + 4 * U * logp.abs())).sum(1) + \
        4 * U * loss.abs() + 1e-30
    c = torch.where(some, dloss.double() * T, 0.0)[:, None]
    full = torch.zeros_like(z).scatter_add_(1, at, torch.where(has, p, 0.0))
    efull = torch.zeros_like(z).scatter_add_(1, at, torch.where(has, p * (ep + k * U), 0.0))
    q = torch.exp(logq)
    dz = c * (q - full)
    edz = c.abs() * (torch.where(q > 0, q * (elogq + 4 * U), 0.0) + efull) + \
        (R[dt] + 4 * U) * dz.abs() + 2.0 ** -126 * c.abs()
    return (loss, dz), (eloss, edz)


def check(got, ref, bound, what):
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fine), what
    d = torch.where(fine, (got.double() - ref).abs(), 0.0)
    bad = ~(d <= torch.where(fine, bound, 0.0) + 1e-35)
    assert not bad.any(), (what, int(bad.sum()), float((d / (bound + 1e-35)).nan_to_num(0).max()))


def inputs(rows, cols, k, dtype, t_dtype=F, seed=0, empty=0.2, distinct=False):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + rows * 101 + cols * 13 + k)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    z = (3 * rn(rows, cols)).to(dtype)
    index = torch.randint(cols, (rows, k), generator=gen, device="cuda")  # repeats among them
    index = torch.where(torch.rand(rows, k, generator=gen, device="cuda") < empty, -1, index)
    t = (2 * rn(rows, k) + 3).to(t_dtype)
    return z, index, t, rn(rows)


def run(z, index, t, dloss, T, **kw):
    loss, stats = agk.distill_topk_fwd(z, index, t, T)
    return loss, agk.distill_topk_bwd(z, index, t, stats, dloss, T, **kw)


SIZES = [(1, 1, 1), (1, 1000, 8), (2, 7, 3), (3, 130, 5), (33, 32001, 64), (2100, 515, 7),
         (5, 131072, 1024), (3, 300001, 70), (9, 2049, 256), (300, 4096, 20), (4, 50257, 257), (40, 8, 300)]


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("t_dtype", [F, BF])
@pytest.mark.parametrize("rows,cols,k", SIZES)
def test_against_fp64(cuda, dtype, t_dtype, rows, cols, k):
    for T in (1.0, 2.5):
        z, index, t, dloss = inputs(rows, cols, k, dtype, t_dtype)
        loss, dz = run(z, index, t, dloss, T)
        assert loss.dtype == F and dz.dtype == dtype
        ref, bound = reference(z, index, t, dloss, T)
        check(loss, ref[0], bound[0], ("loss", rows, cols, k))
        check(dz, ref[1], bound[1], ("dz", rows, cols, k))
        again = run(z, index, t, dloss, T)
        assert torch.equal(again[0], loss) and torch.equal(again[1], dz)


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("rows,cols,k", [(5, 1001, 12), (2100, 260, 4), (3, 20000, 64),
                                         (33, 1003, 200), (7, 5001, 1000), (500, 2051, 70)])
def test_in_place_and_accumulation(cuda, dtype, rows, cols, k):
    z, index, t, dloss = inputs(rows, cols, k, dtype)
    dloss[0] = 0.0
    loss, dz = run(z, index, t, dloss, 2.0)
    zc = z.clone()
    _, stats = agk.distill_topk_fwd(zc, index, t, 2.0)
    agk.distill_topk_bwd(zc, index, t, stats, dloss, 2.0, dz=zc)
    assert torch.equal(zc, dz)
    ref, bound = reference(z, index, t, dloss, 2.0)
    old = torch.randn_like(z)
    got = old.clone()
    agk.distill_topk_bwd(z, index, t, stats, dloss, 2.0, dz=got, accumulate=True)
    want = old.double() + ref[1]
    check(got, want, bound[1] + (R[dtype] + 4 * U) * (want.abs() + old.double().abs()), "dz")
    assert torch.equal(got[0], old[0]) and (dz[0] == 0).all()
    # leading axes
    z3 = z.view(1, rows, cols)
    l3, s3 = agk.distill_topk_fwd(z3, index.view(1, rows, k), t.view(1, rows, k), 2.0)
    assert l3.shape == (1, rows) and torch.equal(l3[0], loss) and s3.shape == (1, rows, 2)


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("cols", [700, 30001])
def test_empty_rows_and_special_values(cuda, dtype, cols):
    rows, k = 24, 16
    z, index, t, dloss = inputs(rows, cols, k, dtype, empty=0.0)
    index[1] = -1                          # no teacher
    index[2] = -(1 << 62)
    t[3] = NEG                             # entries without a probability
    t[4, :8] = NEG
    t[5, 0] = torch.finfo(F).min           # the lowest value: p = 0
    index[6, :] = index[6, 0]              # one column k times
    z[7, ::2] = NEG                        # columns the student excludes
    index[7] = 2 * torch.arange(k, device="cuda") + 1
    z[8, ::2] = torch.finfo(dtype).min
    index[8] = 2 * torch.arange(k, device="cuda") + 1
    z[9] = torch.finfo(dtype).min          # all at the lowest value: uniform
    z[10, 5] = NEG
    index[10, 0] = 5                       # wanted by the teacher, excluded by the student
    index[11, 0] = cols - 1
    index[11, 1] = 0
    T = 0.5
    loss, dz = run(z, index, t, dloss, T)
    ref, bound = reference(z, index, t, dloss, T)
    check(loss, ref[0], bound[0], "loss")
    check(dz, ref[1], bound[1], "dz")
    assert (loss[1:4] == 0).all() and (dz[1:4] == 0).all() and loss[10] == float("inf")
    # without a teacher, or with a zero weight, nothing of z matters
    z[1], z[2, 3], z[12, 4] = float("nan"), float("inf"), float("nan")
    dloss[12] = 0.0
    l2, d2 = run(z, index, t, dloss, T)
    assert (l2[1:4] == 0).all() and (d2[1:4] == 0).all() and (d2[12] == 0).all()
    assert l2[12].isnan()
    keep = torch.arange(rows, device="cuda") > 12
    assert torch.equal(l2[keep], loss[keep]) and torch.equal(d2[keep], dz[keep])
    # a column past the last: a NaN in its row, and only there
    index[15, 3], index[16, 0] = cols, 1 << 62
    l3, d3 = run(z, index, t, dloss, T)
    assert l3[15:17].isnan().all() and d3[15:17].isnan().all()
    assert torch.equal(l3[17:], loss[17:]) and torch.equal(d3[17:], dz[17:])
    # a NaN of the teacher: every p of the row, so the loss and the named columns of dz
    t[20, 2] = float("nan")
    l4, d4 = run(z, index, t, dloss, T)
    named = torch.zeros(cols, dtype=torch.bool, device="cuda")
    named[index[20]] = True
    assert l4[20].isnan() and torch.equal(d4[20].isnan(), named)
    assert torch.equal(l4[21:], loss[21:]) and torch.equal(d4[21:], dz[21:])


def test_k_of_zero_and_one(cuda):
    z, _, _, dloss = inputs(6, 900, 1, F)
    none_i = torch.empty(6, 0, dtype=torch.int64, device="cuda")
    none_t = torch.empty(6, 0, device="cuda")
    loss, dz = run(z, none_i, none_t, dloss, 1.0)
    assert (loss == 0).all() and (dz == 0).all()
    # one entry: the cross entropy of a label
    label = torch.randint(900, (6, 1), device="cuda")
    loss, dz = run(z, label, torch.randn(6, 1, device="cuda"), dloss, 1.0)
    want = -torch.log_softmax(z.double(), 1).gather(1, label)[:, 0]
    assert torch.all((loss.double() - want).abs() <= 100 * U * (1 + want))
    x = agk.linear_cross_entropy_fwd(z, torch.eye(900, device="cuda"), label[:, 0])
    assert torch.all((loss - x[0]).abs() <= 1e-5 * (1 + x[0]))


def test_empty_and_refusals(cuda):
    z = torch.empty(0, 50, device="cuda")
    index = torch.empty(0, 4, dtype=torch.int64, device="cuda")
    loss, dz = run(z, index, torch.empty(0, 4, device="cuda"), torch.empty(0, device="cuda"), 1.0)
    assert loss.numel() == 0 and dz.shape == (0, 50)
    z, index, t, dloss = inputs(4, 50, 3, F)
    _, stats = agk.distill_topk_fwd(z, index, t)
    with pytest.raises(TypeError):
        agk.distill_topk_fwd(z, index.int(), t)
    with pytest.raises(TypeError):
        agk.distill_topk_fwd(z.half(), index, t)
    with pytest.raises(TypeError):
        agk.distill_topk_fwd(z, index, t.half())
    with pytest.raises(ValueError):
        agk.distill_topk_fwd(z, index[:3], t)
    with pytest.raises(ValueError):
        agk.distill_topk_fwd(z, index, t[:, :2])
    with pytest.raises(ValueError):
        agk.distill_topk_fwd(z.t(), index, t)
    with pytest.raises(agk.AgkError):
        agk.distill_topk_fwd(z, index, t, 0.0)
    with pytest.raises(agk.AgkError):
        agk.distill_topk_fwd(z, index.repeat(1, 400), t.repeat(1, 400))
    with pytest.raises(ValueError):
        agk.distill_topk_bwd(z, index, t, stats, dloss[:3])
    with pytest.raises(TypeError):
        agk.distill_topk_bwd(z, index, t, stats, dloss, dz=torch.empty_like(z).bfloat16())
    wide = torch.empty(8, 50, device="cuda")
    with pytest.raises(agk.AgkError):
        agk.distill_topk_bwd(wide[:4], index, t, stats, dloss, dz=wide[2:6])


@pytest.mark.parametrize("rows,cols", [(40, 9000), (2100, 300), (4, 270001)])
def test_graph_and_streams(cuda, rows, cols):
    z, index, t, dloss = inputs(rows, cols, 12, BF)

    def step():
        return run(z, index, t, dloss, 1.5)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        for old, new in zip((z, index, t, dloss), inputs(rows, cols, 12, BF, seed=seed + 1)):
            old.copy_(new)
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


def test_gradient_against_differences(cuda):
    """Central differences of sum(dloss * loss) in fp64 along a random direction of z."""
    T = 1.7
    z, index, t, dloss = inputs(8, 60, 6, F)
    _, dz = run(z, index, t, dloss, T)

    def f(z):
        return (reference(z, index, t, dloss, T)[0][0] * dloss.double()).sum()
    d = torch.randn(z.shape, device="cuda").double()
    h = 1e-5
    want = (f(z.double() + h * d) - f(z.double() - h * d)) / (2 * h)
    terms = dz.double() * d
    assert abs(terms.sum() - want) <= 1e-5 * terms.abs().sum()


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("rows,cols,k", [(1800, 20011, 20), (3100, 1003, 70), (2500, 3, 2),
                                         (1792, 8200, 300), (1791, 8200, 9), (500, 9001, 30),
                                         (768, 9001, 30), (257, 8300, 64)])
def test_many_rows(cuda, dtype, rows, cols, k):
    z, index, t, dloss = inputs(rows, cols, k, dtype, seed=5)
    loss, dz = run(z, index, t, dloss, 1.5)
    ref, bound = reference(z, index, t, dloss, 1.5)
    check(loss, ref[0], bound[0], "loss")
    check(dz, ref[1], bound[1], "dz")


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("cols", [333, 20001])
def test_special_rows_among_many(cuda, dtype, cols):
    rows, k, T = 1830, 12, 2.0
    z, index, t, dloss = inputs(rows, cols, k, dtype, seed=6, empty=0.0)
    r = torch.arange(rows, device="cuda") % 10
    odd = 2 * torch.arange(k, device="cuda") + 1
    index[r == 1] = -1
    t[r == 2] = NEG
    z[r == 1] = float("nan")
    z[r == 2] = float("inf")
    low = r == 3
    z[low] = torch.finfo(dtype).min
    masked = (r == 4).nonzero()[:, 0]
    z[masked, ::2] = NEG
    index[masked] = odd
    low_masked = (r == 5).nonzero()[:, 0]
    z[low_masked, ::2] = torch.finfo(dtype).min
    index[low_masked] = odd
    loss, dz = run(z, index, t, dloss, T)
    empty = (r == 1) | (r == 2)
    assert (loss[empty] == 0).all() and (dz[empty] == 0).all()
    ref, bound = reference(torch.where(empty[:, None], 0.0, z), index, t, dloss, T)
    check(loss, ref[0], bound[0], "loss")
    check(dz, ref[1], bound[1], "dz")
    z[r == 6, 7 % cols] = float("nan")
    index[r == 7, 3] = cols
    l2, d2 = run(z, index, t, dloss, T)
    bad = (r == 6) | (r == 7)
    assert l2[bad].isnan().all() and d2[bad].isnan().any(1).all()
    assert torch.equal(l2[~bad], loss[~bad]) and torch.equal(d2[~bad], dz[~bad])
