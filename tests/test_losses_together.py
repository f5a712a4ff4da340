"""A model's end as it is trained and served: LayerNorm with weight and bias, the vocabulary head's
cross entropy, distillation from a teacher's top logits on the head's logits, and back.

The forward's intermediates (h, z) are taken as stored, so each loss is compared with fp64 from
the same inputs.  The gradients are linear in what comes from above; bounds per element, with u =
2^-24, r the storage type's half step, P(n) = (n + 16) u of the terms' magnitude for an fp32 sum of n
products, and 12 u more for fp32 products on fp16 halves:
- dz: (r + 64 u) |dz| + 64 u |c| q + 2^-126 (its own test has the tight form; k, cols are small);
- G: r (bf16's operand) or 64 u of it, and the logits' error twice;
- dh = dz w + G w: those errors through |w|, P(V) of each, a rounding of the first product and
  of the sum; dw alike through |h|, stored in fp32;
- dx, dgamma, dbeta: linear in dh, dh's bound through the same formula with magnitudes, P(cols) or
  P(rows), one rounding to storage, and the statistics' error (32 u (1 + |mean| rstd) of xhat).
"""
import pytest

torch = pytest.importorskip("torch")

import cgadimpl_amd as agk  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
R = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
BF, F = torch.bfloat16, torch.float32


def model(N, D, V, K, dtype, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x = (rn(N, D) * 2 + 0.5).to(dtype)
    gamma, beta = (1 + 0.3 * rn(D)).to(dtype), (0.3 * rn(D)).to(dtype)
    w = (rn(V, D) * (1.5 / D ** 0.5)).to(dtype)
    labels = torch.randint(V, (N,), generator=gen, device="cuda")
    labels[::5] = -100
    index = torch.stack([torch.randperm(V, generator=gen, device="cuda")[:K] for _ in range(N)])
    index[1::4, K // 2:] = -1
    index[2::7] = -1
    teacher = rn(N, K) * 3
    g1, g2 = torch.full((N,), 0.7 / N, device="cuda"), torch.full((N,), 0.3 / N, device="cuda")
    return x, gamma, beta, w, labels, index, teacher, g1, g2


def product(a, b, dtype, **kw):
    if dtype == BF:
        return agk.gemm_bf16(a, b, workspace=None, **kw)
    return agk.gemm_f32(a, b, **kw)


def forward(x, gamma, beta, w, labels, index, teacher, T, **kw):
    h, mean, rstd = agk.layernorm_affine_fwd(x, gamma, beta, 1e-5, **kw)
    ce, ce_stats = agk.linear_cross_entropy_fwd(h, w, labels, **kw)
    z = product(h, w, x.dtype, trans_b=True, **kw)
    kl, kl_stats = agk.distill_topk_fwd(z, index, teacher, T, **kw)
    return h, mean, rstd, ce, ce_stats, z, kl, kl_stats


def backward(x, gamma, w, labels, index, teacher, T, g1, g2, saved, **kw):
    h, mean, rstd, _, ce_stats, z, _, kl_stats = saved
    dz = agk.distill_topk_bwd(z, index, teacher, kl_stats, g2, T, **kw)
    dh = product(dz, w, x.dtype, **kw)
    dw = torch.empty(w.shape, device="cuda")
    product(dz, h, x.dtype, c=dw, trans_a=True, **kw)
    agk.linear_cross_entropy_bwd(h, w, labels, ce_stats, g1, dx=dh, dw=dw, accumulate=True, **kw)
    return agk.layernorm_affine_bwd(x, gamma, mean, rstd, dh, **kw) + (dw,)


def check(got, ref, bound, what):
    d = (got.double() - ref).abs()
    assert (d <= bound + 1e-30).all(), (what, float((d / (bound + 1e-30)).max()))


def reference(x, gamma, beta, w, labels, index, teacher, T, g1, g2, h, z):
    r, fp = R[x.dtype], (12 * U if x.dtype == F else 0.0)
    r_g = r if x.dtype == BF else 8 * U  # before x turns into fp64
    P = lambda n: (n + 16) * U + fp  # noqa: E731
    (N, D), V = x.shape, w.shape[0]
    x, gamma, beta, w, h, z, t, g1, g2 = (v.double() for v in (x, gamma, beta, w, h, z, teacher,
                                                              g1, g2))
    out, tol = {}, {}
    mean = x.mean(1, keepdim=True)
    rstd = (x.var(1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    xhat = (x - mean) * rstd
    exhat = 32 * U * (1 + mean.abs() * rstd) * (1 + xhat.abs()) + D * U * xhat.abs()
    out["h"] = xhat * gamma + beta
    tol["h"] = exhat * gamma.abs() + 4 * U * ((xhat * gamma).abs() + beta.abs()) + r * out["h"].abs()
    # cross entropy from the stored h
    zz = h @ w.T
    ez = P(D) * (h.abs() @ w.abs().T)
    worst = ez.amax(1, keepdim=True)
    logp = torch.log_softmax(zz, 1)
    keep = (labels >= 0)[:, None]
    at = labels.clamp(min=0)[:, None]
    out["ce"] = torch.where(keep, -logp.gather(1, at), 0.0)[:, 0]
    tol["ce"] = (2 * worst + 256 * U * (1 + zz.abs().amax(1, keepdim=True)))[:, 0]
    p = logp.exp()
    G = torch.where(keep, g1[:, None] * (p - torch.zeros_like(p).scatter_(1, at, 1.0)), 0.0)
    eG = g1.abs()[:, None] * p * (2 * worst + 256 * U * (1 + zz.abs().amax(1, keepdim=True))) + \
        r_g * G.abs()
    # distillation from the stored z
    has = index >= 0
    some = has.any(1, keepdim=True)
    tt = torch.where(has, t / T, float("-inf"))
    pt = torch.where(some, torch.softmax(torch.where(some, tt, 0.0), 1), 0.0)
    pt = torch.where(has, pt, 0.0)
    lq = torch.log_softmax(z / T, 1)
    ci = index.clamp(min=0)
    diff = torch.where(pt > 0, torch.log(torch.where(pt > 0, pt, 1.0)) - lq.gather(1, ci), 0.0)
    out["kl"] = T * T * (pt * diff).sum(1)
    size = 1 + (z.abs().amax(1) + t.abs().amax(1)) / T
    tol["kl"] = 256 * U * T * T * size
    c = torch.where(some[:, 0], g2 * T, 0.0)[:, None]
    full = torch.zeros_like(z).scatter_add_(1, ci, pt)
    dz = c * (lq.exp() - full)
    edz = (r + 4 * U) * dz.abs() + 256 * U * size[:, None] * c.abs() * (lq.exp() + full)
    # back
    dh1, dh = dz @ w, dz @ w + G @ w
    edh = (edz + eG + P(V) * (dz.abs() + G.abs())) @ w.abs() + (r + 8 * U) * (dh1.abs() + dh.abs())
    out["dw"] = dz.T @ h + G.T @ h
    tol["dw"] = (edz + eG + P(N) * (dz.abs() + G.abs())).T @ h.abs() + 8 * U * out["dw"].abs()
    a = dh * gamma
    ea = edh * gamma.abs() + 4 * U * a.abs()
    mx = (a * xhat).mean(1, keepdim=True)
    emx = (ea * xhat.abs() + a.abs() * exhat + P(D) * (a * xhat).abs()).mean(1, keepdim=True)
    ma, ema = a.mean(1, keepdim=True), (ea + P(D) * a.abs()).mean(1, keepdim=True)
    out["dx"] = rstd * (a - ma - xhat * mx)
    tol["dx"] = rstd * (ea + ema + xhat.abs() * emx + exhat * mx.abs() +
                        (64 + D) * U * (a.abs() + ma.abs() + (xhat * mx).abs())) + \
        r * out["dx"].abs()
    out["dgamma"], out["dbeta"] = (dh * xhat).sum(0), dh.sum(0)
    tol["dgamma"] = (edh * xhat.abs() + dh.abs() * exhat + P(N) * (dh * xhat).abs()).sum(0)
    tol["dbeta"] = (edh + P(N) * dh.abs()).sum(0)
    return out, tol


@pytest.mark.parametrize("N,D,V,K,T", [(1, 64, 257, 8, 1.0), (37, 128, 1000, 16, 2.0),
                                       (200, 320, 4099, 65, 0.5), (513, 64, 333, 300, 4.0)])
@pytest.mark.parametrize("dtype", [F, BF])
def test_training_step(cuda, dtype, N, D, V, K, T):
    if dtype == BF:
        N, V = (N + 7) // 8 * 8, (V + 7) // 8 * 8  # the GEMM's
    x, gamma, beta, w, labels, index, teacher, g1, g2 = model(N, D, V, K, dtype, N + V)
    saved = forward(x, gamma, beta, w, labels, index, teacher, T)
    grads = backward(x, gamma, w, labels, index, teacher, T, g1, g2, saved)
    out, tol = reference(x, gamma, beta, w, labels, index, teacher, T, g1, g2, saved[0], saved[5])
    for name, got in (("h", saved[0]), ("ce", saved[3]), ("kl", saved[6]), *zip(
            ("dx", "dgamma", "dbeta", "dw"), grads)):
        check(got, out[name], tol[name], name)


@pytest.mark.parametrize("dtype", [F, BF])
def test_served_and_replayed(cuda, dtype):
    # one captured step, replayed on new inputs between eager steps of the same shapes
    N, D, V, K, T = 24, 128, 2000, 16, 2.0
    sets = [model(N, D, V, K, dtype, s) for s in (1, 2, 3)]
    eager = []
    for x, gamma, beta, w, labels, index, teacher, g1, g2 in sets:
        saved = forward(x, gamma, beta, w, labels, index, teacher, T)
        eager.append(saved + backward(x, gamma, w, labels, index, teacher, T, g1, g2, saved))
    held = [v.clone() for v in sets[0]]
    x, gamma, beta, w, labels, index, teacher, g1, g2 = held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        saved = forward(x, gamma, beta, w, labels, index, teacher, T)
        out = saved + backward(x, gamma, w, labels, index, teacher, T, g1, g2, saved)
    for i in (1, 0, 2, 1):
        for to, of in zip(held, sets[i]):
            to.copy_(of)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager[i]):
            assert torch.equal(a, b)
        a, b = sets[i][:5], sets[i][5:7]
        again = forward(*a, *b, T)
        assert torch.equal(again[3], eager[i][3])


@pytest.mark.parametrize("dtype", [F, BF])
def test_another_stream(cuda, dtype):
    # outputs, workspaces and the zeros of an accumulated gradient are the stream's own: work that
    # the current stream does meanwhile, in memory the calls gave back, reaches none of them
    N, D, V, K, T = 304, 256, 4000, 16, 1.0
    x, gamma, beta, w, labels, index, teacher, g1, g2 = model(N, D, V, K, dtype, 9)
    saved = forward(x, gamma, beta, w, labels, index, teacher, T)
    want = saved + backward(x, gamma, w, labels, index, teacher, T, g1, g2, saved)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    busy = torch.randn(4096, 4096, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(4):
            busy = busy @ busy * 1e-3
    got = forward(x, gamma, beta, w, labels, index, teacher, T, stream=side)
    dx, dw = agk.linear_cross_entropy_bwd(got[0], w, labels, got[4], g1, accumulate=True,
                                          stream=side)
    dz = agk.distill_topk_bwd(got[5], index, teacher, got[7], g2, T, accumulate=True, stream=side)
    ln = agk.layernorm_affine_bwd(x, gamma, got[1], got[2], got[0], accumulate=True, stream=side)
    fill = [torch.full((1 << s,), float("nan"), device="cuda") for s in range(8, 24)]
    torch.cuda.synchronize()
    assert all(bool(f.isnan().all()) for f in fill)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for a, b in zip((dx, dw), agk.linear_cross_entropy_bwd(saved[0], w, labels, saved[4], g1)):
        assert torch.equal(a, b)
    assert torch.equal(dz, agk.distill_topk_bwd(saved[5], index, teacher, saved[7], g2, T))
    for a, b in zip(ln, agk.layernorm_affine_bwd(x, gamma, saved[1], saved[2], saved[0])):
        assert torch.equal(a, b)
