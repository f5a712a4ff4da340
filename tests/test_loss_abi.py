"""Argument checks of the LayerNorm with weight and bias and of the losses, without a GPU:
everything here ends before any kernel is launched."""
import ctypes

import pytest

import cgadimpl_amd as agk

FAKE = 0x10000   # never dereferenced: the call ends before
F32, BF16 = agk.AGK_F32, agk.AGK_BF16
OK, EINVAL, EDTYPE, EWORKSPACE = 0, 1, 2, 3
BIG = 1 << 40


def test_layernorm_affine_validation():
    lib = agk.lib()
    f = lib.agk_layernorm_affine_fwd  # x, gamma, beta, y, mean, rstd, rows, cols, eps, dtype
    assert f(None, FAKE, FAKE, FAKE, FAKE, FAKE, 4, 8, 1e-5, F32, None) == EINVAL
    assert f(FAKE, FAKE, FAKE, None, FAKE, FAKE, 4, 8, 1e-5, F32, None) == EINVAL
    assert f(FAKE, FAKE, FAKE, FAKE, None, FAKE, 4, 8, 1e-5, F32, None) == EINVAL
    assert f(FAKE, FAKE, FAKE, FAKE, FAKE, None, 4, 8, 1e-5, F32, None) == EINVAL
    assert f(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 4, 8, 1e-5, 2, None) == EDTYPE
    assert f(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, -4, 8, 1e-5, F32, None) == EINVAL
    assert f(None, None, None, None, None, None, 0, 8, 1e-5, F32, None) == OK
    assert f(None, None, None, None, None, None, 8, 0, 1e-5, F32, None) == OK

    names = ["x", "gamma", "mean", "rstd", "dy", "dx", "dgamma", "dbeta", "ws", "ws_bytes", "rows",
             "cols", "dtype", "acc"]

    def b(**kw):
        v = dict.fromkeys(names, FAKE)
        v.update(ws_bytes=BIG, rows=4, cols=8, dtype=F32, acc=0)
        v.update(kw)
        return lib.agk_layernorm_affine_bwd(*[v[n] for n in names], None)

    for name in ("x", "mean", "rstd", "dy"):
        assert b(**{name: None}) == EINVAL, name
    assert b(dtype=5) == EDTYPE
    assert b(rows=-1) == EINVAL and b(cols=1 << 31) == EINVAL
    assert b(acc=8) == EINVAL
    assert b(ws=None) == EWORKSPACE
    assert b(ws_bytes=4 * 8 * 8 - 1) == EWORKSPACE
    assert b(ws=FAKE + 2) == EINVAL
    assert b(dx=None, dgamma=None, dbeta=None) == OK
    assert b(cols=0) == OK
    assert b(rows=0, acc=7, x=None, ws=None) == OK
    assert b(rows=0, dgamma=None, dbeta=None, x=None, ws=None) == OK


def test_layernorm_affine_workspace_rule():
    ws = agk.lib().agk_layernorm_affine_bwd_workspace_bytes
    assert ws(0, 8) == 0 and ws(8, 0) == 0 and ws(-1, 8) == 0
    for rows, cols in ((1, 8), (7, 1030), (255, 4), (256, 8192), (100000, 64)):
        assert ws(rows, cols) == min(rows, 256) * cols * 8


def _xent_fwd(**kw):
    names = ["x", "ldx", "w", "ldw", "labels", "loss", "stats", "ws", "ws_bytes", "rows", "vocab",
             "cols", "dtype"]
    v = dict.fromkeys(names, FAKE)
    v.update(ldx=64, ldw=64, ws_bytes=BIG, rows=5, vocab=99, cols=64, dtype=BF16)
    v.update(kw)
    return agk.lib().agk_linear_xent_fwd(*[v[n] for n in names], None)


def _xent_bwd(**kw):
    names = ["x", "ldx", "w", "ldw", "labels", "stats", "dloss", "dx", "dw", "dw_dtype", "ws",
             "ws_bytes", "rows", "vocab", "cols", "piece", "dtype", "acc"]
    v = dict.fromkeys(names, FAKE)
    v.update(ldx=64, ldw=64, dw_dtype=F32, ws_bytes=BIG, rows=5, vocab=99, cols=64, piece=0,
             dtype=BF16, acc=0)
    v.update(kw)
    return agk.lib().agk_linear_xent_bwd(*[v[n] for n in names], None)


@pytest.mark.parametrize("call", [_xent_fwd, _xent_bwd])
def test_linear_xent_validation(call):
    for name in ("x", "w", "labels", "stats"):
        assert call(**{name: None}) == EINVAL, name
    assert call(dtype=2) == EDTYPE
    assert call(rows=-1) == EINVAL and call(rows=1 << 24) == EINVAL
    assert call(vocab=0) == EINVAL and call(cols=0) == EINVAL
    assert call(rows=0, vocab=0) == EINVAL
    assert call(ldx=56) == EINVAL and call(ldw=56) == EINVAL
    assert call(cols=60) == EINVAL                   # bf16: multiples of 8
    assert call(ldx=68) == EINVAL and call(ldw=68) == EINVAL
    assert call(x=FAKE + 8) == EINVAL and call(w=FAKE + 8) == EINVAL
    assert call(x=FAKE + 2, dtype=F32) == EINVAL
    assert call(stats=FAKE + 4) == EINVAL and call(labels=FAKE + 4) == EINVAL
    assert call(rows=(1 << 24) - 1, vocab=1 << 30) == EINVAL   # more tiles than a grid holds
    assert call(ws=None) == EWORKSPACE
    assert call(ws_bytes=0) == EWORKSPACE
    assert call(ws=FAKE + 8) == EINVAL


def test_linear_xent_more_validation():
    assert _xent_fwd(loss=None) == EINVAL
    assert _xent_fwd(rows=0, x=None, w=None, labels=None, loss=None, stats=None, ws=None) == OK
    assert _xent_bwd(dloss=None) == EINVAL
    assert _xent_bwd(dx=None, dw=None) == OK
    assert _xent_bwd(acc=4) == EINVAL and _xent_bwd(piece=-1) == EINVAL
    assert _xent_bwd(dw_dtype=7) == EDTYPE
    assert _xent_bwd(dtype=F32, dw_dtype=BF16) == EDTYPE
    assert _xent_bwd(dx=FAKE + 8) == EINVAL and _xent_bwd(dw=FAKE + 2) == EINVAL
    # rows * ldx past 2^30
    assert _xent_bwd(rows=(1 << 24) - 8, vocab=99, cols=72, ldx=72, ldw=72) == EINVAL
    # G's pieces of at least 256 vocabulary rows, whatever the width
    assert _xent_bwd(rows=(1 << 22) + 1, cols=8, ldx=8, ldw=8) == EINVAL
    assert _xent_bwd(rows=1 << 22, cols=8, ldx=8, ldw=8, ws=None) == EWORKSPACE
    assert _xent_bwd(rows=(1 << 21) + 1, cols=8, ldx=8, ldw=8, dtype=F32) == EINVAL
    assert _xent_bwd(rows=1 << 21, cols=8, ldx=8, ldw=8, dtype=F32, ws=None) == EWORKSPACE
    assert _xent_fwd(loss=FAKE + 2) == EINVAL and _xent_bwd(dloss=FAKE + 2) == EINVAL
    assert _xent_bwd(rows=0, x=None, w=None, dw=None) == OK
    assert _xent_bwd(rows=0, cols=57, x=None, w=None, dw_dtype=BF16) == EINVAL
    assert _xent_bwd(rows=0, x=None, w=None, acc=2) == OK
    f = agk.lib().agk_linear_xent_fwd_workspace_bytes
    b = agk.lib().agk_linear_xent_bwd_workspace_bytes
    for args in ((0, 9, 8), (9, 0, 8), (9, 9, 0), (-1, 9, 8)):
        assert f(*args, BF16) == 0 and b(*args, BF16, 0) == 0
    assert f(9, 9, 8, 3) == 0 and b(9, 9, 8, 3, 0) == 0
    # the logits of all tokens would be 4096 x 131072 x 4 bytes
    assert 0 < f(4096, 131072, 4096, BF16) < 4096 * 131072 * 4 // 16
    assert 0 < b(4096, 131072, 4096, BF16, 0) < 768 << 20
    assert b(4096, 131072, 4096, BF16, 256) < b(4096, 131072, 4096, BF16, 0)
    assert b(4096, 131072, 4096, BF16, 1) == b(4096, 131072, 4096, BF16, 256)


def test_distill_validation():
    lib = agk.lib()
    fn = ["z", "index", "t", "loss", "stats", "ws", "ws_bytes", "rows", "cols", "k", "temperature",
          "dtype", "t_dtype"]
    bn = ["z", "index", "t", "stats", "dloss", "dz", "rows", "cols", "k", "temperature", "dtype",
          "t_dtype", "acc"]
    base = dict.fromkeys(set(fn + bn), FAKE)
    base.update(ws_bytes=BIG, rows=4, cols=100, k=3, temperature=2.0, dtype=F32, t_dtype=BF16,
                acc=0, dz=1 << 30)

    def fwd(**kw):
        v = dict(base, **kw)
        return lib.agk_distill_topk_fwd(*[v[n] for n in fn], None)

    def bwd(**kw):
        v = dict(base, **kw)
        return lib.agk_distill_topk_bwd(*[v[n] for n in bn], None)

    for call in (fwd, bwd):
        for name in ("z", "index", "t", "stats"):
            assert call(**{name: None}) == EINVAL, name
        assert call(dtype=2) == EDTYPE and call(t_dtype=-1) == EDTYPE
        assert call(rows=-1) == EINVAL and call(cols=0) == EINVAL
        assert call(k=-1) == EINVAL and call(k=agk.AGK_DISTILL_MAX_K + 1) == EINVAL
        for t in (0.0, -1.0, 1e-5, 1e5, float("inf"), float("nan")):
            assert call(temperature=t) == EINVAL, t
        assert call(stats=FAKE + 4) == EINVAL and call(index=FAKE + 4) == EINVAL
        assert call(rows=0, z=None) == OK
        assert call(rows=0, cols=0) == OK
    assert fwd(loss=None) == EINVAL
    need = lib.agk_distill_topk_workspace_bytes(4, 1000000, F32)
    assert need > 0
    assert fwd(cols=1000000, ws=None) == EWORKSPACE
    assert fwd(cols=1000000, ws_bytes=need - 1) == EWORKSPACE
    assert fwd(cols=1000000, ws=FAKE + 4) == EINVAL
    assert bwd(dloss=None) == EINVAL and bwd(dz=None) == EINVAL
    assert bwd(acc=2) == EINVAL
    assert bwd(dz=FAKE + 16) == EINVAL               # overlaps z without being it
    ws = lib.agk_distill_topk_workspace_bytes
    assert ws(0, 100, F32) == 0 and ws(100, 0, F32) == 0 and ws(100, 100, 2) == 0
    assert ws(100000, 500000, F32) == 0 and ws(4, 100000, BF16) == 0 and ws(4, 100000, F32) > 0
    assert agk.AGK_DISTILL_MAX_K == 1024 and agk.AGK_ACCUM_DBETA == 4


def test_bindings_refuse_cpu_tensors():
    torch = pytest.importorskip("torch")
    x, w = torch.zeros(4, 8), torch.zeros(16, 8)
    lab = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError):
        agk.layernorm_affine_fwd(x, None, None)
    with pytest.raises(ValueError):
        agk.layernorm_affine_bwd(x, None, x[:, 0], x[:, 0], x)
    with pytest.raises(ValueError):
        agk.linear_cross_entropy_fwd(x, w, lab)
    with pytest.raises(ValueError):
        agk.linear_cross_entropy_bwd(x, w, lab, torch.zeros(4, 2), torch.zeros(4))
    with pytest.raises(ValueError):
        agk.distill_topk_fwd(x, lab[:, None], x[:, :1])
    with pytest.raises(ValueError):
        agk.distill_topk_bwd(x, lab[:, None], x[:, :1], torch.zeros(4, 2), torch.zeros(4))
