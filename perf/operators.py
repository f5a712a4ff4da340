"""The end of a language model as cases to measure: the final layer norm, the vocabulary head
with its loss, and distillation from a teacher's top logits.

Kinds:

- ``layer_norm``  y = (x - mean) / sqrt(var + eps) * gamma + beta over the last axis; with
  ``train`` also its VJP: dx, and dgamma and dbeta summed over the rows;
- ``linear_xent``  the loss of a head, per token: the softmax cross entropy of z = x w^T against a
  label, where a negative label is a token without a loss; with ``train`` also the gradients of
  x and w for a given gradient of each token's loss;
- ``distill_topk``  per row T^2 KL(p || q) of the student's q = softmax(z / T) over all columns from
  the teacher's p = softmax(t / T) over the k columns whose logits the teacher gave (a negative
  column is an empty entry), and with ``train`` the gradient of z.

``run`` computes them in plain torch operations, or through the entry points of
``cgadimpl_amd`` where ``own`` is true.  Sizes are those of the benchmark's configurations and
the tests, or round numbers of the same ranges.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # The final norm while decoding: 16 sequences, one token each.
        dict(name="norm_decode", kind="layer_norm", train=False, dtype="bf16", rows=16, cols=4096),
        # The norm of a training step at an ordinary batch.
        dict(name="norm_train", kind="layer_norm", train=True, dtype="bf16", rows=16384, cols=8192),
        # An odd number of fp32 rows whose width is no multiple of 16 bytes.
        dict(name="norm_train_ragged", kind="layer_norm", train=True, dtype="f32", rows=4099,
             cols=1030),
        # Scoring a handful of tokens: the head's weights are read once for 16 rows.
        dict(name="head_score_few", kind="linear_xent", train=False, dtype="bf16", rows=16,
             hidden=4096, vocab=32000, ignored=0.0),
        # Perplexity of a batch: the forward alone.
        dict(name="head_score_batch", kind="linear_xent", train=False, dtype="bf16", rows=4096,
             hidden=4096, vocab=32000, ignored=0.0),
        # A fine-tuning step: a packed batch of odd length whose prompts carry no loss, a
        # vocabulary that is a multiple of nothing.
        dict(name="head_train_ragged", kind="linear_xent", train=True, dtype="bf16", rows=4099,
             hidden=2048, vocab=50257, ignored=0.3),
        # A training step of a large vocabulary.
        dict(name="head_train_large", kind="linear_xent", train=True, dtype="bf16", rows=8192,
             hidden=4096, vocab=131072, ignored=0.02),
        # A small fp32 model's step.
        dict(name="head_train_f32", kind="linear_xent", train=True, dtype="f32", rows=512,
             hidden=512, vocab=10007, ignored=0.1),
        # A few sequences' last positions, fp32 logits, 64 columns of the teacher.
        dict(name="distill_few", kind="distill_topk", train=True, dtype="f32", rows=32, cols=32000,
             k=64, temperature=2.0, empty=0.0),
        # A training batch over a vocabulary that is a multiple of nothing; rows of the teacher
        # are of unequal length, some empty.
        dict(name="distill_train", kind="distill_topk", train=True, dtype="bf16", rows=8192,
             cols=50257, k=64, temperature=2.0, empty=0.1),
        # Validation of the same loss on fp32 logits, forward alone.
        dict(name="distill_validate", kind="distill_topk", train=False, dtype="f32", rows=2048,
             cols=50257, k=20, temperature=1.0, empty=0.0),
        # Few very wide rows and many columns of the teacher.
        dict(name="distill_wide", kind="distill_topk", train=True, dtype="bf16", rows=96,
             cols=131072, k=256, temperature=1.5, empty=0.05),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row width: half of them a multiple of 16 bytes in either type, half anything."""
    w = _log_int(rng, lo, hi)
    return max(8, w // 8 * 8) if rng.random() < 0.5 else w


def draw(rng):
    kind = rng.choice(["layer_norm", "linear_xent", "distill_topk"])
    train = rng.random() < 0.7
    dtype = rng.choice(["f32", "bf16"])
    if kind == "layer_norm":
        cols = _width(rng, 64, 16384)
        rows = min(_log_int(rng, 1, 65536), (1 << 27) // cols)
        return dict(kind=kind, train=train, dtype=dtype, rows=rows, cols=cols)
    if kind == "linear_xent":
        ignored = rng.choice([0.0, 0.02, 0.3, 0.7])
        if dtype == "f32":
            return dict(kind=kind, train=train, dtype=dtype, rows=_log_int(rng, 1, 1024),
                        hidden=_width(rng, 64, 1024), vocab=_width(rng, 500, 32000),
                        ignored=ignored)
        return dict(kind=kind, train=train, dtype=dtype, rows=_log_int(rng, 1, 8192),
                    hidden=8 * _log_int(rng, 8, 512), vocab=_width(rng, 1000, 131072),
                    ignored=ignored)
    cols = _width(rng, 1000, 151936)
    rows = min(_log_int(rng, 1, 8192), (1 << 28) // cols)
    return dict(kind=kind, train=train, dtype=dtype, rows=rows, cols=cols, k=_log_int(rng, 1, 256),
                temperature=rng.choice([1.0, 1.5, 2.0, 4.0]), empty=rng.choice([0.0, 0.1, 0.5]))


# ---- inputs -------------------------------------------------------------------

class _Gen:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape, dtype, std=1.0):
        t = torch.randn(*shape, generator=self.gen, device="cuda")
        return (t.mul_(std) if std != 1.0 else t).to(dtype)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.gen, device="cuda")

    def integers(self, hi, *shape):
        return torch.randint(hi, shape, generator=self.gen, device="cuda")


def prepare(case, seed):
    g = _Gen(seed)
    dt = DTYPES[case["dtype"]]
    k, rows = case["kind"], case["rows"]
    s = {"kind": k, "train": case["train"]}
    if k == "layer_norm":
        cols = case["cols"]
        s["x"] = g.normal(rows, cols, dtype=dt).add_(0.25)
        s["gamma"] = (g.uniform(cols) + 0.5).to(dt)
        s["beta"] = g.normal(cols, dtype=dt, std=0.1)
        if case["train"]:
            s["dy"] = g.normal(rows, cols, dtype=dt)
    elif k == "linear_xent":
        hidden, vocab = case["hidden"], case["vocab"]
        # normed activations, and weights that give logits of a few units
        s["x"] = g.normal(rows, hidden, dtype=dt)
        s["w"] = g.normal(vocab, hidden, dtype=dt, std=2.0 / math.sqrt(hidden))
        labels = g.integers(vocab, rows)
        ignored = g.uniform(rows) < case["ignored"]
        ignored[0] = False  # a batch has a token with a loss
        s["labels"] = torch.where(ignored, -100, labels)
        if case["train"]:
            has = s["labels"] >= 0
            s["dloss"] = has.float() / has.sum().clamp(min=1)  # the mean over the tokens with a loss
    else:
        cols, kk = case["cols"], case["k"]
        s["temperature"] = case["temperature"]
        s["z"] = g.normal(rows, cols, dtype=dt, std=3.0)
        # k different columns a row, one from each of k ranges (modulo the width) where
        # the row has that many
        step = max(1, cols // kk)
        at = g.integers(cols, rows, 1) + step * torch.arange(kk, device="cuda")
        at = (at + (g.uniform(rows, kk) * step).long()) % cols
        # the teacher thinks much as the student does, and is surer of its best columns
        t = s["z"].gather(1, at).float() + 4.0 + g.normal(rows, kk, dtype=torch.float32)
        length = torch.where(g.uniform(rows) < case["empty"],
                             (g.uniform(rows) * kk).long(), kk)
        length[0] = kk
        s["index"] = torch.where(torch.arange(kk, device="cuda") < length[:, None], at, -1)
        s["teacher"] = t.to(dt)
        if case["train"]:
            s["dloss"] = torch.full((rows,), 1.0 / rows, device="cuda")
    return s


# ---- plain forms --------------------------------------------------------------

def _layer_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    xhat = d * rstd
    gamma = s["gamma"].float()
    y = (xhat * gamma + s["beta"].float()).to(s["x"].dtype)
    if not s["train"]:
        return y
    dy = s["dy"].float()
    h = dy * gamma
    dx = rstd * (h - h.mean(1, keepdim=True) - xhat * (h * xhat).mean(1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * xhat).sum(0), dy.sum(0)


def _linear_xent(s):
    x, w = s["x"].float(), s["w"].float()
    has = s["labels"] >= 0
    at = s["labels"].clamp(min=0)[:, None]
    z = torch.mm(x, w.t())
    top = z.amax(1, keepdim=True)
    picked = (z.gather(1, at) - top)[:, 0]
    e = z.sub_(top).exp_()
    total = e.sum(1, keepdim=True)
    loss = torch.where(has, torch.log(total[:, 0]) - picked, 0.0)
    if not s["train"]:
        return loss
    dloss = torch.where(has, s["dloss"], 0.0)[:, None]
    dz = e.mul_(dloss / total)
    dz.scatter_add_(1, at, -dloss)
    dx = torch.mm(dz, w).to(s["x"].dtype)
    dw = torch.mm(dz.t(), x).to(s["w"].dtype)
    return loss, dx, dw


def _distill_topk(s):
    temp = s["temperature"]
    z = s["z"].float() / temp
    has = s["index"] >= 0
    at = s["index"].clamp(min=0)
    some = has.any(1)
    t = torch.where(has, s["teacher"].float() / temp, -math.inf)
    t = t - torch.where(some, t.amax(1), 0.0)[:, None]
    e = torch.exp(t)
    total = torch.where(some, e.sum(1), 1.0)[:, None]
    p = e / total
    logp = torch.where(has, t - torch.log(total), 0.0)
    z = z - z.amax(1, keepdim=True)
    ez = torch.exp(z)
    sz = ez.sum(1, keepdim=True)
    logq = z.gather(1, at) - torch.log(sz)
    loss = temp * temp * (p * (logp - logq)).sum(1)
    if not s["train"]:
        return loss
    c = torch.where(some, s["dloss"] * temp, 0.0)[:, None]
    dz = ez * (c / sz)
    dz.scatter_add_(1, at, -c * p)
    return loss, dz.to(s["z"].dtype)


# ---- the framework's calls ------------------------------------------------------

def _layer_norm_own(s):
    import cgadimpl_amd as agk
    y, mean, rstd = agk.layernorm_affine_fwd(s["x"], s["gamma"], s["beta"], EPS)
    if not s["train"]:
        return y
    dx, dgamma, dbeta = agk.layernorm_affine_bwd(s["x"], s["gamma"], mean, rstd, s["dy"])
    return y, dx, dgamma, dbeta


def _linear_xent_own(s):
    import cgadimpl_amd as agk
    loss, stats = agk.linear_cross_entropy_fwd(s["x"], s["w"], s["labels"])
    if not s["train"]:
        return loss
    dx, dw = agk.linear_cross_entropy_bwd(s["x"], s["w"], s["labels"], stats, s["dloss"],
                                          dw_dtype=s["w"].dtype)
    return loss, dx, dw


def _distill_topk_own(s):
    import cgadimpl_amd as agk
    loss, stats = agk.distill_topk_fwd(s["z"], s["index"], s["teacher"], s["temperature"])
    if not s["train"]:
        return loss
    dz = agk.distill_topk_bwd(s["z"], s["index"], s["teacher"], stats, s["dloss"],
                              s["temperature"])
    return loss, dz


def run(state):
    k = state["kind"]
    if k == "layer_norm":
        return _layer_norm_own(state) if own else _layer_norm(state)
    if k == "linear_xent":
        return _linear_xent_own(state) if own else _linear_xent(state)
    return _distill_topk_own(state) if own else _distill_topk(state)


# ---- what a pass cannot do without ------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    rows, train = case["rows"], case["train"]
    if case["kind"] == "layer_norm":
        n, cols = rows * case["cols"], case["cols"]
        return {"bytes": (4 if train else 2) * n * size + 2 * cols * size + (8 * cols if train else 0),
                "flops": n * (22 if train else 8)}
    if case["kind"] == "linear_xent":
        hidden, vocab = case["hidden"], case["vocab"]
        operands = (rows + vocab) * hidden * size
        # the logits; with their gradients, dx and dw too (the logits a second time,
        # where they are not kept, are not counted)
        return {"bytes": (2 if train else 1) * operands + rows * (16 if train else 12),
                "flops": 2 * rows * vocab * hidden * (3 if train else 1)}
    n = rows * case["cols"]
    return {"bytes": (2 if train else 1) * n * size + rows * case["k"] * (8 + size) +
            rows * (8 if train else 4),
            "flops": n * (8 if train else 4)}


# ---- the definitions in 64 bits -----------------------------------------------------

def _exact_layer_norm(s):
    x = s["x"].double()
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    xhat = (x - mean) / torch.sqrt(var + EPS)
    y = torch.addcmul(s["beta"].double(), xhat, s["gamma"].double())
    if not s["train"]:
        return y
    dy = s["dy"].double()
    h = dy * s["gamma"].double()
    n = x.shape[1]
    dx = n * h - h.sum(1, keepdim=True) - xhat * (h * xhat).sum(1, keepdim=True)
    dx /= n * torch.sqrt(var + EPS)
    return y, dx, (dy * xhat).sum(0), dy.sum(0)


def _exact_linear_xent(s):
    # token by token blocks, from the log-probabilities
    x, w = s["x"].double(), s["w"].double()
    rows = x.shape[0]
    loss = torch.zeros(rows, dtype=torch.float64, device="cuda")
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for r in range(0, rows, 1024):
        b = slice(r, min(rows, r + 1024))
        keep = torch.nonzero(s["labels"][b] >= 0)[:, 0] + r
        if keep.numel() == 0:
            continue
        z = x[keep] @ w.T
        z -= torch.logsumexp(z, 1, keepdim=True)
        lab = s["labels"][keep]
        one = torch.arange(keep.numel(), device="cuda")
        loss[keep] = -z[one, lab]
        if s["train"]:
            z.exp_()
            z[one, lab] -= 1.0
            z *= s["dloss"][keep].double()[:, None]
            dx[keep] = z @ w
            dw.addmm_(z.T, x[keep])
    return (loss, dx, dw) if s["train"] else loss


def _exact_distill_topk(s):
    temp = s["temperature"]
    rows, cols = s["z"].shape
    loss = torch.zeros(rows, dtype=torch.float64, device="cuda")
    dz = torch.zeros(rows, cols, dtype=torch.float64, device="cuda") if s["train"] else None
    for r in range(0, rows, 512):
        b = slice(r, min(rows, r + 512))
        logq = torch.log_softmax(s["z"][b].double() / temp, 1)
        # an empty entry is a column past the last, whose probability is dropped
        index = torch.where(s["index"][b] < 0, cols, s["index"][b])
        t = s["teacher"][b].double() / temp
        t[s["index"][b] < 0] = -math.inf
        p = torch.nan_to_num(torch.softmax(t, 1))
        logq1 = torch.cat([logq, torch.zeros_like(logq[:, :1])], 1)
        loss[b] = temp ** 2 * (torch.special.xlogy(p, p) - p * logq1.gather(1, index)).sum(1)
        if s["train"]:
            full = torch.zeros_like(logq1).scatter_add_(1, index, p)[:, :cols]
            mass = full.sum(1, keepdim=True)  # 1, or 0 for a row without a teacher
            dz[b] = (logq.exp() * (mass > 0.5) - full) * (s["dloss"][b].double()[:, None] * temp)
    return (loss, dz) if s["train"] else loss


def exact(case, seed):
    s = prepare(case, seed)
    return {"layer_norm": _exact_layer_norm, "linear_xent": _exact_linear_xent,
            "distill_topk": _exact_distill_topk}[s["kind"]](s)
