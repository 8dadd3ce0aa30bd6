"""The operators of a language model's last part: the affine layer norm, the
LM head with its softmax cross entropy (the logits are never kept whole), and
distillation from a teacher's top logits.

Each case names its operator in "op".  With `own` false, `run` computes the
plain form in elementary torch operations; with `own` true it calls the
malus_b200 entry points on the same tensors.  Everything is f32, the one
floating type of the runtime; token ids are i32 or i64.

  norm     y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis;
           "train" also gives dx, dweight, dbias for an incoming dy.
  head     logits = x weight^T (tied: weight [V, D], the embedding) or
           x weight (weight [D, V]); nll = logsumexp(logits) - logits[target]
           per row, the loss is its mean over the rows whose target is not
           negative (0 when there is none); "train" also gives dx, dweight.
  distill  p = softmax of the teacher's K logits over T, q = softmax of the
           student's V logits over T; the row's value is T^2 KL(p || q), the
           loss its mean over the rows with an entry (an id below 0 or a
           teacher logit of -inf is no entry); "train" also gives dlogits.
"""
import math

import numpy as np
import torch

own = False


# ------------------------------------------------------------------- cases

def listed():
    return [
        # one token being sampled from the GPT-2-small shape: latency of one call
        dict(name="norm_token", op="norm", n=1, d=768, bias=True, train=False),
        # a training batch of the character-level model (64 x 256 tokens)
        dict(name="norm_train_c4", op="norm", n=16384, d=384, bias=True, train=True),
        # a training batch of the GPT-2-small shape (8 x 1024 tokens)
        dict(name="norm_train_c5", op="norm", n=8192, d=768, bias=True, train=True),
        # a wide model's ragged batch, odd in both sizes, weight without bias
        dict(name="norm_train_odd", op="norm", n=4099, d=5001, bias=False, train=True),
        # scoring one token against the GPT-2 vocabulary
        dict(name="head_token", op="head", n=1, d=768, v=50304, tied=True, ids="i32", masked=0.0, train=False),
        # the character-level model's head over a whole batch
        dict(name="head_train_chars", op="head", n=16384, d=384, v=65, tied=False, ids="i32", masked=0.0, train=True),
        # perplexity of one sequence of the GPT-2-small shape
        dict(name="head_eval", op="head", n=1024, d=768, v=50304, tied=True, ids="i64", masked=0.0, train=False),
        # a fine-tuning batch: prompt tokens masked out, odd sizes, untied head
        dict(name="head_train_odd", op="head", n=1999, d=500, v=10007, tied=False, ids="i64", masked=0.3, train=True),
        # a training batch of the GPT-2-small shape with its tied head
        dict(name="head_train_c5", op="head", n=8192, d=768, v=50304, tied=True, ids="i32", masked=0.0, train=True),
        # a character-level student
        dict(name="distill_chars", op="distill", n=256, v=65, k=8, t=2.0, ids="i32", padded=0.0, train=True),
        # a GPT-2-vocabulary student, two sequences, the teacher's 64 best
        dict(name="distill_train", op="distill", n=2048, v=50304, k=64, t=2.0, ids="i32", padded=0.0, train=True),
        # validation over another vocabulary, ragged lists of entries, odd sizes
        dict(name="distill_eval_odd", op="distill", n=1021, v=32003, k=20, t=1.0, ids="i64", padded=0.3, train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "head", "distill"])
    if op == "norm":
        d = _log(rng, 16, 8192)
        n = _log(rng, 1, min(32768, 20_000_000 // d))
        return dict(op=op, n=n, d=d, bias=rng.random() < 0.7, train=rng.random() < 0.7)
    if op == "head":
        d, v = _log(rng, 32, 1024), _log(rng, 50, 50304)
        n = _log(rng, 1, min(16384, 200_000_000_000 // (d * v)))
        return dict(op=op, n=n, d=d, v=v, tied=rng.random() < 0.5, ids=rng.choice(["i32", "i64"]),
                    masked=rng.choice([0.0, round(rng.uniform(0.05, 0.9), 2)]), train=rng.random() < 0.7)
    v = _log(rng, 50, 65536)
    n = _log(rng, 1, min(8192, 100_000_000 // v))
    return dict(op=op, n=n, v=v, k=min(v, _log(rng, 1, 64)), t=round(rng.uniform(0.5, 4.0), 2),
                ids=rng.choice(["i32", "i64"]), padded=rng.choice([0.0, round(rng.uniform(0.05, 0.9), 2)]),
                train=rng.random() < 0.7)


def work(case):
    c = case
    if c["op"] == "norm":
        nd, vec = c["n"] * c["d"], c["d"] * (2 if c["bias"] else 1)
        if not c["train"]:
            return {"bytes": 4 * (2 * nd + vec), "flops": 8 * nd}
        # x, dy in; y, dx, dweight (dbias) out
        return {"bytes": 4 * (4 * nd + 2 * vec), "flops": 20 * nd}
    idb = 4 if c["ids"] == "i32" else 8
    if c["op"] == "head":
        n, d, v = c["n"], c["d"], c["v"]
        one = 4 * (n * d + v * d)
        if not c["train"]:
            return {"bytes": one + (idb + 4) * n, "flops": 2 * n * d * v}
        return {"bytes": 2 * one + (idb + 4) * n, "flops": 6 * n * d * v}
    n, v, k = c["n"], c["v"], c["k"]
    b = 4 * n * v * (2 if c["train"] else 1) + (idb + 4) * n * k + 4 * n
    return {"bytes": b, "flops": (8 if c["train"] else 5) * n * v}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def prepare(case, seed):
    c, g = case, _gen(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)

    def randint(hi, *shape):
        t = torch.randint(0, hi, shape, generator=g, device="cuda", dtype=torch.int64)
        return t.to(torch.int32) if c["ids"] == "i32" else t

    s = dict(case=dict(c))
    if c["op"] == "norm":
        n, d = c["n"], c["d"]
        # a residual stream: rows of different scale, channels with their own
        # offset, a few of them far larger than the rest
        x = randn(n, d) * (0.5 + rand(n, 1) * 3.0) + randn(1, d) * 0.3
        x[:, :: max(1, d // 3)] *= 8.0
        s["x"], s["weight"] = x, 1.0 + 0.2 * randn(d)
        s["bias"] = 0.1 * randn(d) if c["bias"] else None
        s["dy"] = randn(n, d) * 0.01 if c["train"] else None
    elif c["op"] == "head":
        n, d, v = c["n"], c["d"], c["v"]
        # normalised activations and a head some way into training
        s["x"] = randn(n, d) * (1.0 + 0.2 * randn(1, d))
        w = randn(v, d) * (1.5 / math.sqrt(d))
        s["weight"] = w if c["tied"] else w.t().contiguous()
        tgt = randint(v, n)
        if c["masked"]:
            tgt[rand(n) < c["masked"]] = -1
        s["targets"] = tgt
    else:
        n, v, k = c["n"], c["v"], c["k"]
        s["logits"] = randn(n, v) * 2.0
        s["ids"] = randint(v, n, k)
        s["teacher"] = torch.sort(randn(n, k) * 2.0 + 6.0, dim=1, descending=True).values
        # the student already leans the teacher's way
        s["logits"].scatter_add_(1, s["ids"].long(), 0.7 * s["teacher"])
        if c["padded"]:
            s["ids"][rand(n, k) < c["padded"]] = -1
    return s


# -------------------------------------------------------------- plain forms

def _norm_plain(s):
    c, x, w = s["case"], s["x"], s["weight"]
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + 1e-5)
    xhat = xc * rstd
    y = xhat * w
    if s["bias"] is not None:
        y = y + s["bias"]
    if not c["train"]:
        return {"y": y}
    dy = s["dy"]
    g = dy * w
    dx = (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True)) * rstd
    out = {"y": y, "dx": dx, "dweight": (dy * xhat).sum(0)}
    if s["bias"] is not None:
        out["dbias"] = dy.sum(0)
    return out


def _head_plain(s):
    c, x, w = s["case"], s["x"], s["weight"]
    tgt = s["targets"].long()
    counted = tgt >= 0
    at = torch.where(counted, tgt, torch.zeros_like(tgt)).unsqueeze(1)
    inv = 1.0 / counted.sum().clamp(min=1).float()
    logits = x @ (w.t() if c["tied"] else w)
    m = logits.max(1, keepdim=True).values
    e = torch.exp(logits - m)
    z = e.sum(1, keepdim=True)
    nll = torch.log(z) - (logits.gather(1, at) - m)
    nll = torch.where(counted, nll.squeeze(1), torch.zeros_like(z.squeeze(1)))
    out = {"loss": (nll.sum() * inv).reshape(1), "nll": nll}
    if c["train"]:
        row = counted.float().unsqueeze(1)
        dl = (e / z) * row
        dl.scatter_add_(1, at, -row)
        dl *= inv
        out["dx"] = dl @ (w if c["tied"] else w.t())
        out["dweight"] = dl.t() @ x if c["tied"] else x.t() @ dl
    return out


def _distill_plain(s):
    c, t = s["case"], s["case"]["t"]
    ids = s["ids"].long()
    there = (ids >= 0) & (s["teacher"] != -math.inf)
    at = torch.where(there, ids, torch.zeros_like(ids))
    counted = there.any(1)
    inv = 1.0 / counted.sum().clamp(min=1).float()
    te = torch.where(there, s["teacher"] / t, torch.full_like(s["teacher"], -math.inf))
    tm = torch.where(counted, te.max(1).values, torch.zeros_like(te[:, 0])).unsqueeze(1)
    pe = torch.exp(te - tm)
    pz = pe.sum(1, keepdim=True)
    pz = torch.where(pz > 0, pz, torch.ones_like(pz))
    p = pe / pz
    z = s["logits"] / t
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    ez = e.sum(1, keepdim=True)
    log_p = te - tm - torch.log(pz)
    log_q = z.gather(1, at) - m - torch.log(ez)
    kl = (t * t) * torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)).sum(1)
    out = {"loss": (kl.sum() * inv).reshape(1), "kl": kl}
    if c["train"]:
        dl = e / ez * counted.float().unsqueeze(1)
        dl.scatter_add_(1, at, -p)
        out["dlogits"] = dl * (t * inv)
    return out


# ---------------------------------------------------- the framework's calls

def _malus():
    import malus_b200
    return malus_b200


_NP = {torch.float32: np.float32, torch.int32: np.int32, torch.int64: np.int64}


def _in(t):
    return None if t is None else _malus().Tensor.wrap(t.data_ptr(), t.shape, _NP[t.dtype])


def _out(t):
    return torch.as_tensor(t, device="cuda")


def _norm_own(s):
    c, x, w = s["case"], _in(s["x"]), _in(s["weight"])
    y, stats = _malus().layernorm_affine(x, w, _in(s["bias"]), eps=1e-5)
    if not c["train"]:
        return {"y": _out(y)}
    dx, dw, db = _malus().layernorm_affine_bwd(x, w, stats, _in(s["dy"]))
    out = {"y": _out(y), "dx": _out(dx), "dweight": _out(dw)}
    if s["bias"] is not None:
        out["dbias"] = _out(db)
    return out


def _head_own(s):
    c = s["case"]
    loss, nll, dx, dw = _malus().linear_xent(_in(s["x"]), _in(s["weight"]), _in(s["targets"]), tied=c["tied"],
                                             grad=c["train"])
    out = {"loss": _out(loss), "nll": _out(nll)}
    if c["train"]:
        out["dx"], out["dweight"] = _out(dx), _out(dw)
    return out


def _distill_own(s):
    c = s["case"]
    loss, kl, dl = _malus().distill(_in(s["logits"]), _in(s["ids"]), _in(s["teacher"]), temperature=c["t"],
                                    grad=c["train"])
    out = {"loss": _out(loss), "kl": _out(kl)}
    if c["train"]:
        out["dlogits"] = _out(dl)
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _norm_own, "head": _head_own, "distill": _distill_own}[op](state)
    return {"norm": _norm_plain, "head": _head_plain, "distill": _distill_plain}[op](state)


# ------------------------------------------------- 64-bit values, by rows

def _norm_exact(s):
    x, w = s["x"].double(), s["weight"].double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    sigma = (var + 1e-5).sqrt()
    y = torch.addcmul(torch.zeros_like(w) if s["bias"] is None else s["bias"].double(), (x - mean) / sigma, w)
    out = {"y": y}
    if s["dy"] is not None:
        d = x.shape[1]
        dy = s["dy"].double()
        u = (x - mean) / sigma
        # dx = J^T (w dy) with J = (I - 1 1^T / d - u u^T / d) / sigma
        h = w * dy
        out["dx"] = (h - (h.sum(1, keepdim=True) + u * torch.einsum("nd,nd->n", h, u).unsqueeze(1)) / d) / sigma
        out["dweight"] = torch.einsum("nd,nd->d", dy, u)
        if s["bias"] is not None:
            out["dbias"] = torch.einsum("nd->d", dy)
    return out


def _head_exact(s):
    c, x = s["case"], s["x"].double()
    w = s["weight"].double()
    if not c["tied"]:
        w = w.t()
    n, v = x.shape[0], w.shape[0]
    tgt = s["targets"].long()
    rows = torch.nonzero(tgt >= 0).squeeze(1)
    count = max(1, rows.numel())
    nll = torch.zeros(n, dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for part in rows.split(1024):
        logq = torch.log_softmax(x[part] @ w.t(), dim=1)
        nll[part] = -logq[torch.arange(part.numel(), device=x.device), tgt[part]]
        if c["train"]:
            q = logq.exp_()
            dx[part] = (q @ w - w[tgt[part]]) / count
            dw.addmm_(q.t(), x[part], alpha=1.0 / count)
            dw.index_add_(0, tgt[part], x[part], alpha=-1.0 / count)
    out = {"loss": (nll.sum() / count).reshape(1), "nll": nll}
    if c["train"]:
        out["dx"], out["dweight"] = dx, dw if c["tied"] else dw.t().contiguous()
    return out


def _distill_exact(s):
    c, t = s["case"], float(s["case"]["t"])
    n, v = s["logits"].shape
    ids = s["ids"].long()
    there = (ids >= 0) & torch.isfinite(s["teacher"])
    rows = torch.nonzero(there.sum(1) > 0).squeeze(1)
    count = max(1, rows.numel())
    kl = torch.zeros(n, dtype=torch.float64, device=ids.device)
    dl = torch.zeros(n, v, dtype=torch.float64, device=ids.device) if c["train"] else None
    for part in rows.split(512):
        logq = torch.log_softmax(s["logits"][part].double() / t, dim=1)
        te = (s["teacher"][part].double() / t).masked_fill(~there[part], -1e300)
        logp = torch.log_softmax(te, dim=1)
        p = logp.exp().masked_fill(~there[part], 0.0)
        idx = ids[part].clamp(min=0)
        kl[part] = t * t * (p * (logp.masked_fill(~there[part], 0.0) - logq.gather(1, idx))).sum(1)
        if c["train"]:
            dl[part] = (logq.exp() - torch.zeros_like(logq).scatter_add_(1, idx, p)) * (t / count)
    out = {"loss": (kl.sum() / count).reshape(1), "kl": kl}
    if c["train"]:
        out["dlogits"] = dl
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _norm_exact, "head": _head_exact, "distill": _distill_exact}[case["op"]](s)
