"""Cases of the operators at the end of a token model: layer normalisation of any width, log probabilities of given
tokens with entropy and top alternatives, and distillation from a teacher's top log probabilities.

``own`` false: the operators in elementary torch operations, in 32 bits (64 where a difference from one is taken),
rounded once at the end.  ``own`` true: the calls that a program makes of scmomer_amd.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
WIDTH = {"f32": 4, "bf16": 2, "fp16": 2}
IGNORE = -100
GENES = 16906          # genes of a cell
BINS = 7               # expression classes of the RNA model


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one position of a wide model, as each step of single-token use normalises it: launch latency
        dict(name="norm_token", op="norm", rows=1, dim=1024, dtype="bf16", train=False),
        # the RNA encoder's own width over five cells, the f32 residual stream, forward and backward
        dict(name="norm_genes", op="norm", rows=5 * GENES, dim=200, dtype="f32", train=True),
        # a wide student, one large micro-batch of a training step
        dict(name="norm_wide", op="norm", rows=8192, dim=4096, dtype="bf16", train=True),
        # odd width, odd number of rows: no row but the first is aligned
        dict(name="norm_ragged", op="norm", rows=4001, dim=1111, dtype="fp16", train=True),
        # every gene of four cells scored under the RNA model's bins, with the two most likely bins
        dict(name="score_genes", op="score", rows=4 * GENES, vocab=BINS, dtype="f32", k=2, tau=1.0, masked=0.0, train=False),
        # three positions in flight over a large vocabulary of which a rule forbids a part (-inf)
        dict(name="score_token", op="score", rows=3, vocab=131072, dtype="bf16", k=20, tau=0.7, masked=0.3, train=False),
        # a whole prompt scored, and a teacher's alternatives taken from it
        dict(name="score_prompt", op="score", rows=2048, vocab=65536, dtype="bf16", k=8, tau=1.0, masked=0.0, train=False),
        # a policy-gradient step: log probabilities and entropy, and the gradient of both; odd vocabulary
        dict(name="score_train", op="score", rows=1021, vocab=50001, dtype="f32", k=0, tau=1.0, masked=0.0, train=True),
        # the masked genes of four cells distilled from another RNA model's three most likely bins
        dict(name="distill_genes", op="distill", rows=4 * GENES, vocab=BINS, dtype="f32", k=3, tau=1.0, tail=True, kept=0.15, fused=False),
        # a short padded batch over a small vocabulary, renormalised, at a temperature
        dict(name="distill_small", op="distill", rows=37, vocab=1000, dtype="fp16", k=16, tau=2.0, tail=False, kept=0.9, fused=False),
        # an ordinary step over a large vocabulary through autograd
        dict(name="distill_vocab", op="distill", rows=4096, vocab=65536, dtype="bf16", k=32, tau=1.0, tail=True, kept=0.95, fused=False),
        # the same step without autograd between loss and gradient: both from one call
        dict(name="distill_step", op="distill", rows=2048, vocab=131072, dtype="bf16", k=64, tau=1.5, tail=True, kept=0.95, fused=True),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "score", "distill"))
    dtype = rng.choice(("f32", "bf16", "fp16"))
    if op == "norm":
        dim = _spread(rng, 1, 16384)
        rows = _spread(rng, 1, max(1, min(100000, 33000000 // dim)))
        return dict(op=op, rows=rows, dim=dim, dtype=dtype, train=rng.random() < 0.7)
    vocab = _spread(rng, 2, 131072)
    rows = _spread(rng, 1, max(1, min(80000, 120000000 // vocab)))
    k = min(vocab, rng.choice((0, 1, 2, 5, 8, 20, 32, 50, 64)) if op == "score" else _spread(rng, 1, 64))
    tau = rng.choice((1.0, 1.0, 0.7, 1.5, 2.0))
    if op == "score":
        return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, k=k, tau=tau, masked=rng.choice((0.0, 0.0, 0.3)),
                    train=rng.random() < 0.4)
    return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, k=k, tau=tau, tail=rng.random() < 0.7,
                kept=rng.choice((1.0, 0.9, 0.15)), fused=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _logits(case, gen):
    t, v = case["rows"], case["vocab"]
    return torch.randn((t, v), generator=gen, device="cuda", dtype=torch.float32).mul_(2.0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    t = case["rows"]

    def normal(*size):
        return torch.randn(size, generator=gen, device="cuda", dtype=torch.float32)

    if case["op"] == "norm":
        d = case["dim"]
        x = (normal(t, d) * (0.5 + 2 * torch.rand((t, 1), generator=gen, device="cuda")) + 0.5 * normal(t, 1)).to(dt)
        st = {"case": case, "x": x, "w": 1 + 0.2 * normal(d), "b": 0.1 * normal(d)}
        if case["train"]:
            st["dy"] = (0.05 * normal(t, d)).to(dt)
        return st
    v, k = case["vocab"], case["k"]
    x = _logits(case, gen)
    if case["op"] == "score":
        target = torch.randint(0, v, (t,), generator=gen, device="cuda")
        x.scatter_add_(1, target[:, None], 4 * torch.rand((t, 1), generator=gen, device="cuda"))     # a model that has learnt some
        if case["masked"]:
            ban = torch.rand((t, v), generator=gen, device="cuda") < case["masked"]
            ban.scatter_(1, target[:, None], False)
            x.masked_fill_(ban, -math.inf)
            del ban
        if t > 8:
            target = torch.where(torch.rand((t,), generator=gen, device="cuda") < 0.1, IGNORE, target)   # padding
        st = {"case": case, "x": x.to(dt), "target": target}
        if case["train"]:
            st["g_logprob"] = normal(t) / t
            st["g_entropy"] = torch.full((t,), 0.01 / t, device="cuda")
        return st
    # a teacher's entries: distinct indices, log probabilities in descending order, some mass left over
    step = torch.randint(1, max(2, (v - 1) // max(1, k - 1) + 1) if k > 1 else 2, (t, 1), generator=gen, device="cuda")
    start = torch.randint(0, v, (t, 1), generator=gen, device="cuda")
    index = (start + step * torch.arange(k, device="cuda")) % v
    score = torch.cat([2 * normal(t, k) + 2, normal(t, 1)], 1)
    lp = torch.log_softmax(score.double(), 1).float()[:, :k]
    lp = lp.sort(dim=1, descending=True).values
    x.scatter_add_(1, index, lp.clamp(min=-6) + 8 + 0.5 * normal(t, k))
    weight = (torch.rand((t,), generator=gen, device="cuda") < case["kept"]).float()
    weight[0] = 1.0
    return {"case": case, "x": x.to(dt), "index": index.contiguous(), "lp": lp.contiguous(), "weight": weight}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return (_run_own if own else _run_plain)[case["op"]](state, case)


def _norm_plain(s, case):
    x = s["x"].float()
    xc = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + 1e-5)
    xh = xc * rstd
    y = (xh * s["w"] + s["b"]).to(s["x"].dtype)
    if not case["train"]:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * s["w"]
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dw": (dy * xh).sum(0), "db": dy.sum(0)}


def _norm_own(s, case):
    from scmomer_amd.norm import layer_norm
    if not case["train"]:
        return {"y": layer_norm(s["x"], s["w"], s["b"], 1e-5)}
    x, w, b = (s[n].detach().requires_grad_() for n in ("x", "w", "b"))
    y = layer_norm(x, w, b, 1e-5)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _top(x, k):
    """the k largest of each row, the lowest index first among equals"""
    bits = x.float().add(0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -2147483648 - bits, bits)                  # the order of the values
    key = order * 4294967296 + (4294967295 - torch.arange(x.shape[1], device=x.device))
    return torch.topk(key, k, dim=1).indices


def _score_plain(s, case):
    x, target, k = s["x"], s["target"], case["k"]
    z = x.float() / case["tau"]
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    logp = z - lse
    p = e / total
    ent = -torch.where(p > 0, p * logp, 0).sum(1)
    used = target != IGNORE
    at = torch.where(used, target, 0)[:, None]
    lp = torch.where(used, logp.gather(1, at)[:, 0], 0)
    out = {"logprob": lp, "entropy": ent, "lse": lse[:, 0]}
    if k:
        top = _top(x, k)
        out["top_logprob"], out["top_index"] = logp.gather(1, top), top
    if case["train"]:
        g = torch.where(used, s["g_logprob"], 0)[:, None]
        dz = -p * g - torch.where(p > 0, s["g_entropy"][:, None] * p * (logp + ent[:, None]), 0)
        dz.scatter_add_(1, at, g)
        out["dx"] = (dz / case["tau"]).to(x.dtype)
    return out


def _score_own(s, case):
    from scmomer_amd.logits import token_logprobs
    x = s["x"].detach().requires_grad_() if case["train"] else s["x"]
    r = token_logprobs(x, s["target"], k=case["k"], temperature=case["tau"], ignore_index=IGNORE)
    out = {"logprob": r.logprob, "entropy": r.entropy, "lse": r.lse}
    if case["k"]:
        out["top_logprob"], out["top_index"] = r.top_logprob, r.top_index
    if case["train"]:
        out["dx"], = torch.autograd.grad((r.logprob, r.entropy), (x,), (s["g_logprob"], s["g_entropy"]))
        out = {n: t.detach() for n, t in out.items()}
    return out


def _distill_plain(s, case):
    x, index, lp, w = s["x"], s["index"], s["lp"], s["weight"]
    z = x.float() / case["tau"]
    q = torch.exp(lp)
    if case["tail"]:
        r = (1 - torch.exp(lp.double()).sum(1, keepdim=True)).clamp(min=0).float()
    else:
        lp = lp - torch.log(q.sum(1, keepdim=True))
        q = torch.exp(lp)
        r = torch.zeros_like(q[:, :1])
    m = z.max(1, keepdim=True).values
    lse = m + torch.log(torch.exp(z - m).sum(1, keepdim=True))
    rest = z.scatter(1, index, -math.inf)
    mr = rest.max(1, keepdim=True).values
    some = mr > -math.inf
    mr = torch.where(some, mr, 0)
    er = torch.exp(rest - mr)
    sr = er.sum(1, keepdim=True)
    r = torch.where(some, r, 0)
    lse_rest = torch.where(some, mr + torch.log(sr), 0)
    zi = z.gather(1, index)
    row = (q * (lp - zi + lse)).sum(1) + torch.where(r > 0, r * (torch.log(r) - lse_rest + lse), 0)[:, 0]
    wsum = w.sum()
    dz = (q.sum(1, keepdim=True) + r) * torch.exp(z - lse) - torch.where(some, r * er / sr, 0)
    dz.scatter_add_(1, index, -q)
    dz *= (w / wsum)[:, None]
    return {"loss": torch.where(w > 0, w * row, 0).sum() / wsum, "dx": (dz / case["tau"]).to(x.dtype)}


def _distill_own(s, case):
    from scmomer_amd.logits import topk_distillation, topk_distillation_grad
    kw = dict(temperature=case["tau"], tail=case["tail"], weight=s["weight"])
    if case["fused"]:
        loss, dx = topk_distillation_grad(s["x"], s["index"], s["lp"], **kw)
        return {"loss": loss, "dx": dx}
    x = s["x"].detach().requires_grad_()
    loss = topk_distillation(x, s["index"], s["lp"], **kw)
    dx, = torch.autograd.grad(loss, (x,))
    return {"loss": loss.detach(), "dx": dx}


_run_plain = {"norm": _norm_plain, "score": _score_plain, "distill": _distill_plain}
_run_own = {"norm": _norm_own, "score": _score_own, "distill": _distill_own}


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    t, b = case["rows"], WIDTH[case["dtype"]]
    if case["op"] == "norm":
        d = case["dim"]
        n = t * d
        if case["train"]:     # x and dy read; y and dx written; the weight, the bias and their gradients
            return {"bytes": 4 * n * b + 16 * d, "flops": 19 * n}
        return {"bytes": 2 * n * b + 8 * d, "flops": 7 * n}
    n, k = t * case["vocab"], case["k"]
    if case["op"] == "score":     # logits and targets read; three numbers and the alternatives a row written
        byt, fl = n * b + t * (8 + 12 + 12 * k), 7 * n
        if case["train"]:
            byt, fl = byt + n * b + 8 * t, fl + 6 * n
        return {"bytes": byt, "flops": fl}
    return {"bytes": 2 * n * b + t * (4 + 12 * k), "flops": 11 * n}     # logits and entries read, the gradient written


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s, case)
    width = max(1, (1 << 26) // case["vocab"])
    total = s["weight"].double().sum() if case["op"] == "distill" else None
    blocks = []
    for lo in range(0, case["rows"], width):
        part = {n: (v[lo:lo + width] if torch.is_tensor(v) else v) for n, v in s.items()}
        blocks.append(_exact_score(part, case) if case["op"] == "score" else _exact_distill(part, case, total))
    out = {n: torch.cat([blk[n] for blk in blocks]) for n in blocks[0] if n != "loss"}
    if case["op"] == "distill":
        out = {"loss": torch.stack([blk["loss"] for blk in blocks]).sum(), "dx": out["dx"]}
    return out


def _exact_norm(s, case):
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    sd = torch.sqrt(var + 1e-5)
    unit = (x - mean) / sd
    out = {"y": unit * w + b}
    if case["train"]:
        d = case["dim"]
        dy = s["dy"].double()
        a = dy * w
        out["dx"] = (d * a - a.sum(1, keepdim=True) - unit * (a * unit).sum(1, keepdim=True)) / (d * sd)
        out["dw"], out["db"] = (dy * unit).sum(0), dy.sum(0)
    return out


def _exact_score(s, case):
    x = s["x"].double()
    logp = torch.log_softmax(x / case["tau"], dim=1)
    lse = torch.logsumexp(x / case["tau"], dim=1)
    p = logp.exp()
    surprise = torch.nan_to_num(logp, neginf=0.0)
    ent = -(p * surprise).sum(1)
    pad = s["target"] == IGNORE
    t = s["target"].clamp(min=0)
    out = {"logprob": logp.gather(1, t[:, None]).squeeze(1).masked_fill(pad, 0.0), "entropy": ent, "lse": lse}
    if case["k"]:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["k"]]
        out["top_logprob"], out["top_index"] = logp.gather(1, order), order
    if case["train"]:
        g = s["g_logprob"].double().masked_fill(pad, 0.0)
        dz = -p * (g[:, None] + s["g_entropy"].double()[:, None] * (surprise + ent[:, None]))
        dz[torch.arange(len(t), device=t.device), t] += g
        out["dx"] = dz / case["tau"]
    return out


def _exact_distill(s, case, total):
    logp = torch.log_softmax(s["x"].double() / case["tau"], dim=1)
    p = logp.exp()
    q = s["lp"].double().exp()
    named = torch.zeros_like(p, dtype=torch.bool).scatter_(1, s["index"], True)
    target = torch.zeros_like(p)
    if case["tail"]:
        r = (1 - q.sum(1)).clamp(min=0) * (~named).any(1)
    else:
        q, r = q / q.sum(1, keepdim=True), torch.zeros_like(q[:, 0])
    target.scatter_(1, s["index"], q)
    p_rest = p.masked_fill(named, 0).sum(1)
    share = torch.where(p_rest > 0, r / p_rest, 0)
    row = (torch.special.xlogy(q, q) - q * logp.gather(1, s["index"])).sum(1)
    row = row + torch.special.xlogy(r, r) - torch.special.xlogy(r, p_rest)
    w = s["weight"].double()
    target = target + p.masked_fill(named, 0) * share[:, None]
    dz = ((q.sum(1) + r)[:, None] * p - target) * (w / total)[:, None]
    return {"loss": (w * row).sum() / total, "dx": dz / case["tau"]}
