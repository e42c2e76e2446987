"""
Cases for the operators a language model needs around its matrix products: layer
normalisation and its gradient, the embedding lookup and its gradient, and two costs on
the logits with their gradient (distillation from a teacher's largest logits, and a clipped
policy cost with a KL term).

``own`` False computes them in elementary torch operations in 32 bits; ``own`` True makes the
calls of this package's backend.  Orders: "rows" keeps the features (or the vocabulary) of
one item next to each other, memory shape (items, features); "cols" is neon's own order,
memory shape (features, items).  The backend's tensors always have the shape (features,
items); a "rows" buffer is handed over as its transposed view.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-5
_CLIP_LOW, _CLIP_HIGH, _KL = 0.2, 0.28, 0.05
_be = None


def listed():
    return [
        # one decoding step of a small batch: latency is all there is
        {"name": "ln_fprop step", "op": "ln_fprop", "order": "rows", "dtype": "bf16", "params": "f32",
         "features": 1024, "items": 32},
        # a training batch of 16 sequences of 2048 tokens
        {"name": "ln_fprop large", "op": "ln_fprop", "order": "rows", "dtype": "bf16", "params": "f32",
         "features": 4096, "items": 32768},
        # a batch in neon's own order, an odd width, fp32
        {"name": "ln_bprop cols", "op": "ln_bprop", "order": "cols", "dtype": "f32", "params": "f32",
         "features": 1001, "items": 4096},
        {"name": "ln_bprop large", "op": "ln_bprop", "order": "rows", "dtype": "bf16", "params": "f32",
         "features": 4096, "items": 32768},
        # tokens of one decoding step
        {"name": "lut_fprop step", "op": "lut_fprop", "order": "rows", "dtype": "f32", "vocab": 10000,
         "features": 512, "items": 64},
        {"name": "lut_fprop large", "op": "lut_fprop", "order": "rows", "dtype": "bf16", "vocab": 50257,
         "features": 2048, "items": 65536},
        # a text classifier's table: 20000 words, 128 features, 128 sentences of 16 words
        {"name": "lut_bprop small", "op": "lut_bprop", "order": "cols", "dtype": "f32", "params": "f32",
         "vocab": 20000, "features": 128, "items": 2048},
        # a training batch, word frequencies as in text
        {"name": "lut_bprop large", "op": "lut_bprop", "order": "rows", "dtype": "bf16", "params": "f32",
         "vocab": 50257, "features": 1024, "items": 131072},
        # an odd vocabulary in fp16, teacher's 50 largest logits
        {"name": "distill odd", "op": "distill", "order": "rows", "dtype": "f16", "vocab": 32003, "items": 1000,
         "top": 50, "grad": True},
        {"name": "distill large", "op": "distill", "order": "rows", "dtype": "bf16", "vocab": 131072, "items": 4096,
         "top": 64, "grad": True},
        # a batch of sampled answers
        {"name": "policy rows", "op": "policy", "order": "rows", "dtype": "bf16", "vocab": 50257, "items": 2048,
         "grad": True},
        # a word model in neon's own order: 10000 words, 64 sequences of 20 steps
        {"name": "policy cols", "op": "policy", "order": "cols", "dtype": "f32", "vocab": 10000, "items": 1280,
         "grad": True},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["ln_fprop", "ln_bprop", "lut_fprop", "lut_bprop", "distill", "policy"])
    case = {"op": op, "order": rng.choice(["rows", "rows", "cols"]), "dtype": rng.choice(["f32", "f16", "bf16", "bf16"])}
    if op in ("ln_fprop", "ln_bprop"):
        case["params"] = rng.choice(["f32", case["dtype"]])
        case["features"] = _log_uniform(rng, 64, 16384)
        if rng.random() < 0.6:                       # widths of models are mostly whole multiples
            case["features"] = max(64, case["features"] // 64 * 64)
        most = 1 << (26 if case["dtype"] == "f32" else 27)
        case["items"] = _log_uniform(rng, 1, min(65536, most // case["features"]))
    elif op in ("lut_fprop", "lut_bprop"):
        case["features"] = _log_uniform(rng, 32, 4096)
        if rng.random() < 0.7:
            case["features"] = max(32, case["features"] // 32 * 32)
        most = 1 << (26 if case["dtype"] == "f32" or op == "lut_bprop" else 27)
        case["vocab"] = _log_uniform(rng, 256, min(262144, most // case["features"]))
        case["items"] = _log_uniform(rng, 1, min(262144, most // case["features"]))
        if op == "lut_bprop":
            case["params"] = rng.choice(["f32", case["dtype"]])
    else:
        case["vocab"] = _log_uniform(rng, 256, 131072)
        if rng.random() < 0.6:
            case["vocab"] = max(256, case["vocab"] // 64 * 64)
        most = 1 << (27 if case["dtype"] == "f32" else 28)
        case["items"] = _log_uniform(rng, 1, min(16384, most // case["vocab"]))
        if op == "distill":
            case["top"] = _log_uniform(rng, 1, 128)
        case["grad"] = rng.random() < 0.75
    return case


# ---------------------------------------------------------------- inputs
def _word_probabilities(vocab):
    """Frequencies of words by rank, as in text: 1 / (rank + 2.7)."""
    p = 1.0 / (np.arange(vocab, dtype=np.float64) + 2.7)
    return p / p.sum()


def _words(gen, vocab, items):
    """Word numbers with those frequencies; frequent words lie anywhere in the vocabulary."""
    cdf = torch.from_numpy(np.cumsum(_word_probabilities(vocab))).cuda()
    u = torch.rand(items, generator=gen, device="cuda", dtype=torch.float64)
    rank = torch.searchsorted(cdf, u).clamp_(max=vocab - 1)
    place = torch.randperm(vocab, generator=gen, device="cuda")
    return place[rank].to(torch.int32)


def _memory(case, features, items):
    return (items, features) if case["order"] == "rows" else (features, items)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    items, op = case["items"], case["op"]

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype).mul_(scale)

    t = {}
    if op in ("ln_fprop", "ln_bprop"):
        f, pt = case["features"], _DTYPES[case["params"]]
        along = 1 if case["order"] == "rows" else 0
        shape = _memory(case, f, items)
        # activations: every item with a scale and an offset of its own
        per_item = (items, 1) if along else (1, items)
        x = normal(*shape) * (0.5 + torch.rand(*per_item, generator=gen, device="cuda")) + normal(*per_item, scale=0.3)
        t["x"] = x.to(dt)
        t["gamma"] = (1 + normal(f, scale=0.1)).to(pt)
        if op == "ln_fprop":
            t["beta"] = normal(f, scale=0.1).to(pt)
            t["y"] = torch.empty(shape, dtype=dt, device="cuda")
            t["mean"] = torch.empty(items, device="cuda")
            t["rstd"] = torch.empty(items, device="cuda")
        else:
            xf = t["x"].float()
            t["mean"] = xf.mean(along).contiguous()
            t["rstd"] = torch.rsqrt(xf.var(along, unbiased=False) + _EPS).contiguous()
            del xf
            t["error"] = normal(*shape).to(dt)
            t["delta"] = torch.empty(shape, dtype=dt, device="cuda")
            t["grad_gamma"] = torch.empty(f, dtype=pt, device="cuda")
            t["grad_beta"] = torch.empty(f, dtype=pt, device="cuda")
    elif op == "lut_fprop":
        t["W"] = normal(case["vocab"], case["features"], scale=0.02).to(dt)
        t["ids"] = _words(gen, case["vocab"], items)
        t["out"] = torch.empty(_memory(case, case["features"], items), dtype=dt, device="cuda")
    elif op == "lut_bprop":
        t["ids"] = _words(gen, case["vocab"], items)
        t["error"] = normal(*_memory(case, case["features"], items)).to(dt)
        if case["order"] == "cols":                  # the layer's buffer for the transposed error
            t["error_t"] = torch.empty(items, case["features"], dtype=dt, device="cuda")
        t["dW"] = torch.empty(case["vocab"], case["features"], dtype=_DTYPES[case["params"]], device="cuda")
    else:
        v = case["vocab"]
        shape = _memory(case, v, items)
        z = normal(*shape, scale=2.0, dtype=dt)
        rows = z if case["order"] == "rows" else z.t()
        # items that pad the batch have weight 0; half-precision gradients are scaled up, as in training
        weight = 64.0 if case["dtype"] == "f16" else 1.0 / items
        t["weights"] = (torch.rand(items, generator=gen, device="cuda") < 0.85).float() * weight
        t["weights"][0] = weight
        if op == "distill":
            k = min(case["top"], v)
            # the teacher's words are all different, from a random progression through the vocabulary
            step = v // k
            first = torch.randint(0, v, (items, 1), generator=gen, device="cuda")
            ids = (first + step * torch.arange(k, device="cuda")) % v
            top = torch.gather(rows, 1, ids).float() + normal(items, k) + 2.0
            top, by = torch.sort(top, dim=1, descending=True)
            ids = torch.gather(ids, 1, by).to(torch.int32)
            if case["order"] == "cols":
                ids, top = ids.t(), top.t()
            t["top_ids"], t["top"] = ids.contiguous(), top.to(dt).contiguous()
        else:
            actions = torch.randint(0, v, (items,), generator=gen, device="cuda")
            logp = torch.gather(rows, 1, actions[:, None])[:, 0].float()
            for at in range(0, items, 1024):         # in pieces, for the memory that 32 bits take
                logp[at:at + 1024] -= torch.logsumexp(rows[at:at + 1024].float(), 1)
            t["actions"] = actions.to(torch.int32)
            t["old"] = logp + normal(items, scale=0.2)
            t["ref"] = logp + normal(items, scale=0.3)
            t["advantages"] = normal(items)
            t["logp"] = torch.empty(items, device="cuda")
        t["z"] = z
        t["cost"] = torch.empty(items, device="cuda")
        if case["grad"]:
            t["delta"] = torch.empty(shape, dtype=dt, device="cuda")
    state = {"case": dict(case), "t": t}
    if own:
        state["b"] = _backend_tensors(case, t)       # the same memory as tensors of the backend
    return state


def _backend_tensors(case, t):
    global _be
    from neon_b200 import gen_backend
    from neon_b200.tensor import B200Tensor, bfloat16
    if _be is None:
        _be = gen_backend(backend="b200", rng_seed=0)
    types = {torch.float32: np.float32, torch.float16: np.float16, torch.bfloat16: bfloat16, torch.int32: np.int32}

    def view(name, x):
        if x.dim() == 1:                             # one value per feature, or one per item
            shape = (x.shape[0], 1) if name in ("gamma", "beta", "grad_gamma", "grad_beta") else (1, x.shape[0])
            return B200Tensor(_be, shape, dtype=types[x.dtype], gpudata=x.data_ptr())
        b = B200Tensor(_be, tuple(x.shape), dtype=types[x.dtype], gpudata=x.data_ptr())
        return b.T if case["order"] == "rows" and name not in ("W", "dW") else b

    return {name: view(name, x) for name, x in t.items()}


# ---------------------------------------------------------------- one pass
def run(state):
    case, t = state["case"], state["t"]
    op = case["op"]
    if own:
        b = state["b"]
        if op == "ln_fprop":
            _be.compound_fprop_ln(b["x"], b["mean"], b["rstd"], b["gamma"], b["beta"], b["y"], _EPS)
            return {"y": t["y"], "mean": t["mean"], "rstd": t["rstd"]}
        if op == "ln_bprop":
            _be.compound_bprop_ln(b["delta"], b["grad_gamma"], b["grad_beta"], b["error"], b["x"], b["mean"],
                                  b["rstd"], b["gamma"])
            return {"delta": t["delta"], "grad_gamma": t["grad_gamma"], "grad_beta": t["grad_beta"]}
        if op == "lut_fprop":
            _be.compound_fprop_lut(b["ids"], b["W"], b["out"], scale=math.sqrt(case["features"]))
            return {"out": t["out"]}
        if op == "lut_bprop":
            _be.compound_bprop_lut(1, b["ids"], b["error"], b.get("error_t"), b["dW"], pad_idx=0,
                                   alpha=math.sqrt(case["features"]))
            return {"dW": t["dW"]}
        if op == "distill":
            _be.compound_distill(b["z"], b["top_ids"], b["top"], b["cost"], b.get("delta"), weights=b["weights"],
                                 temperature=2.0)
            out = {"cost": t["cost"]}
        else:
            _be.compound_policy(b["z"], b["actions"], b["old"], b["advantages"], b["cost"], b.get("delta"),
                                logp=b["logp"], ref_logp=b["ref"], weights=b["weights"],
                                clip=(_CLIP_LOW, _CLIP_HIGH), kl_coef=_KL)
            out = {"cost": t["cost"], "logp": t["logp"]}
        if case["grad"]:
            out["delta"] = t["delta"]
        return out
    if op == "ln_fprop":
        return _plain_ln_fprop(case, t)
    if op == "ln_bprop":
        return _plain_ln_bprop(case, t)
    if op == "lut_fprop":
        out = (t["W"][t["ids"].long()].float() * math.sqrt(case["features"])).to(t["W"].dtype)
        return {"out": out if case["order"] == "rows" else out.t().contiguous()}
    if op == "lut_bprop":
        return _plain_lut_bprop(case, t)
    return _plain_distill(case, t) if op == "distill" else _plain_policy(case, t)


def _plain_ln_fprop(case, t):
    along = 1 if case["order"] == "rows" else 0
    wide = (1, -1) if along else (-1, 1)
    x = t["x"].float()
    mean = x.mean(along, keepdim=True)
    x = x - mean
    rstd = 1.0 / torch.sqrt((x * x).mean(along, keepdim=True) + _EPS)
    y = x * rstd * t["gamma"].float().view(wide) + t["beta"].float().view(wide)
    return {"y": y.to(t["x"].dtype), "mean": mean.view(-1), "rstd": rstd.view(-1)}


def _plain_ln_bprop(case, t):
    along = 1 if case["order"] == "rows" else 0
    wide, tall = ((1, -1), (-1, 1)) if along else ((-1, 1), (1, -1))
    rstd = t["rstd"].view(tall)
    xhat = (t["x"].float() - t["mean"].view(tall)) * rstd
    dy = t["error"].float()
    grad_gamma, grad_beta = (dy * xhat).sum(1 - along), dy.sum(1 - along)
    g = dy * t["gamma"].float().view(wide)
    delta = rstd * (g - g.mean(along, keepdim=True) - xhat * (g * xhat).mean(along, keepdim=True))
    return {"delta": delta.to(t["x"].dtype),
            "grad_gamma": grad_gamma.to(t["gamma"].dtype), "grad_beta": grad_beta.to(t["gamma"].dtype)}


def _plain_lut_bprop(case, t):
    error = t["error"].float()
    if case["order"] == "cols":
        error = error.t()
    error = error * (t["ids"] != 0)[:, None]
    dw = torch.zeros(case["vocab"], case["features"], device="cuda")
    dw.index_add_(0, t["ids"], error)
    return {"dW": (dw * math.sqrt(case["features"])).to(t["dW"].dtype)}


def _plain_softmax(z, scale):
    """(softmax of the rows of z * scale, log of the sum, largest) in 32 bits."""
    z = z * scale
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    s = e.sum(1, keepdim=True)
    return e / s, torch.log(s), top


def _plain_distill(case, t):
    rows = case["order"] == "rows"
    z = (t["z"] if rows else t["z"].t()).float()
    ids, top = (t["top_ids"], t["top"]) if rows else (t["top_ids"].t(), t["top"].t())
    ids, w, temp = ids.long(), t["weights"][:, None], 2.0
    p, log_sum, largest = _plain_softmax(top.float(), 1.0 / temp)
    log_p = top.float() / temp - largest - log_sum
    q, log_sum, largest = _plain_softmax(z, 1.0 / temp)
    log_q = torch.gather(z, 1, ids) / temp - largest - log_sum
    out = {"cost": (w * (temp * temp * (p * (log_p - log_q)).sum(1, keepdim=True))).view(-1)}
    if case["grad"]:
        delta = q.scatter_add_(1, ids, -p).mul_(temp * w).to(t["z"].dtype)
        out["delta"] = delta if rows else delta.t().contiguous()
    return out


def _plain_policy(case, t):
    rows = case["order"] == "rows"
    z = (t["z"] if rows else t["z"].t()).float()
    act = t["actions"].long()[:, None]
    q, log_sum, largest = _plain_softmax(z, 1.0)
    # ratios next to the border of the clip: 64 bits
    logp = torch.gather(z, 1, act).double() - largest.double() - log_sum.double()
    ratio = torch.exp(logp - t["old"][:, None].double())
    adv, w = t["advantages"][:, None].double(), t["weights"][:, None].double()
    free, held = ratio * adv, ratio.clamp(1 - _CLIP_LOW, 1 + _CLIP_HIGH) * adv
    gap = t["ref"][:, None].double() - logp
    cost = w * (_KL * (torch.exp(gap) - gap - 1) - torch.minimum(free, held))
    out = {"cost": cost.float().view(-1), "logp": logp.float().view(-1)}
    if case["grad"]:
        slope = w * (_KL * (1 - torch.exp(gap)) - torch.where(free <= held, free, torch.zeros_like(free)))
        slope = slope.float()
        delta = (q * -slope).scatter_add_(1, act, slope).to(t["z"].dtype)
        out["delta"] = delta if rows else delta.t().contiguous()
    return out


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    t = prepare(case, seed)["t"]
    rows, op, n = case["order"] == "rows", case["op"], case["items"]

    def item_major(x):
        return x if rows else x.t()

    def laid_out(x):
        return x if rows else x.t().contiguous()

    if op in ("ln_fprop", "ln_bprop"):
        x, gamma = item_major(t["x"]).double(), t["gamma"].double()
        f = x.shape[1]
        if op == "ln_fprop":
            var, mean = torch.var_mean(x, dim=1, correction=0)
            rstd = (var + _EPS).pow(-0.5)
            y = torch.addcmul(t["beta"].double(), (x - mean[:, None]).mul_(rstd[:, None]), gamma)
            return {"y": laid_out(y), "mean": mean, "rstd": rstd}
        mean, rstd, dy = t["mean"].double(), t["rstd"].double(), item_major(t["error"]).double()
        hat = torch.empty_like(x)
        torch.sub(x, mean[:, None], out=hat)
        hat.mul_(rstd[:, None])
        # the Jacobian of one item is rstd * (1 - 1/f - hat hat'/f), applied to gamma * dy
        a = dy @ gamma / f
        b = torch.einsum("ij,ij,j->i", dy, hat, gamma) / f
        return {"delta": laid_out((dy * gamma - a[:, None] - hat * b[:, None]) * rstd[:, None]),
                "grad_gamma": torch.einsum("ij,ij->j", dy, hat), "grad_beta": torch.einsum("ij->j", dy)}
    if op == "lut_fprop":
        return {"out": laid_out(torch.index_select(t["W"].double(), 0, t["ids"]) * float(case["features"]) ** 0.5)}
    if op == "lut_bprop":
        order = torch.argsort(t["ids"].long(), stable=True)
        run_sum = torch.cumsum(torch.bincount(t["ids"].long(), minlength=case["vocab"]), 0)
        error = item_major(t["error"])
        dw = torch.zeros(case["vocab"], case["features"], dtype=torch.float64, device="cuda")
        cols = max(1, (1 << 26) // max(1, n))
        for c in range(0, case["features"], cols):      # differences of running sums, a few columns at a time
            s = torch.cumsum(error[:, c:c + cols].double()[order], 0)
            s = torch.cat([torch.zeros_like(s[:1]), s])
            s = s[run_sum]
            dw[:, c:c + cols] = torch.diff(s, dim=0, prepend=torch.zeros_like(s[:1]))
        dw[0] = 0
        return {"dW": dw * float(case["features"]) ** 0.5}
    z = item_major(t["z"])
    cost = torch.empty(n, dtype=torch.float64, device="cuda")
    logp = torch.empty(n, dtype=torch.float64, device="cuda")
    delta = torch.empty(n, case["vocab"], dtype=torch.float64, device="cuda") if case["grad"] else None
    for i in range(0, n, 512):
        part = slice(i, min(n, i + 512))
        w = t["weights"][part].double()
        if op == "distill":
            log_q = torch.log_softmax(z[part].double() / 2.0, 1)
            log_p = torch.log_softmax(item_major(t["top"])[part].double() / 2.0, 1)
            ids = item_major(t["top_ids"])[part].long()
            p = log_p.exp()
            cost[part] = 4.0 * w * (p * (log_p - log_q.gather(1, ids))).sum(1)
            if delta is not None:
                full = torch.zeros_like(log_q)
                full.scatter_add_(1, ids, p)
                delta[part] = 2.0 * w[:, None] * (log_q.exp() - full)
        else:
            log_q = torch.log_softmax(z[part].double(), 1)
            act = t["actions"][part].long()
            at = torch.arange(act.numel(), device="cuda")
            lp = log_q[at, act]
            adv, r = t["advantages"][part].double(), (lp - t["old"][part].double()).exp()
            d = t["ref"][part].double() - lp
            held = torch.where(adv >= 0, r > 1 + _CLIP_HIGH, r < 1 - _CLIP_LOW)
            limit = torch.where(adv >= 0, torch.full_like(r, 1 + _CLIP_HIGH), torch.full_like(r, 1 - _CLIP_LOW))
            cost[part] = w * (_KL * (torch.expm1(d) - d) - adv * torch.where(held, limit, r))
            logp[part] = lp
            if delta is not None:
                slope = w * (-_KL * torch.expm1(d) - torch.where(held, torch.zeros_like(r), adv * r))
                g = log_q.exp().mul_(-slope[:, None])
                g[at, act] += slope
                delta[part] = g
    out = {"cost": cost} if op == "distill" else {"cost": cost, "logp": logp}
    if delta is not None:
        out["delta"] = laid_out(delta)
    return out


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    n, op, size = case["items"], case["op"], _SIZE[case["dtype"]]
    if op in ("ln_fprop", "ln_bprop"):
        f = case["features"]
        tensors, per_feature = (2, 2) if op == "ln_fprop" else (3, 3)
        return {"bytes": tensors * f * n * size + per_feature * f * _SIZE[case["params"]] + 8 * n,
                "flops": (8 if op == "ln_fprop" else 14) * f * n}
    if op in ("lut_fprop", "lut_bprop"):
        f, v = case["features"], case["vocab"]
        if op == "lut_bprop":
            return {"bytes": f * n * size + f * v * _SIZE[case["params"]] + 4 * n, "flops": f * n + f * v}
        # rows of the table that are looked up at least once
        rows = float(-np.expm1(n * np.log1p(-_word_probabilities(v))).sum())
        return {"bytes": f * n * size + f * rows * size + 4 * n, "flops": f * n}
    v, grad = case["vocab"], case["grad"]
    per_item = case.get("top", 0) * (4 + size) + 8 if op == "distill" else 28
    return {"bytes": v * n * size * (2 if grad else 1) + per_item * n, "flops": (4 + 4 * grad) * v * n}
