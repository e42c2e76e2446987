"""
The language-model operators from their formulas in numpy float64, and how far a kernel that
computes them in fp32 may be off: u = 2^-24 per rounding, `depth` roundings for a sum whose
longest chain has that many additions, and half a step of the stored type on top.
"""
import numpy as np

U = 2.0 ** -24
# ex2.approx and exp2f are within 2 ulp; expf and logf as well
EXP = 2.0 ** -22


def half_step(dtype):
    """Half a step relative to the value, and half of the smallest subnormal step."""
    name = np.dtype(dtype).name
    return {"float32": (U, 0.0), "float16": (2.0 ** -11, 2.0 ** -25), "bfloat16": (2.0 ** -8, 0.0)}[name]


def stored(value, tol, dtype):
    """Tolerance of ``value`` (known to ``tol``) after rounding to dtype."""
    rel, tiny = half_step(dtype)
    return tol + rel * (np.abs(value) + tol) + tiny


def depth(n):
    """Longest chain of additions of a sum over n values: at most n, and for long sums a share of
    it per thread plus the partial sums of the blocks."""
    return min(n, n // 128 + 700) + 16


def ln_fprop(x, gamma, beta, eps, dtype):
    """{name: (value, tolerance)} of y, mean, rstd."""
    x = x.astype(np.float64)
    f = x.shape[0]
    mean = x.mean(axis=0, keepdims=True)
    var = ((x - mean) ** 2).mean(axis=0, keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    h = (x - mean) * rstd
    g = 1.0 if gamma is None else gamma.astype(np.float64)
    b = 0.0 if beta is None else beta.astype(np.float64)
    y = h * g + b
    d = depth(f)
    tmean = (d + 2) * U * np.abs(x).mean(axis=0, keepdims=True)
    rel = (d + 8) * U + tmean * rstd * np.abs(h).mean(axis=0, keepdims=True) + (tmean * rstd) ** 2
    th = rstd * tmean + np.abs(h) * (rel + 4 * U)
    ty = np.abs(g) * th + 3 * U * (np.abs(h * g) + np.abs(b))
    return {"y": (y, stored(y, ty, dtype)), "mean": (mean, tmean + U * np.abs(mean)), "rstd": (rstd, rstd * (rel + 4 * U))}


def ln_bprop(e, x, mean, rstd, gamma, dtype, pdtype):
    """mean and rstd are the fp32 vectors that the kernel is given."""
    e, x, mean, rstd = (a.astype(np.float64) for a in (e, x, mean, rstd))
    f, n = x.shape
    h = (x - mean) * rstd
    g = e if gamma is None else e * gamma.astype(np.float64)
    a, b = g.mean(axis=0, keepdims=True), (g * h).mean(axis=0, keepdims=True)
    delta = rstd * (g - a - h * b)
    d = depth(f)
    ta = (d + 3) * U * np.abs(g).mean(axis=0, keepdims=True)
    tb = (d + 6) * U * np.abs(g * h).mean(axis=0, keepdims=True)
    td = rstd * (ta + np.abs(h) * tb + 8 * U * (np.abs(g) + np.abs(a) + np.abs(h * b)))
    d = depth(n)
    gg, gb = (e * h).sum(axis=1, keepdims=True), e.sum(axis=1, keepdims=True)
    return {"delta": (delta, stored(delta, td, dtype)),
            "grad_gamma": (gg, stored(gg, (d + 4) * U * np.abs(e * h).sum(axis=1, keepdims=True), pdtype)),
            "grad_beta": (gb, stored(gb, d * U * np.abs(e).sum(axis=1, keepdims=True), pdtype))}


def lut_fprop(ids, w, scale, dtype):
    w = w.astype(np.float64)
    ids = np.asarray(ids).reshape(-1)
    ok = (ids >= 0) & (ids < w.shape[0])
    out = np.where(ok, w[np.where(ok, ids, 0)].T * scale, 0.0)
    return {"out": (out, stored(out, 2 * U * np.abs(out), dtype))}


def lut_bprop(ids, e, dw, pad, alpha, beta, dtype):
    e = e.astype(np.float64)
    ids = np.asarray(ids).reshape(-1)
    out = np.zeros(dw.shape)
    size = np.zeros(dw.shape)
    for n, v in enumerate(ids):
        if 0 <= v < dw.shape[0] and v != pad:
            out[v] += e[:, n]
            size[v] += np.abs(e[:, n])
    count = np.bincount(ids[(ids >= 0) & (ids < dw.shape[0])], minlength=dw.shape[0])[:, None]
    old = beta * dw.astype(np.float64) if beta else 0.0
    value = alpha * out + old
    return {"dW": (value, stored(value, U * (abs(alpha) * (count + 4) * size + 3 * np.abs(old)), dtype))}


def _log_softmax(z):
    """log softmax over axis 0 of float64 logits, and the error bound of an fp32 evaluation."""
    with np.errstate(invalid="ignore"):
        top = z.max(axis=0, keepdims=True)
        s = np.exp(z - top).sum(axis=0, keepdims=True)
        logq = z - top - np.log(s)
    with np.errstate(all="ignore"):
        far = np.where(np.isfinite(z) & (z - top > -100), top - z, 0.0).max(axis=0, keepdims=True)
        size = np.abs(np.where(np.isfinite(top), top, 0.0))
    # arguments of the exponentials: 4 roundings of at most `far`; the sum; the logarithms; the maximum
    return logq, U * (4 * far + 2 * size + depth(z.shape[0]) + 16) + 4 * EXP


def distill(z, ids, top, w, temp, dtype):
    v, n = z.shape
    z, top = z.astype(np.float64), top.astype(np.float64)
    w = np.ones((1, n)) if w is None else w.reshape(1, -1).astype(np.float64)
    logq, tq = _log_softmax(z / temp)
    cost, tcost = np.zeros((1, n)), np.zeros((1, n))
    delta, tdelta = np.zeros((v, n)), np.zeros((v, n))
    for i in range(n):
        if w[0, i] == 0:
            continue
        use = (ids[:, i] >= 0) & (ids[:, i] < v) & (top[:, i] != -np.inf)
        if not use.any():
            continue
        at = ids[use, i]
        t = top[use, i] / temp
        lp = t - t.max() - np.log(np.exp(t - t.max()).sum())
        p = np.exp(lp)
        tp = U * (8 * np.abs(lp).max() + 2 * np.abs(t).max() + use.size + 16) + 4 * EXP
        scale = w[0, i] * temp * temp
        live = p > 0
        terms = p[live] * (lp[live] - logq[at[live], i])
        cost[0, i] = scale * terms.sum()
        lq = np.abs(logq[at[live], i])
        tcost[0, i] = abs(scale) * (p[live] * (tp * (2 + np.abs(lp[live]) + lq) + tq[0, i] + 8 * U * (np.abs(lp[live]) + lq))).sum()
        q = np.exp(logq[:, i])
        mass, tmass = np.zeros(v), np.zeros(v)
        np.add.at(mass, at, p)
        np.add.at(tmass, at, p * (tp + (use.size + 8) * U))
        delta[:, i] = w[0, i] * temp * (q - mass)
        tdelta[:, i] = abs(w[0, i]) * temp * (q * (tq[0, i] + 8 * U) + tmass)
    return {"cost": (cost, tcost + 2 * U * np.abs(cost)), "delta": (delta, stored(delta, tdelta, dtype))}


def policy(z, act, old, ref, adv, w, low, high, kl, dtype):
    v, n = z.shape
    z = z.astype(np.float64)
    row = lambda a: a.reshape(-1).astype(np.float64)                   # noqa: E731
    act, old, adv = act.reshape(-1), row(old), row(adv)
    ref = row(ref) if ref is not None and kl else None
    w = np.ones(n) if w is None else row(w)
    logq, tq = _log_softmax(z)
    cost, logp, delta = np.zeros((1, n)), np.zeros((1, n)), np.zeros((v, n))
    tc, tl, td = np.zeros((1, n)), np.zeros((1, n)), np.zeros((v, n))
    for i in range(n):
        a = act[i]
        if a < 0 or a >= v:
            continue
        l, t = logq[a, i], tq[0, i]
        logp[0, i], tl[0, i] = l, t + 4 * U * abs(l)
        if w[i] == 0:
            continue
        t = tl[0, i]
        r = np.exp(l - old[i])
        tr = r * (t + 2 * U * abs(l - old[i]) + 2 * EXP)
        free, held = r * adv[i], np.clip(r, 1 - low, 1 + high) * adv[i]
        c, s = -min(free, held), (-free if free <= held else 0.0)
        ec, es = abs(adv[i]) * tr + 4 * U * abs(free), abs(adv[i]) * tr + 4 * U * abs(free)
        if ref is not None:
            d = ref[i] - l
            ec += abs(kl) * (abs(np.expm1(d)) * (t + 2 * U * abs(d)) + (8 * U + 2 * EXP) * (np.exp(d) + abs(d) + 1))
            es += abs(kl) * (np.exp(d) * (t + 2 * U * abs(d) + 2 * EXP) + 8 * U)
            c, s = c + kl * (np.exp(d) - d - 1), s + kl * (1 - np.exp(d))
        cost[0, i], tc[0, i] = w[i] * c, abs(w[i]) * (ec + 4 * U * abs(c))
        hit = np.zeros(v)
        hit[a] = 1
        q = np.exp(logq[:, i])
        s, es = w[i] * s, abs(w[i]) * (es + 4 * U * abs(s))
        delta[:, i] = s * (hit - q)
        td[:, i] = es * (hit + q) + abs(s) * (q * (tq[0, i] + 8 * U) + 2 * U * hit)
    return {"cost": (cost, tc), "logp": (logp, tl), "delta": (delta, stored(delta, td, dtype))}


def check(name, got, want):
    """``want`` is (value, tolerance); infinities and NaN have to be where the value has them."""
    value, tol = (np.broadcast_to(np.asarray(a, np.float64), got.shape) for a in want)
    got = got.astype(np.float64)
    fine = np.isfinite(value)
    assert np.array_equal(got[~fine], value[~fine], equal_nan=True), "%s: infinities or NaN differ" % name
    assert np.isfinite(got[fine]).all(), "%s: not finite" % name
    off = np.abs(got[fine] - value[fine])
    bad = off > tol[fine]
    assert not bad.any(), "%s: %d of %d off, worst %.3g times the tolerance" % (
        name, bad.sum(), bad.size, (off[bad] / np.maximum(tol[fine][bad], 1e-300)).max())
