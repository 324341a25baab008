"""The fine-tuning losses and the clipping in float64 numpy, from the formulas in include/znn_cuda.h (the reference has no
counterpart).  Checker only."""
import numpy as np


def rows(x, targets, inv_temp=1.0):
    """(logp, entropy, p, log p, in_use, bad) of the logits x [M, N]; rows that are not in use hold zeros."""
    x = np.asarray(x, np.float64)
    t = np.asarray(targets, np.int64)
    M, N = x.shape
    bad, in_use = t >= N, (t >= 0) & (t < N)
    logp, ent = np.zeros(M), np.zeros(M)
    p, lp = np.zeros((M, N)), np.full((M, N), -np.inf)
    for i in np.flatnonzero(in_use):
        r = x[i]
        if np.all(r == -np.inf):
            logp[i] = -np.inf
            continue
        with np.errstate(invalid="ignore", divide="ignore"):
            d = (r - np.max(r)) * inv_temp
            e = np.exp(d)
            s = e.sum()
            lp[i], p[i] = d - np.log(s), e / s
            logp[i] = lp[i, t[i]]
            ent[i] = np.log(s) - np.where(e > 0, d * e, 0.0).sum() / s if np.isfinite(s) else np.nan
    logp[bad] = np.nan
    return logp, ent, p, lp, in_use, bad


def rows_grad(x, targets, dlogp, dentropy, inv_temp=1.0):
    """d/dx of sum_i dlogp_i logp_i + dentropy_i entropy_i"""
    logp, ent, p, lp, in_use, _ = rows(x, targets, inv_temp)
    out = np.zeros_like(p)
    for i in np.flatnonzero(in_use):
        if np.all(np.asarray(x[i]) == -np.inf):
            continue
        hot = np.zeros(p.shape[1])
        hot[targets[i]] = 1.0
        with np.errstate(invalid="ignore"):
            inner = np.where(p[i] > 0, p[i] * (lp[i] + ent[i]), 0.0)
            out[i] = inv_temp * (np.where(hot == p[i], 0.0, dlogp[i] * (hot - p[i])) - dentropy[i] * inner)   # 0 times an infinite slope is 0
    return out


def policy(x, targets, old, adv, ref=None, weights=None, clip=(0.2, 0.2), kl=0.0, ce=0.0, inv_temp=1.0):
    logp, ent, _, _, in_use, bad = rows(x, targets, inv_temp)
    M = len(logp)
    w = np.ones(M) if weights is None else np.asarray(weights, np.float64)
    counted = (in_use | bad) & (w != 0)
    use = in_use & (w != 0)
    n = int(counted.sum())
    if weights is None:
        w = np.full(M, 1.0 / max(n, 1))
    token, g, h = np.zeros(M), np.zeros(M), np.zeros(M)
    for i in np.flatnonzero(use):
        A = float(adv[i])
        if A != 0.0:
            r = np.exp(logp[i] - float(old[i]))
            a, b = r * A, min(max(r, 1.0 - clip[0]), 1.0 + clip[1]) * A
            token[i] -= min(a, b)
            g[i] -= a if a <= b else 0.0
        if kl != 0.0:
            with np.errstate(invalid="ignore", over="ignore"):
                q = float(ref[i]) - logp[i]
                token[i] += kl * (np.exp(q) - q - 1.0 if q < np.inf else q)   # the limit, not inf - inf
                g[i] += kl * (1.0 - np.exp(q))
        token[i] -= ce * ent[i]
        h[i] = -ce
    used_logp = np.where(use | (bad & counted), logp, 0.0)
    grad = rows_grad(x, np.where(use, targets, -1), np.where(use, w * g, 0.0), np.where(use, w * h, 0.0), inv_temp)
    token = np.where(bad & counted, np.nan, token)
    loss = float((w * token)[counted].sum()) if n else 0.0
    return {"loss": loss, "rows": n, "token_loss": token, "logp": used_logp, "entropy": np.where(use, ent, 0.0), "dlogits": grad}


def preference(logp, offsets, ref=None, targets=None, beta=0.1, smoothing=0.0, margin=0.0, by_length=False, dlogp=None):
    logp = np.asarray(logp, np.float64)
    M, P = len(logp), (len(offsets) - 1) // 2
    d = logp if ref is None else logp - np.asarray(ref, np.float64)
    kept = np.ones(M, bool) if targets is None else np.asarray(targets) >= 0
    out = np.zeros(M) if dlogp is None else np.array(dlogp, np.float64)
    rewards, pair = np.zeros(2 * P), np.zeros(P)
    for p in range(P):
        o = [int(v) for v in offsets[2 * p:2 * p + 3]]
        if o[0] < 0 or o[1] < o[0] or o[2] < o[1] or o[2] > M:
            rewards[2 * p:2 * p + 2] = pair[p] = np.nan
            continue
        share = []
        for k in range(2):
            sl = slice(o[k], o[k + 1])
            n = kept[sl].sum()
            share.append(beta / n if by_length and n else 0.0 if by_length else beta)
            rewards[2 * p + k] = share[k] * d[sl][kept[sl]].sum()
        m = rewards[2 * p] - rewards[2 * p + 1] - margin
        pair[p] = (1 - smoothing) * np.logaddexp(0, -m) + (smoothing * np.logaddexp(0, m) if smoothing else 0.0)   # 0 of an infinite margin
        slope = (smoothing * np.exp(-np.logaddexp(0, -m)) - (1 - smoothing) * np.exp(-np.logaddexp(0, m))) / P
        for k, sign in ((0, 1.0), (1, -1.0)):
            sl = slice(o[k], o[k + 1])
            out[sl] = np.where(kept[sl], sign * slope * share[k], 0.0)
    return {"loss": pair.mean(), "pair_loss": pair, "rewards": rewards, "dlogp": out}


def grad_norm(grads, max_norm=np.inf, grad_scale=1.0):
    with np.errstate(invalid="ignore"):
        norm = abs(grad_scale) * np.sqrt(sum(float((np.asarray(g, np.float64) ** 2).sum()) for g in grads))
    return norm, 0.0 if not np.isfinite(norm) else max_norm / norm if norm > max_norm else 1.0
