"""Losses over vocabulary logits in float64 numpy: values and gradients from the formulas.

Every function takes logits [n, V] (any float dtype, read as float64) and returns its outputs in the order of the
kdn_b200 function of that name, the gradient last.  A row whose label is ``ignore`` (whose first teacher id is
negative) counts for nothing.
"""

import numpy as np


def _log_softmax(x):
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(axis=-1, keepdims=True)
        d = x - m
        return d - np.log(np.exp(d).sum(axis=-1, keepdims=True))


def _rows(logits, labels, temperature, ignore):
    lq = _log_softmax(np.asarray(logits, np.float64) / temperature)
    labels = np.asarray(labels, np.int64)
    live = labels != ignore
    y = np.where(live, labels, 0)
    return lq, y, live, np.where(live, lq[np.arange(len(y)), y], 0.0)


def _through(lq, y, live, dlogps, temperature):
    """sum_t dlogps_t d logp_t / dz"""
    c = np.where(live, dlogps, 0.0) / temperature
    with np.errstate(invalid="ignore"):
        g = -c[:, None] * np.exp(lq)
    g[np.arange(len(y)), y] += c
    return np.where((c != 0.0)[:, None], g, 0.0)


def token_logprobs(logits, labels, dlogps, temperature=1.0, ignore=-100):
    lq, y, live, logps = _rows(logits, labels, temperature, ignore)
    return logps, _through(lq, y, live, np.asarray(dlogps, np.float64), temperature)


def _weights(weights, live):
    w = np.full(live.shape, 1.0 / max(1, int(live.sum()))) if weights is None else np.asarray(weights, np.float64)
    return np.where(live, w, 0.0)


def policy_loss(logits, actions, old_logps, advantages, ref_logps=None, weights=None, clip_low=0.2, clip_high=0.2,
                kl_coef=0.0, entropy_coef=0.0, temperature=1.0, ignore=-100):
    lq, y, live, logps = _rows(logits, actions, temperature, ignore)
    w = _weights(weights, live)
    with np.errstate(invalid="ignore", over="ignore"):
        plogp = np.where(lq == -np.inf, 0.0, np.exp(lq) * lq)
        H = np.where(live, -plogp.sum(-1), 0.0)
        r = np.exp(logps - np.asarray(old_logps, np.float64))
        a = np.asarray(advantages, np.float64)
        free, clipped = r * a, np.clip(r, 1.0 - clip_low, 1.0 + clip_high) * a
        each = -np.minimum(free, clipped) - entropy_coef * H
        slope = -np.where(free > clipped, 0.0, free)  # NaN where free is
        if ref_logps is not None and kl_coef:
            g = np.asarray(ref_logps, np.float64) - logps
            each = each + kl_coef * (np.expm1(g) - g)
            slope = slope - kl_coef * np.expm1(g)
        loss = np.where(w != 0.0, w * each, 0.0).sum()
        d = _through(lq, y, live, np.where(w != 0.0, w * slope, 0.0), temperature)
        bonus = plogp + np.exp(lq) * H[:, None]
        d = d + np.where((w != 0.0)[:, None], (w * entropy_coef / temperature)[:, None] * bonus, 0.0)
    return loss, logps, H, d


def preference_loss(logits, labels, cu_seqlens, ref_logps=None, beta=0.1, label_smoothing=0.0,
                    length_normalised=False, temperature=1.0, ignore=-100):
    lq, y, live, logps = _rows(logits, labels, temperature, ignore)
    gap = logps if ref_logps is None else np.where(live, logps - np.asarray(ref_logps, np.float64), 0.0)
    cu = [int(c) for c in cu_seqlens]
    pairs = (len(cu) - 1) // 2
    size = [max(1, int(live[cu[s]:cu[s + 1]].sum())) if length_normalised else 1 for s in range(2 * pairs)]
    ratios = np.array([gap[cu[s]:cu[s + 1]].sum() / size[s] for s in range(2 * pairs)])
    h = beta * (ratios[0::2] - ratios[1::2])
    log_sigmoid = lambda v: -np.logaddexp(0.0, -v)
    eps = label_smoothing
    loss = -((1 - eps) * log_sigmoid(h) + eps * log_sigmoid(-h)).mean()
    dh = (np.exp(log_sigmoid(h)) - (1 - eps)) * beta / pairs
    dlogps = np.zeros(len(y))
    for s in range(2 * pairs):
        dlogps[cu[s]:cu[s + 1]] = (dh[s // 2] if s % 2 == 0 else -dh[s // 2]) / size[s]
    return loss, ratios, logps, _through(lq, y, live, dlogps, temperature)


def distillation_loss(logits, teacher_logits, teacher_ids, teacher_lse=None, weights=None, temperature=1.0):
    z = np.asarray(logits, np.float64) / temperature
    t = np.asarray(teacher_logits, np.float64) / temperature
    ids = np.asarray(teacher_ids, np.int64)
    n, V = z.shape
    w = _weights(weights, ids[:, 0] >= 0)
    divergence, d = np.zeros(n), np.zeros((n, V))
    for r in range(n):
        if ids[r, 0] < 0:
            continue
        at = ids[r][(ids[r] >= 0) & (ids[r] < V)]
        tr = t[r][(ids[r] >= 0) & (ids[r] < V)]
        if at.size == 0:
            continue
        lq = _log_softmax(z[r][None])[0]
        q = np.exp(lq)
        lp = _log_softmax(tr[None])[0] if teacher_lse is None else tr - float(teacher_lse[r])
        p = np.exp(lp)
        divergence[r] = sum(pi * (li - lq[i]) for pi, li, i in zip(p, lp, at) if pi > 0)
        g = q * p.sum()
        if teacher_lse is not None:
            outside = np.ones(V, bool)
            outside[at] = False
            p_rest, log_q_rest = max(0.0, 1.0 - p.sum()), np.logaddexp.reduce(lq[outside], initial=-np.inf)
            g = q * (p.sum() + p_rest)
            if p_rest > 0:  # the share of an entry in the rest: q / q_rest, which both may be too small for
                divergence[r] += p_rest * (np.log(p_rest) - log_q_rest)
                if log_q_rest != -np.inf:
                    g[outside] -= p_rest * np.exp(lq[outside] - log_q_rest)
        np.add.at(g, at, -p)
        if w[r] != 0.0:
            d[r] = w[r] * temperature * g
    loss = temperature ** 2 * np.where(w != 0.0, w * divergence, 0.0).sum()
    return loss, divergence, d
