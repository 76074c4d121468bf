"""The operators on a network's answers (dosma_amd.models.answers) in 64 bits, straight from their definitions: numpy, one
softmax per row, no attention to speed.  Test infrastructure only.

``z``: (rows, C) float64.  Every function takes the categories' scores with the implicit background already in front."""
import numpy as np

EPS32 = 2.0 ** -24  # half a step of float32, relative


def with_background(z):
    return np.concatenate([np.zeros(z.shape[:-1] + (1,)), z], axis=-1)


def log_softmax(z, T):
    """(log p, M, ln s); empty rows: log p = -inf."""
    with np.errstate(all="ignore"):
        M = np.max(z, axis=-1)
        d = (z - np.where(np.isinf(M) & (M < 0), 0.0, M)[..., None]) / T
        ls = np.log(np.sum(np.exp(d), axis=-1))
        lp = np.where(np.isneginf(z) & ~np.isnan(ls)[..., None], -np.inf, d - ls[..., None])
    return lp, np.where(np.isnan(ls), np.nan, M), ls  # a row with NaN or +inf: every result is NaN


def xlogx(p, lp):
    return np.where(p == 0, 0.0, p * np.where(p == 0, 0.0, lp))


def scores(z, T=1.0, labels=None, top=0, ignore=-1):
    lp, M, ls = log_softmax(z, T)
    cats = z.shape[-1]
    p = np.exp(lp)
    out = {"entropy": -np.sum(xlogx(p, lp), axis=-1), "norm": np.stack([M, ls], -1), "lp": lp}
    if labels is not None:
        labels = labels.astype(np.int64)
        ok = (labels >= 0) & (labels < cats)
        got = np.take_along_axis(lp, np.where(ok, labels, 0)[..., None], -1)[..., 0]
        out["log_prob"] = np.where(labels == ignore, 0.0, np.where(ok, got, np.nan))
    if top:
        order = np.argsort(-z, axis=-1, kind="stable")[..., :top]
        v = np.take_along_axis(z, order, -1)
        out["top_label"] = np.where(np.isneginf(v), -1, order).astype(np.int32)
        out["top_log_prob"] = np.take_along_axis(lp, order, -1)
    return out


def scores_grad(z, T=1.0, labels=None, a=None, b=None, ignore=-1):
    lp, M, _ = log_softmax(z, T)
    p = np.exp(lp)
    g = np.zeros_like(p)
    if a is not None:
        labels = labels.astype(np.int64)
        ok = (labels >= 0) & (labels < z.shape[-1]) & (labels != ignore)
        aa = np.where(labels == ignore, 0.0, np.where(ok, a, np.nan))[..., None]
        hit = np.zeros_like(p)
        np.put_along_axis(hit, np.where(ok, labels, 0)[..., None], ok[..., None].astype(float), -1)
        g = aa * (hit - p)
    if b is not None:
        H = -np.sum(xlogx(p, lp), axis=-1, keepdims=True)
        g = g - b[..., None] * (xlogx(p, lp) + p * H)
    return np.where(np.isneginf(M)[..., None], 0.0, g / T)


def teacher(labels, values, cats, T, tail):
    """(usable entry, q, log q, rest)."""
    ok = (labels >= 0) & (labels < cats)
    v = np.where(ok, values.astype(np.float64), -np.inf)
    with np.errstate(all="ignore"):
        if tail:
            q, lq = np.exp(v), v
            rest = 1.0 - q.sum(-1)
            rest = np.where((rest > labels.shape[-1] * EPS32) & ok.any(-1), rest, 0.0)
            return ok, q, lq, rest, ok.any(-1)
        m = v.max(-1, keepdims=True)
        e = np.exp((v - np.where(np.isneginf(m), 0.0, m)) / T)
        s = e.sum(-1, keepdims=True)
        q = np.where(ok & (s != 0), e / s, 0.0)
        return ok, q, np.log(q), np.zeros(labels.shape[:-1]), (s[..., 0] != 0)


def distill(z, labels, values, T=1.0, tail=False, w=None):
    """-> loss, log p(tail) and, with ``w``, the gradient of sum(w * loss)."""
    lp, M, _ = log_softmax(z, T)
    cats = z.shape[-1]
    ok, q, lq, rest, some = teacher(labels, values, cats, T, tail)
    idx = np.where(ok, labels, 0).astype(np.int64)
    inside = np.zeros(z.shape, dtype=bool)
    weight = np.zeros(z.shape)
    for k in range(labels.shape[-1]):  # (the same label twice: one after the other)
        old = np.take_along_axis(inside, idx[..., k:k + 1], -1)
        np.put_along_axis(inside, idx[..., k:k + 1], old | ok[..., k:k + 1], -1)
        acc = np.take_along_axis(weight, idx[..., k:k + 1], -1)
        np.put_along_axis(weight, idx[..., k:k + 1], acc + q[..., k:k + 1] * ok[..., k:k + 1], -1)
    with np.errstate(all="ignore"):
        lpk = np.take_along_axis(lp, idx, -1)
        loss = np.sum(np.where(q == 0, 0.0, q * (lq - lpk)), -1)
        outside = np.where(inside, -np.inf, lp)
        mo = outside.max(-1, keepdims=True)
        lt = (np.where(np.isneginf(mo), 0.0, mo) + np.log(np.sum(np.exp(outside - np.where(np.isneginf(mo), 0.0, mo)), -1, keepdims=True)))[..., 0]
        loss = loss + np.where(rest == 0, 0.0, rest * (np.log(rest) - lt))
        empty = np.isneginf(M) | ~some
        res = {"loss": np.where(empty, 0.0, loss), "log_tail": lt, "q": q, "rest": rest}
        if w is not None:
            p = np.exp(lp)
            g = (q.sum(-1) + rest)[..., None] * p - weight
            g = g - np.where(inside | (rest == 0)[..., None] | (p == 0), 0.0, rest[..., None] * np.exp(lp - lt[..., None]))
            res["grad"] = np.where(empty[..., None], 0.0, g * (w / T)[..., None])
    return res
