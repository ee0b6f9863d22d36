"""Row-by-row statements in 64 bits of the operators over vocabulary logits (top entries with the rest's log-mass, filtered
sampling, distillation), written from their definitions for the tests."""
import math

import numpy as np
import torch


def clean(x):
    """float64 rows as the operators order them: NaN is -inf, -0 is +0."""
    x = x.detach().cpu().to(torch.float64).numpy()
    return np.where(np.isnan(x), -np.inf, x) + 0.0


def order(row):
    return np.lexsort((np.arange(len(row)), -row))  # by value, then by index


def log_sum(z):
    if len(z) == 0 or z.max() == -np.inf:
        return -np.inf
    m = z.max()
    return np.inf if m == np.inf else m + math.log(np.exp(z - m).sum())


def top_logits(x, k, tau):
    rows = clean(x)
    vals, ids, rest = [], [], []
    for r in rows:
        o = order(r)
        vals.append(r[o[:k]])
        ids.append(o[:k])
        rest.append(log_sum(r[o[k:]] / tau))
    return np.array(vals), np.array(ids), np.array(rest)


def sample_row(row, q, temp, k, p, least):
    """(token, probability) of one cleaned float64 row."""
    o = order(row)
    m = row[o[0]]
    if m == -np.inf:
        return -1, 0.0
    if not temp > 0:
        return int(o[0]), 1.0
    V = len(row)
    n = min(k, V) if k > 0 else V
    with np.errstate(invalid="ignore"):
        w = np.where(row[o] == m, 1.0, np.exp((row[o] - m) / temp))
    w = np.where(row[o] == -np.inf, 0.0, w)
    keep = n
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[:n])[:-1]])
        keep = max(1, int(np.count_nonzero(before < p * w[:n].sum())))
    if least > 0:
        with np.errstate(invalid="ignore"):
            ok = (row[o] == m) | (row[o] - m >= temp * math.log(min(least, 1.0)))
        keep = min(keep, int(np.count_nonzero(ok)))
    keep = min(keep, int(np.count_nonzero(row[o] > -np.inf)))
    with np.errstate(divide="ignore", invalid="ignore"):
        race = np.where(w[:keep] > 0, w[:keep] / q[o[:keep]], 0.0)
    best = race.max()
    i = min(int(o[j]) for j in range(keep) if race[j] == best)
    j = int(np.nonzero(o == i)[0][0])
    return i, w[j] / w[:keep].sum()


def sample(x, q, temp, k, p, least):
    rows, q = clean(x), q.cpu().double().numpy()
    T = len(rows)
    get = lambda v, t: np.broadcast_to(np.asarray(v.cpu() if torch.is_tensor(v) else v, t), (T,))  # noqa: E731
    temp, p, least = (get(v, np.float32).astype(np.float64) for v in (temp, p, least))
    k = get(k, np.int32)
    out = [sample_row(rows[t], q[t], temp[t], int(k[t]), p[t], least[t]) for t in range(T)]
    return np.array([a for a, _ in out]), np.array([b for _, b in out])


def distill(x, values, ids, rest, tau, w):
    """Row losses, d sum(losses)/dx (both float64), and per row / element the sizes the error bounds are made of:
    (loss scale, gradient scale)."""
    x = x.detach().cpu().double().numpy()
    values, ids = clean(values), ids.cpu().numpy().astype(np.int64)
    T, V = x.shape
    loss, grad = np.zeros(T), np.zeros((T, V))
    lscale, gscale = np.zeros(T), np.zeros((T, V))
    for t in range(T):
        wt = 1.0 if w is None else float(w[t])
        ok = (ids[t] >= 0) & (ids[t] < V) & (values[t] > -np.inf)
        if wt == 0.0 or not ok.any() or (x[t] == -np.inf).all():
            continue
        if np.isnan(x[t]).any() or (x[t] == np.inf).any():
            loss[t], grad[t] = np.nan, np.nan
            continue
        i, v = ids[t][ok], values[t][ok] / tau
        z = (x[t] - x[t].max()) / tau  # (the loss does not change; a row at the type's lowest value keeps its digits)
        lse = log_sum(z)
        s = np.exp(z - lse)
        r = -np.inf if rest is None else float(rest[t])
        most = max(v.max(), r if r < np.inf else -np.inf)  # (as z: at temperature 2^-40 an entry of 11 is 1.2e13, spaced by 2^-9)
        v, r = v - most, r - most
        lt = log_sum(np.append(v, r))
        te, tr = np.exp(v - lt), math.exp(r - lt) if r > -np.inf else 0.0
        out = np.ones(V, bool)
        out[i] = False
        lse_o = log_sum(z[out])
        with np.errstate(invalid="ignore"):
            terms = np.where(te > 0, te * ((v - lt) - (z[i] - lse)), 0.0)
        loss[t] = terms.sum()
        lscale[t] = np.sum(np.where(te > 0, te * (np.abs(v - v.max()) + np.abs(z[i] - z.max())), 0.0)) + abs(lse - z.max()) + abs(lt - v.max()) + 1
        g = s.copy()
        gs = s.copy()
        if tr > 0:
            loss[t] += tr * ((r - lt) - (lse_o - lse)) if lse_o > -np.inf else np.inf
            lscale[t] += tr * (abs(r - lt) + abs(lse_o - lse)) if lse_o > -np.inf else 0
            if lse_o > -np.inf:
                share = np.where(out, np.exp(z - lse_o), 0.0)
                g -= tr * share
                gs += (tr + math.exp(lse_o - lse)) * share
        for e, p in zip(i, te):
            g[e] -= p
            gs[e] += p
        loss[t] *= wt * tau * tau
        lscale[t] *= abs(wt) * tau * tau
        grad[t] = wt * tau * g
        gscale[t] = abs(wt) * tau * gs
    return loss, grad, lscale, gscale
