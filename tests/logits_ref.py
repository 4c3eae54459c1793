"""The vocabulary-row operators in 64 bits, row by row, with error bounds.

Each function returns its results and, for every float result, how far an fp32
computation of the stated form may be off.  u = 2^-24 is fp32's half step.

  d_v = (z_v - m)/t in fp32: a subtraction, the rounded 1/t (or log2(e)/t) and a
  product, so |err| <= 4 u |d_v|.
  e_v = exp(d_v): relative 4 u |d_v| from its argument and 4 u of its own.
  s: a sum of positive terms, at most CHAIN additions one after another on any
  term (64 values a thread, then trees); sum_v p_v |d_v| <= log s <= log V, so
  s is off by at most A = (4 log V + 4 + CHAIN) u relative, log s by A and its
  own rounding, log p by that and 4 u |d|.
"""
import numpy as np

U = 2.0 ** -24
CHAIN = 96
TAIL_MIN = 2.0 ** -20


def half_step(dtype):
    """(relative half step, absolute) of a result type.  fp16's smallest step is 2^-24.  An
    exponential below 2^-126 may be taken as 0: with factors up to 2^26 that is 2^-100 at most."""
    return {"f32": (2.0 ** -24, 2.0 ** -100), "bf16": (2.0 ** -8, 2.0 ** -100),
            "f16": (2.0 ** -11, 2.0 ** -25)}[dtype]


def a_bound(V):
    return (4 * np.log(max(V, 2)) + 4 + CHAIN) * U


def log_softmax(row, tau):
    """log p in 64 bits (None for a row without a distribution), the largest logit, log of the sum."""
    if np.isnan(row).any() or (row == np.inf).any():
        return None, np.nan, np.nan
    m = row.max()
    if m == -np.inf:
        return np.full(row.shape, -np.inf), m, -np.inf
    with np.errstate(over="ignore"):
        y = (row - m) / tau
    ls = np.log(np.exp(y).sum())
    return y - ls, m, ls


def logp_bound(logp, V):
    """|err| of log p: d's, log s's and the final subtraction's."""
    lp = np.where(np.isfinite(logp), np.abs(logp), 0.0)
    return a_bound(V) + 8 * U * (lp + np.log(max(V, 2))) + 4 * U


def entropy(logp):
    fin = np.isfinite(logp)
    return float(-(np.exp(logp[fin]) * logp[fin]).sum())


def entropy_bound(V):
    """H = log s - t/s, t a sum of e d with sum p |d| <= log V: relative A each."""
    lv = np.log(max(V, 2))
    return a_bound(V) * (2 + 3 * lv) + 8 * U * (1 + lv)


def score(z, ids, tau, K):
    """logp, entropy, top_ids, top_logp of rows z [N, V] (64-bit copies of the inputs)."""
    N, V = z.shape
    lp, H = np.zeros(N), np.zeros(N)
    ti, tl = np.full((N, K), -1, np.int64), np.full((N, K), -np.inf)
    lp_tol, tl_tol = np.zeros(N), np.zeros((N, K))
    for n in range(N):
        logp, _, _ = log_softmax(z[n], tau)
        given = 0 <= ids[n] < V
        if logp is None:
            lp[n] = np.nan if given else 0.0
            H[n] = np.nan
            tl[n] = np.nan
            continue
        if given:
            lp[n] = logp[ids[n]]
            lp_tol[n] = logp_bound(logp[ids[n]], V)
        H[n] = entropy(logp)
        order = np.argsort(-z[n], kind="stable")[:K]
        order = order[z[n][order] > -np.inf]
        ti[n, :len(order)] = order
        tl[n, :len(order)] = logp[order]
        tl_tol[n, :len(order)] = logp_bound(logp[order], V)
    return {"logp": lp, "entropy": H, "top_ids": ti, "top_logp": tl, "logp_tol": lp_tol,
            "entropy_tol": entropy_bound(V), "top_logp_tol": tl_tol}


def score_grad(z, ids, tau, a, b, dtype):
    """Gradient of sum a logp + b entropy; a or b may be None."""
    N, V = z.shape
    d, tol = np.zeros((N, V)), np.zeros((N, V))
    for n in range(N):
        given = 0 <= ids[n] < V
        an = float(a[n]) if a is not None and given else 0.0
        bn = float(b[n]) if b is not None else 0.0
        if an == 0.0 and bn == 0.0:
            continue
        logp, m, _ = log_softmax(z[n], tau)
        if logp is None:
            d[n] = np.nan
            continue
        if m == -np.inf:
            continue
        p, H = np.exp(logp), entropy(logp)
        lp0 = np.where(np.isfinite(logp), logp, 0.0)
        d[n] = -p * (an + bn * (lp0 + H))
        err = logp_bound(logp, V) + 8 * U
        tol[n] = p * (abs(an) * err + abs(bn) * (np.abs(lp0 + H) * err + err + entropy_bound(V)))
        if given:
            d[n, ids[n]] += an
            tol[n, ids[n]] += 2 * U * abs(an)
        tol[n] += 4 * U * np.abs(d[n])
    rel, least = half_step(dtype)
    return d / tau, (tol / tau) * (1 + rel) + rel * np.abs(d / tau) + least


def distill(z, t_ids, t_vals, tau, tail, w, scale, dtype):
    """loss [N] and the gradient [N, V] of scale * sum loss."""
    N, V = z.shape
    K = t_ids.shape[1]
    loss, d = np.zeros(N), np.zeros((N, V))
    ltol, dtol = np.zeros(N), np.zeros((N, V))
    for n in range(N):
        wn = 1.0 if w is None else float(w[n])
        if wn == 0.0:
            continue
        ok = (t_ids[n] >= 0) & (t_ids[n] < V)
        ids, t = t_ids[n][ok], t_vals[n][ok].astype(np.float64)
        if np.isnan(t).any() or (t == np.inf).any():
            loss[n], d[n] = np.nan, np.nan
            continue
        if tail:
            q = np.exp(t)
        else:
            q = np.exp((t - t.max()) / tau) if len(t) and t.max() > -np.inf else np.zeros(len(t))
            q = q / q.sum() if q.sum() > 0 else q
        fin = t[np.isfinite(t)]
        qrel = (K + 24 + 4 * (np.ptp(fin) if len(fin) else 0.0) / tau) * U
        dense = np.zeros(V)
        np.add.at(dense, ids, q)
        qr, qr_err = 0.0, 0.0
        if tail:
            qr = 1.0 - q.sum()
            qr_err = (K + 8) * U
            qr = 0.0 if qr < TAIL_MIN else qr
        logp, m, _ = log_softmax(z[n], tau)
        if logp is None:
            loss[n], d[n] = np.nan, np.nan
            continue
        if m == -np.inf:
            loss[n] = wn * (np.inf if q.sum() + qr > 0 else 0.0)
            continue
        p, err = np.exp(logp), logp_bound(logp, V) + 8 * U
        on = dense > 0
        with np.errstate(divide="ignore", invalid="ignore"):
            terms = dense[on] * (np.log(dense[on]) - logp[on])
        L = terms.sum()
        fin = np.where(np.isfinite(logp[on]), np.abs(logp[on]), 0.0)
        size = dense[on] * (np.abs(np.log(dense[on])) + fin + 1)
        Lt = (size * (qrel + 8 * U)).sum() + (dense[on] * err[on]).sum() + (K + 8) * U * size.sum()
        total = q.sum() + qr
        g = total * p - dense
        gt = p * total * (err + 8 * U + qrel) + dense * (qrel + 4 * U)
        if qr > 0.0:
            rest = np.ones(V, bool)
            rest[ids] = False
            with np.errstate(divide="ignore"):
                lr = np.log(p[rest].sum())
                L += qr * (np.log(qr) - lr)
            if np.isfinite(lr):
                size = abs(np.log(qr)) + abs(lr) + 1
                Lt += qr_err * size + qr * (2 * err[np.isfinite(logp)].max() + 8 * U * size)
                share = p[rest] * qr / np.exp(lr)
                g[rest] -= share
                gt[rest] += share * (2 * err[rest] + 8 * U + qr_err / qr) + p[rest] * qr_err
        loss[n], ltol[n] = wn * L, abs(wn) * (Lt + 4 * U * abs(L) if np.isfinite(L) else 0.0)
        k = wn * scale / tau
        d[n], dtol[n] = k * g, abs(k) * (gt + 4 * U * np.abs(g))
    rel, least = half_step(dtype)
    return loss, ltol, d, dtol * (1 + rel) + rel * np.abs(d) + least


def close(got, want, tol, what):
    """got equals want within tol; infinities and NaN have to be in the same places."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    tol = np.broadcast_to(tol, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    inf = np.isinf(want)
    assert np.array_equal(inf, np.isinf(got)) and np.array_equal(got[inf], want[inf]), f"{what}: infinities differ"
    fin = np.isfinite(want)
    err = np.abs(got[fin] - want[fin])
    over = err > tol[fin]
    assert not over.any(), (f"{what}: {over.sum()} of {over.size} outside; worst {err.max():.3e} where "
                            f"{tol[fin][int(np.argmax(err - tol[fin]))]:.3e} is allowed")
