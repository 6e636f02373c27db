"""Float64 rows of the divergence from a teacher's best entries, by differences from the maxima throughout, so that neither far logits nor a
rest of tiny mass lose digits, with the error bounds that go with it."""
import numpy as np


def distill_far(z, ids, teacher, kind, T):
    """(L, dL/dz, bound of L, bound of dL/dz) of one row.

    Bounds: as in test_gpu_distill.py, but in what the logarithms come to and not in |z| / T: a distance from a maximum is exact but for
    the roundings of log2(e) / T and of its product, 2^-23 of itself, so log p, log q and log Q are off by 2^-21 of themselves plus
    2^-21 (ln V + 4), and p by 2^-24 (3 |d| + 8) of itself with d its teacher's distance from the best (none for given log-probabilities, whose
    exponential is off by 2^-24).  What the hardware's exponential flushes lies below 2^-126."""
    z, T = np.asarray(z, np.float64), float(T)
    V = z.size
    ids = np.asarray(ids)
    valid = (ids >= 0) & (ids < V)
    ids, t = ids[valid].astype(np.int64), np.asarray(teacher, np.float64)[valid]
    with np.errstate(invalid="ignore", divide="ignore", over="ignore", under="ignore"):
        y = (z - z.max()) / T
        lse = np.log(np.exp(y).sum())
        logq, q = y - lse, np.exp(y - lse)
        if kind == "logits":
            d = (t - t.max()) / T
            logp = d - np.log(np.exp(d).sum())
            P, perr = 0.0, 2.0 ** -24 * (3 * np.abs(np.maximum(d, -1e30)) + 8)
        else:
            logp = t
            P, perr = 1.0 - np.exp(logp).sum(), np.full(t.size, 2.0 ** -23)
        p = np.exp(logp)
        target, near = np.zeros(V), np.zeros(V)
        np.add.at(target, ids, p)
        np.add.at(near, ids, p * perr)
        some = p > 0
        L = (p * (logp - logq[ids]))[some].sum()
        far = np.abs(logp[some]) + np.abs(logq[ids][some])
        tolL = 2.0 ** -21 * ((p[some] * far).sum() + p.sum() * (np.log(V) + 4)) + (p[some] * perr[some] * (far + 1)).sum()
        g = p.sum() * q - target
        away = np.where(np.isfinite(y), -y, 0.0)
        tolg = max(p.sum(), 1.0) * q * 2.0 ** -21 * (4 + away) + near + 2.0 ** -22 * (q + target)
        if kind == "logprobs" and P > 0:
            free = np.ones(V, bool)
            free[ids] = False
            share = np.zeros(V)
            mr = z[free].max() if free.any() else -np.inf
            if mr == -np.inf:
                L = np.inf
            else:
                yr = (z[free] - mr) / T
                logR = np.log(np.exp(yr).sum())
                logQ = (mr - z.max()) / T + logR - lse
                L += P * (np.log(P) - logQ)
                tolL += 2.0 ** -21 * P * (np.abs(np.log(P)) + np.abs(logQ) + 2 * np.log(V) + 4)
                share[free] = P * np.exp(yr - logR)
                fall = np.zeros(V)
                fall[free] = np.where(np.isfinite(yr), -yr, 0.0)
                tolg = tolg + share * 2.0 ** -21 * (4 + fall)
            g = q - target - share
    return L, g / T, tolL, (tolg + 2.0 ** -126) / T


def rows_of(z, ids, teacher, kind, T):
    zn = z.double().numpy()
    rows = [distill_far(zn[r], ids[r], teacher[r], kind, T) for r in range(len(zn))]
    return tuple(np.stack([x[i] for x in rows]) for i in range(4))
