"""Float64 restatement of the operators over rows of logits (include/flowrl_hip.h: frl_logits_constrain / _choose,
frl_distill_fwd / _bwd), row by row and token by token.  PARITY UNPINNED by the reference, which has none of them; tests only."""
from __future__ import annotations

import numpy as np


def _at(v, r):
    return float(np.asarray(v).reshape(-1)[r]) if np.ndim(v) else float(v)


def constrain_row(z, r, *, history=None, lengths=None, prompt_lengths=None, repetition=1.0, frequency=0.0, presence=0.0, bias=None,
                  bias_tokens=None, bias_values=None, allowed=None):
    """(constrained logits of row r, the magnitudes that went into each element: the scale of its rounding errors)"""
    x = np.asarray(z[r], np.float64).copy()
    V = x.size
    size = np.abs(x)
    if history is not None:
        n = history.shape[1] if lengths is None else min(max(int(lengths[r]), 0), history.shape[1])
        first = 0 if prompt_lengths is None else min(max(int(prompt_lengths[r]), 0), n)
        rep, freq, pres = _at(repetition, r), _at(frequency, r), _at(presence, r)
        count = {}
        for t in range(n):
            v = int(history[r, t])
            if 0 <= v < V:
                count[v] = count.get(v, 0) + (1 if t >= first else 0)
        for v, c in count.items():
            x[v] = x[v] / rep if x[v] > 0 else x[v] * rep
            x[v] -= freq * c + (pres if c > 0 else 0.0)
            size[v] = size[v] * max(rep, 1.0 / rep) + abs(freq * c) + abs(pres)
    if bias is not None:
        b = np.asarray(bias, np.float64) if np.ndim(bias) == 1 else np.asarray(bias[r], np.float64)
        x, size = x + b, size + np.abs(b)
    if bias_tokens is not None:
        for v, b in zip(bias_tokens if np.ndim(bias_tokens) == 1 else bias_tokens[r], bias_values if np.ndim(bias_values) == 1 else bias_values[r]):
            if 0 <= v < V:
                x[v] += float(b)
                size[v] += abs(float(b))
    if allowed is not None:
        ok = np.asarray(allowed if np.ndim(allowed) == 1 else allowed[r])
        x[~ok] = -np.inf
        size[~ok] = 0.0
    return x, size


def keys_of(x, temperature, noise):
    """(y, key) of a constrained row"""
    if noise is None or not temperature > 0:
        return x, x
    y = x / (1e-6 + float(temperature))
    return y, np.where(y == -np.inf, -np.inf, y + np.asarray(noise, np.float64))


def choose_row(y, key):
    if np.isnan(key).any():
        return int(np.flatnonzero(np.isnan(key))[0]), np.nan
    if (y == -np.inf).all():
        return -1, -np.inf
    v = int(np.argmax(key))
    with np.errstate(invalid="ignore"):
        m = y.max()
        return v, float(y[v] - m - np.log(np.exp(y - m).sum()))


def distill_row(z, ids, teacher, kind, temperature):
    """(L, dL/dz, q, dict of what the error bounds need) of one row"""
    z = np.asarray(z, np.float64)
    V, T = z.size, float(temperature)
    valid = (ids >= 0) & (ids < V)
    ids, t = np.asarray(ids)[valid].astype(np.int64), np.asarray(teacher, np.float64)[valid]
    y = z / T
    m = y.max()
    e = np.exp(y - m)
    s = e.sum()
    q, logq = e / s, y - m - np.log(s)
    named = np.zeros(V, bool)
    named[ids] = True
    P = 0.0
    if kind == "logits":
        if ids.size == 0:
            return 0.0, np.zeros(V), q, dict(P=0.0, Q=1.0, logp=np.zeros(0))
        t = t / T
        logp = t - t.max() - np.log(np.exp(t - t.max()).sum())
    else:
        logp = t
        P = 1.0 - np.exp(logp).sum()
    p = np.exp(logp)
    with np.errstate(invalid="ignore", divide="ignore"):
        L = float(np.where(p > 0, p * (logp - logq[ids]), 0.0).sum())
        target = np.zeros(V)
        np.add.at(target, ids, p)
        g = p.sum() * q - target
        Q = e[~named].sum() / s
        if kind == "logprobs" and P > 0:
            L += P * np.log(P / Q)
            g = np.where(named, q - target, q * (1.0 - P / Q))
    return L, g / T, q, dict(P=max(P, 0.0), Q=Q, logp=logp)
