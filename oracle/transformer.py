"""The transformer operators in float64 NumPy, and how far a float32 evaluation may lie.

Each function returns values and, where it says so, bounds on the error of an evaluation
with float32 products and sums (u = 2^-24, half a step of float32): a dot product of n
terms is off by at most (n + 8) u sum |x y| in any order, 8 u covering operands held as
a sum of two shorter numbers; an exponential by 4 u.
"""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
def rotary(x, positions, rotated, interleaved=False, inverse=False, base=10000.0, factor=1.0, original=0.0, low=1.0,
           high=32.0, magnitude=1.0):
    """x [b, t, h, d] in any type, positions [b, t]; values and bounds.

    A turned feature is two products and a sum with rounded cosines and sines: at most
    4 u (|x1| + |x2|) magnitude."""
    x = np.asarray(x, np.float64)
    f = base ** (-np.arange(0, rotated, 2) / max(1, rotated))
    if factor != 1.0:
        keep = np.clip((original * f / (2 * np.pi) - low) / (high - low), 0, 1) if original else np.zeros_like(f)
        f = f * (keep + (1 - keep) / factor)
    angle = np.asarray(positions, np.float64)[:, :, None, None] * f
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle) * (-1 if inverse else 1)
    one, two = (slice(0, rotated, 2), slice(1, rotated, 2)) if interleaved else \
        (slice(0, rotated // 2), slice(rotated // 2, rotated))
    y, bound = x.copy(), np.zeros_like(x)
    y[..., one], y[..., two] = x[..., one] * c - x[..., two] * s, x[..., two] * c + x[..., one] * s
    size = 4 * U * abs(magnitude) * (np.abs(x[..., one]) + np.abs(x[..., two]))
    bound[..., one] = bound[..., two] = size
    return y, bound


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def visible(m, n, q_len, kv_len, causal, window):
    """[q_len, kv_len] truth: which keys each query sees, m and n positions being valid."""
    i, j = np.arange(q_len)[:, None], np.arange(kv_len)[None]
    p = i + n - m
    see = (i < m) & (j < n)
    if causal:
        see &= j <= p
    if window:
        see &= (j > p - window) & (j < p + window)
    return see


def _norm(x):
    return np.sqrt((x * x).sum(-1))


def attention(q, k, v, dout=None, causal=False, window=0, scale=None, q_lens=None, kv_lens=None):
    """q [b, t, h, d], k and v [b, n, hk, d]; a dict of values `out lse (dq dk dv)` and, under
    the same names with `_tol`, bounds."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    b, t, h, d = q.shape
    n, hk = k.shape[1], k.shape[2]
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    r = {"out": np.zeros_like(q), "lse": np.full((b, h, t), -np.inf)}
    r["out_tol"], r["lse_tol"] = np.zeros_like(q), np.zeros((b, h, t))
    if dout is not None:
        dout = np.asarray(dout, np.float64)
        for name, like in (("dq", q), ("dk", k), ("dv", v)):
            r[name], r[name + "_tol"] = np.zeros_like(like), np.zeros_like(like)
    for e in range(b):
        m = t if q_lens is None else int(np.clip(q_lens[e], 0, t))
        w = n if kv_lens is None else int(np.clip(kv_lens[e], 0, n))
        see = visible(m, w, t, n, causal, window)[:m, :w]
        for g in range(h):
            x, y, z = q[e, :m, g], k[e, :w, g // (h // hk)], v[e, :w, g // (h // hk)]
            s = np.where(see, scale * (x @ y.T), -np.inf)
            alive = see.any(1)
            top = np.where(alive, s.max(1, initial=-np.inf), 0.0)
            p = np.exp(s - top[:, None])
            total = np.where(alive, p.sum(1), 1.0)
            p /= total[:, None]
            lse = np.where(alive, top + np.log(total), -np.inf)
            out = p @ z
            r["out"][e, :m, g], r["lse"][e, g, :m] = out, lse
            # relative error of a weight: the score's dot product and its scaling, the
            # exponential, and the same of the sum that divides
            fs = np.where(see, s, 0.0)
            es = abs(scale) * (d + 8) * U * _norm(x)[:, None] * _norm(y)[None] + 3 * U * np.abs(fs)
            ep = np.where(see, es, 0).max(1, initial=0)[:, None] + 8 * U
            count = see.sum(1)[:, None]
            rel = 2 * ep + (2 * count + 8) * U
            r["out_tol"][e, :m, g] = out_tol = rel * (p @ np.abs(z)) + 1e-37
            r["lse_tol"][e, g, :m] = lse_tol = np.where(alive, (ep + (count + 4) * U)[:, 0] + 2 * U * np.abs(
                np.where(alive, lse, 0)), 0)
            if dout is None:
                continue
            go = dout[e, :m, g]
            dp, delta = go @ z.T, (go * out).sum(1, keepdims=True)
            ds = scale * p * (dp - delta)
            kg = g // (h // hk)
            r["dq"][e, :m, g] = ds @ y
            r["dk"][e, :w, kg] += ds.T @ x
            r["dv"][e, :w, kg] += p.T @ go
            rp = ep + lse_tol[:, None] + 2 * U              # the recomputed weight's relative error
            edp = (d + 8) * U * _norm(go)[:, None] * _norm(z)[None]
            edelta = ((d + 8) * U * np.abs(go * out) + np.abs(go) * out_tol).sum(1, keepdims=True)
            eds = np.abs(scale) * p * ((rp + 4 * U) * (np.abs(dp) + np.abs(delta)) + edp + edelta)
            rows = see.sum(0)[:, None] * (h // hk)
            r["dq_tol"][e, :m, g] = eds @ np.abs(y) + (count + 8) * U * (np.abs(ds) @ np.abs(y)) + 1e-37
            r["dk_tol"][e, :w, kg] += eds.T @ np.abs(x) + (rows + 8) * U * (np.abs(ds).T @ np.abs(x)) + 1e-37
            r["dv_tol"][e, :w, kg] += (rp * p).T @ np.abs(go) + (rows + 8) * U * (p.T @ np.abs(go)) + 1e-37
    return r


# ---------------------------------------------------------------------------
# the orthogonalised update
# ---------------------------------------------------------------------------
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalize(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """One matrix; its orthogonalisation and a bound on the Frobenius norm of the error.

    The rounding errors of a dot product of n terms are taken as independent: 4 sqrt(n) u of
    the sum of magnitudes instead of n u (Higham and Mary's probabilistic bound with
    lambda = 4).  An error of X grows by at most the polynomial's slope on the singular
    values at hand; for an error across singular directions that is the largest divided
    difference, which the slope bounds too."""
    a, b, c = coefficients
    x = np.asarray(x, np.float64)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (np.linalg.norm(x) + eps)
    err = 4 * U * np.linalg.norm(x)
    lam = lambda n: (4 * np.sqrt(n) + 8) * U  # noqa: E731
    for _ in range(steps):
        g = x @ x.T
        big = np.linalg.norm(g, 2) if g.size else 0.0
        s = np.linspace(0, np.sqrt(big) * 1.01, 200)
        slope = np.abs(a + 3 * b * s ** 2 + 5 * c * s ** 4).max()
        poly = b * g + c * (g @ g)
        eg = lam(x.shape[1]) * np.linalg.norm(np.abs(x) @ np.abs(x).T)
        ep = (abs(b) + 2 * abs(c) * big) * eg + lam(x.shape[0]) * abs(c) * np.linalg.norm(np.abs(g) @ np.abs(g)) \
            + 4 * U * (abs(b) * np.linalg.norm(g) + np.linalg.norm(poly))
        y = a * x + poly @ x
        err = slope * err + np.sqrt(big) * ep + lam(x.shape[0]) * np.linalg.norm(np.abs(poly) @ np.abs(x)) \
            + 4 * U * (abs(a) * np.linalg.norm(x) + np.linalg.norm(y))
        x = y
    return (x.T if tall else x), err


def muon(w, m, g, lr, momentum, nesterov, weight_decay, scale, **kw):
    """New w and m of one matrix, and the bound on w's error beside its own roundings (norm)."""
    w, m, g = (np.asarray(x, np.float64) for x in (w, m, g))
    m = momentum * m + g
    o, err = orthogonalize(g + momentum * m if nesterov else m, **kw)
    return (1 - lr * weight_decay) * w - lr * scale * o, m, lr * scale * err
