"""How far attention's results may lie from their definition, measured by what plain float32 does.

`compare` evaluates the formulas in float64 and in NumPy's float32 on the same inputs.  The
float32 run's own error, row by row, is the unit: a kernel with float32 products and sums in
another order, operands held as two float16 numbers (22 bits, 2^-23 at most, against float32's
2^-24) and matrix instructions that truncate (2^-23 of the partial sum each, where rounding is
off by 2^-24 at most) is off by a few times as much, so FACTOR is 8.  A row whose float32 error
is small by chance, or whose terms cancel (one visible key), gets a floor beside it: FLOOR
roundings of each of its terms, u (half a step) of the term's size before cancellation, as
independent errors: in length the root of the sum of squares, not the sum.

For dv, whose last key may have a single row's weight to be made of, the floor counts what the
weight exp(s - lse) is off by when lse is a float32 number, as the interface has it.  Its exponent
is off by at most u |s| (the factor that takes the score to the exponent's base), u |lse| (lse
itself), u |lse| (in that base) and u |s - lse| (the difference), each half a step of a number of
that size, and the weight relatively by as much: |s| 4, |lse| 6, |s - lse| 10 make 26 u.
"""
from __future__ import annotations

import numpy as np

from oracle import transformer as T

U = T.U
FACTOR, FLOOR = 8.0, 8.0
NAMES = ("out", "dq", "dk", "dv")


def _len(x):
    return np.sqrt((x.astype(np.float64) ** 2).sum(-1))


def _head(q, k, v, go, see, scale, dtype):
    """One head in one type: out, dq, dk, dv."""
    q, k, v, go = (x.astype(dtype) for x in (q, k, v, go))
    scale = dtype(scale)
    s = np.where(see, (q @ k.T) * scale, dtype(-np.inf))
    alive = see.any(1)
    top = np.where(alive, s.max(1, initial=-np.inf), 0).astype(dtype)
    p = np.exp(s - top[:, None])
    p /= np.where(alive, p.sum(1, dtype=dtype), 1).astype(dtype)[:, None]
    out = p @ v
    delta = (go * out).sum(1, keepdims=True, dtype=dtype)
    dp = go @ v.T
    ds = p * (dp - delta) * scale
    return {"out": out, "dq": ds @ k, "dk": ds.T @ q, "dv": p.T @ go, "p": p, "delta": delta}


def _floors(q, k, v, go, see, scale, r):
    """u times the length of a row's terms before cancellation."""
    q, k, v, go = (x.astype(np.float64) for x in (q, k, v, go))
    p, lq, lk, lv, lg = r["p"], _len(q), _len(k), _len(v), _len(go)
    term = abs(scale) * p * (lg[:, None] * lv[None] + np.abs(r["delta"]))      # of dS
    s = np.where(see, scale * (q @ k.T), 0.0)
    with np.errstate(divide="ignore"):
        away = np.where(p > 0, -np.log(p), 0.0)                                # lse - s
    weight = p * (1 + (np.abs(s) + 2 * np.abs(np.where(see, s + away, 0)) + away) / FLOOR)
    # an error of delta is one for the whole row: it meets the sum of the weighted keys
    shared = abs(scale) * lg * _len(r["out"]) * _len(p @ k)
    return {"out": U * np.sqrt((p * p) @ (lv * lv)), "dv": U * np.sqrt((weight * weight).T @ (lg * lg)),
            "dq": U * (np.sqrt((term * term) @ (lk * lk)) + shared), "dk": U * np.sqrt((term * term).T @ (lq * lq))}


def compare(got, q, k, v, go, causal=False, window=0, scale=None, names=NAMES, features=None):
    """Per name: (error of the whole head over its bound, worst row's error over its bound), as the
    largest over batch entries and heads.  features: the last dimension of got[name] has just these,
    whose own size is the measure then (the floors are those of rows of all features, and left out)."""
    b, t, h, d = q.shape
    n, hk = k.shape[1], k.shape[2]
    group = h // hk
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    see = T.visible(t, n, t, n, causal, window)
    worst = {x: [0.0, 0.0] for x in names}
    pick = features or {}
    for e in range(b):
        for g in range(hk):
            sums = {}
            for i in range(group):
                a = (q[e, :, g * group + i], k[e, :, g], v[e, :, g], go[e, :, g * group + i], see, scale)
                exact, plain = _head(*a, np.float64), _head(*a, np.float32)
                floor = _floors(*a, exact)
                for x in ("out", "dq"):
                    if x in names:
                        _worse(worst[x], got[x][e, :, g * group + i], exact[x], plain[x], floor[x], pick.get(x))
                for x in ("dk", "dv"):
                    w = sums.setdefault(x, [0.0, 0.0, 0.0])
                    w[0], w[1], w[2] = w[0] + exact[x], w[1] + plain[x].astype(np.float64), w[2] + floor[x] ** 2
            for x in ("dk", "dv"):
                if x in names:
                    _worse(worst[x], got[x][e, :, g], sums[x][0], sums[x][1], np.sqrt(sums[x][2]), pick.get(x))
    return worst


def _worse(at, got, exact, plain, floor, features=None):
    if features is not None:          # as a whole only: a row of few features can be near by chance
        exact, plain = exact[:, features], plain[:, features]
        off, own = (np.sqrt(((x - exact) ** 2).sum()) for x in (got, plain))
        at[0] = max(at[0], float(off / (FACTOR * own)))
        return
    off, own = _len(got - exact), _len(plain - exact)
    off = np.where(np.isfinite(off), off, np.inf)
    bound = FACTOR * own + FLOOR * floor + 1e-42 * np.sqrt(exact.shape[-1])
    whole = FACTOR * np.sqrt((own ** 2).sum()) + np.sqrt((floor ** 2).sum()) + 1e-42 * np.sqrt(exact.size)
    at[0] = max(at[0], np.sqrt((off ** 2).sum()) / whole)
    at[1] = max(at[1], float((off / bound).max(initial=0.0)))


def hold(got, *inputs, **kw):
    worst = compare(got, *inputs, **kw)
    assert all(max(w) <= 1 for w in worst.values()), {x: [round(float(y), 3) for y in w] for x, w in worst.items()}
