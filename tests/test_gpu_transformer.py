"""The transformer operators on the GPU against their float64 definitions (oracle.transformer),
within the bounds that the oracle derives for float32 arithmetic."""
import ctypes
import math

import numpy as np
import pytest

from directcompute_torch_b200 import _abi
from oracle import transformer as T

pytestmark = pytest.mark.gpu

ERR = {v: k for k, v in _abi.ERRORS.items()}


def _at(shape, stride, offset, data, room):
    """A flat float32 buffer of `room` words, NaN but for `data` at offset + strides."""
    flat = np.full(room, np.nan, np.float32)
    np.lib.stride_tricks.as_strided(flat[offset:], shape, [4 * s for s in stride] + [4])[...] = data
    return flat


def _packed(shape):
    b, t, h, d = shape
    return (t * h * d, h * d, d)


def _max_over(err, tol):
    """How many times its bound the worst element is off (NaN counts as infinite)."""
    with np.errstate(invalid="ignore", divide="ignore"):
        r = np.where(err == 0, 0.0, err / tol)
    return float(np.max(np.nan_to_num(r, nan=np.inf), initial=0))


# ---------------------------------------------------------------------------
# rotary
# ---------------------------------------------------------------------------
ROTARY = [
    # batch, length, heads, dim, rotated, interleaved, options
    (2, 5, 3, 64, 64, False, {}),
    (2, 5, 3, 64, 64, True, {}),
    (1, 1, 1, 2, 2, False, {}),
    (3, 7, 2, 10, 6, True, {}),
    (3, 7, 2, 10, 6, False, {"start": 12345}),
    (1, 33, 5, 96, 32, False, {"factor": 4.0}),
    (2, 9, 4, 80, 80, False, {"factor": 8.0, "original": 2048, "low": 1.0, "high": 32.0, "magnitude": 1.2}),
    (1, 3, 40, 128, 128, True, {"base": 5e5}),
    (1, 2, 1, 512, 256, False, {}),
    (1, 300, 1, 16, 0, False, {}),
    (1, 300, 1, 4, 4, True, {}),
]


@pytest.mark.parametrize("case", ROTARY)
@pytest.mark.parametrize("inverse", [0, 1])
@pytest.mark.parametrize("positions", [False, True])
def test_rotary(dev, case, inverse, positions):
    b, t, h, d, rotated, inter, kw = case
    kw = dict(kw)
    r = np.random.default_rng(7)
    x = r.normal(size=(b, t, h, d)).astype(np.float32)
    start = kw.pop("start", 0)
    pos = r.integers(-3, 2 ** 31 - 1, (b, t)).astype(np.int32) if positions else np.broadcast_to(start + np.arange(t), (b, t))
    want, tol = T.rotary(x, pos, rotated, inter, bool(inverse), **kw)
    full = {"base": 10000.0, "factor": 1.0, "low": 1.0, "high": 32.0, "original": 0.0, "magnitude": 1.0, **kw}
    p = _abi.Rotary(batch=b, length=t, heads=h, head_dim=d, x_stride=_packed(x.shape), y_stride=_packed(x.shape),
                    rotated=rotated, interleaved=inter, inverse=inverse, start=start, **full)
    hx, hy = dev.buf(x), dev.empty(x.size, fill=np.nan)
    hp = dev.buf(pos) if positions else None
    try:
        _abi.check(dev.lib, dev.lib.dct_rotary(ctypes.byref(p), hx, hp, hy))
        # float64 angles of far positions: position * f is off by 2^-52 of itself, in radians
        tol = tol + 2.0 ** -51 * np.abs(pos.astype(np.float64))[..., None, None] * np.abs(want).max()
        assert _max_over(np.abs(dev.read(hy).reshape(x.shape) - want), tol + 1e-37) <= 1
        _abi.check(dev.lib, dev.lib.dct_rotary(ctypes.byref(p), hx, hp, hx))            # in place
        assert np.array_equal(dev.read(hx), dev.read(hy))
    finally:
        dev.free(hx, hy, *([hp] if hp else []))


@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 3), (4, 4)])
@pytest.mark.parametrize("inter", [0, 1])
def test_rotary_strides(dev, offset, pad, inter):
    """A head of a packed projection, whole and at an offset that no vector load fits."""
    b, t, h, d = 2, 6, 3, 32
    r = np.random.default_rng(8)
    x = r.normal(size=(b, t, h, d)).astype(np.float32)
    xs, ys = (t * (3 * h * d + pad), 3 * h * d + pad, d), (d, b * d, t * b * d)
    hx, hy = dev.buf(_at(x.shape, xs, offset, x, offset + b * xs[0])), dev.empty(x.size)
    try:
        hw = dev.lib.dct_wrap_device_ptr(dev.lib.dct_buffer_device_ptr(hx) + 4 * offset, b * xs[0])
        p = _abi.Rotary(batch=b, length=t, heads=h, head_dim=d, x_stride=xs, y_stride=ys, rotated=d, interleaved=inter,
                        base=10000.0, factor=1.0, magnitude=1.0)
        _abi.check(dev.lib, dev.lib.dct_rotary(ctypes.byref(p), hw, None, hy))
        want, tol = T.rotary(x, np.broadcast_to(np.arange(t), (b, t)), d, bool(inter))
        got = np.lib.stride_tricks.as_strided(dev.read(hy), x.shape, [4 * s for s in ys] + [4])
        assert _max_over(np.abs(got - want), tol + 1e-37) <= 1
        dev.free(hw)
    finally:
        dev.free(hx, hy)


def test_rotary_refuses(dev):
    lib = dev.lib
    hx, hy, hw = dev.empty(64), dev.empty(64), dev.empty(3)

    def call(x=hx, pos=None, y=hy, **kw):
        f = {"batch": 1, "length": 4, "heads": 2, "head_dim": 8, "x_stride": (64, 16, 8), "y_stride": (64, 16, 8),
             "rotated": 8, "base": 1e4, "factor": 1.0, "magnitude": 1.0, **kw}
        return lib.dct_rotary(ctypes.byref(_abi.Rotary(**f)), x, pos, y)
    try:
        assert call() == 0
        assert call(rotated=7) == ERR["ARG"] and call(rotated=10) == ERR["ARG"]
        assert call(base=0.0) == ERR["ARG"] and call(base=math.nan) == ERR["ARG"] and call(factor=-1.0) == ERR["ARG"]
        assert call(factor=2.0, original=10.0, low=3.0, high=3.0) == ERR["ARG"]
        assert call(x_stride=(64, -16, 8)) == ERR["ARG"]
        assert call(y_stride=(64, 4, 8)) == ERR["ARG"]                       # outputs overlap
        assert call(y=hx, y_stride=(64, 8, 32)) == ERR["ARG"]                # in place with other strides
        assert call(length=5) == ERR["SIZE"] and call(pos=hw) == ERR["SIZE"]
        assert call(x=12345) == ERR["HANDLE"] and call(y=None) == ERR["HANDLE"] and call(pos=999) == ERR["HANDLE"]
        assert call(batch=0) == 0 and call(length=0) == 0
        assert lib.dct_rotary(None, hx, None, hy) == ERR["ARG"]
    finally:
        dev.free(hx, hy, hw)
        dev.clear_error()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attention(dev, q, k, v, go=None, strides=None, offset=0, lse=True, **kw):
    """Both calls (the second where go is given); a dict of arrays."""
    lib = dev.lib
    b, t, h, d = q.shape
    n, hk = k.shape[1], k.shape[2]
    st = {"q": _packed(q.shape), "k": _packed(k.shape), "v": _packed(v.shape), "o": _packed(q.shape),
          "dq": _packed(q.shape), "dk": _packed(k.shape), "dv": _packed(k.shape), **(strides or {})}
    shapes = {"q": q.shape, "k": k.shape, "v": v.shape, "o": q.shape, "dq": q.shape, "dk": k.shape, "dv": k.shape}
    room = {x: 4 + offset + sum((a - 1) * s for a, s in zip(shapes[x][:3], st[x])) + d for x in st}
    hold = []

    def up(x, data=None):
        flat = np.full(room[x], np.nan, np.float32) if data is None else _at(shapes[x], st[x], offset, data, room[x])
        base = dev.buf(flat)
        w = lib.dct_wrap_device_ptr(lib.dct_buffer_device_ptr(base) + 4 * offset, max(1, room[x] - offset))
        hold.extend((w, base))
        return w, base
    p = _abi.Attention(batch=b, q_heads=h, kv_heads=hk, q_len=t, kv_len=n, head_dim=d, causal=kw.get("causal", False),
                       window=kw.get("window", 0), scale=kw.get("scale") or 0.0, **{x + "_stride": s for x, s in st.items()})
    words = []
    for name in ("q_lens", "kv_lens"):
        x = kw.get(name)
        words.append(dev.buf(np.asarray(x, np.int32)) if x is not None else None)
        hold.extend(w for w in words[-1:] if w)
    try:
        hq, hk_, hv = up("q", q)[0], up("k", k)[0], up("v", v)[0]
        ho, base_o = up("o")
        hl = dev.empty(max(1, b * h * t), fill=np.nan)
        hold.append(hl)

        def read(x, base):
            flat = dev.read(base)
            view = np.lib.stride_tricks.as_strided(flat[offset:], shapes[x], [4 * s for s in st[x]] + [4])
            got = view.copy()
            view[...] = np.nan
            assert np.isnan(flat).all(), f"{x}: words behind the tensor were written"
            return got
        _abi.check(lib, lib.dct_attention_forward(ctypes.byref(p), hq, hk_, hv, *words, ho, hl if lse else None))
        r = {"out": read("o", base_o), "lse": dev.read(hl)[:b * h * t].reshape(b, h, t)}
        if go is not None:
            b2 = dev.buf(_at(shapes["o"], st["o"], offset, go, room["o"]))
            hg = lib.dct_wrap_device_ptr(lib.dct_buffer_device_ptr(b2) + 4 * offset, max(1, room["o"] - offset))
            hold.extend((hg, b2))
            outs = {x: up(x) for x in ("dq", "dk", "dv")}
            _abi.check(lib, lib.dct_attention_backward(ctypes.byref(p), hq, hk_, hv, *words, ho, hl, hg,
                                                       *(outs[x][0] for x in ("dq", "dk", "dv"))))
            for x in outs:
                r[x] = read(x, outs[x][1])
        return r
    finally:
        dev.free(*hold)


def _inputs(b, t, n, h, hk, d, seed=3):
    r = np.random.default_rng(seed)
    return tuple(r.normal(size=s).astype(np.float32) for s in ((b, t, h, d), (b, n, hk, d), (b, n, hk, d), (b, t, h, d)))


def _hold(got, want, names):
    for x in names:
        fine = np.isfinite(want[x])
        assert np.array_equal(got[x][~fine], want[x][~fine].astype(np.float32)), x
        worst = _max_over(np.abs(got[x][fine] - want[x][fine]), want[x + "_tol"][fine])
        assert worst <= 1, (x, worst)


ALL = ("out", "lse", "dq", "dk", "dv")
SHAPES = [
    # batch, q_len, kv_len, q_heads, kv_heads, dim
    (1, 1, 1, 1, 1, 1), (2, 5, 7, 2, 1, 9), (1, 64, 64, 2, 2, 64), (2, 65, 63, 4, 2, 64), (1, 130, 257, 2, 1, 128),
    (1, 127, 128, 3, 3, 80), (3, 33, 200, 8, 2, 32), (1, 300, 300, 2, 2, 96), (1, 17, 1000, 6, 3, 128),
    (2, 129, 129, 1, 1, 127), (1, 256, 31, 2, 1, 16), (1, 400, 400, 4, 1, 128),
]
MASKS = [{}, {"causal": True}, {"causal": True, "window": 40}, {"window": 17}]


@pytest.mark.parametrize("mask", MASKS, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention(dev, shape, mask):
    q, k, v, go = _inputs(*shape)
    _hold(_attention(dev, q, k, v, go, **mask), T.attention(q, k, v, go, **mask), ALL)


@pytest.mark.parametrize("size", [(90, 150, 64), (260, 270, 128), (200, 330, 64)])
@pytest.mark.parametrize("mask", MASKS, ids=str)
def test_attention_ragged(dev, mask, size):
    """Lengths of 0, 1, whole ones and ones past the end (clamped), queries fewer and more than keys."""
    t, n, d = size
    q, k, v, go = _inputs(7, t, n, 4, 2, d)
    lens = {"q_lens": [t, 0, 1, 37, 64, t + 9, t], "kv_lens": [n, n, 1, 20, 65, 1000, 0]}
    want = T.attention(q, k, v, go, **mask, **lens)
    _hold(_attention(dev, q, k, v, go, **mask, **lens), want, ALL)


@pytest.mark.parametrize("bad", [np.nan, np.inf, 3e38])
@pytest.mark.parametrize("shape", [(2, 70, 140, 4, 2, 64), (2, 1, 300, 4, 2, 128), (2, 5, 300, 2, 2, 32),
                                   (2, 210, 400, 4, 2, 64), (2, 300, 300, 4, 1, 100)], ids=str)
def test_attention_masked_places_do_not_reach_results(dev, bad, shape):
    q, k, v, go = _inputs(*shape)
    t, n = shape[1], shape[2]
    lens = {"q_lens": [t, max(1, t // 2)], "kv_lens": [n // 2, n]}
    want = T.attention(q, k, v, go, causal=True, **lens)
    k[0, n // 2:], v[0, n // 2:] = bad, bad
    q[1, max(1, t // 2):], go[1, max(1, t // 2):] = bad, bad
    _hold(_attention(dev, q, k, v, go, causal=True, **lens), want, ALL)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("t", [200, 520])
def test_attention_later_keys_do_not_reach_earlier_queries(dev, bad, t):
    """A value that a causal mask hides from a query does not reach it, inside a tile too."""
    q, k, v, go = _inputs(1, t, t, 2, 2, 64)
    want = T.attention(q, k, v, go, causal=True)
    v[0, 150, 1], k[0, 170, 1] = bad, bad
    got = _attention(dev, q, k, v, causal=True)
    assert _max_over(np.abs(got["out"][:, :150] - want["out"][:, :150]), want["out_tol"][:, :150]) <= 1
    assert _max_over(np.abs(got["out"][:, :, 0] - want["out"][:, :, 0]), want["out_tol"][:, :, 0]) <= 1
    assert not np.isfinite(got["out"][0, 150:, 1]).any() if np.isnan(bad) else not np.isfinite(got["out"][0, 150, 1]).any()


@pytest.mark.parametrize("spread", [0, 8, 13, 30])
@pytest.mark.parametrize("t", [150, 520])
def test_attention_far_apart_magnitudes(dev, spread, t):
    """Rows whose sizes lie 2^spread apart, and inputs far from 1."""
    q, k, v, go = _inputs(1, t, t, 2, 1, 64)
    r = np.random.default_rng(5)
    for x in (v, go):
        x *= np.exp2(-r.integers(0, spread + 1, x.shape[:3] + (1,))).astype(np.float32)
    q *= np.float32(2.0 ** 40)
    k *= np.float32(2.0 ** -40)
    v *= np.float32(2.0 ** -60)
    _hold(_attention(dev, q, k, v, go), T.attention(q, k, v, go), ALL)


@pytest.mark.parametrize("offset", [0, 1, 4])
@pytest.mark.parametrize("t,d", [(100, 64), (300, 64), (260, 128), (280, 50)])
def test_attention_strides(dev, offset, t, d):
    """Packed projections and heads before positions, at aligned and unaligned starts; nothing is
    written between an output's rows."""
    b, h, hk = 2, 4, 2
    q, k, v, go = _inputs(b, t, t, h, hk, d)
    w = (h + 2 * hk) * d + 4
    st = {"q": (t * w, w, d), "k": (t * w, w, d), "v": (hk * t * d, d, t * d), "o": (h * t * d, d, t * d),
          "dq": (t * w, w, d), "dk": (hk * t * (d + 4), d + 4, t * (d + 4)), "dv": (t * w, w, d)}
    want = T.attention(q, k, v, go, causal=True)
    _hold(_attention(dev, q, k, v, go, strides=st, offset=offset, causal=True), want, ALL)


@pytest.mark.parametrize("group", [1, 4, 8])
@pytest.mark.parametrize("n", [1, 31, 129, 4097])
@pytest.mark.parametrize("d", [64, 128, 100])
def test_attention_one_new_token(dev, group, n, d):
    q, k, v, _ = _inputs(3, 1, n, 2 * group, 2, d)
    kw = {"causal": True, "kv_lens": [n, max(1, n // 3), 0]}
    _hold(_attention(dev, q, k, v, **kw), T.attention(q, k, v, **kw), ("out", "lse"))


@pytest.mark.parametrize("shape,mask", [
    ((2, 192, 192, 8, 2, 64), {"causal": True, "window": 50}), ((3, 16, 1500, 16, 4, 128), {"causal": True}),
    ((1, 700, 900, 6, 6, 72), {"window": 300}), ((2, 5, 3000, 16, 2, 128), {"causal": True}),
    ((4, 260, 260, 8, 1, 33), {"causal": True}), ((1, 1, 5000, 8, 1, 128), {}), ((2, 300, 2000, 4, 4, 128), {"window": 1}),
    ((1, 1000, 130, 4, 2, 64), {"causal": True}), ((2, 385, 385, 4, 4, 112), {})], ids=str)
def test_attention_larger(dev, shape, mask):
    """Sizes that take the tensor cores, forward with the keys split where rows are few."""
    q, k, v, go = _inputs(*shape)
    _hold(_attention(dev, q, k, v, go, **mask), T.attention(q, k, v, go, **mask), ALL)


@pytest.mark.parametrize("bad", ["nan", "inf", "rows", "values", "scores"])
@pytest.mark.parametrize("t", [40, 300])
def test_attention_heads_apart(dev, bad, t):
    """One key head that float16 pairs cannot hold leaves the other heads as they were, and is right itself."""
    q, k, v, go = _inputs(2, t, 1500, 4, 2, 64)
    fine = _attention(dev, q, k, v, go, causal=True)
    if bad in ("nan", "inf"):
        v[1, 700, 1, 3] = np.nan if bad == "nan" else np.inf
    elif bad == "rows":
        k[1, 130, 1] *= np.float32(2.0 ** -30)
    elif bad == "values":
        v[1, 128:, 1] *= np.float32(2.0 ** -80)
    else:
        q[1, :, 2:] *= 3e4
    got = _attention(dev, q, k, v, go, causal=True)
    for x in ALL[2:] + ("out",):
        heads = 2 if x in ("out", "dq") else 1
        assert np.array_equal(got[x][0], fine[x][0]) and np.array_equal(got[x][1][:, :heads], fine[x][1][:, :heads])
    if bad in ("rows", "values"):
        _hold(got, T.attention(q, k, v, go, causal=True), ALL)
    elif bad == "scores":
        _hold(got, T.attention(q, k, v, go, causal=True), ("out", "lse"))
    else:
        first = max(0, 700 - (1500 - t))                     # queries that see key 700
        assert not np.isfinite(got["out"][1, first:, 2:, 3]).any()


@pytest.mark.parametrize("d", [64, 128, 37])
def test_attention_of_a_single_key_has_no_gradient_of_its_score(dev, d):
    """softmax of one score is 1 whatever it is: dq and dk are exactly 0, dv is the sum of dout."""
    q, k, v, go = _inputs(3, 5, 1, 4, 2, d)
    got = _attention(dev, q, k, v, go)
    assert not got["dq"].any() and not got["dk"].any()
    assert np.array_equal(got["out"], np.repeat(v, 2, 2) + 0 * q)
    _hold(got, T.attention(q, k, v, go), ALL)
    q, k, v, go = _inputs(2, 30, 30, 4, 2, d)
    got = _attention(dev, q, k, v, go, window=1)
    assert not got["dq"].any() and not got["dk"].any()


def test_attention_over_a_cache_with_room(dev):
    """Keys in a cache longer than its valid part, heads before positions."""
    b, t, n, h, hk, d, room = 3, 20, 900, 8, 2, 64, 1024
    q, k, v, go = _inputs(b, t, n, h, hk, d)
    st = {x: (hk * room * d, d, room * d) for x in ("k", "v", "dk", "dv")}
    kw = {"causal": True, "kv_lens": [900, 1, 555]}
    _hold(_attention(dev, q, k, v, go, strides=st, **kw), T.attention(q, k, v, go, **kw), ALL)


@pytest.mark.parametrize("t", [190, 350])
def test_attention_is_the_same_from_run_to_run(dev, t):
    q, k, v, go = _inputs(2, t, t, 4, 2, 64)
    one, two = (_attention(dev, q, k, v, go, causal=True) for _ in range(2))
    assert all(np.array_equal(one[x], two[x]) for x in ALL)
    none = _attention(dev, q, k, v, causal=True, lse=False)
    assert np.array_equal(none["out"], one["out"]) and np.isnan(none["lse"]).all()


@pytest.mark.parametrize("t", [70, 520])
def test_attention_scale_of_either_sign(dev, t):
    q, k, v, go = _inputs(1, t, t, 2, 2, 64)
    for scale in (0.5, -0.1, 1e-20):
        _hold(_attention(dev, q, k, v, go, scale=scale), T.attention(q, k, v, go, scale=scale), ALL)


def test_attention_empty(dev):
    for shape in ((0, 3, 4, 2, 1, 8), (2, 0, 4, 2, 1, 8), (2, 3, 0, 2, 1, 8)):
        q, k, v, go = _inputs(*shape)
        if 0 in shape[:2] or shape[2] == 0:
            b, t, h, d = q.shape
            lib = dev.lib
            bufs = [dev.empty(max(1, x.size), fill=7.0) for x in (q, k, v, q, q, q, k, v)]
            hl = dev.empty(max(1, b * h * t), fill=7.0)
            p = _abi.Attention(batch=b, q_heads=h, kv_heads=1, q_len=t, kv_len=shape[2], head_dim=d,
                               **{x + "_stride": _packed(y.shape) for x, y in (
                                   ("q", q), ("k", k), ("v", v), ("o", q), ("dq", q), ("dk", k), ("dv", v))})
            try:
                _abi.check(lib, lib.dct_attention_forward(ctypes.byref(p), *bufs[:3], None, None, bufs[3], hl))
                _abi.check(lib, lib.dct_attention_backward(ctypes.byref(p), *bufs[:3], None, None, bufs[3], hl, *bufs[4:]))
                if b and t:
                    assert not dev.read(bufs[3]).any() and np.isneginf(dev.read(hl)).all() and not dev.read(bufs[5]).any()
                if b and shape[2]:
                    assert not dev.read(bufs[6]).any() and not dev.read(bufs[7]).any()
            finally:
                dev.free(*bufs, hl)


def test_attention_refuses(dev):
    lib = dev.lib
    n = 2 * 3 * 2 * 8
    h = [dev.empty(n) for _ in range(9)]
    words, short = dev.empty(2), dev.empty(1)
    st = (48, 16, 8)

    def call(back=False, swap=None, lens=(None, None), params=True, **kw):
        f = {"batch": 2, "q_heads": 2, "kv_heads": 2, "q_len": 3, "kv_len": 3, "head_dim": 8,
             **{x + "_stride": st for x in ("q", "k", "v", "o", "dq", "dk", "dv")}, **kw}
        b = list(h)
        for i, x in (swap or {}).items():
            b[i] = x
        p = ctypes.byref(_abi.Attention(**f)) if params else None
        if back:
            return lib.dct_attention_backward(p, *b[:3], *lens, b[3], b[4], *b[5:])
        return lib.dct_attention_forward(p, *b[:3], *lens, b[3], b[4])
    try:
        for back in (False, True):
            assert call(back) == 0
            assert call(back, params=False) == ERR["ARG"]
            assert call(back, head_dim=0) == ERR["ARG"] and call(back, head_dim=129) == ERR["ARG"]
            assert call(back, kv_heads=0) == ERR["ARG"] and call(back, q_heads=3) == ERR["ARG"]
            assert call(back, scale=math.nan) == ERR["ARG"] and call(back, scale=math.inf) == ERR["ARG"]
            assert call(back, q_stride=(48, -16, 8)) == ERR["ARG"]
            assert call(back, kv_len=4) == ERR["SIZE"] and call(back, k_stride=(49, 16, 8)) == ERR["SIZE"]
            assert call(back, swap={1: 77}) == ERR["HANDLE"] and call(back, swap={3: None}) == ERR["HANDLE"]
            assert call(back, lens=(short, None)) == ERR["SIZE"] and call(back, lens=(words, 5)) == ERR["HANDLE"]
            assert call(back, batch=1 << 20, q_len=1 << 20) == ERR["ARG"]
        assert call(o_stride=(48, 4, 8)) == ERR["ARG"] and call(True, dq_stride=(48, 16, 4)) == ERR["ARG"]
        assert call(swap={3: h[0]}) == ERR["ARG"] and call(swap={4: h[1]}) == ERR["ARG"]
        assert call(True, swap={6: h[5]}) == ERR["ARG"] and call(True, swap={4: None}) == ERR["HANDLE"]
        assert call(True, swap={6: h[4]}) == ERR["ARG"]
    finally:
        dev.free(*h, words, short)
        dev.clear_error()


# ---------------------------------------------------------------------------
# orthogonalisation
# ---------------------------------------------------------------------------
def _muon(shape, **kw):
    b, r, c = shape
    return _abi.Muon(batch=b, rows=r, cols=c, **{"steps": 5, "eps": 1e-7, **kw})


MATRICES = [(1, 1, 1), (1, 1, 9), (2, 9, 1), (1, 17, 33), (3, 64, 64), (1, 127, 333), (1, 333, 127), (2, 128, 256),
            (1, 260, 130), (5, 96, 200), (1, 513, 700), (1, 700, 513), (2, 256, 1025), (1, 128, 2560), (2, 2561, 128),
            (1, 129, 640), (3, 64, 321), (1, 5, 3000), (1, 2100, 1), (40, 100, 70), (1, 1030, 1300), (3, 600, 600),
            (1, 2048, 2050)]


@pytest.mark.parametrize("shape", MATRICES, ids=str)
@pytest.mark.parametrize("steps", [0, 1, 5])
def test_orthogonalize(dev, shape, steps):
    r = np.random.default_rng(11)
    x = (1e-3 * r.normal(size=shape)).astype(np.float32)
    hx, hy = dev.buf(x), dev.empty(x.size, fill=np.nan)
    try:
        p = _muon(shape, steps=steps)
        _abi.check(dev.lib, dev.lib.dct_orthogonalize(ctypes.byref(p), hx, hy))
        got = dev.read(hy).reshape(shape)
        for i in range(shape[0]):
            want, tol = T.orthogonalize(x[i], steps)
            assert np.linalg.norm(got[i] - want) <= tol
        _abi.check(dev.lib, dev.lib.dct_orthogonalize(ctypes.byref(p), hx, hx))
        assert np.array_equal(dev.read(hx), got.ravel())
    finally:
        dev.free(hx, hy)


@pytest.mark.parametrize("nesterov", [0, 1])
@pytest.mark.parametrize("shape", [(1, 40, 24), (2, 130, 257), (3, 128, 128)], ids=str)
def test_muon_step(dev, shape, nesterov):
    r = np.random.default_rng(12)
    w, m, g = (r.normal(size=shape).astype(np.float32) for _ in range(3))
    hw, hm, hg = dev.buf(w), dev.buf(m), dev.buf(g)
    kw = {"lr": 0.05, "momentum": 0.9, "weight_decay": 0.1}
    try:
        p = _muon(shape, nesterov=nesterov, **kw)
        _abi.check(dev.lib, dev.lib.dct_muon(ctypes.byref(p), hw, hm, hg))
        gw, gm = dev.read(hw).reshape(shape), dev.read(hm).reshape(shape)
        scale = math.sqrt(max(1.0, shape[1] / shape[2]))
        exact = {k: float(np.float32(v)) for k, v in kw.items()}     # as the call holds them
        for i in range(shape[0]):
            ww, mm, tol = T.muon(w[i], m[i], g[i], nesterov=bool(nesterov), scale=scale, **exact)
            assert (np.abs(gm[i] - mm) <= 2 * T.U * (np.abs(mm) + np.abs(0.9 * m[i]))).all()
            assert np.linalg.norm(gw[i] - ww) <= tol + 4 * T.U * (np.linalg.norm(w[i]) + np.linalg.norm(ww))
        assert np.array_equal(dev.read(hg).reshape(shape), g)
    finally:
        dev.free(hw, hm, hg)


@pytest.mark.parametrize("size", [1e-30, 1e-7, 1e30])
def test_orthogonalize_any_magnitude(dev, size):
    x = np.random.default_rng(13).normal(size=(1, 70, 90)) * size
    x = x.astype(np.float32)
    hx = dev.buf(x)
    try:
        _abi.check(dev.lib, dev.lib.dct_orthogonalize(ctypes.byref(_muon(x.shape, eps=0.0)), hx, hx))
        want, tol = T.orthogonalize(x[0], eps=0.0)
        assert np.linalg.norm(dev.read(hx).reshape(70, 90) - want) <= tol
    finally:
        dev.free(hx)


@pytest.mark.parametrize("coefficients", [(1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375)], ids=str)
def test_orthogonalize_other_polynomials(dev, coefficients):
    """Polynomials that take singular values to 1 itself."""
    x = np.random.default_rng(15).normal(size=(1, 140, 90)).astype(np.float32)
    hx = dev.buf(x)
    a, b, c = coefficients
    try:
        _abi.check(dev.lib, dev.lib.dct_orthogonalize(ctypes.byref(_muon(x.shape, a=a, b=b, c=c, steps=12)), hx, hx))
        want, tol = T.orthogonalize(x[0], 12, coefficients)
        assert np.linalg.norm(dev.read(hx).reshape(140, 90) - want) <= tol
    finally:
        dev.free(hx)


def test_orthogonalize_zero_and_nan(dev):
    """A zero matrix stays zero; a NaN stays in its matrix of the batch."""
    x = np.random.default_rng(14).normal(size=(3, 66, 40)).astype(np.float32)
    x[0], x[1, 3, 5] = 0, np.nan
    hx = dev.buf(x)
    try:
        _abi.check(dev.lib, dev.lib.dct_orthogonalize(ctypes.byref(_muon(x.shape)), hx, hx))
        got = dev.read(hx).reshape(x.shape)
        assert not got[0].any() and np.isnan(got[1]).all()
        want, tol = T.orthogonalize(x[2])
        assert np.linalg.norm(got[2] - want) <= tol
    finally:
        dev.free(hx)


def test_orthogonalize_refuses(dev):
    lib = dev.lib
    h = [dev.empty(24) for _ in range(3)]

    def call(x=h[0], y=h[1], **kw):
        return lib.dct_orthogonalize(ctypes.byref(_muon((1, 4, 6), **kw)), x, y)
    try:
        assert call() == 0 and call(y=h[0]) == 0
        assert lib.dct_orthogonalize(None, h[0], h[1]) == ERR["ARG"]
        assert call(steps=17) == ERR["ARG"] and call(eps=-1.0) == ERR["ARG"] and call(a=math.nan) == ERR["ARG"]
        assert call(a=100.0, b=0.0, c=1.0) == ERR["ARG"]
        assert call(x=None) == ERR["HANDLE"] and call(y=31) == ERR["HANDLE"]
        assert lib.dct_orthogonalize(ctypes.byref(_muon((2, 4, 6))), h[0], h[1]) == ERR["SIZE"]
        assert lib.dct_orthogonalize(ctypes.byref(_muon((70000, 4, 6))), h[0], h[1]) == ERR["ARG"]
        assert lib.dct_orthogonalize(ctypes.byref(_muon((0, 4, 6))), h[0], h[1]) == 0
        assert lib.dct_muon(ctypes.byref(_muon((1, 4, 6))), h[0], h[1], h[0]) == ERR["ARG"]
        assert lib.dct_muon(ctypes.byref(_muon((1, 4, 6))), h[0], h[1], h[2]) == 0
    finally:
        dev.free(*h)
        dev.clear_error()


# ---------------------------------------------------------------------------
# the operators together, through the Python ops
# ---------------------------------------------------------------------------
def test_a_training_step(dev):
    """Rotary queries and keys, causal attention, its gradient through both, and an
    orthogonalised update of the projections."""
    from directcompute_torch_b200 import ops
    r = np.random.default_rng(21)
    b, t, h, hk, d = 2, 48, 4, 2, 32
    q, k, v = (r.normal(size=s).astype(np.float32) for s in ((b, t, h, d), (b, t, hk, d), (b, t, hk, d)))
    go = r.normal(size=q.shape).astype(np.float32)
    tq, tk, tv = (ops.tensor(x, requires_grad=True) for x in (q, k, v))
    out = ops.attention(ops.rotary(tq), ops.rotary(tk), tv, causal=True, kv_lens=[t, 40], q_lens=[t, 40])
    out.backward(ops.tensor(go))
    pos = np.broadcast_to(np.arange(t), (b, t))
    rq, rk = (T.rotary(x, pos, d)[0] for x in (q, k))
    want = T.attention(rq, rk, v, go, causal=True, q_lens=[t, 40], kv_lens=[t, 40])
    # beside the bounds, the turned inputs' own rounding (4 u of each, through scores of order 1)
    slack = 64 * T.U * d * max(np.abs(want[x]).max() for x in ALL[2:])
    assert _max_over(np.abs(ops.to_numpy(out) - want["out"]), want["out_tol"] + slack) <= 1
    for x, g in (("dq", tq), ("dk", tk), ("dv", tv)):
        full = want[x] if x == "dv" else T.rotary(want[x], pos, d, inverse=True)[0]
        assert _max_over(np.abs(ops.to_numpy(g.grad) - full), want[x + "_tol"].max() + slack) <= 1
    w = r.normal(size=(t, hk * d)).astype(np.float32)
    g0 = ops.to_numpy(tk.grad)[0].reshape(t, hk * d)
    tw, tm = ops.tensor(w), ops.tensor(np.zeros_like(w))
    ops.muon_step(tw, tm, ops.tensor(g0), lr=0.1)
    ww, mm, tol = T.muon(w, np.zeros_like(w), g0, float(np.float32(0.1)), float(np.float32(0.95)), True, 0.0, 1.0)
    assert np.linalg.norm(ops.to_numpy(tw) - ww) <= tol + 4 * T.U * np.linalg.norm(w)


def test_ops_orthogonalize_and_shapes(dev):
    from directcompute_torch_b200 import ops
    x = np.random.default_rng(22).normal(size=(2, 3, 20, 30)).astype(np.float32)
    got = ops.to_numpy(ops.orthogonalize(ops.tensor(x)))
    for i in np.ndindex(2, 3):
        want, tol = T.orthogonalize(x[i])
        assert np.linalg.norm(got[i] - want) <= tol
    t = ops.tensor(x)
    for f in (lambda: ops.rotary(ops.tensor(x[0])), lambda: ops.attention(t, t, ops.tensor(x[:1])),
              lambda: ops.orthogonalize(ops.tensor(x[0, 0, 0])), lambda: ops.muon_step(t, t, ops.tensor(x[0])),
              lambda: ops.rotary(t, positions=[0.5])):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(RuntimeError):
        ops.rotary(t, rotated=7)


@pytest.mark.parametrize("call", ["rotary", "attention", "muon"])
def test_refused_while_the_stream_is_captured(dev, call):
    torch = pytest.importorskip("torch")
    lib = dev.lib
    h = [dev.empty(64) for _ in range(4)]
    dev.sync()
    try:
        s = torch.cuda.ExternalStream(lib.dct_stream())
        g = torch.cuda.CUDAGraph()
        seen = []
        with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
            if call == "rotary":
                p = _abi.Rotary(batch=1, length=1, heads=1, head_dim=8, rotated=8, base=1e4, factor=1, magnitude=1)
                seen.append(lib.dct_rotary(ctypes.byref(p), h[0], None, h[1]))
            elif call == "attention":
                p = _abi.Attention(batch=1, q_heads=1, kv_heads=1, q_len=1, kv_len=1, head_dim=8)
                seen.append(lib.dct_attention_forward(ctypes.byref(p), *h[:3], None, None, h[3], None))
            else:
                seen.append(lib.dct_orthogonalize(ctypes.byref(_muon((1, 4, 4))), h[0], h[1]))
        assert seen == [ERR["UNSUPPORTED"]]
    finally:
        dev.sync()
        dev.free(*h)
        dev.clear_error()


# ---------------------------------------------------------------------------
# gradients in one buffer
# ---------------------------------------------------------------------------
def test_attention_gradients_packed(dev):
    """dq, dk and dv interleaved in one buffer are those of three buffers; shared elements are refused."""
    lib = dev.lib
    b, t, h, d = 2, 5, 2, 8
    q, k, v, go = _inputs(b, t, t, h, h, d)
    apart = _attention(dev, q, k, v, go)
    st, packed = _packed(q.shape), (3 * t * h * d, 3 * h * d, d)
    hold = [dev.buf(x.ravel()) for x in (q, k, v, go)]
    out, lse, base = dev.empty(q.size), dev.empty(b * h * t), dev.empty(3 * q.size, fill=np.nan)
    hold += [out, lse, base]
    part = []
    for x in range(3):
        at = x * h * d
        part.append(lib.dct_wrap_device_ptr(lib.dct_buffer_device_ptr(base) + 4 * at, 3 * q.size - at))
    hold += part

    def back(dq, dk, dv, **kw):
        p = _abi.Attention(batch=b, q_heads=h, kv_heads=h, q_len=t, kv_len=t, head_dim=d,
                           **{x + "_stride": st for x in "qkvo"},
                           **{**{x + "_stride": packed for x in ("dq", "dk", "dv")}, **kw})
        return lib.dct_attention_backward(ctypes.byref(p), *hold[:3], None, None, out, lse, hold[3], dq, dk, dv)
    try:
        p = _abi.Attention(batch=b, q_heads=h, kv_heads=h, q_len=t, kv_len=t, head_dim=d,
                           **{x + "_stride": st for x in "qkvo"})
        _abi.check(lib, lib.dct_attention_forward(ctypes.byref(p), *hold[:3], None, None, out, lse))
        for order in ((0, 1, 2), (2, 0, 1)):
            _abi.check(lib, back(*(part[i] for i in order)))
            got = dev.read(base).reshape(b, t, 3, h, d)
            for name, i in zip(("dq", "dk", "dv"), order):
                assert np.array_equal(got[:, :, i], apart[name]), (name, order)
        assert back(part[0], part[1], part[1]) == ERR["ARG"]
        assert back(part[0], part[0], part[2]) == ERR["ARG"]
        assert back(part[0], part[1], part[2], dv_stride=(packed[0], h * d, d)) == ERR["ARG"]
        near = lib.dct_wrap_device_ptr(lib.dct_buffer_device_ptr(base) + 4 * (h * d - 1), 3 * q.size - h * d + 1)
        hold.append(near)
        assert back(part[0], near, part[2]) == ERR["ARG"]
    finally:
        dev.free(*reversed(hold))
        dev.clear_error()


def test_attention_refuses_log_sums_over_the_lengths(dev):
    lib = dev.lib
    h = [dev.empty(96) for _ in range(4)]
    lse = dev.empty(12)
    tail = lib.dct_wrap_device_ptr(lib.dct_buffer_device_ptr(lse) + 4 * 10, 2)
    st = (48, 16, 8)
    p = _abi.Attention(batch=2, q_heads=2, kv_heads=2, q_len=3, kv_len=3, head_dim=8,
                       **{x + "_stride": st for x in "qkvo"})
    try:
        for lens in ((lse, None), (None, lse), (tail, None), (None, tail)):
            assert lib.dct_attention_forward(ctypes.byref(p), *h[:3], *lens, h[3], lse) == ERR["ARG"], lens
        assert lib.dct_attention_forward(ctypes.byref(p), *h[:3], tail, None, h[3], None) == 0
    finally:
        dev.free(tail, lse, *h)
        dev.clear_error()


def test_attention_refuses_too_many_heads_without_positions(dev):
    """Heads and batch entries are bounded where the lengths are 0 as well."""
    lib = dev.lib
    h = [dev.empty(8) for _ in range(9)]
    try:
        for size in ({"q_heads": 1 << 31}, {"batch": 1 << 31}, {"batch": 1 << 20, "q_heads": 1 << 20},
                     {"q_heads": 1 << 28, "kv_heads": 1 << 28}, {"batch": (1 << 32) - 1}):
            p = _abi.Attention(**{"batch": 1, "q_heads": 1, "kv_heads": 1, "q_len": 0, "kv_len": 0, "head_dim": 8,
                                  **size})
            assert lib.dct_attention_forward(ctypes.byref(p), *h[:3], None, None, h[3], h[4]) == ERR["ARG"], size
            assert lib.dct_attention_backward(ctypes.byref(p), *h[:3], None, None, h[3], h[4], *h[5:9]) == \
                ERR["ARG"], size
    finally:
        dev.free(*h)
        dev.clear_error()


@pytest.mark.parametrize("rows", [False, True])
def test_attention_window_over_a_long_cache_of_many_query_heads(dev, rows):
    """Keys times query heads of a key head past 2^31: the rows that see an early key are none, as
    32-bit numbers too.  rows: a head that float16 pairs cannot hold."""
    n, h, d, w, near = 600_000, 4096, 4, 100, 200
    q, k, v, go = _inputs(1, 1, near, h, 1, d)
    if rows:
        k[0, -1] *= np.float32(2.0 ** -30)
    far_k, far_v = (np.concatenate((np.ones((1, n - near, 1, d), np.float32), x), 1) for x in (k, v))
    kw = {"causal": True, "window": w}
    got = _attention(dev, q, far_k, far_v, go, **kw)
    assert not got["dk"][:, :n - near].any() and not got["dv"][:, :n - near].any()
    got["dk"], got["dv"] = got["dk"][:, n - near:], got["dv"][:, n - near:]
    _hold(got, T.attention(q, k, v, go, **kw), ALL)


def test_orthogonalize_many_short_matrices(dev):
    """More clusters of one and two chunks a block than there are SMs, which no two may share."""
    r = np.random.default_rng(2)
    for shape in ((400, 16, 60), (300, 90, 100), (160, 40, 500)):
        x = r.normal(size=shape).astype(np.float32)
        h, y = dev.buf(x), dev.empty(x.size)
        try:
            _abi.check(dev.lib, dev.lib.dct_orthogonalize(ctypes.byref(_muon(shape, steps=2)), h, y))
            got = dev.read(y).reshape(shape)
        finally:
            dev.free(h, y)
        for i in range(0, len(x), 37):
            want, err = T.orthogonalize(x[i], steps=2)
            assert np.linalg.norm(got[i] - want) <= err


@pytest.mark.parametrize("shape,update", [((4000, 4, 2600), False), ((4000, 2600, 4), True), ((11000, 2, 2500), False),
                                          ((11000, 2500, 2), True)], ids=str)
def test_orthogonalize_of_a_batch_in_groups(dev, shape, update):
    """Thin matrices whose scratch would be far more than their data: a bounded part of it, in turn."""
    import torch
    r = np.random.default_rng(8)
    x = r.normal(size=shape).astype(np.float32)
    w = r.normal(size=shape).astype(np.float32)
    hs = [dev.buf(x), dev.buf(w), dev.buf(np.zeros(shape, np.float32))]
    before = torch.cuda.mem_get_info()[0]
    try:
        p = _muon(shape, steps=2, lr=0.5, momentum=0.9, scale=1.0)
        if update:
            _abi.check(dev.lib, dev.lib.dct_muon(ctypes.byref(p), hs[1], hs[2], hs[0]))
        else:
            _abi.check(dev.lib, dev.lib.dct_orthogonalize(ctypes.byref(p), hs[0], hs[1]))
        got, m = dev.read(hs[1]).reshape(shape), dev.read(hs[2]).reshape(shape)
        assert before - torch.cuda.mem_get_info()[0] < 5 << 30
    finally:
        dev.free(*hs)
    for i in (0, 1, len(x) // 2 - 1, len(x) // 2, len(x) // 2 + 1, len(x) - 1):
        want, err = T.orthogonalize(x[i], steps=2)
        if update:
            assert np.array_equal(m[i], x[i])
            want, err = w[i] - 0.5 * want, 0.5 * err + T.U * 2 * (np.linalg.norm(w[i]) + np.linalg.norm(want))
        assert np.linalg.norm(got[i] - want) <= err


def test_scaling_alone_takes_no_scratch_of_its_steps(dev):
    """Without steps a thin matrix is only divided by its norm."""
    import torch
    shape = (2, 1, 1 << 23)
    x = np.ones(shape, np.float32)
    hs = [dev.buf(x), dev.empty(x.size)]
    before = torch.cuda.mem_get_info()[0]
    try:
        _abi.check(dev.lib, dev.lib.dct_orthogonalize(ctypes.byref(_muon(shape, steps=0)), *hs))
        got = dev.read(hs[1])
        assert before - torch.cuda.mem_get_info()[0] < 1 << 30
    finally:
        dev.free(*hs)
    assert np.abs(got * np.sqrt(1 << 23) - 1).max() <= 4 * T.U


def test_a_gradient_of_the_log_sums_is_refused(dev):
    """It has no formula here: refused where one reaches them, not left out of the sum."""
    from directcompute_torch_b200 import ops
    q, k, v, go = _inputs(1, 5, 7, 2, 1, 8)
    t = [ops.tensor(x, requires_grad=True) for x in (q, k, v)]
    out, lse = ops.attention(*t, return_lse=True)
    want = T.attention(q, k, v, go)
    assert _max_over(np.abs(ops.to_numpy(lse) - want["lse"]), want["lse_tol"]) <= 1
    with pytest.raises(NotImplementedError):
        ops.add(ops.mul(out, out), ops.sum(ops.exp(lse))).backward()
    for x in t:
        x.grad = None
    out, lse = ops.attention(*t, return_lse=True)            # beside a backward pass that leaves them out
    out.backward(ops.tensor(go))
    got = {x: ops.to_numpy(y.grad) for x, y in zip(("dq", "dk", "dv"), t)}
    _hold(got, want, ("dq", "dk", "dv"))
    assert not ops.attention(*(ops.tensor(x) for x in (q, k, v)), return_lse=True)[1].requires_grad
