"""The measured cases of the transformer operators: rotary positions, attention with its
gradient, and the orthogonalised optimizer update.

`listed()` names the cases, `draw(rng)` gives others of the same ranges, `prepare(case, seed)`
makes a case's tensors on the GPU, and `run(state)` makes one pass: in plain torch operations
(`own` false) or through libdct_cuda's entry points (`own` true).  `work(case)` counts what a
pass cannot do without, and `exact(case, seed)` gives its result in 64 bits.

All tensors are float32 with the features of a head adjacent in memory, [batch, position,
head, feature]; index tensors are int32.  The library's calls take buffer handles; a program
that holds torch tensors wraps their device pointers for the call.
"""
import ctypes
import math

import torch

own = False


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one new token for each of 32 sequences, at far positions of its own: a step of generation
        {"name": "rotary_step", "op": "rotary", "batch": 32, "length": 1, "heads": 32, "dim": 128, "rotated": 128,
         "interleaved": False, "gradient": False, "positions": True, "packed": False, "factor": 1.0, "original": 0},
        # the queries of a training batch, half layout, frequencies scaled by parts for a longer context
        {"name": "rotary_long", "op": "rotary", "batch": 2, "length": 4096, "heads": 32, "dim": 128, "rotated": 128,
         "interleaved": False, "gradient": False, "positions": False, "packed": False, "factor": 8.0, "original": 8192},
        # the gradient for heads that are half rotated, interleaved, inside a packed projection of odd length
        {"name": "rotary_gradient", "op": "rotary", "batch": 3, "length": 1531, "heads": 12, "dim": 96, "rotated": 48,
         "interleaved": True, "gradient": True, "positions": False, "packed": True, "factor": 1.0, "original": 0},
        # one new token for each of 16 sequences against long ragged keys and values, four queries sharing a head
        {"name": "attend_step", "op": "attend", "batch": 16, "q_len": 1, "kv_len": 8191, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "causal": True, "window": 0, "ragged": True, "packed": False},
        # a chunk of new tokens after a context, odd lengths and a head width that is no power of two
        {"name": "attend_chunk", "op": "attend", "batch": 4, "q_len": 131, "kv_len": 2501, "q_heads": 16,
         "kv_heads": 16, "dim": 80, "causal": True, "window": 0, "ragged": True, "packed": False},
        # a whole prompt, causal, packed projection
        {"name": "attend_prompt", "op": "attend", "batch": 1, "q_len": 8192, "kv_len": 8192, "q_heads": 16,
         "kv_heads": 4, "dim": 128, "causal": True, "window": 0, "ragged": False, "packed": True},
        # training on short padded sequences, both directions visible (an encoder over image patches)
        {"name": "train_short", "op": "train", "batch": 8, "q_len": 197, "kv_len": 197, "q_heads": 12, "kv_heads": 12,
         "dim": 64, "causal": False, "window": 0, "ragged": True, "packed": True},
        # training with a sliding window
        {"name": "train_window", "op": "train", "batch": 2, "q_len": 2048, "kv_len": 2048, "q_heads": 12,
         "kv_heads": 6, "dim": 64, "causal": True, "window": 500, "ragged": False, "packed": False},
        # training on long causal sequences, four query heads to a key head
        {"name": "train_long", "op": "train", "batch": 2, "q_len": 4096, "kv_len": 4096, "q_heads": 16, "kv_heads": 4,
         "dim": 128, "causal": True, "window": 0, "ragged": False, "packed": False},
        # one small tall matrix of odd sides
        {"name": "orthogonalize_small", "op": "orthogonalize", "batch": 1, "rows": 333, "cols": 127},
        # the attention projections of a stack of layers, updated together
        {"name": "muon_layers", "op": "muon", "batch": 12, "rows": 768, "cols": 768},
        # a large feed-forward matrix
        {"name": "muon_large", "op": "muon", "batch": 1, "rows": 2048, "cols": 8192},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rotary", "attend", "attend", "train", "train", "orthogonalize", "muon"])
    if op == "rotary":
        dim = 2 * rng.randint(8, 64)
        length = _log_int(rng, 1, 4096)
        heads = rng.randint(1, 32)
        batch = max(1, min(rng.randint(1, 32), (1 << 25) // (length * heads * dim)))
        scaled = rng.random() < 0.4
        return {"op": op, "batch": batch, "length": length, "heads": heads, "dim": dim,
                "rotated": rng.choice([dim, dim, 2 * rng.randint(1, dim // 2)]), "interleaved": rng.random() < 0.5,
                "gradient": rng.random() < 0.5, "positions": rng.random() < 0.5, "packed": rng.random() < 0.5,
                "factor": round(rng.uniform(1.5, 16), 2) if scaled else 1.0,
                "original": rng.choice([0, 2048, 8192]) if scaled else 0}
    if op in ("attend", "train"):
        kv_heads = rng.choice([1, 2, 4, 6, 8])
        group = rng.choice([1, 1, 2, 4])
        kv_len = _log_int(rng, 1, 4096)
        q_len = kv_len if op == "train" and rng.random() < 0.7 else rng.choice([1, _log_int(rng, 1, kv_len), kv_len])
        batch = max(1, min(rng.randint(1, 12), (1 << 28) // (kv_heads * group * q_len * kv_len)))
        return {"op": op, "batch": batch, "q_len": q_len, "kv_len": kv_len, "q_heads": kv_heads * group,
                "kv_heads": kv_heads, "dim": rng.choice([32, 64, 64, 80, 96, 128, 128, rng.randint(9, 128)]),
                "causal": rng.random() < 0.6, "window": rng.choice([0, 0, rng.randint(1, kv_len)]),
                "ragged": rng.random() < 0.4, "packed": q_len == kv_len and rng.random() < 0.5}
    rows, cols = _log_int(rng, 16, 2048), _log_int(rng, 16, 8192)
    batch = max(1, min(rng.choice([1, 1, 2, 4, 12]), (1 << 34) // (min(rows, cols) * rows * cols)))
    rows, cols = (cols, rows) if rng.random() < 0.5 else (rows, cols)
    return {"op": op, "batch": batch, "rows": rows, "cols": cols}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
BASE = 10000.0
LOW, HIGH = 1.0, 32.0                        # rotations over the original context between which frequencies blend
COEFFICIENTS = (3.4445, -4.7750, 2.0315)     # the quintic of the Newton-Schulz steps
STEPS, EPS = 5, 1e-7
RATE, MOMENTUM, DECAY = 0.02, 0.95, 0.01


def _lengths(case):
    """(q lengths, key lengths) of a ragged batch: from full ones down to a sequence with a third of the keys."""
    n, q, k = case["batch"], case["q_len"], case["kv_len"]
    share = [1.0 - 2.0 * ((7 * b) % n) / (3.0 * n) for b in range(n)]
    kv = [max(1, int(round(k * s))) for s in share]
    return [min(q, x) if case["op"] == "train" or q > 1 else q for x in kv], kv


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    s = dict(case)
    if case["op"] == "rotary":
        b, t, h, d = case["batch"], case["length"], case["heads"], case["dim"]
        s["x"] = normal(b, t, 3, h, d)[:, :, 1] if case["packed"] else normal(b, t, h, d)
        s["where"] = torch.randint(0, 1 << 20, (b, t), generator=g, device="cuda",
                                   dtype=torch.int32) if case["positions"] else None
        s["y"] = torch.empty((b, t, h, d), device="cuda")
    elif case["op"] in ("attend", "train"):
        b, q, k, hq, hk, d = (case[n] for n in ("batch", "q_len", "kv_len", "q_heads", "kv_heads", "dim"))
        if case["packed"]:                   # one projection holds q, k and v side by side
            qkv = normal(b, q, hq + 2 * hk, d)
            s["q"], s["k"], s["v"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk], qkv[:, :, hq + hk:]
        else:
            s["q"], s["k"], s["v"] = normal(b, q, hq, d), normal(b, k, hk, d), normal(b, k, hk, d)
        s["q_lens"] = s["kv_lens"] = None
        if case["ragged"]:
            s["q_lens"], s["kv_lens"] = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in _lengths(case))
        s["out"], s["lse"] = torch.empty((b, q, hq, d), device="cuda"), torch.empty((b, hq, q), device="cuda")
        if case["op"] == "train":
            s["dout"] = normal(b, q, hq, d)
            s["dq"], s["dk"], s["dv"] = (torch.empty(x.shape, device="cuda") for x in (s["q"], s["k"], s["v"]))
    else:
        n, r, c = case["batch"], case["rows"], case["cols"]
        # a gradient of few strong directions over weak noise
        few = max(1, min(r, c) // 8)
        s["g"] = 1e-3 * (torch.bmm(normal(n, r, few), normal(n, few, c)) / math.sqrt(few) + 0.3 * normal(n, r, c))
        if case["op"] == "orthogonalize":
            s["y"] = torch.empty_like(s["g"])
        else:
            s["w"], s["m"] = 0.02 * normal(n, r, c), 1e-3 * normal(n, r, c)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _frequencies(s, device):
    """Angle per position of each pair, in 64 bits."""
    r = s["rotated"]
    f = BASE ** (-torch.arange(0, r, 2, dtype=torch.float64, device=device) / r)
    if s["factor"] != 1.0:
        keep = torch.zeros_like(f) if not s["original"] else \
            ((s["original"] * f / (2 * math.pi) - LOW) / (HIGH - LOW)).clamp(0, 1)
        f = f * (keep + (1 - keep) / s["factor"])
    return f


def _magnitude(s):
    return 0.1 * math.log(s["factor"]) + 1.0 if s["factor"] != 1.0 and s["original"] else 1.0


def _plain_rotary(s):
    x, r = s["x"], s["rotated"]
    where = s["where"] if s["where"] is not None else torch.arange(x.shape[1], device=x.device)[None]
    angle = where.double()[:, :, None, None] * _frequencies(s, x.device)
    c, n = (_magnitude(s) * angle.cos()).float(), (_magnitude(s) * angle.sin()).float()
    n = -n if s["gradient"] else n
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if s["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
    u, v = a * c - b * n, b * c + a * n
    turned = torch.stack((u, v), -1).flatten(-2) if s["interleaved"] else torch.cat((u, v), -1)
    return torch.cat((turned, x[..., r:]), -1)


def _visible(s, device):
    """[batch or 1, q_len, kv_len]: the keys that each query sees."""
    i = torch.arange(s["q_len"], device=device)[None, :, None]
    j = torch.arange(s["kv_len"], device=device)[None, None, :]
    m = s["q_lens"][:, None, None].long() if s["q_lens"] is not None else s["q_len"]
    n = s["kv_lens"][:, None, None].long() if s["kv_lens"] is not None else s["kv_len"]
    at = i + n - m
    seen = (i < m) & (j < n)
    if s["causal"]:
        seen = seen & (j <= at)
    if s["window"]:
        seen = seen & (j > at - s["window"]) & (j < at + s["window"])
    return seen


def _grouped(x, heads):
    """[b, t, h, d] as [b, heads, h / heads * t, d]: the query heads of one key head side by side."""
    b, t, h, d = x.shape
    return x.reshape(b, t, heads, h // heads, d).permute(0, 2, 3, 1, 4).reshape(b, heads, h // heads * t, d)


def _spread(x, t):
    """The reverse of _grouped."""
    b, heads, gt, d = x.shape
    return x.reshape(b, heads, gt // t, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, heads * (gt // t), d)


def _plain_attention(s):
    b, t, hq, d = s["q"].shape
    hk = s["k"].shape[2]
    q, k, v = _grouped(s["q"], hk), s["k"].transpose(1, 2), s["v"].transpose(1, 2)
    scale = 1.0 / math.sqrt(d)
    seen = _visible(s, q.device)[:, None].repeat(1, 1, hq // hk, 1)
    x = torch.matmul(q, k.transpose(2, 3)).mul_(scale).masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total > 0, total.log() + top, -math.inf)
    p = p.div_(total.masked_fill(total == 0, 1.0))
    out = torch.matmul(p, v)
    lse = lse.reshape(b, hq, t)
    if s["op"] == "attend":
        return _spread(out, t), lse
    do = _grouped(s["dout"], hk)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3)).sub_((do * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3), q)
    return _spread(out, t), lse, _spread(dq, t), dk.transpose(1, 2).contiguous(), dv.transpose(1, 2).contiguous()


def _plain_orthogonalize(g):
    a, b, c = COEFFICIENTS
    x = g / (g.double().square().sum((1, 2), keepdim=True).sqrt().float() + EPS)
    tall = g.shape[1] > g.shape[2]
    x = x.transpose(1, 2) if tall else x
    for _ in range(STEPS):
        y = torch.matmul(x, x.transpose(1, 2))
        x = a * x + torch.matmul(b * y + c * torch.matmul(y, y), x)
    return x.transpose(1, 2).contiguous() if tall else x


def _plain_muon(s):
    m = s["m"].mul_(MOMENTUM).add_(s["g"])
    o = _plain_orthogonalize(s["g"] + MOMENTUM * m)
    scale = math.sqrt(max(1.0, s["rows"] / s["cols"]))
    return s["w"].mul_(1 - RATE * DECAY).sub_(RATE * scale * o), m


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------
def _library():
    """The library.  Its calls are ordered on its own stream and on no other, so torch's work goes there from
    the first call on: what torch has written is there for a call, and what a call writes for torch."""
    from directcompute_torch_b200 import load_library
    lib = load_library()
    if not hasattr(_library, "stream"):
        if not lib.InitEngine():
            raise RuntimeError("libdct_cuda: " + lib.dct_last_error().decode())
        _library.stream = torch.cuda.ExternalStream(lib.dct_stream(), device=lib.dct_device())
        _library.stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(_library.stream)
    return lib


def _call(function, struct, *tensors):
    """One library call over torch tensors: their device pointers wrapped as handles for its time."""
    from directcompute_torch_b200 import _abi
    lib = _library()
    handles = [None if t is None else lib.dct_wrap_device_ptr(t.data_ptr(), 1 + sum(
        (n - 1) * st for n, st in zip(t.shape, t.stride()))) for t in tensors]
    status = getattr(lib, function)(ctypes.byref(struct), *handles)
    for h in handles:
        if h is not None:
            lib.ReleaseBuffer(h)
    _abi.check(lib, status, function)


def _own_rotary(s):
    from directcompute_torch_b200 import _abi
    x, y = s["x"], s["y"]
    p = _abi.Rotary(batch=s["batch"], length=s["length"], heads=s["heads"], head_dim=s["dim"],
                    x_stride=x.stride()[:3], y_stride=y.stride()[:3], rotated=s["rotated"],
                    interleaved=s["interleaved"], inverse=s["gradient"], start=0, base=BASE, factor=s["factor"],
                    original=s["original"], low=LOW, high=HIGH, magnitude=_magnitude(s))
    _call("dct_rotary", p, x, s["where"], y)
    return y


def _own_attention(s):
    from directcompute_torch_b200 import _abi
    q, k, v, out = s["q"], s["k"], s["v"], s["out"]
    p = _abi.Attention(batch=s["batch"], q_heads=s["q_heads"], kv_heads=s["kv_heads"], q_len=s["q_len"],
                       kv_len=s["kv_len"], head_dim=s["dim"], causal=s["causal"], window=s["window"],
                       q_stride=q.stride()[:3], k_stride=k.stride()[:3], v_stride=v.stride()[:3],
                       o_stride=out.stride()[:3], dq_stride=out.stride()[:3], scale=0.0)
    if s["op"] == "attend":
        _call("dct_attention_forward", p, q, k, v, s["q_lens"], s["kv_lens"], out, s["lse"])
        return out, s["lse"]
    p.dq_stride[:], p.dk_stride[:], p.dv_stride[:] = (s[n].stride()[:3] for n in ("dq", "dk", "dv"))
    _call("dct_attention_forward", p, q, k, v, s["q_lens"], s["kv_lens"], out, s["lse"])
    _call("dct_attention_backward", p, q, k, v, s["q_lens"], s["kv_lens"], out, s["lse"], s["dout"], s["dq"],
          s["dk"], s["dv"])
    return out, s["lse"], s["dq"], s["dk"], s["dv"]


def _own_orthogonalize(s):
    from directcompute_torch_b200 import _abi
    a, b, c = COEFFICIENTS
    p = _abi.Muon(batch=s["batch"], rows=s["rows"], cols=s["cols"], steps=STEPS, a=a, b=b, c=c, eps=EPS)
    if s["op"] == "orthogonalize":
        _call("dct_orthogonalize", p, s["g"], s["y"])
        return s["y"]
    p.lr, p.momentum, p.weight_decay, p.nesterov = RATE, MOMENTUM, DECAY, 1
    p.scale = math.sqrt(max(1.0, s["rows"] / s["cols"]))
    _call("dct_muon", p, s["w"], s["m"], s["g"])
    return s["w"], s["m"]


def run(state):
    if own:
        return _own_rotary(state) if state["op"] == "rotary" else \
            _own_attention(state) if state["op"] in ("attend", "train") else _own_orthogonalize(state)
    if state["op"] == "rotary":
        return _plain_rotary(state)
    if state["op"] in ("attend", "train"):
        return _plain_attention(state)
    return _plain_orthogonalize(state["g"]) if state["op"] == "orthogonalize" else _plain_muon(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _pairs(case):
    """(query, key) pairs that are visible, over the batch, for one head."""
    total = 0
    lengths = zip(*_lengths(case)) if case["ragged"] else [(case["q_len"], case["kv_len"])] * case["batch"]
    w = case["window"]
    for m, n in lengths:
        i = torch.arange(m, dtype=torch.int64) + n - m
        low = (i - w + 1).clamp(min=0) if w else torch.zeros_like(i)
        high = (i + 1).clamp(max=n) if case["causal"] else ((i + w).clamp(max=n) if w else torch.full_like(i, n))
        total += int((high - low).clamp(min=0).sum())
    return total


def work(case):
    if case["op"] == "rotary":
        n = case["batch"] * case["length"] * case["heads"] * case["dim"]
        return {"bytes": 8 * n + (4 * case["batch"] * case["length"] if case["positions"] else 0), "flops": 3 * n}
    if case["op"] in ("attend", "train"):
        q_lens, kv_lens = _lengths(case) if case["ragged"] else ([case["q_len"]] * case["batch"],
                                                                 [case["kv_len"]] * case["batch"])
        d, hq, hk = case["dim"], case["q_heads"], case["kv_heads"]
        rows = case["batch"] * case["q_len"] * hq
        read = 4 * d * (sum(q_lens) * hq + 2 * sum(kv_lens) * hk)
        n = {"bytes": read + 4 * rows * (d + 1), "flops": 4 * d * hq * _pairs(case)}
        if case["op"] == "train":    # reads dout, writes dq, dk and dv; five products beside the forward pass's two
            n["bytes"] += 4 * d * (2 * rows + 2 * case["batch"] * case["kv_len"] * hk)
            n["flops"] += 10 * d * hq * _pairs(case)
        return n
    r, c = sorted((case["rows"], case["cols"]))
    n = case["batch"]
    # the two products with symmetric results need one triangle of them
    flops = STEPS * n * (r * (r + 1) * c + r * r * (r + 1) + 2 * r * r * c)
    return {"bytes": 4 * n * r * c * (2 if case["op"] == "orthogonalize" else 5), "flops": flops}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rotary(s):
    x = s["x"].double()
    r, half = s["rotated"], s["rotated"] // 2
    out = x.clone()
    where = s["where"].double() if s["where"] is not None else \
        torch.arange(s["length"], dtype=torch.float64, device=x.device).expand(s["batch"], -1)
    for j in range(half):
        f = BASE ** (-2.0 * j / r)
        if s["factor"] != 1.0:
            blend = min(1.0, max(0.0, (s["original"] * f / (2 * math.pi) - LOW) / (HIGH - LOW))) if s["original"] else 0.0
            f = (1 - blend) * f / s["factor"] + blend * f
        turn = torch.polar(torch.full_like(where, _magnitude(s)), (-1.0 if s["gradient"] else 1.0) * where * f)
        one, two = (2 * j, 2 * j + 1) if s["interleaved"] else (j, j + half)
        z = torch.complex(x[..., one], x[..., two]) * turn[..., None]
        out[..., one], out[..., two] = z.real, z.imag
    return out


def _exact_attention(s):
    """Head by head and sequence by sequence, the gradients by differentiation."""
    train = s["op"] == "train"
    b, t, hq, d = s["q"].shape
    hk, n = s["k"].shape[2], s["k"].shape[1]
    new = lambda x: torch.zeros(x.shape, dtype=torch.float64, device=x.device)  # noqa: E731
    out, lse = new(s["q"]), torch.full((b, hq, t), -math.inf, dtype=torch.float64, device=s["q"].device)
    dq, dk, dv = new(s["q"]), new(s["k"]), new(s["v"])
    for e in range(b):
        m = int(s["q_lens"][e]) if s["q_lens"] is not None else t
        k_n = int(s["kv_lens"][e]) if s["kv_lens"] is not None else n
        gap = (torch.arange(m)[:, None] + (k_n - m) - torch.arange(k_n)[None]).to(out.device)
        hide = torch.zeros_like(gap, dtype=torch.bool)
        if s["causal"]:
            hide |= gap < 0
        if s["window"]:
            hide |= gap.abs() >= s["window"] if not s["causal"] else gap >= s["window"]
        alive = ~hide.all(1)
        for h in range(hq):
            q, k, v = (x[e, :y, z].double().requires_grad_(train) for x, y, z in (
                (s["q"], m, h), (s["k"], k_n, h // (hq // hk)), (s["v"], k_n, h // (hq // hk))))
            scores = (q @ k.t() / math.sqrt(d))[alive].masked_fill(hide[alive], -math.inf)
            o = torch.softmax(scores, 1) @ v
            out[e, :m, h][alive] = o.detach()
            lse[e, h, :m][alive] = torch.logsumexp(scores.detach(), 1)
            if train and bool(alive.any()):
                gq, gk, gv = torch.autograd.grad(o, (q, k, v), s["dout"][e, :m, h].double()[alive])
                dq[e, :m, h] += gq
                dk[e, :k_n, h // (hq // hk)] += gk
                dv[e, :k_n, h // (hq // hk)] += gv
    return (out, lse, dq, dk, dv) if train else (out, lse)


def _exact_orthogonalize(u):
    """Through the polynomial in each matrix's Gram matrix on its shorter side."""
    a, b, c = COEFFICIENTS
    x = u / (torch.linalg.vector_norm(u, dim=(1, 2), keepdim=True) + EPS)
    wide = u.shape[1] <= u.shape[2]
    eye = torch.eye(min(u.shape[1:]), dtype=torch.float64, device=u.device)
    for _ in range(STEPS):
        g = x @ x.mT if wide else x.mT @ x
        poly = a * eye + g @ (b * eye + c * g)
        x = poly @ x if wide else x @ poly
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(s)
    if case["op"] in ("attend", "train"):
        return _exact_attention(s)
    if case["op"] == "orthogonalize":
        return _exact_orthogonalize(s["g"].double())
    m = MOMENTUM * s["m"].double() + s["g"].double()
    o = _exact_orthogonalize(s["g"].double() + MOMENTUM * m)
    scale = math.sqrt(max(1.0, case["rows"] / case["cols"]))
    return (1 - RATE * DECAY) * s["w"].double() - RATE * scale * o, m
