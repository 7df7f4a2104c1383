"""Sequence operators of a splat predictor: what is measured, and their plain forms.

A network that predicts Gaussians from a stream of posed views works on one
token per 16 x 16 tile of a view, the rasterizer's own tile grid: 1200 tokens
for a 640 x 480 frame, 8160 for full HD, 2500 for each of 16 views of 800².
Its blocks are a root-mean-square norm with the residual's addition, a gated
linear recurrence and attention with a sliding window in which the stream's
first tokens stay visible.  With ``own`` true, ``run`` calls them through
``gaussian_splats_hip.sequence``; with ``own`` false it computes them with
elementary torch operations in float32.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = Path(__file__).resolve().parents[1] / "gaussian-splats_amd"
if str(_PACKAGE) not in sys.path:
    sys.path.insert(0, str(_PACKAGE))

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}


def _attention(name, batch, tq, tk, heads, kv_heads, dim, window, sinks, dtype, grad, ragged=False):
    case = {"op": "attention", "batch": batch, "tq": tq, "tk": tk, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks, "dtype": dtype,
            "grad": grad, "ragged": ragged}
    return {"name": name, **case} if name else case


def _step(name, batch, heads, kv_heads, dim, window, sinks, dtype, ragged=False):
    case = {"op": "attention_step", "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "window": window, "sinks": sinks, "dtype": dtype, "ragged": ragged}
    return {"name": name, **case} if name else case


def _scan(name, batch, tokens, channels, dtype, grad, state):
    case = {"op": "scan", "batch": batch, "tokens": tokens, "channels": channels, "dtype": dtype,
            "grad": grad, "state": state}
    return {"name": name, **case} if name else case


def _scan_step(name, batch, channels, dtype):
    case = {"op": "scan_step", "batch": batch, "channels": channels, "dtype": dtype}
    return {"name": name, **case} if name else case


def _norm(name, rows, width, dtype, residual, grad, quant=""):
    case = {"op": "norm", "rows": rows, "width": width, "dtype": dtype, "residual": residual,
            "grad": grad, "quant": quant}
    return {"name": name, **case} if name else case


def listed():
    return [
        # A training step's attention over one 640 x 480 frame.
        _attention("frame attention", 1, 1200, 1200, 8, 8, 64, 300, 4, "bf16", True),
        # The same over a batch of 16 views of 800² in stream order: a window
        # of two views, shared key heads.
        _attention("view stream attention", 1, 40000, 40000, 12, 4, 64, 5000, 16, "bf16", True),
        # Two full-HD frames taken into a stream, one of them shorter: forward only.
        _attention("full HD prefill", 2, 8160, 8160, 16, 4, 128, 2040, 8, "f16", False, True),
        # Small fits in float32, the rasterizer's own type, at odd sizes.
        _attention("odd attention f32", 2, 777, 777, 6, 2, 40, 131, 3, "f32", True),
        # One new token of one stream: latency.
        _step("one stream's step", 1, 8, 8, 64, 2500, 4, "bf16"),
        # One new token of each of many streams, their caches filled to
        # different lengths, some of them wrapped around.
        _step("many streams' step", 32, 32, 8, 128, 8160, 16, "bf16", True),
        # The recurrence's training step over two full-HD frames.
        _scan("full HD scan", 2, 8160, 1024, "bf16", True, True),
        # The same over 16 views of 800² at one token per 8 x 8 pixels.
        _scan("long scan", 1, 160000, 768, "bf16", True, False),
        # Small fits in float32 at odd sizes.
        _scan("odd scan f32", 3, 1201, 331, "f32", True, True),
        # One new token of each of many streams.
        _scan_step("scan step", 32, 1024, "f16"),
        # The norm's training step on the view stream, the residual kept in float32.
        _norm("norm step", 40000, 768, "bf16", "f32", True),
        # The norm before an 8-bit product while streaming: few rows, latency.
        _norm("norm int8", 32, 4096, "bf16", "bf16", False, "int8"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "attention_step", "scan", "scan",
                     "scan_step", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4])
        dim = rng.choice([32, 40, 64, 64, 80, 128])
        batch = rng.choice([1, 1, 2, 3])
        tk = _log_int(rng, 64, 40000)
        tq = tk if rng.random() < 0.8 else max(1, tk // rng.choice([2, 3, 5]))
        window = min(tk, _log_int(rng, 16, 8192))
        # Float32 runs at a sixteenth of the 16-bit rate.
        budget = 40000 * 5000 * 12 * 64 // (16 if dtype == "f32" else 1)
        while batch * heads * tq * window * dim > budget:
            window, tq = max(16, window // 2), max(16, (tq * 3) // 4)
        sinks = rng.choice([0, 1, 4, 16, 67])
        return _attention(None, batch, tq, tk, heads, kv_heads, dim, window, sinks, dtype,
                          rng.random() < 0.7, rng.random() < 0.3)
    if op == "attention_step":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 7, 8])
        dim = rng.choice([64, 80, 128])
        batch, window = _log_int(rng, 1, 32), _log_int(rng, 64, 8160)
        return _step(None, batch, heads, kv_heads, dim, window, rng.choice([0, 4, 16]),
                     rng.choice(["bf16", "f16"]), rng.random() < 0.6)
    if op == "scan":
        channels = _log_int(rng, 64, 2048)
        tokens = _log_int(rng, 16, 160000)
        batch = rng.choice([1, 2, 3, 8])
        while batch * tokens * channels * SIZES[dtype] > 160000 * 768 * 2:
            tokens = max(1, tokens // 2)
        return _scan(None, batch, tokens, channels, dtype, rng.random() < 0.7, rng.random() < 0.5)
    if op == "scan_step":
        return _scan_step(None, _log_int(rng, 1, 256), _log_int(rng, 64, 4096), dtype)
    width = _log_int(rng, 64, 8192)
    if rng.random() < 0.7:
        width = -(-width // 8) * 8
    rows = _log_int(rng, 1, 40000)
    while rows * width > 40000 * 2048:
        rows = max(1, rows // 2)
    quant = rng.choice(["", "", "int8", "e4m3"])
    residual = rng.choice([dtype, "f32", ""])
    return _norm(None, rows, width, dtype, residual, not quant and rng.random() < 0.7, quant)


def _visible_pairs(tq, tk, window, sinks, length):
    """Number of (query, key) pairs of one head that the mask leaves."""
    p = torch.arange(tk - tq, tk, dtype=torch.int64)
    top = torch.minimum(p + 1, torch.tensor(length)).clamp_min(0)
    low = torch.minimum((p + 1 - window).clamp_min(0), top)
    return int((top - low + torch.minimum(low, torch.tensor(sinks))).sum())


def _lengths(case):
    """Keys of each sequence that exist, fixed by the case."""
    b, tk = case["batch"], case["tk"]
    return [tk - (tk * 2 * i) // (5 * b) if case["ragged"] else tk for i in range(b)]


def _positions(case):
    """Position of each stream's new token: half filled up to wrapped around."""
    b, n = case["batch"], case["sinks"] + case["window"]
    if not case["ragged"]:
        return [n + n // 3] * b
    return [n // 2 + (n * 3 * i) // (2 * b) for i in range(b)]


def work(case):
    if case["op"] == "scan":
        n = case["batch"] * case["tokens"] * case["channels"]
        ends = case["batch"] * case["channels"] * 4
        arrays = 6 if case["grad"] else 3
        return {"bytes": n * arrays * SIZES[case["dtype"]] + ends * (5 if case["grad"] else 2),
                "flops": n * (20 if case["grad"] else 8)}
    if case["op"] == "scan_step":
        n = case["batch"] * case["channels"]
        return {"bytes": n * (3 * SIZES[case["dtype"]] + 8), "flops": n * 8}
    if case["op"] == "norm":
        n, e = case["rows"] * case["width"], SIZES[case["dtype"]]
        s = SIZES[case["residual"]] if case["residual"] else 0
        moved = n * (e + 2 * s)  # x and the residual in, their sum out
        moved += n + 4 * case["rows"] if case["quant"] else n * e
        if case["grad"]:  # both outputs' gradients in, the inputs' out
            moved += n * (2 * e + s + (s or e))
        return {"bytes": moved, "flops": n * (16 if case["grad"] else 6)}
    e, d = SIZES[case["dtype"]], case["dim"]
    if case["op"] == "attention_step":
        seen = sum(min(p + 1, case["sinks"] + case["window"]) for p in _positions(case))
        io = case["batch"] * (2 * case["heads"] + 4 * case["kv_heads"]) * d
        return {"bytes": (2 * seen * case["kv_heads"] * d + io) * e,
                "flops": 4 * seen * case["heads"] * d}
    pairs = case["heads"] * sum(_visible_pairs(case["tq"], case["tk"], case["window"],
                                               case["sinks"], n) for n in _lengths(case))
    nq = case["batch"] * case["tq"] * case["heads"] * d
    nk = case["batch"] * case["tk"] * case["kv_heads"] * d
    arrays = (4 * nq + 4 * nk) if case["grad"] else (2 * nq + 2 * nk)
    return {"bytes": arrays * e, "flops": pairs * d * (14 if case["grad"] else 4)}


def _data(case, seed):
    """Inputs of a case from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(TYPES[dtype])

    t = case["dtype"]
    if case["op"] == "attention":
        b, tq, tk, h, hk, d = (case[k] for k in ("batch", "tq", "tk", "heads", "kv_heads", "dim"))
        s = {"q": normal((b, tq, h, d), t), "k": normal((b, tk, hk, d), t),
             "v": normal((b, tk, hk, d), t)}
        if case["grad"]:
            s["grad"] = normal((b, tq, h, d), t, 0.1)
        if case["ragged"]:
            s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        return s
    if case["op"] == "attention_step":
        b, h, hk, d = (case[k] for k in ("batch", "heads", "kv_heads", "dim"))
        n = case["sinks"] + case["window"]
        return {"q": normal((b, h, d), t), "k": normal((b, hk, d), t), "v": normal((b, hk, d), t),
                "k_cache": normal((b, n, hk, d), t), "v_cache": normal((b, n, hk, d), t),
                "positions": torch.tensor(_positions(case), dtype=torch.int32, device="cuda")}
    if case["op"] == "scan":
        shape = (case["batch"], case["tokens"], case["channels"])
        # Gates around sigmoid(3): memories of some twenty tokens, some far longer.
        s = {"x": normal(shape, t), "gate": normal(shape, t, 2.0, 3.0)}
        if case["state"]:
            s["state"] = normal((shape[0], shape[2]), "f32")
        if case["grad"]:
            s["grad"] = normal(shape, t, 0.1)
            s["grad_last"] = normal((shape[0], shape[2]), "f32", 0.1)
        return s
    if case["op"] == "scan_step":
        shape = (case["batch"], case["channels"])
        return {"x": normal(shape, t), "gate": normal(shape, t, 2.0, 3.0),
                "state": normal(shape, "f32")}
    shape = (case["rows"], case["width"])
    s = {"x": normal(shape, t), "weight": normal(shape[1:], t, 0.1, 1.0)}
    if case["residual"]:
        s["residual"] = normal(shape, case["residual"], 2.0)
    if case["grad"]:
        s["grad"] = normal(shape, t, 0.1)
        s["grad_sum"] = normal(shape, case["residual"] or t, 0.1)
    return s


#: What a training step takes gradients of, in the order in which run() returns them.
LEAVES = {"attention": ("q", "k", "v"), "scan": ("x", "gate", "state"),
          "norm": ("x", "residual", "weight")}


def prepare(case, seed):
    data = _data(case, seed)
    if case.get("grad"):
        for name in LEAVES[case["op"]]:
            if name in data:
                data[name].requires_grad_(True)
    return {"case": case, **data}


def _own(s):
    from gaussian_splats_hip import sequence

    case, op = s["case"], s["case"]["op"]
    if op == "attention":
        outputs = (sequence.window_attention(s["q"], s["k"], s["v"], case["window"], case["sinks"],
                                             lengths=s.get("lengths")),)
        grads = (s.get("grad"),)
    elif op == "attention_step":
        out = sequence.window_attention_step(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"],
                                             s["positions"], case["window"], case["sinks"])
        return out, s["k_cache"], s["v_cache"]
    elif op == "scan":
        outputs = sequence.gated_scan(s["x"], s["gate"], s.get("state"))
        grads = (s.get("grad"), s.get("grad_last"))
    elif op == "scan_step":
        return sequence.gated_scan_step(s["x"], s["gate"], s["state"])
    elif case["quant"]:
        codes, scales, total = sequence.add_rms_norm_quant(s["x"], s.get("residual"), s["weight"],
                                                           EPS, case["quant"])
        # Eight bits come back as the values that they stand for.
        return (codes.float() * scales[:, None]).to(torch.bfloat16), scales, total
    else:
        outputs = sequence.add_rms_norm(s["x"], s.get("residual"), s["weight"], EPS)
        grads = (s.get("grad"), s.get("grad_sum"))
    if not case["grad"]:
        return outputs
    leaves = [s[n] for n in LEAVES[op] if n in s]
    return tuple(o.detach() for o in outputs) + torch.autograd.grad(outputs, leaves, grads)


def _plain_attention(s):
    """Blocks of queries against the keys that their windows reach, and against
    the first tokens."""
    case = s["case"]
    b, tq, tk, h, hk, d = (case[k] for k in ("batch", "tq", "tk", "heads", "kv_heads", "dim"))
    g, dev = h // hk, s["q"].device
    window, sinks = min(case["window"], tk), min(case["sinks"], tk)
    n = min(tq, 512, max(64, window))  # queries of a block
    nb = -(-tq // n)
    pad = nb * n - tq
    scale = 1.0 / math.sqrt(d)

    def rows(t):  # [B, Tq, H, D] -> [B, Hkv, blocks, G * n, D]
        t = torch.cat([t.float(), t.new_zeros((b, pad, h, d), dtype=torch.float32)], 1)
        return t.view(b, nb, n, hk, g, d).permute(0, 3, 1, 4, 2, 5).reshape(b, hk, nb, g * n, d)

    def back(t):
        t = t.view(b, hk, nb, g, n, d).permute(0, 2, 4, 1, 3, 5).reshape(b, nb * n, h, d)
        return t[:, :tq]

    q = rows(s["q"])
    first = tk - tq + torch.arange(nb, device=dev)[:, None] * n
    p = first + torch.arange(n, device=dev)  # [blocks, n]
    near = first - window + 1 + torch.arange(n + window - 1, device=dev)  # [blocks, L]
    length = (s["lengths"] if "lengths" in s else torch.full((1,), tk, device=dev)).view(-1, 1, 1, 1)
    seen = ((near[:, None] <= p[..., None]) & (near[:, None] > p[..., None] - window)
            & (near[:, None] >= 0) & (near[:, None] < length))  # [B or 1, blocks, n, L]
    # The first tokens, where the window does not hold them already.
    j = torch.arange(sinks, device=dev)
    seen_first = ((j <= p[..., None] - window) & (j < length)).expand(seen.shape[0], nb, n, sinks)
    seen = torch.cat([seen, seen_first], -1)[:, None, :, None].expand(-1, -1, -1, g, -1, -1)
    seen = seen.reshape(seen.shape[0], 1, nb, g * n, -1)
    index = torch.cat([near.clamp(0, tk - 1), j.expand(nb, sinks)], 1)  # [blocks, L + S]
    k = s["k"].float().transpose(1, 2)[:, :, index]  # [B, Hkv, blocks, L + S, D]
    v = s["v"].float().transpose(1, 2)[:, :, index]
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min_(-1e30)
    probs = scores.sub_(top).exp_()
    total = probs.sum(-1, keepdim=True)
    probs = probs.div_(total.clamp_min(1e-30))
    out = torch.matmul(probs, v)
    result = (back(out).to(s["q"].dtype),)
    if not case["grad"]:
        return result
    grad = rows(s["grad"])
    at = index.reshape(-1)

    def gather(t):  # [B, Hkv, blocks, L + S, D] -> [B, Tk, Hkv, D]
        whole = torch.zeros((b, hk, tk, d), device=dev)
        return whole.index_add_(2, at, t.reshape(b, hk, -1, d)).transpose(1, 2)

    dv = gather(torch.matmul(probs.transpose(-1, -2), grad))
    ds = torch.matmul(grad, v.transpose(-1, -2)).sub_((grad * out).sum(-1, keepdim=True))
    ds = ds.mul_(probs).mul_(scale)
    dq = back(torch.matmul(ds, k))
    dk = gather(torch.matmul(ds.transpose(-1, -2), q))
    return result + tuple(t.to(s["q"].dtype) for t in (dq, dk, dv))


def _plain_step(s):
    case = s["case"]
    b, h, hk, d = (case[k] for k in ("batch", "heads", "kv_heads", "dim"))
    sinks, window = case["sinks"], case["window"]
    pos = s["positions"].long()
    slot = torch.where(pos < sinks, pos, sinks + (pos - sinks) % window)
    each = torch.arange(b, device=pos.device)
    s["k_cache"][each, slot] = s["k"]
    s["v_cache"][each, slot] = s["v"]
    q = s["q"].float().view(b, hk, h // hk, d)
    k = s["k_cache"].float().transpose(1, 2)
    v = s["v_cache"].float().transpose(1, 2)
    seen = torch.arange(sinks + window, device=pos.device) <= pos[:, None]
    scores = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(d)
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    probs = (scores - scores.amax(-1, keepdim=True)).exp()
    out = torch.matmul(probs / probs.sum(-1, keepdim=True), v)
    return out.view(b, h, d).to(s["q"].dtype), s["k_cache"], s["v_cache"]


def _doubling(a, b):
    """All h_t = a_t h_{t-1} + b_t along dimension 1, h_{-1} = 0, by doubling."""
    step, tokens = 1, a.shape[1]
    while step < tokens:
        b = torch.cat([b[:, :step], a[:, step:] * b[:, :-step] + b[:, step:]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _plain_scan(s):
    x, gate = s["x"].float(), s["gate"].float()
    a, keep = torch.sigmoid(gate), torch.sigmoid(-gate)
    start = s["state"] if "state" in s else torch.zeros_like(x[:, 0])
    b = keep * x
    b[:, 0] += a[:, 0] * start
    h = _doubling(a, b)
    result = (h.to(s["x"].dtype), h[:, -1].clone())
    if not s["case"]["grad"]:
        return result
    dy = s["grad"].float()
    dy = torch.cat([dy[:, :-1], dy[:, -1:] + s["grad_last"][:, None]], 1)
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    total = _doubling(later.flip(1), dy.flip(1)).flip(1)
    before = torch.cat([start[:, None], h[:, :-1]], 1)
    dx, dgate = keep * total, total * (before - x) * a * keep
    result += (dx.to(s["x"].dtype), dgate.to(s["x"].dtype))
    return result + ((a[:, 0] * total[:, 0],) if "state" in s else ())


def _plain_scan_step(s):
    gate = s["gate"].float()
    h = torch.sigmoid(gate) * s["state"] + torch.sigmoid(-gate) * s["x"].float()
    return h.to(s["x"].dtype), h


def _plain_norm(s):
    case = s["case"]
    x, w = s["x"].float(), s["weight"].float()
    total = x + s["residual"].float() if "residual" in s else x
    inverse = 1.0 / torch.sqrt((total * total).mean(-1, keepdim=True) + EPS)
    unit = total * inverse
    y = unit * w
    kept = total.to(TYPES[case["residual"] or case["dtype"]])
    if case["quant"]:
        top = 127.0 if case["quant"] == "int8" else 448.0
        scale = y.abs().amax(-1, keepdim=True) / top
        ratio = y / torch.where(scale > 0, scale, torch.ones_like(scale))
        codes = (ratio.round().clamp(-127, 127) if case["quant"] == "int8"
                 else ratio.clamp(-448, 448).to(torch.float8_e4m3fn).float())
        return (codes * scale).to(torch.bfloat16), scale[:, 0], kept
    result = (y.to(s["x"].dtype), kept)
    if not case["grad"]:
        return result
    dy = s["grad"].float()
    t = dy * w
    ds = inverse * (t - unit * (t * unit).mean(-1, keepdim=True)) + s["grad_sum"].float()
    result += (ds.to(s["x"].dtype),)
    if "residual" in s:
        result += (ds.to(s["residual"].dtype),)
    return result + ((dy * unit).sum(0).to(s["weight"].dtype),)


PLAIN = {"attention": _plain_attention, "attention_step": _plain_step, "scan": _plain_scan,
         "scan_step": _plain_scan_step, "norm": _plain_norm}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return PLAIN[state["case"]["op"]](state)


def _exact_attention(case, s):
    """Every row against every key, a slice of rows of one key head at a time,
    with the mask written out."""
    b, tq, tk, h, hk, d = (case[k] for k in ("batch", "tq", "tk", "heads", "kv_heads", "dim"))
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    dout = s["grad"].double() if case["grad"] else None
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    lengths = _lengths(case)
    keys = torch.arange(tk, device=q.device)
    rows = max(1, min(tq, (1 << 28) // tk))
    for i in range(b):
        for head in range(h):
            kk, vv, of = k[i, :, head * hk // h], v[i, :, head * hk // h], head * hk // h
            for r in range(0, tq, rows):
                e = min(tq, r + rows)
                p = torch.arange(tk - tq + r, tk - tq + e, device=q.device)[:, None]
                hidden = (keys > p) | (keys >= lengths[i])
                hidden |= (keys <= p - case["window"]) & (keys >= case["sinks"])
                w = torch.softmax((q[i, r:e, head] @ kk.T / d ** 0.5)
                                  .masked_fill_(hidden, -1e300), -1).masked_fill_(hidden, 0.0)
                out[i, r:e, head] = w @ vv
                if dout is None:
                    continue
                go = dout[i, r:e, head]
                dv[i, :, of] += w.T @ go
                z = w * (go @ vv.T - (go * out[i, r:e, head]).sum(-1, keepdim=True)) / d ** 0.5
                dq[i, r:e, head] = z @ kk
                dk[i, :, of] += z.T @ q[i, r:e, head]
    return (out, dq, dk, dv) if case["grad"] else (out,)


def _exact_step(case, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, p in enumerate(_positions(case)):
        slot = p if p < case["sinks"] else case["sinks"] + (p - case["sinks"]) % case["window"]
        s["k_cache"][i, slot], s["v_cache"][i, slot] = s["k"][i], s["v"][i]
        n = min(p + 1, case["sinks"] + case["window"])
        for head in range(case["heads"]):
            of = head * case["kv_heads"] // case["heads"]
            z = s["k_cache"][i, :n, of].double() @ s["q"][i, head].double() / case["dim"] ** 0.5
            out[i, head] = torch.softmax(z, 0) @ s["v_cache"][i, :n, of].double()
    return out, s["k_cache"].double(), s["v_cache"].double()


def _exact_scan(case, s):
    """Token after token."""
    x, gate = s["x"].double(), s["gate"].double()
    a = 1 / (1 + torch.exp(-gate))
    h = s["state"].double() if "state" in s else torch.zeros_like(x[:, 0])
    start, y = h, torch.empty_like(x)
    for t in range(case["tokens"]):
        h = torch.lerp(x[:, t], h, a[:, t])
        y[:, t] = h
    result = (y, h)
    if not case["grad"]:
        return result
    dx, da = s["grad"].double(), torch.empty_like(x)
    carry = s["grad_last"].double()
    for t in range(case["tokens"] - 1, -1, -1):
        dx[:, t] += carry
        carry = a[:, t] * dx[:, t]
    da[:, 1:] = dx[:, 1:] * (y[:, :-1] - x[:, 1:])
    da[:, 0] = dx[:, 0] * (start - x[:, 0])
    slope = torch.exp(-gate) * a * a
    result += (dx / (1 + torch.exp(gate)), da * slope)
    return result + ((carry,) if "state" in s else ())


def _exact_norm(case, s):
    x, w = s["x"].double(), s["weight"].double()
    total = x + s["residual"].double() if "residual" in s else x
    r = (total.square().sum(1, keepdim=True) / case["width"] + EPS).rsqrt()
    y = total * r * w
    if case["quant"]:
        scale = y.abs().max(1, keepdim=True).values / (127 if case["quant"] == "int8" else 448)
        z = y / scale
        if case["quant"] == "int8":
            return z.round() * scale, scale[:, 0], total
        # Four bits of mantissa, the smallest normal value 2^-6.
        unit = torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6))) - 3)
        return (z / unit).round() * unit * scale, scale[:, 0], total
    if not case["grad"]:
        return y, total
    dy = s["grad"].double()
    dr = (dy * w * total).sum(1, keepdim=True)
    ds = dy * w * r - total * dr * r ** 3 / case["width"] + s["grad_sum"].double()
    dw = (dy * total * r).sum(0)
    return (y, total, ds, ds, dw) if "residual" in s else (y, total, ds, dw)


def exact(case, seed):
    s = _data(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "attention_step":
        return _exact_step(case, s)
    if case["op"] == "scan":
        return _exact_scan(case, s)
    if case["op"] == "scan_step":
        a = 1 / (1 + torch.exp(-s["gate"].double()))
        h = torch.lerp(s["x"].double(), s["state"].double(), a)
        return h, h
    return _exact_norm(case, s)
