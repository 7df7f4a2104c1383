"""Operators of a splat predictor's training and streaming: what is measured,
and their plain forms.

Beside the operators of ``perf/operators.py``, a network that predicts splats
from a stream of posed views (one token per 16 x 16 tile: 1200 for a 640 x 480
frame, 8160 for full HD, 2500 for each of 16 views of 800²) has a recurrence
whose state is a matrix per head (the gated delta rule), a window cache held in
4 bits while it streams, and a training step that clips its gradients' norm.
With ``own`` true, ``run`` calls them through ``gaussian_splats_hip.sequence``
and ``.training``; with ``own`` false it computes them with elementary torch
operations in float32.
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

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}


def _delta(name, batch, tokens, heads, key_heads, key_dim, dim, dtype, grad, state=False, ragged=False):
    case = {"op": "delta", "batch": batch, "tokens": tokens, "heads": heads, "key_heads": key_heads,
            "key_dim": key_dim, "dim": dim, "dtype": dtype, "grad": grad, "state": state,
            "ragged": ragged}
    return {"name": name, **case} if name else case


def _delta_step(name, batch, heads, key_heads, key_dim, dim, dtype):
    case = {"op": "delta_step", "batch": batch, "heads": heads, "key_heads": key_heads,
            "key_dim": key_dim, "dim": dim, "dtype": dtype}
    return {"name": name, **case} if name else case


def _cache_step(name, batch, heads, kv_heads, dim, window, sinks, dtype, ragged=False):
    case = {"op": "cache_step", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "window": window, "sinks": sinks, "dtype": dtype, "ragged": ragged}
    return {"name": name, **case} if name else case


def _cache_fill(name, batch, tokens, kv_heads, dim, window, sinks, dtype, ragged=False):
    case = {"op": "cache_fill", "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "dim": dim,
            "window": window, "sinks": sinks, "dtype": dtype, "ragged": ragged}
    return {"name": name, **case} if name else case


def _clip(name, width, blocks, dtype):
    case = {"op": "clip", "width": width, "blocks": blocks, "dtype": dtype}
    return {"name": name, **case} if name else case


def _clipped_adam(name, splats, sh):
    case = {"op": "clipped_adam", "splats": splats, "sh": sh}
    return {"name": name, **case} if name else case


def listed():
    return [
        # A training step's delta rule over one 640 x 480 frame.
        _delta("frame delta", 1, 1200, 8, 8, 64, 64, "bf16", True),
        # The same over 16 views of 800² in stream order, keys shared by three heads.
        _delta("view stream delta", 1, 40000, 12, 4, 64, 64, "bf16", True),
        # Two full-HD frames taken into running streams, one of them shorter: forward only.
        _delta("full HD delta prefill", 2, 8160, 16, 16, 128, 128, "f16", False, True, True),
        # Small fits in float32, the rasterizer's own type, at odd sizes.
        _delta("odd delta f32", 2, 777, 6, 2, 40, 72, "f32", True, True),
        # One new token of one stream: latency.
        _delta_step("one stream's delta step", 1, 8, 8, 64, 64, "bf16"),
        # One new token of each of many streams.
        _delta_step("many streams' delta step", 32, 32, 16, 128, 128, "bf16"),
        # One new token of one stream over a cache in 4 bits: latency.
        _cache_step("one stream's 4-bit step", 1, 8, 8, 64, 2500, 4, "bf16"),
        # One new token of each of many streams, their caches filled to different
        # lengths, some of them wrapped around.
        _cache_step("many streams' 4-bit step", 32, 32, 8, 128, 8160, 16, "bf16", True),
        # Two full-HD frames taken into caches of half a frame's window, one of them shorter.
        _cache_fill("full HD 4-bit fill", 2, 8160, 4, 128, 4080, 16, "f16", True),
        # The gradients of a predictor, weights in bfloat16 and norms in float32,
        # whose norm is within the limit: the usual step of a run that goes well.
        _clip("predictor clip", 1024, 5, "bf16"),
        # Adam on the parameters of a scene of a small fit, the gradients clipped.
        _clipped_adam("clipped Adam 20k", 20_011, 2),
        # The same at the size of the rasterizer's headline step.
        _clipped_adam("clipped Adam 1M", 1_000_000, 3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["delta", "delta", "delta", "delta_step", "cache_step", "cache_step", "cache_fill",
                     "clip", "clipped_adam"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "delta":
        key_heads = rng.choice([1, 2, 4, 8])
        heads = key_heads * rng.choice([1, 1, 2, 3])
        key_dim, dim = rng.choice([32, 40, 64, 64, 96, 128]), rng.choice([24, 64, 64, 80, 128])
        batch, tokens = rng.choice([1, 1, 2, 4]), _log_int(rng, 16, 40000)
        grad = rng.random() < 0.7
        budget = 40000 * 12 * 64 * 64 // (8 if dtype == "f32" else 1)
        while batch * tokens * heads * max(64, key_dim) * max(64, dim) > budget:
            tokens = max(1, tokens * 2 // 3)
        return _delta(None, batch, tokens, heads, key_heads, key_dim, dim, dtype, grad,
                      rng.random() < 0.5, rng.random() < 0.3)
    if op == "delta_step":
        key_heads = rng.choice([1, 2, 4, 8, 16])
        heads = key_heads * rng.choice([1, 2])
        return _delta_step(None, _log_int(rng, 1, 32), heads, key_heads, rng.choice([32, 40, 64, 96, 128]),
                           rng.choice([24, 64, 80, 128]), dtype)
    if op == "cache_step":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4])
        return _cache_step(None, _log_int(rng, 1, 32), heads, kv_heads, rng.choice([32, 64, 64, 96, 128]),
                           _log_int(rng, 64, 8160), rng.choice([0, 4, 16]), rng.choice(["bf16", "f16"]),
                           rng.random() < 0.6)
    if op == "cache_fill":
        tokens = _log_int(rng, 16, 16000)
        return _cache_fill(None, rng.choice([1, 2, 4]), tokens, rng.choice([1, 2, 4, 8]),
                           rng.choice([32, 64, 96, 128]), _log_int(rng, 16, 8160), rng.choice([0, 4, 16]),
                           dtype, rng.random() < 0.5)
    if op == "clip":
        return _clip(None, 8 * _log_int(rng, 4, 160), rng.randint(1, 5), dtype)
    return _clipped_adam(None, _log_int(rng, 100, 1_000_000), rng.choice([0, 1, 2, 3]))


def _lengths(case):
    """Tokens of each sequence that exist, fixed by the case."""
    b, t = case["batch"], case["tokens"]
    return [t - (t * 2 * i) // (5 * b) if case["ragged"] else t for i in range(b)]


def _positions(case):
    """Position of each stream's new token: half filled up to wrapped around."""
    b, n = case["batch"], case["sinks"] + case["window"]
    if not case["ragged"]:
        return [n + n // 3] * b
    return [n // 2 + (n * 3 * i) // (2 * b) for i in range(b)]


def _tensor_shapes(case):
    """A predictor's parameters: [(shape, type)], as its blocks have them."""
    w, t = case["width"], case["dtype"]
    shapes = [((w, 774), t), ((w,), t)]
    for _ in range(case["blocks"]):
        shapes += [((3, w), "f32"), ((2 * w, w), t), ((2 * w,), t), ((w, w), t), ((2 * w, w), t), ((w, w), t),
                   ((4 * w, w), t), ((4 * w,), t), ((w, 4 * w), t), ((w,), t)]
    return shapes + [((w,), "f32"), ((60, w), t), ((60,), t)]


def _splat_shapes(case):
    n = case["splats"]
    return {"mean": (n, 3), "rotation": (n, 4), "scale": (n, 3), "opacity": (n, 1),
            "color": (n, (case["sh"] + 1) ** 2, 3)}


def work(case):
    op = case["op"]
    if op == "delta":
        e, d, dv = SIZES[case["dtype"]], case["key_dim"], case["dim"]
        tokens = sum(_lengths(case))
        rows = case["batch"] * case["tokens"]
        moved = rows * e * (2 * case["key_heads"] * d + case["heads"] * (2 * dv + 2))
        states = case["batch"] * case["heads"] * d * dv * 4
        moved += states * (2 if case["state"] else 1)
        if case["grad"]:  # the output's gradient in, the inputs' out
            moved += rows * e * (2 * case["key_heads"] * d + case["heads"] * (2 * dv + 2))
            moved += states * (2 if case["state"] else 1)
        return {"bytes": moved, "flops": tokens * case["heads"] * d * dv * (20 if case["grad"] else 6)}
    if op == "delta_step":
        e, d, dv = SIZES[case["dtype"]], case["key_dim"], case["dim"]
        states = case["batch"] * case["heads"] * d * dv
        io = case["batch"] * (2 * case["key_heads"] * d + case["heads"] * (2 * dv + 2))
        return {"bytes": 8 * states + io * e, "flops": 6 * states}
    if op == "cache_step":
        d, n = case["dim"], case["sinks"] + case["window"]
        seen = sum(min(p + 1, n) for p in _positions(case))
        io = case["batch"] * (2 * case["heads"] + 2 * case["kv_heads"]) * d * SIZES[case["dtype"]]
        return {"bytes": 2 * seen * case["kv_heads"] * (d // 2 + d // 32) + io,
                "flops": 4 * seen * case["heads"] * d}
    if op == "cache_fill":
        d, n = case["dim"], case["sinks"] + case["window"]
        kept = sum(min(t, n) for t in _lengths(case)) * case["kv_heads"]
        return {"bytes": 2 * kept * (d * SIZES[case["dtype"]] + d // 2 + d // 32), "flops": 8 * kept * d}
    if op == "clip":
        sizes = [(math.prod(s), SIZES[t]) for s, t in _tensor_shapes(case)]
        return {"bytes": sum(n * e for n, e in sizes), "flops": 2 * sum(n for n, _ in sizes)}
    n = sum(math.prod(s) for s in _splat_shapes(case).values())
    # The norm has to be known before the first parameter moves: gradients twice.
    return {"bytes": n * 32, "flops": n * 16}


LIMIT = 1.0
RATE, BETAS, EPS, STEP = 1e-3, (0.9, 0.999), 1e-15, 100


def _data(case, seed):
    """Inputs of a case from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(TYPES[dtype])

    def unit(shape, dtype):
        t = torch.randn(shape, generator=g, device="cuda")
        return (t / t.square().sum(-1, keepdim=True).sqrt()).to(TYPES[dtype])

    op, t = case["op"], case.get("dtype")
    if op in ("delta", "delta_step"):
        tokens = (case["tokens"],) if op == "delta" else ()
        b, h, hk, d, dv = (case[n] for n in ("batch", "heads", "key_heads", "key_dim", "dim"))
        s = {"q": unit((b, *tokens, hk, d), t), "k": unit((b, *tokens, hk, d), t),
             "v": normal((b, *tokens, h, dv), t),
             # Memories of some twenty tokens, some far longer.
             "gate": normal((b, *tokens, h), t, 2.0, 3.0), "beta": normal((b, *tokens, h), t)}
        if op == "delta_step" or case["state"]:
            s["state"] = normal((b, h, d, dv), "f32", 0.3)
        if op == "delta" and case["grad"]:
            s["grad"] = normal((b, *tokens, h, dv), t, 0.1)
            s["grad_last"] = normal((b, h, d, dv), "f32", 0.1)
        if op == "delta" and case["ragged"]:
            s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        return s
    if op in ("cache_step", "cache_fill"):
        b, hk, d, n = case["batch"], case["kv_heads"], case["dim"], case["sinks"] + case["window"]
        s = {}
        for name in ("k", "v"):
            # Codes of the sizes that a filled cache has: powers of two around a quarter.
            s[name + "_codes"] = torch.randint(0, 256, (b, hk, n, d // 2), generator=g, device="cuda",
                                               dtype=torch.uint8)
            s[name + "_exponents"] = torch.randint(123, 127, (b, hk, n, d // 32), generator=g, device="cuda",
                                                   dtype=torch.uint8)
        if op == "cache_fill":
            s["k"], s["v"] = (normal((b, case["tokens"], hk, d), t) for _ in range(2))
            if case["ragged"]:
                s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        else:
            s["q"], s["k"], s["v"] = normal((b, case["heads"], d), t), normal((b, hk, d), t), normal((b, hk, d), t)
            s["positions"] = torch.tensor(_positions(case), dtype=torch.int32, device="cuda")
        return s
    if op == "clip":
        shapes = _tensor_shapes(case)
        total = sum(math.prod(shape) for shape, _ in shapes)
        size = 0.7 * LIMIT / math.sqrt(total)
        return {"grads": [normal(shape, kind, size) for shape, kind in shapes]}
    shapes = _splat_shapes(case)
    return {"params": [normal(shape, "f32") for shape in shapes.values()],
            "grads": [normal(shape, "f32", 1e-2) for shape in shapes.values()],
            "exp_avg": [normal(shape, "f32", 1e-5) for shape in shapes.values()],
            "exp_avg_sq": [normal(shape, "f32", 1e-5).square() for shape in shapes.values()]}


#: What a training step takes gradients of, in the order in which run() returns them.
LEAVES = ("q", "k", "v", "gate", "beta", "state")


def prepare(case, seed):
    data = _data(case, seed)
    if case.get("grad"):
        for name in LEAVES:
            if name in data:
                data[name].requires_grad_(True)
    if case["op"] == "clip":
        data["params"] = [torch.nn.Parameter(torch.empty_like(g)) for g in data["grads"]]
    if case["op"] == "clipped_adam":
        data["params"] = [torch.nn.Parameter(p) for p in data["params"]]
        data["steps"] = STEP
    for p, g in zip(data.get("params", ()), data.get("grads", ())):
        p.grad = g
    return {"case": case, **data}


def _own(s):
    from gaussian_splats_hip import sequence, training

    case, op = s["case"], s["case"]["op"]
    if op == "delta":
        outputs = sequence.delta_scan(s["q"], s["k"], s["v"], s["gate"], s["beta"], s.get("state"),
                                      lengths=s.get("lengths"))
        if not case["grad"]:
            return outputs
        leaves = [s[n] for n in LEAVES if n in s]
        return tuple(o.detach() for o in outputs) + torch.autograd.grad(
            outputs, leaves, (s["grad"], s["grad_last"]))
    if op == "delta_step":
        return sequence.delta_scan_step(s["q"], s["k"], s["v"], s["gate"], s["beta"], s["state"])
    if op in ("cache_step", "cache_fill"):
        cache = (s["k_codes"], s["k_exponents"], s["v_codes"], s["v_exponents"])
        if op == "cache_fill":
            sequence.window_cache_fill_quant(s["k"], s["v"], *cache, case["window"], case["sinks"],
                                             s.get("lengths"))
            return cache
        return (sequence.window_attention_step_quant(s["q"], s["k"], s["v"], *cache, s["positions"],
                                                     case["window"], case["sinks"]), *cache)
    if op == "clip":
        norm = training.clip_grad_norm(s["params"], LIMIT)
        return norm, [p.grad for p in s["params"]]
    # The optimiser that a program keeps, made at its first step.
    if "optimizer" not in s:
        s["optimizer"] = training.FusedAdam(s["params"], lr=RATE, betas=BETAS, eps=EPS, max_norm=LIMIT)
        for p, m, v in zip(s["params"], s["exp_avg"], s["exp_avg_sq"]):
            s["optimizer"].state[p].update(step=torch.tensor(float(s["steps"])), exp_avg=m, exp_avg_sq=v)
    s["optimizer"].step()
    return (s["optimizer"].grad_norm, [p.detach() for p in s["params"]], s["exp_avg"], s["exp_avg_sq"])


CHUNK = 64


def _chunks(t, tokens):
    """[B, T, H, ...] as [B, H, chunks, CHUNK, ...] in float32, zeros behind the last token."""
    count = -(-tokens // CHUNK)
    pad = t.new_zeros((t.shape[0], count * CHUNK - tokens, *t.shape[2:]), dtype=torch.float32)
    t = torch.cat([t.float(), pad], 1)
    return t.view(t.shape[0], count, CHUNK, *t.shape[2:]).movedim(3, 1)


def _tokens(t, tokens):
    """Back to [B, T, H, ...]."""
    t = t.movedim(1, 3)
    return t.reshape(t.shape[0], -1, *t.shape[3:])[:, :tokens]


def _plain_delta(s):
    """Chunks of 64 tokens: within a chunk the updates solve a triangular
    system, between chunks the state goes on one chunk after the other."""
    case = s["case"]
    tokens, h, hk = case["tokens"], case["heads"], case["key_heads"]
    scale, group = 1.0 / math.sqrt(case["key_dim"]), h // hk
    there = torch.ones((case["batch"], tokens, 1), dtype=torch.bool, device=s["q"].device)
    if "lengths" in s:
        there = torch.arange(tokens, device=s["q"].device)[None, :, None] < s["lengths"][:, None, None]
    q, k, v = (_chunks(torch.where(there[..., None], t, torch.zeros_like(t)), tokens)
               for t in (s["q"].repeat_interleave(group, 2), s["k"].repeat_interleave(group, 2), s["v"]))
    gate = s["gate"].float()
    # Tokens behind a sequence's last one change nothing: a = 1, b = 0.
    log_a = _chunks(torch.where(there, torch.nn.functional.logsigmoid(gate), torch.zeros_like(gate)), tokens)
    b = _chunks(torch.where(there, torch.sigmoid(s["beta"].float()), torch.zeros_like(gate)), tokens)
    total = log_a.double().cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = (total[..., :, None] - total[..., None, :]).masked_fill(~lower, -math.inf).exp().float()
    up, last = total.exp().float()[..., None], total[..., -1:]
    down, whole = (last - total).exp().float()[..., None], last.exp().float()[..., None]
    system = b[..., None] * decay * torch.matmul(k, k.mT.contiguous())
    system = system.tril(-1)
    # (I + system)^-1, its powers from the 64th on being zero.
    eye = torch.eye(CHUNK, device=q.device)
    solve, power = eye - system, torch.matmul(system, system)
    for _ in range(5):
        solve, power = torch.matmul(solve, eye + power), torch.matmul(power, power)
    w = torch.matmul(solve, b[..., None] * up * k)
    free = torch.matmul(solve, b[..., None] * v)
    state = (s["state"].detach() if "state" in s
             else torch.zeros((*q.shape[:2], q.shape[-1], v.shape[-1]), device=q.device))
    starts, updates = torch.empty((*q.shape[:3], *state.shape[2:]), device=q.device), torch.empty_like(v)
    write = (down * k).mT.contiguous()
    for c in range(q.shape[2]):
        starts[:, :, c] = state
        updates[:, :, c] = free[:, :, c] - torch.matmul(w[:, :, c], state)
        state = whole[:, :, c] * state + torch.matmul(write[:, :, c], updates[:, :, c])
    scores = torch.matmul(q, k.mT.contiguous()) * decay * scale
    out = torch.matmul(q * (up * scale), starts) + torch.matmul(scores, updates)
    out = torch.where(there[..., None], _tokens(out, tokens), 0.0)
    result = (out.to(s["v"].dtype), state)
    if not case["grad"]:
        return result
    grad = _chunks(torch.where(there[..., None], s["grad"], torch.zeros_like(s["grad"])), tokens)
    free = torch.matmul(scores.mT.contiguous(), grad)
    read = torch.matmul((q * (up * scale)).mT.contiguous(), grad)
    ends, dstate = torch.empty_like(starts), s["grad_last"]
    du, wt = torch.empty_like(updates), w.mT.contiguous()
    for c in range(q.shape[2] - 1, -1, -1):
        ends[:, :, c] = dstate
        du[:, :, c] = free[:, :, c] + down[:, :, c] * torch.matmul(k[:, :, c], dstate)
        dstate = whole[:, :, c] * dstate + read[:, :, c] - torch.matmul(wt[:, :, c], du[:, :, c])
    dr = torch.matmul(solve.mT.contiguous(), du)
    ut = updates.mT.contiguous()
    ds = torch.matmul(grad, ut) * decay * scale
    da = (torch.matmul(dr, ut) * decay).tril(-1)
    starts_t, ends_t = starts.mT.contiguous(), ends.mT.contiguous()
    dq = up * scale * torch.matmul(grad, starts_t) + torch.matmul(ds, k)
    # What the keys read with, before b, and what they write with.
    read_k = -(up * torch.matmul(dr, starts_t) + torch.matmul(da, k))
    write_k = (down * torch.matmul(updates, ends_t) + torch.matmul(ds.mT.contiguous(), q)
               - torch.matmul((b[..., None] * da).mT.contiguous(), k))
    db = (dr * v).sum(-1) + (read_k * k).sum(-1)
    read_k = read_k * b[..., None]
    slope = ((q * dq).sum(-1) + (k * (read_k - write_k)).sum(-1)).double()
    after = torch.cat([starts[:, :, 1:], state[:, :, None]], 2)
    slope[..., -1] += (after.double() * ends).sum((-1, -2))
    dlog = slope.flip(-1).cumsum(-1).flip(-1).float()

    def shared(t):  # heads that share a key
        t = _tokens(t, tokens)
        return t.reshape(*t.shape[:2], hk, group, -1).sum(3)

    beta = s["beta"].float()
    grads = [shared(dq), shared(read_k + write_k), _tokens(b[..., None] * dr, tokens),
             _tokens(dlog, tokens) * torch.sigmoid(-gate),
             _tokens(db, tokens) * torch.sigmoid(beta) * torch.sigmoid(-beta)]
    grads = [torch.where(there if t.dim() == 3 else there[..., None], t, 0.0).to(s["q"].dtype) for t in grads]
    return result + tuple(grads) + ((dstate,) if "state" in s else ())


def _plain_delta_step(s):
    group = s["case"]["heads"] // s["case"]["key_heads"]
    q, k = (s[n].float().repeat_interleave(group, 1)[..., None] for n in ("q", "k"))
    a, b = torch.sigmoid(s["gate"].float())[..., None], torch.sigmoid(s["beta"].float())[..., None]
    state = a[..., None] * s["state"]
    update = b * (s["v"].float() - (state * k).sum(-2))
    state = state + k * update[..., None, :]
    return ((state * q).sum(-2) / math.sqrt(s["case"]["key_dim"])).to(s["v"].dtype), state


def _encode(x):
    """Codes [.., dim / 2] and exponents [.., dim / 32] of rows: blocks of 32 share
    the power of two two below their largest value's; 4-bit values of one bit of
    mantissa, ties to even, the largest one 6."""
    x = x.float().unflatten(-1, (-1, 32))
    top = torch.frexp(x.abs().amax(-1, keepdim=True)).exponent - 3
    top = torch.where(x.abs().amax(-1, keepdim=True) > 0, top.clamp(-127, 127), -127)
    y = torch.ldexp(x.abs(), -top)
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5)
            + (y > 5.0) + 8 * torch.signbit(x))
    code = code.to(torch.uint8).flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), (top[..., 0] + 127).to(torch.uint8)


def _decode(codes, exponents):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    table = torch.cat([table, -table])
    x = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()].unflatten(-1, (-1, 32))
    return torch.ldexp(x, exponents.int()[..., None] - 127).flatten(-2)


def _plain_cache_step(s):
    case = s["case"]
    b, h, hk, d = (case[k] for k in ("batch", "heads", "kv_heads", "dim"))
    sinks, window = case["sinks"], case["window"]
    pos = s["positions"].long()
    slot = torch.where(pos < sinks, pos, sinks + (pos - sinks) % window)
    each = torch.arange(b, device=pos.device)
    for name in ("k", "v"):
        codes, exponents = _encode(s[name])
        s[name + "_codes"][each, :, slot] = codes
        s[name + "_exponents"][each, :, slot] = exponents
    q = s["q"].float().view(b, hk, h // hk, d)
    k = _decode(s["k_codes"], s["k_exponents"])
    seen = torch.arange(sinks + window, device=pos.device) <= pos[:, None]
    scores = torch.matmul(q, k.mT.contiguous()) / math.sqrt(d)
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    probs = (scores - scores.amax(-1, keepdim=True)).exp()
    out = torch.matmul(probs / probs.sum(-1, keepdim=True), _decode(s["v_codes"], s["v_exponents"]))
    # The cache's whole bytes: powers of two and ties to even leave no doubt about a code.
    return (out.view(b, h, d).to(s["q"].dtype), s["k_codes"], s["k_exponents"], s["v_codes"],
            s["v_exponents"])


def _plain_cache_fill(s):
    case = s["case"]
    sinks, window, tokens = case["sinks"], case["window"], case["tokens"]
    n = torch.tensor(_lengths(case), device=s["k"].device)
    slot = torch.arange(sinks + window, device=n.device)
    behind = n[:, None] - 1 - slot  # the ring's slot has the last of slot, slot + window, ..
    ring = slot + behind.div(window, rounding_mode="floor") * window
    token = torch.where(slot < sinks, slot, ring).clamp(0, tokens - 1)
    filled = (behind >= 0)[:, None, :, None]
    index = token[:, :, None, None]
    for name in ("k", "v"):
        rows = torch.take_along_dim(s[name], index, 1).transpose(1, 2)
        codes, exponents = _encode(rows)
        torch.where(filled, codes, s[name + "_codes"], out=s[name + "_codes"])
        torch.where(filled, exponents, s[name + "_exponents"], out=s[name + "_exponents"])
    return s["k_codes"], s["k_exponents"], s["v_codes"], s["v_exponents"]


def _norm(tensors):
    return torch.stack([t.float().square().sum(dtype=torch.float64) for t in tensors]).sum().sqrt()


def _plain_clip(s):
    grads = [p.grad for p in s["params"]]
    norm = _norm(grads)
    factor = (LIMIT / (norm + 1e-6)).clamp(max=1.0)
    for g in grads:
        g.copy_(g.float() * factor.float())
    return norm.float(), grads


def _plain_clipped_adam(s):
    norm = _norm(s["grads"])
    factor = (LIMIT / (norm + 1e-6)).clamp(max=1.0).float()
    s["steps"] += 1
    size = RATE / (1 - BETAS[0] ** s["steps"])
    root = math.sqrt(1 - BETAS[1] ** s["steps"])
    for p, g, m, v in zip(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"]):
        g = g * factor
        m.add_((g - m) * (1 - BETAS[0]))
        v.mul_(BETAS[1]).add_(g * g * (1 - BETAS[1]))
        p.sub_(size * (m / (v.sqrt() / root + EPS)))
    return norm.float(), [p.detach() for p in s["params"]], s["exp_avg"], s["exp_avg_sq"]


PLAIN = {"delta": _plain_delta, "delta_step": _plain_delta_step, "cache_step": _plain_cache_step,
         "cache_fill": _plain_cache_fill, "clip": _plain_clip, "clipped_adam": _plain_clipped_adam}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return PLAIN[state["case"]["op"]](state)


def _exact_delta(case, s):
    """Token after token, forwards and back, every state kept."""
    tokens, h, hk = case["tokens"], case["heads"], case["key_heads"]
    of = torch.arange(h, device="cuda") * hk // h
    q, k = (s[n].double()[:, :, of] for n in ("q", "k"))
    v, gate, beta = (s[n].double() for n in ("v", "gate", "beta"))
    a, b = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(-beta))
    there = torch.tensor([[t < n for t in range(tokens)] for n in _lengths(case)], device="cuda")
    a, b = torch.where(there[..., None], a, 1.0), torch.where(there[..., None], b, 0.0)
    scale = case["key_dim"] ** -0.5
    shape = (case["batch"], h, case["key_dim"], case["dim"])
    states = torch.empty((tokens + 1, *shape), dtype=torch.float64, device="cuda")
    states[0] = s["state"].double() if "state" in s else 0.0
    u = torch.empty_like(v)
    for t in range(tokens):
        kept = states[t] * a[:, t, :, None, None]
        u[:, t] = b[:, t, :, None] * (v[:, t] - (k[:, t, :, None] @ kept)[:, :, 0])
        torch.addcmul(kept, k[:, t, :, :, None], u[:, t, :, None], out=states[t + 1])
    out = torch.empty_like(v)
    for i in range(case["batch"]):
        for r in range(0, tokens, 1024):
            e = min(tokens, r + 1024)
            out[i, r:e] = scale * (q[i, r:e, :, None] @ states[r + 1:e + 1, i])[:, :, 0]
    out *= there[..., None, None]
    if not case["grad"]:
        return out, states[-1]
    do = s["grad"].double() * there[..., None, None]
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    da, db = torch.empty_like(a), torch.empty_like(b)
    ds = s["grad_last"].double().clone()
    for t in range(tokens - 1, -1, -1):
        dot = do[:, t, :, :, None]
        dq[:, t] = scale * (states[t + 1] @ dot)[..., 0]
        ds = torch.addcmul(ds, q[:, t, :, :, None], do[:, t, :, None], value=scale)
        kt, ut = k[:, t, :, :, None], u[:, t, :, :, None]
        du = (kt.mT.contiguous() @ ds)[:, :, 0]
        seen = (kt.mT.contiguous() @ states[t])[:, :, 0] * a[:, t, :, None]
        db[:, t] = (du * (v[:, t] - seen)).sum(-1)
        dv[:, t] = b[:, t, :, None] * du
        dk[:, t] = (ds @ ut)[..., 0] - a[:, t, :, None] * (states[t] @ dv[:, t, :, :, None])[..., 0]
        ds = torch.addcmul(ds, kt, dv[:, t, :, None], value=-1.0)
        da[:, t] = (states[t] * ds).sum((-1, -2))
        ds = ds * a[:, t, :, None, None]
    last = states[-1].clone()
    del states
    lost = there[..., None]
    share = lambda t: (t * lost[..., None]).unflatten(2, (hk, h // hk)).sum(3)  # noqa: E731
    grads = (share(dq), share(dk), dv * lost[..., None], da * a * (1 / (1 + torch.exp(gate))) * lost,
             db * b * (1 / (1 + torch.exp(beta))) * lost)
    return (out, last, *grads) + ((ds,) if "state" in s else ())


def _values(codes, exponents):
    """What codes stand for, in 64 bits."""
    c = torch.stack([codes % 16, codes // 16], -1).flatten(-2).long()
    size, mantissa = (c % 8) // 2, (c % 2).double()
    x = torch.where(size == 0, mantissa / 2, (1 + mantissa / 2) * torch.exp2(size.double() - 1))
    x = torch.where(c >= 8, -x, x)
    return x * torch.exp2(exponents.double() - 127).repeat_interleave(32, -1)


def _nearest(x):
    """The values that a row's codes will stand for, in 64 bits."""
    x = x.double().unflatten(-1, (-1, 32))
    unit = torch.exp2(torch.floor(torch.log2(x.abs().amax(-1, keepdim=True))) - 2)
    levels = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0], dtype=torch.float64, device=x.device)
    # Even codes first, so that of two levels as near the even one is taken.
    y = (x.abs() / unit)[..., None]
    return (levels[(y - levels).abs().argmin(-1)] * torch.sign(x) * unit).flatten(-2)


def _exact_cache_step(case, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    k_new, v_new = _nearest(s["k"]), _nearest(s["v"])
    for i, p in enumerate(_positions(case)):
        slot = p if p < case["sinks"] else case["sinks"] + (p - case["sinks"]) % case["window"]
        n = min(p + 1, case["sinks"] + case["window"])
        for of in range(case["kv_heads"]):
            k = _values(s["k_codes"][i, of, :n], s["k_exponents"][i, of, :n])
            v = _values(s["v_codes"][i, of, :n], s["v_exponents"][i, of, :n])
            k[slot], v[slot] = k_new[i, of], v_new[i, of]
            g = case["heads"] // case["kv_heads"]
            z = s["q"][i, of * g:(of + 1) * g].double() @ k.T.contiguous() / case["dim"] ** 0.5
            out[i, of * g:(of + 1) * g] = torch.softmax(z, -1) @ v
    return out, None, None, None, None


def exact(case, seed):
    s = _data(case, seed)
    op = case["op"]
    if op == "delta":
        return _exact_delta(case, s)
    if op == "delta_step":
        of = torch.arange(case["heads"], device="cuda") * case["key_heads"] // case["heads"]
        q, k = s["q"].double()[:, of], s["k"].double()[:, of]
        a, b = (1 / (1 + torch.exp(-s[n].double()))[..., None] for n in ("gate", "beta"))
        kept = s["state"].double() * a[..., None]
        u = b * (s["v"].double() - (k[:, :, None] @ kept)[:, :, 0])
        state = kept + k[..., None] * u[:, :, None]
        return (q[:, :, None] @ state)[:, :, 0] * case["key_dim"] ** -0.5, state
    if op == "cache_step":
        return _exact_cache_step(case, s)
    if op == "cache_fill":
        return None
    squares = [g.double().square().sum() for g in s["grads"]]
    norm = torch.stack(squares).sum().sqrt()
    factor = torch.clamp(LIMIT / (norm + 1e-6), max=1.0)
    if op == "clip":
        return norm, [g.double() * factor for g in s["grads"]]
    params, first, second = [], [], []
    for p, g, m, v in zip(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"]):
        g = g.double() * factor
        first.append(BETAS[0] * m.double() + (1 - BETAS[0]) * g)
        second.append(BETAS[1] * v.double() + (1 - BETAS[1]) * g * g)
        rate = RATE / (1 - BETAS[0] ** (STEP + 1))
        root = (second[-1] / (1 - BETAS[1] ** (STEP + 1))).sqrt()
        params.append(p.double() - rate * first[-1] / (root + EPS))
    return norm, params, first, second
