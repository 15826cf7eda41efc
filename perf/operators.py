"""Cases that measure the attention and dropout operators, with their plain forms.

Three passes of a decoder's attention block are measured:

* ``train``: sliding-window attention with sinks, forward and backward (``direction``
  "train"), or the forward alone over a chunk of a longer prompt ("forward");
* ``step``: the same attention for one new token per sequence over a key / value cache;
* ``dropout``: residual + dropout(x + bias) from a counter-based generator, forward and
  backward, with no stored mask.

``own`` chooses between the plain form (elementary torch operations in 32 bits, rounded once
at the end) and the package's calls. Key j is visible to the query at position p of a
sequence of ``length`` keys when j < length, j <= p and (p - j < window or j < sinks); a
query that sees no key gives zeros. Element e of a dropout is dropped when word e mod 4 of
Philox4x32-7(counter = (e // 4, offset), key = seed) is below p * 2^32.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
DEVICE = "cuda"
# Share of the longest length that sequence b of a ragged batch has, in turn.
RAGGED = (1.0, 0.37, 0.82, 0.05, 0.66, 0.93, 0.0, 0.5)


def attention(name, batch, heads, kv_heads, queries, keys, dim, dtype, window, sinks, ragged=False, offset=0,
              direction="train"):
    return {"name": name, "op": "attention", "batch": batch, "heads": heads, "kv_heads": kv_heads, "queries": queries,
            "keys": keys, "dim": dim, "dtype": dtype, "window": window, "sinks": sinks, "ragged": ragged,
            "offset": offset, "direction": direction}


def step(name, batch, heads, kv_heads, capacity, dim, dtype, window, sinks, longest, ragged=True):
    return {"name": name, "op": "step", "batch": batch, "heads": heads, "kv_heads": kv_heads, "capacity": capacity,
            "dim": dim, "dtype": dtype, "window": window, "sinks": sinks, "longest": longest, "ragged": ragged}


def dropout(name, rows, width, dtype, p, bias=True, residual=True):
    return {"name": name, "op": "dropout", "rows": rows, "width": width, "dtype": dtype, "p": p, "bias": bias,
            "residual": residual}


def listed():
    return [
        # One layer of the 124M model (12 heads of 64, 1024 tokens, batch 8), attention
        # limited to the last 256 tokens and the first 4.
        attention("train_124m", 8, 12, 12, 1024, 1024, 64, "bf16", 256, 4),
        # One layer of the 1.3B model (width 2048 as 16 heads of 128, 2048 tokens).
        attention("train_1p3b", 2, 16, 16, 2048, 2048, 128, "bf16", 512, 4),
        # A long document with grouped heads.
        attention("train_long_grouped", 1, 16, 4, 8192, 8192, 128, "bf16", 1024, 16),
        # No window: the ordinary causal attention of the same model, the largest product.
        attention("train_full_causal", 1, 16, 16, 4096, 4096, 128, "bf16", 0, 0),
        # A padded batch of odd lengths (one sequence shorter than its window, one empty),
        # head width 80, float16.
        attention("train_ragged_f16", 8, 6, 2, 777, 777, 80, "f16", 100, 3, ragged=True),
        # The 4-layer model of width 256 in float32.
        attention("train_small_f32", 4, 4, 4, 256, 256, 64, "f32", 64, 2),
        # Serving: a chunk of 512 prompt tokens after 7680 that are already in the cache.
        attention("prefill_chunk", 1, 16, 4, 512, 8192, 128, "bf16", 2048, 4, offset=7680, direction="forward"),
        # Serving, one sequence of the 124M model: the latency of one token.
        step("step_short", 1, 12, 12, 1024, 64, "bf16", 256, 4, 700, ragged=False),
        # Serving, a batch with long histories and a wide window.
        step("step_window", 32, 16, 4, 8192, 128, "bf16", 4096, 4, 8192),
        # Serving without a window: everything that is in the cache is read.
        step("step_full", 8, 16, 4, 32768, 128, "f16", 0, 0, 32768),
        # A small batch of odd width in float32.
        dropout("dropout_small_odd", 257, 769, "f32", 0.1),
        # The residual stream of the 1.3B model, 8 sequences of 2048 tokens.
        dropout("dropout_1p3b", 16384, 2048, "bf16", 0.1),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """A case of the same ranges; none costs more than the largest listed one."""
    kind = rng.choice(("attention", "attention", "step", "dropout"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "dropout":
        width = _log(rng, 64, 4096)
        rows = _log(rng, 1, max(2, (1 << 25) // width))
        case = dropout("", rows, width, dtype, round(rng.uniform(0.02, 0.6), 3), rng.random() < 0.7, rng.random() < 0.8)
    elif kind == "step":
        group, kv_heads = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 8, 12))
        dim = rng.choice((64, 64, 80, 128, 128, 40))
        batch, capacity = _log(rng, 1, 48), _log(rng, 16, 32768)
        while batch * kv_heads * capacity * dim * SIZE[dtype] > 8 * 4 * 32768 * 128 * 2:
            capacity //= 2
        window = 0 if rng.random() < 0.3 else _log(rng, 1, capacity)
        case = step("", batch, group * kv_heads, kv_heads, capacity, dim, dtype, window, rng.choice((0, 1, 4, 16)),
                    max(1, int(capacity * rng.uniform(0.3, 1.0))), rng.random() < 0.7)
    else:
        group, kv_heads = rng.choice((1, 1, 2, 4)), rng.choice((1, 2, 3, 4, 8))
        dim = rng.choice((64, 64, 80, 128, 128, 40))
        keys = _log(rng, 1, 8192 if dtype != "f32" else 2048)
        batch = _log(rng, 1, 8)
        while batch * group * kv_heads * keys * keys > 16 * 4096 * 4096:
            if batch > 1:
                batch //= 2
            else:
                keys //= 2
        direction = rng.choice(("train", "train", "forward"))
        queries = keys if direction == "train" or rng.random() < 0.3 else _log(rng, 1, keys)
        window = 0 if rng.random() < 0.25 else _log(rng, 1, keys)
        case = attention("", batch, group * kv_heads, kv_heads, queries, keys, dim, dtype, window,
                         rng.choice((0, 1, 4, 16, 130)), rng.random() < 0.4, keys - queries, direction)
    del case["name"]
    return case


def _lengths(case):
    """Visible keys of each sequence, as the case alone gives them."""
    longest = case["longest"] if case["op"] == "step" else case["keys"]
    if not case["ragged"]:
        return [longest] * case["batch"]
    return [int(longest * RAGGED[b % len(RAGGED)]) for b in range(case["batch"])]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dt = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=dt)

    if case["op"] == "dropout":
        shape = (case["rows"], case["width"])
        state = {"case": case, "seed": int(seed) * 2654435761 % (1 << 62), "offset": int(seed) % 1000003,
                 "x": normal(*shape).requires_grad_(), "grad": normal(*shape)}
        state["bias"] = normal(case["width"]).requires_grad_() if case["bias"] else None
        state["residual"] = normal(*shape).requires_grad_() if case["residual"] else None
        return state
    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)
    b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    state = {"case": case, "lengths": lengths, "window": case["window"] or None, "sinks": case["sinks"]}
    if case["op"] == "step":
        state.update(q=normal(b, h, d), k=normal(b, hk, case["capacity"], d), v=normal(b, hk, case["capacity"], d))
        return state
    # Views of one packed projection [batch, tokens, (heads + 2 kv_heads) * dim] where there
    # are as many queries as keys; else the keys and values of a cache.
    tq, tk = case["queries"], case["keys"]
    if tq == tk:
        packed = normal(b, tk, h + 2 * hk, d)
        q, k, v = (t.transpose(1, 2) for t in packed.split((h, hk, hk), dim=2))
    else:
        q, k, v = normal(b, tq, h, d).transpose(1, 2), normal(b, hk, tk, d), normal(b, hk, tk, d)
    state.update(q=q, k=k, v=v)
    if case["direction"] == "train":
        state.update({n: state[n].detach().requires_grad_() for n in "qkv"})
        state["grad"] = normal(b, tq, h, d).transpose(1, 2)
    if not case["ragged"]:
        state["lengths"] = None
    return state


def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


# ---- the package's calls ----------------------------------------------------------------

def _own_attention(s):
    from namitorch_b200.nn import functional as F
    options = {"window": s["window"], "sinks": s["sinks"], "lengths": s["lengths"],
               "query_position_offset": s["case"]["offset"]}
    out = F.sliding_window_attention(s["q"], s["k"], s["v"], **options)
    if s["case"]["direction"] == "forward":
        return {"out": out}
    dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["grad"])
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _own_step(s):
    from namitorch_b200.nn import functional as F
    return {"out": F.sliding_window_attention_step(s["q"], s["k"], s["v"], s["lengths"], window=s["window"],
                                                   sinks=s["sinks"])}


def _own_dropout(s):
    from namitorch_b200.nn import functional as F
    y = F.dropout(s["x"], s["case"]["p"], seed=s["seed"], offset=s["offset"], bias=s["bias"], residual=s["residual"])
    wanted = {n: s[n] for n in ("x", "bias", "residual") if s[n] is not None}
    grads = torch.autograd.grad(y, tuple(wanted.values()), s["grad"])
    return {"out": y, **{"d" + n: t for n, t in zip(wanted, grads)}}


# ---- the plain forms ---------------------------------------------------------------------

def _visible(positions, keys, lengths, window, sinks):
    """[batch or 1, queries, keys] bool: which keys each query sees."""
    p, j = positions[..., None], torch.arange(keys, device=DEVICE)
    seen = j <= p
    if window:
        seen = seen & ((p - j < window) | (j < sinks))
    if lengths is not None:
        seen = seen & (j < lengths[:, None, None])
    return seen


def _softmax(scores, seen):
    scores = torch.where(seen, scores, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


@torch.no_grad()
def _plain_attention(s):
    c, dt = s["case"], s["q"].dtype
    group, scale = c["heads"] // c["kv_heads"], c["dim"] ** -0.5
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    positions = c["offset"] + torch.arange(c["queries"], device=DEVICE)
    seen = _visible(positions[None], c["keys"], s["lengths"], s["window"], s["sinks"])[:, None]
    p = _softmax(torch.matmul(q, kk.transpose(-1, -2)) * scale, seen)
    out = torch.matmul(p, vv)
    if c["direction"] == "forward":
        return {"out": out.to(dt)}
    g = s["grad"].float()
    dv = torch.matmul(p.transpose(-1, -2), g)
    dp = torch.matmul(g, vv.transpose(-1, -2))
    ds = p * (dp - (g * out).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, kk)
    dk = torch.matmul(ds.transpose(-1, -2), q)
    dk, dv = (t.unflatten(1, (c["kv_heads"], group)).sum(2) for t in (dk, dv))
    return {"out": out.to(dt), "dq": dq.to(dt), "dk": dk.to(dt), "dv": dv.to(dt)}


@torch.no_grad()
def _plain_step(s):
    c, dt = s["case"], s["q"].dtype
    group = c["heads"] // c["kv_heads"]
    q = s["q"].float().unflatten(1, (c["kv_heads"], group)) * c["dim"] ** -0.5
    seen = _visible((s["lengths"] - 1)[:, None], c["capacity"], s["lengths"], s["window"], s["sinks"])[:, None]
    p = _softmax(torch.matmul(q, s["k"].float().transpose(-1, -2)), seen)
    return {"out": torch.matmul(p, s["v"].float()).flatten(1, 2).to(dt)}


def _philox(counter, offset, seed):
    """The four 32-bit words (int64, [n, 4]) of Philox4x32-7 at (counter, offset) under seed."""
    low = 0xFFFFFFFF
    a, b = counter & low, counter >> 32
    c, d = torch.full_like(a, offset & low), torch.full_like(a, offset >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(7):
        x, y = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = ((y >> 32) & low) ^ b ^ k0, y & low, ((x >> 32) & low) ^ d ^ k1, x & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((a, b, c, d), -1)


@torch.no_grad()
def _plain_dropout(s):
    c, dt = s["case"], s["x"].dtype
    n = c["rows"] * c["width"]
    words = _philox(torch.arange((n + 3) // 4, device=DEVICE), s["offset"], s["seed"]).flatten()[:n]
    keep = (words >= int(c["p"] * 4294967296.0)).view(c["rows"], c["width"])
    factor = keep.float() * (1.0 / (1.0 - c["p"]))
    x = s["x"].float()
    y = (x if s["bias"] is None else x + s["bias"].float()) * factor
    if s["residual"] is not None:
        y = y + s["residual"].float()
    dx = s["grad"].float() * factor
    got = {"out": y.to(dt), "dx": dx.to(dt)}
    if s["bias"] is not None:
        got["dbias"] = dx.sum(0).to(dt)
    if s["residual"] is not None:
        got["dresidual"] = s["grad"]
    return got


_own = {"attention": _own_attention, "step": _own_step, "dropout": _own_dropout}
_plain = {"attention": _plain_attention, "step": _plain_step, "dropout": _plain_dropout}


# ---- what a pass cannot do without --------------------------------------------------------

def _pairs(case):
    """Visible (query, key) pairs of all sequences, one head."""
    if case["op"] == "step":
        return sum(min(n, case["window"] + min(case["sinks"], max(0, n - case["window"]))) if case["window"] else n
                   for n in _lengths(case))
    p = case["offset"] + np.arange(case["queries"], dtype=np.int64)
    total = 0
    for n in _lengths(case):
        end = np.minimum(n, p + 1)
        start = np.minimum(np.maximum(0, p + 1 - case["window"]), end) if case["window"] else np.zeros_like(p)
        total += int((end - start + (np.minimum(case["sinks"], start) if case["window"] else 0)).sum())
    return total


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "dropout":
        n = case["rows"] * case["width"]
        # x, residual and the upstream gradient in; y and dx out (the residual's gradient is
        # the upstream gradient itself); the bias in and its gradient out.
        return {"bytes": size * (n * (4 + case["residual"]) + 2 * case["bias"] * case["width"]),
                "flops": n * (3 + 2 * case["bias"] + case["residual"])}
    b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "step":
        pairs = _pairs(case)
        return {"bytes": size * d * (2 * hk * pairs + 2 * b * h), "flops": 4 * d * h * pairs}
    pairs, train = _pairs(case), case["direction"] == "train"
    q, kv = b * h * case["queries"] * d, b * hk * case["keys"] * d
    if not train and case["window"]:
        # A chunk reads the keys that some query of it sees.
        kv = min(kv, b * hk * d * (case["queries"] + case["window"] - 1 + case["sinks"]))
    return {"bytes": size * ((4 * q + 4 * kv) if train else (2 * q + 2 * kv)),
            "flops": (14 if train else 4) * d * h * pairs}


# ---- the definitions in 64 bits ------------------------------------------------------------

def _rows(p, length, window, sinks, keys):
    """Additive mask [queries, keys] in 64 bits: 0 where visible, -inf elsewhere."""
    p, j = np.asarray(p)[:, None], np.arange(keys)[None, :]
    near = np.ones((p.shape[0], keys), bool) if not window else (j > p - window) | (j < sinks)
    return torch.from_numpy(np.where(near & (j <= p) & (j < length), 0.0, -np.inf)).to(DEVICE)


def _exact_attention(case, s):
    c, train = case, case["direction"] == "train"
    b, h, hk, d = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    q, k, v = (s[n].detach().double() for n in "qkv")
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i, length in enumerate(_lengths(c)):
        mask = _rows(c["offset"] + np.arange(c["queries"]), length, c["window"], c["sinks"], c["keys"])
        some = torch.isfinite(mask).any(1)
        if not bool(some.any()):
            continue
        for n in range(h):
            m = n // (h // hk)
            log_p = torch.log_softmax((q[i, n] @ k[i, m].T / math.sqrt(d) + mask)[some], -1)
            p = torch.zeros_like(mask)
            p[some] = torch.exp(log_p)
            out[i, n] = p @ v[i, m]
            if train:
                g = s["grad"][i, n].double()
                dp = g @ v[i, m].T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(d)
                dv[i, m] += p.T @ g
                dq[i, n] = ds @ k[i, m]
                dk[i, m] += ds.T @ q[i, n]
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if train else {"out": out}


def _exact_step(case, s):
    c = case
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    for i, n in enumerate(_lengths(c)):
        if n == 0:
            continue
        j = np.arange(n)
        j = torch.from_numpy(j[(j > n - 1 - c["window"]) | (j < c["sinks"])] if c["window"] else j).to(DEVICE)
        for head in range(c["heads"]):
            m = head // (c["heads"] // c["kv_heads"])
            p = torch.softmax(s["k"][i, m, j].double() @ s["q"][i, head].double() / math.sqrt(c["dim"]), 0)
            out[i, head] = p @ s["v"][i, m, j].double()
    return {"out": out}


def _exact_dropout(case, s):
    c, n = case, case["rows"] * case["width"]
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    counter = np.arange((n + 3) // 4, dtype=np.uint64)
    w = [counter & low, counter >> shift, np.full_like(counter, s["offset"] & 0xFFFFFFFF),
         np.full_like(counter, s["offset"] >> 32)]
    key = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32]
    for r in range(7):
        k0, k1 = ((key[i] + r * c32) & 0xFFFFFFFF for i, c32 in enumerate((0x9E3779B9, 0xBB67AE85)))
        x, y = w[0] * np.uint64(0xD2511F53), w[2] * np.uint64(0xCD9E8D57)
        w = [(y >> shift) ^ w[1] ^ np.uint64(k0), y & low, (x >> shift) ^ w[3] ^ np.uint64(k1), x & low]
    keep = torch.from_numpy(np.stack(w, 1).reshape(-1)[:n].reshape(c["rows"], c["width"]) >= int(c["p"] * 2.0 ** 32))
    weight = keep.to(DEVICE).double() / (1.0 - c["p"])
    x = s["x"].detach().double()
    if s["bias"] is not None:
        x = x + s["bias"].detach().double()
    dx = weight * s["grad"].double()
    got = {"out": weight * x, "dx": dx}
    if s["bias"] is not None:
        got["dbias"] = dx.sum(0)
    if s["residual"] is not None:
        got["out"] = got["out"] + s["residual"].detach().double()
        got["dresidual"] = s["grad"].double()
    return got


def exact(case, seed):
    table = {"attention": _exact_attention, "step": _exact_step, "dropout": _exact_dropout}
    with torch.no_grad():
        return table[case["op"]](case, prepare(case, seed))
