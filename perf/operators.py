"""Cases of the 8-bit projections and the cross attention, with plain forms of both.

Three operators are timed and compared here:

* ``linear``: ``act(x w^T + bias)`` with x quantised to 8-bit integers per token and w
  held in 8-bit integers with a scale per output channel.
* ``ffn``: the encoder's feed-forward half, ``h = LayerNorm(a + residual)`` and
  ``o = down(gelu(up(h)))``, both projections in 8-bit integers.
* ``cross``: queries of packed sequences attending to the packed states of an encoder,
  whose sequences have lengths of their own; from single tokens to prompts.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def linear(name, m, k, n, act="none", dtype="bf16"):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "act": act, "dtype": dtype}


def ffn(name, m, h, i, dtype="bf16"):
    return {"name": name, "op": "ffn", "m": m, "h": h, "i": i, "dtype": dtype}


def cross(name, seqs, q_min, q_max, kv_min, kv_max, heads, kv_heads, d, dtype="bf16", empty=False):
    return {"name": name, "op": "cross", "seqs": seqs, "q_min": q_min, "q_max": q_max, "kv_min": kv_min,
            "kv_max": kv_max, "heads": heads, "kv_heads": kv_heads, "d": d, "dtype": dtype, "empty": empty,
            "lengths": 1}


def listed():
    return [
        # one pooled row through a square projection: latency
        linear("linear_one_row", 1, 1024, 1024),
        # a few hundred tokens, no size a multiple of a tile
        linear("linear_odd", 333, 1000, 771, dtype="f16"),
        # the serving batch's tokens through the FFN up projection and its GELU
        linear("linear_up", 17410, 1024, 4096, act="gelu"),
        # a batch of 64 rows of 256 tokens through the wide encoder's up projection
        linear("linear_wide", 16384, 2560, 10240, dtype="f16"),
        # a small request's feed-forward half
        ffn("ffn_small", 64, 1024, 4096),
        # the serving batch's feed-forward half
        ffn("ffn_serve", 17410, 1024, 4096),
        # one token of one request reading one short text: latency
        cross("token_one", 1, 1, 1, 77, 77, 16, 16, 64),
        # one decoding step of 64 requests over texts of a serving batch, one of them empty
        cross("token_batch", 64, 1, 1, 32, 512, 16, 16, 64, empty=True),
        # one step of 32 requests over long documents, four query heads to a key head
        cross("token_long", 32, 1, 1, 64, 8192, 32, 8, 128, dtype="f16"),
        # short prompts over a serving batch's texts
        cross("prompt_batch", 64, 1, 128, 32, 512, 16, 16, 64, empty=True),
        # the wide encoder's heads
        cross("prompt_wide", 16, 64, 300, 32, 512, 32, 32, 80, dtype="f16"),
        # long prompts over long documents
        cross("prompt_long", 8, 256, 1024, 1024, 8192, 16, 16, 64),
    ]


def spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "ffn", "cross", "cross"])
    while True:
        if op == "linear":
            case = linear("", spread(rng, 1, 20000), spread(rng, 16, 10240), spread(rng, 8, 10240),
                          rng.choice(["none", "gelu"]), rng.choice(["bf16", "f16", "f32"]))
            if case["m"] * case["k"] * case["n"] > 16384 * 2560 * 10240:
                continue
        elif op == "ffn":
            case = ffn("", spread(rng, 1, 20000), 8 * spread(rng, 8, 320), 8 * spread(rng, 8, 1280),
                       rng.choice(["bf16", "f16"]))
            if case["m"] * case["h"] * case["i"] > 17410 * 1024 * 4096:
                continue
        else:
            kv_heads = rng.randint(1, 16)
            heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
            q_max = rng.choice([1, 1, spread(rng, 1, 1024)])
            kv_max = spread(rng, 1, 8192)
            case = cross("", spread(rng, 1, 64), rng.randint(1, q_max), q_max, rng.randint(1, kv_max), kv_max, heads,
                         kv_heads, 8 * rng.randint(4, 16), rng.choice(["bf16", "f16"]), rng.random() < 0.3)
            case["lengths"] = rng.randint(1, 1 << 30)
            if case["seqs"] * heads * q_max * kv_max > 8 * 16 * 1024 * 8192:
                continue
            if case["seqs"] * kv_heads * case["d"] * kv_max > 32 * 8 * 128 * 8192:
                continue
        del case["name"]
        return case


def lengths(case):
    """The query and key lengths of a cross case's sequences."""
    rng = random.Random(case["lengths"])
    q = [rng.randint(case["q_min"], case["q_max"]) for _ in range(case["seqs"])]
    kv = [rng.randint(case["kv_min"], case["kv_max"]) for _ in range(case["seqs"])]
    if case["empty"]:
        kv[rng.randrange(case["seqs"])] = 0
    return q, kv


def activations(gen, m, k, dtype):
    """Activations as an encoder's layers see them: normal, one channel in 64 of them
    twelve times as large, tokens of differing size."""
    x = torch.randn(m, k, device="cuda", generator=gen)
    x[:, ::64] *= 12.0
    x *= torch.rand(m, 1, device="cuda", generator=gen) + 0.5
    return x.to(dtype)


def weight8(gen, n, k):
    """A weight in 8-bit integers with a scale per output channel."""
    w = torch.randn(n, k, device="cuda", generator=gen) * k ** -0.5
    scale = w.abs().amax(1) / 127.0
    return torch.round(w / scale[:, None]).to(torch.int8), scale


def inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "linear":
        s["x"] = activations(gen, case["m"], case["k"], dtype)
        s["w"], s["ws"] = weight8(gen, case["n"], case["k"])
        s["bias"] = torch.randn(case["n"], device="cuda", generator=gen).to(dtype)
    elif case["op"] == "ffn":
        h, i = case["h"], case["i"]
        s["a"] = activations(gen, case["m"], h, dtype)
        s["residual"] = torch.randn(case["m"], h, device="cuda", generator=gen).to(dtype)
        s["gamma"] = (1.0 + 0.1 * torch.randn(h, device="cuda", generator=gen)).to(dtype)
        s["beta"] = (0.1 * torch.randn(h, device="cuda", generator=gen)).to(dtype)
        s["up"], s["ups"] = weight8(gen, i, h)
        s["up_bias"] = (0.1 * torch.randn(i, device="cuda", generator=gen)).to(dtype)
        s["down"], s["downs"] = weight8(gen, h, i)
        s["down_bias"] = (0.1 * torch.randn(h, device="cuda", generator=gen)).to(dtype)
    else:
        q, kv = lengths(case)
        d, heads, kv_heads = case["d"], case["heads"], case["kv_heads"]
        s["q"] = torch.randn(sum(q), heads * d, device="cuda", generator=gen).to(dtype)
        both = torch.randn(sum(kv), 2 * kv_heads * d, device="cuda", generator=gen).to(dtype)
        # keys and values are the two halves of one projection of the encoder's states
        s["k"], s["v"] = both[:, :kv_heads * d], both[:, kv_heads * d:]
        s["q_lengths"], s["kv_lengths"] = q, kv
    return s


def prepare(case, seed):
    s = inputs(case, seed)
    if case["op"] == "cross":
        # where the sequences' rows lie, as (sequence, place) grids, and which places hold a row
        for side in ("q", "kv"):
            n = np.asarray(s[side + "_lengths"])
            at = np.arange(max(1, n.max()))
            rows = (np.cumsum(n) - n)[:, None] + np.minimum(at, np.maximum(n - 1, 0)[:, None])
            rows = np.minimum(rows, max(0, n.sum() - 1))
            s[side + "_rows"] = torch.from_numpy(rows).cuda()
            s[side + "_held"] = torch.from_numpy(at < n[:, None]).cuda()
    if own:
        from latefuse_b200 import Int8Weight, cross_batch

        if case["op"] == "linear":
            s["weight"] = Int8Weight(s["w"], s["ws"])
        elif case["op"] == "ffn":
            s["up_weight"], s["down_weight"] = Int8Weight(s["up"], s["ups"]), Int8Weight(s["down"], s["downs"])
        else:
            s["batch"] = cross_batch(s["q_lengths"], s["kv_lengths"], s["q"].device)
    return s


def gelu(v):
    return v * 0.5 * (1.0 + torch.erf(v * math.sqrt(0.5)))


def plain_linear(x, w, ws, bias, act):
    """Each row of x rounded to whole multiples of its largest magnitude / 127 (in 64 bits:
    a ratio next to a half decides a step), the whole numbers multiplied, scaled, biased."""
    top = x.float().abs().amax(1, keepdim=True)
    steps = x.double() * 127.0 / torch.where(top > 0, top, torch.ones_like(top)).double()
    y = torch.round(steps).float() @ w.float().t()
    y = y * (top / 127.0) * ws + bias.float()
    return (gelu(y) if act == "gelu" else y).to(x.dtype)


def plain_ffn(s):
    a = s["a"]
    t = (a.float() + s["residual"].float()).to(a.dtype).float()
    t = t - t.mean(1, keepdim=True)
    t = t / torch.sqrt((t * t).mean(1, keepdim=True) + 1e-5)
    h = (t * s["gamma"].float() + s["beta"].float()).to(a.dtype)
    mid = plain_linear(h, s["up"], s["ups"], s["up_bias"], "gelu")
    return h, plain_linear(mid, s["down"], s["downs"], s["down_bias"], "none")


def plain_cross(s):
    d, kv_heads = s["case"]["d"], s["case"]["kv_heads"]
    if not s["k"].shape[0]:
        return torch.zeros_like(s["q"])
    q = s["q"].float()[s["q_rows"]].unflatten(2, (kv_heads, -1, d))
    k = s["k"].float()[s["kv_rows"]].unflatten(2, (kv_heads, d))
    v = s["v"].float()[s["kv_rows"]].unflatten(2, (kv_heads, d))
    score = torch.einsum("sqhgd,skhd->shgqk", q, k) * d ** -0.5
    held = s["kv_held"][:, None, None, None, :]
    score = torch.where(held, score, torch.full_like(score, -1e30))
    p = torch.exp(score - score.amax(4, keepdim=True)) * held
    o = torch.einsum("shgqk,skhd->sqhgd", p, v)
    total = p.sum(4).permute(0, 3, 1, 2)[..., None]
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.flatten(2)[s["q_held"]].to(s["q"].dtype)


def run(s):
    case = s["case"]
    if own:
        from latefuse_b200 import cross_attention_varlen, ffn_int8, linear_int8

        if case["op"] == "linear":
            return linear_int8(s["x"], s["weight"], s["bias"], act=1 if case["act"] == "gelu" else 0)
        if case["op"] == "ffn":
            return ffn_int8(s["a"], s["residual"], s["gamma"], s["beta"], 1e-5, s["up_weight"], s["up_bias"],
                            s["down_weight"], s["down_bias"])
        return cross_attention_varlen(s["q"], s["k"], s["v"], s["batch"], case["heads"], case["kv_heads"])
    if case["op"] == "linear":
        return plain_linear(s["x"], s["w"], s["ws"], s["bias"], case["act"])
    if case["op"] == "ffn":
        return plain_ffn(s)
    return plain_cross(s)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": size * (m * k + n + m * n) + n * k + 4 * n, "flops": 2 * m * n * k}
    if case["op"] == "ffn":
        m, h, i = case["m"], case["h"], case["i"]
        # both inputs, the state and the output; the weights with their scales and biases
        return {"bytes": size * 4 * m * h + 2 * h * i + (4 + size) * (h + i) + size * 2 * h, "flops": 4 * m * h * i}
    q, kv = lengths(case)
    d, heads, kv_heads = case["d"], case["heads"], case["kv_heads"]
    pairs = sum(a * b for a, b in zip(q, kv))
    return {"bytes": size * (2 * sum(q) * heads * d + 2 * sum(kv) * kv_heads * d), "flops": 4 * pairs * heads * d}


def exact_rows(x):
    """The whole numbers and the steps of the rows of x: round(127 x / max |x|), max |x| / 127."""
    x = x.to(torch.float64)
    top = x.abs().max(dim=1, keepdim=True).values
    whole = torch.where(top > 0, (127.0 * x / top).round(), torch.zeros_like(x))
    return whole, top / 127.0


def exact_projection(x, w, ws, bias, act):
    parts = []
    for rows in x.split(4096):
        whole, step = exact_rows(rows)
        y = torch.mm(whole, w.to(torch.float64).T) * step * ws.to(torch.float64) + bias.to(torch.float64)
        parts.append(torch.special.ndtr(y) * y if act == "gelu" else y)
    return torch.cat(parts)


def exact(case, seed):
    s = inputs(case, seed)
    if case["op"] == "linear":
        return exact_projection(s["x"], s["w"], s["ws"], s["bias"], case["act"])
    if case["op"] == "ffn":
        t = (s["a"].to(torch.float64) + s["residual"].to(torch.float64)).to(s["a"].dtype).to(torch.float64)
        centred = t - t.mean(dim=1, keepdim=True)
        h = centred * (centred.pow(2).mean(dim=1, keepdim=True) + 1e-5).rsqrt()
        h = h * s["gamma"].to(torch.float64) + s["beta"].to(torch.float64)
        mid = exact_projection(h.to(s["a"].dtype), s["up"], s["ups"], s["up_bias"], "gelu")
        return h, exact_projection(mid.to(s["a"].dtype), s["down"], s["downs"], s["down_bias"], "none")
    d, heads, kv_heads = case["d"], case["heads"], case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for nq, nk in zip(s["q_lengths"], s["kv_lengths"]):
        q = s["q"][q0:q0 + nq].to(torch.float64).view(nq, heads, d)
        k = s["k"][k0:k0 + nk].to(torch.float64).reshape(nk, kv_heads, d)
        v = s["v"][k0:k0 + nk].to(torch.float64).reshape(nk, kv_heads, d)
        for h in range(heads if nk else 0):
            g = h * kv_heads // heads
            p = torch.softmax(q[:, h] @ k[:, g].T / math.sqrt(d), dim=1)
            out[q0:q0 + nq, h * d:(h + 1) * d] = p @ v[:, g]
        q0, k0 = q0 + nq, k0 + nk
    return out
