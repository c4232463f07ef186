"""The 8-bit serving operators (row quantiser, residual + RMSNorm, scaled linear layer,
paged key-value cache and the attention that reads it) as measurable cases.

Each case is a dict of plain values.  `prepare` makes what a serving program holds before
the call, `run` makes one pass (in elementary torch operations, or through the library's
entry points when `own` is set), `exact` computes the same outputs from the definitions in
64 bits, and `work` says which bytes and operations a pass cannot do without.

e4m3 codes are returned as torch.float8_e4m3fn tensors beside their scales.
"""
import math
import random

import numpy as np
import torch

own = False

E4M3_MAX = 448.0
TINY = 2.0 ** -110  # the smallest row maximum that sets a scale
EPS = 1e-6
F8 = torch.float8_e4m3fn


# ------------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of a Qwen3-0.6B-shaped encoder (hidden 1024): latency alone
        {"name": "norm-one-row", "op": "norm", "rows": 1, "dim": 1024, "y": "bf16"},
        # the bge-large benchmark batch's token count, hidden 1024
        {"name": "norm-batch", "op": "norm", "rows": 26508, "dim": 1024, "y": "bf16"},
        # a weight matrix (4096 x 1024, fp32 as loaded) quantised per output channel
        {"name": "quant-weight-f32", "op": "quant", "rows": 4096, "dim": 1024, "x": "f32"},
        # attention outputs of the Qwen3 benchmark batch (71,550 tokens, 16 heads x 128) ahead of the out-projection
        {"name": "quant-attn-out", "op": "quant", "rows": 71550, "dim": 2048, "x": "bf16"},
        # eight single tokens through a 1024 -> 4096 projection: bound by reading the weight
        {"name": "linear-few-rows", "op": "linear", "rows": 8, "n": 4096, "k": 1024, "epilogue": "bias", "out": "bf16"},
        # the FFN up-projection of the bge-large batch
        {"name": "linear-ffn-gelu", "op": "linear", "rows": 26508, "n": 4096, "k": 1024, "epilogue": "bias_gelu", "out": "bf16"},
        # an FFN down-projection onto the fp32 residual stream, odd row count
        {"name": "linear-down-residual", "op": "linear", "rows": 4099, "n": 1024, "k": 4096, "epilogue": "bias_residual",
         "out": "f32"},
        # 64 sequences, each with one new token
        {"name": "append-single-tokens", "op": "append", "batch": 64, "past": 2000, "new": 1, "page": 64, "q_heads": 16,
         "kv_heads": 8, "hd": 128, "ragged": 1},
        # prompts of up to 4,000 tokens behind a cached prefix that ends inside a page
        {"name": "append-prompts", "op": "append", "batch": 16, "past": 77, "new": 4000, "page": 64, "q_heads": 16,
         "kv_heads": 8, "hd": 128, "ragged": 2},
        # one token of one sequence over a short cache: latency
        {"name": "attend-one-token", "op": "attend", "batch": 1, "past": 500, "new": 1, "page": 64, "q_heads": 16,
         "kv_heads": 8, "hd": 128, "causal": True, "ragged": 0},
        # 32 sequences, one token each, over caches of up to 16k tokens: bound by reading the cache
        {"name": "attend-single-tokens", "op": "attend", "batch": 32, "past": 16000, "new": 1, "page": 64, "q_heads": 16,
         "kv_heads": 8, "hd": 128, "causal": True, "ragged": 3},
        # prompts of up to 2,000 tokens behind a cached prefix of up to 1,000
        {"name": "attend-prompts", "op": "attend", "batch": 8, "past": 1000, "new": 2000, "page": 64, "q_heads": 16,
         "kv_heads": 8, "hd": 128, "causal": True, "ragged": 4},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "quant", "linear", "append", "attend", "attend"])
    if op in ("norm", "quant"):
        rows = _log(rng, 1, 71550 if op == "quant" else 26508)
        # even the odd widths of the range stay within the largest listed case
        most = (146_000_000 if op == "quant" else 27_000_000) // rows
        dim = max(1, min(_log(rng, 64, 4096), most))
        if rng.random() < 0.8:
            dim = max(8, dim // 8 * 8)
        return {"op": op, "rows": rows, "dim": dim, "y" if op == "norm" else "x": rng.choice(["bf16", "f32"])}
    if op == "linear":
        epi, out = rng.choice([("none", "bf16"), ("none", "f32"), ("bias", "bf16"), ("bias_gelu", "bf16"),
                               ("bias_relu", "bf16"), ("bias_swish", "bf16"), ("bias_residual", "f32"),
                               ("swiglu", "bf16"), ("geglu", "bf16")])
        rows, k = _log(rng, 1, 26508), max(16, _log(rng, 64, 4096) // 16 * 16)
        step = 128 if epi in ("swiglu", "geglu") else 8
        n = min(_log(rng, 128, 4096), 111_000_000_000 // (rows * k))
        return {"op": op, "rows": rows, "n": max(step, n // step * step), "k": k, "epilogue": epi, "out": out}
    kv_heads = rng.choice([1, 2, 4, 8])
    case = {"op": op, "page": rng.choice([16, 32, 64, 128]), "kv_heads": kv_heads, "q_heads": kv_heads * rng.choice([1, 2, 3, 4]),
            "hd": rng.choice([64, 128, 256]), "ragged": rng.randrange(1 << 20)}
    if op == "append":
        case["new"] = rng.choice([1, _log(rng, 2, 4000)])
        case["past"] = rng.choice([0, _log(rng, 1, 4000)])
        most = 64 * 1024 * 8 * 128 // (kv_heads * case["hd"] * (case["new"] + 64))
        case["batch"] = _log(rng, 1, max(1, min(64, most)))
        return case
    case["causal"] = rng.random() < 0.75
    if rng.random() < 0.5:  # few new tokens over a long cache
        case["new"], case["past"] = rng.choice([1, 1, _log(rng, 2, 16)]), _log(rng, 1, 16000)
    else:
        case["new"], case["past"] = _log(rng, 17, 2000), rng.choice([0, _log(rng, 1, 1000)])
    tokens = case["new"] + case["past"]
    most = min(32 * 16000 * 8 * 128 // (tokens * kv_heads * case["hd"]),
               8 * 2000 * 3000 * 16 * 128 // (case["new"] * tokens * case["q_heads"] * case["hd"]))
    case["batch"] = _log(rng, 1, max(1, min(32, most)))
    return case


def _lengths(case):
    """(new tokens, past tokens) of each sequence: the case's own maximum first, the others
    spread from half of it upwards.  A matter of the case alone."""
    rng = random.Random(case["ragged"])
    new, past = [], []
    for b in range(case["batch"]):
        if case["ragged"] == 0 or b == 0:
            n, p = case["new"], case["past"]
        else:
            n, p = rng.randint((case["new"] + 1) // 2, case["new"]), rng.randint(case["past"] // 2, case["past"])
        new.append(n)
        past.append(p)
    return new, past


def _pages(case):
    """(pages in the pool, page-table width): each sequence's own pages and a few spare ones."""
    new, past = _lengths(case)
    own_pages = [-(-(n + p) // case["page"]) for n, p in zip(new, past)]
    return sum(own_pages) + 3, max(own_pages) + 1


# ---------------------------------------------------------------------- prepare
def _codes(x):
    """fp32 [..., tokens, hd] -> (codes, scale [...]): power-of-two scale of the block."""
    m, e = torch.frexp(x.abs().amax((-1, -2)))
    scale = torch.ldexp(torch.ones_like(m), e - torch.where(m <= 0.875, 9, 8))
    return (x / scale[..., None, None]).to(F8), scale


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    op = case["op"]
    if op == "norm":
        h = randn(case["rows"], case["dim"]) * 2.0
        h[:, :: 97] *= 12.0  # the few wide channels of a residual stream
        y = randn(case["rows"], case["dim"])
        return {"case": case, "h": h, "y": y.to(torch.bfloat16) if case["y"] == "bf16" else y,
                "w": 1.0 + 0.2 * randn(case["dim"])}
    if op == "quant":
        x = randn(case["rows"], case["dim"]) * torch.exp(0.5 * randn(case["rows"], 1))
        return {"case": case, "x": x.to(torch.bfloat16) if case["x"] == "bf16" else x * 0.02}
    if op == "linear":
        x, w = randn(case["rows"], case["k"]), randn(case["n"], case["k"]) / math.sqrt(case["k"])
        state = {"case": case}
        for name, v in (("x", x), ("w", w)):
            s = v.abs().amax(-1) / E4M3_MAX
            state[name], state[name + "s"] = (v / s[:, None]).to(F8), s
        state["bias"] = 0.1 * randn(case["n"]) if case["epilogue"].startswith("bias") else None
        state["residual"] = randn(case["rows"], case["n"]) if case["epilogue"] == "bias_residual" else None
        return state

    new, past = _lengths(case)
    pool, width = _pages(case)
    page, hkv, hd = case["page"], case["kv_heads"], case["hd"]
    total = sum(new)
    heads = case["q_heads"] + 2 * hkv
    spread = torch.exp(0.4 * randn(heads, hd))  # keys and values have wide and narrow channels
    qkv = (randn(total, heads, hd) * spread).to(torch.bfloat16).view(total, heads * hd)
    order = torch.randperm(pool, device=dev, generator=g).to(torch.int32)
    table = np.full((case["batch"], width), 0, np.int64)
    at = 0
    for b in range(case["batch"]):
        n = -(-(new[b] + past[b]) // page)
        table[b, :n] = np.arange(at, at + n)
        at += n
    state = {"case": case, "qkv": qkv, "new": new, "past": past, "max_new": max(new),
             "max_kv": max(n + p for n, p in zip(new, past)),
             "cu": torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=dev),
             "past_lens": torch.tensor(past, dtype=torch.int32, device=dev),
             "table": order[torch.from_numpy(table).to(dev)].contiguous()}
    for i, name in enumerate("kv"):  # what earlier calls have left in the pages
        lo = case["q_heads"] + i * hkv
        codes, scales = [], []
        step = max(1, 60_000_000 // (hkv * page * hd))
        for p0 in range(0, pool, step):
            c, s = _codes(randn(min(step, pool - p0), hkv, page, hd) * spread[lo:lo + hkv, None, :])
            codes.append(c.view(torch.uint8))
            scales.append(s)
        state[name] = torch.cat(codes).view(F8)
        state[name + "s"] = torch.cat(scales)
    return state


# -------------------------------------------------------------------- plain forms
def _quantize(v):
    """Row scales and codes of fp32 rows; what is not finite takes the NaN code."""
    finite = torch.isfinite(v)
    s = torch.where(finite, v.abs(), 0.0).amax(-1).clamp_min(TINY) / E4M3_MAX
    return torch.where(finite, v / s[:, None], math.nan).to(F8), s


def _plain_norm(s):
    h = s["h"].add_(s["y"].float())
    n = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["w"]
    q, scale = _quantize(n)
    return h, q, scale


def _gelu(z):
    return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))


def _silu(z):
    return z / (1.0 + torch.exp(-z))


def _epilogue(z, bias, residual, epilogue):
    if epilogue in ("swiglu", "geglu"):  # rows of w alternate 32 gates and 32 inputs
        z = z.view(z.shape[0], -1, 2, 32)
        gate = _silu(z[:, :, 0]) if epilogue == "swiglu" else _gelu(z[:, :, 0])
        return (gate * z[:, :, 1]).reshape(z.shape[0], -1)
    z = z if bias is None else z + bias
    if epilogue == "bias_gelu":
        return _gelu(z)
    if epilogue == "bias_relu":
        return z.clamp_min(0.0)
    if epilogue == "bias_swish":
        return _silu(z)
    return z if residual is None else z + residual


def _plain_linear(s):
    z = (s["x"].float() * s["xs"][:, None]) @ (s["w"].float() * s["ws"][:, None]).T
    y = _epilogue(z, s["bias"], s["residual"], s["case"]["epilogue"])
    return y.to(torch.bfloat16) if s["case"]["out"] == "bf16" else y


def _touched(s):
    """(sequence, page ordinal) of every page that the new tokens reach."""
    page = s["case"]["page"]
    new, past = np.asarray(s["new"]), np.asarray(s["past"])
    first, last = past // page, (past + new - 1) // page
    count = np.where(new > 0, last - first + 1, 0)
    seq = np.repeat(np.arange(len(new)), count)
    ordinal = np.arange(count.sum()) - np.repeat(np.cumsum(count) - count, count) + first[seq]
    return torch.from_numpy(np.stack([seq, ordinal])).to(s["qkv"].device)


def _plain_append(s):
    case = s["case"]
    page, hkv, hd = case["page"], case["kv_heads"], case["hd"]
    seq, ordinal = _touched(s)
    at = s["table"][seq, ordinal].long()
    pos = ordinal[:, None] * page + torch.arange(page, device=at.device)
    past, cu = s["past_lens"].long()[seq, None], s["cu"].long()
    old = pos < past
    token = cu[seq, None] + pos - past
    fresh = ~old & (token < cu[seq + 1, None])
    rows = s["qkv"].view(-1, case["q_heads"] + 2 * hkv, hd)[token.clamp(0, s["qkv"].shape[0] - 1)]
    for i, name in enumerate("kv"):
        x = rows[:, :, case["q_heads"] + i * hkv: case["q_heads"] + (i + 1) * hkv].float().transpose(1, 2)
        x = torch.where(fresh[:, None, :, None], x, 0.0)
        m, e = torch.frexp(x.abs().amax((-1, -2)))
        need = torch.where(m > 0, torch.ldexp(torch.ones_like(m), e - torch.where(m <= 0.875, 9, 8)), 0.0)
        before = torch.where(old[:, :1], s[name + "s"][at], 0.0)
        scale = torch.maximum(need, before)
        inv = torch.where(scale > 0, 1.0 / scale, 0.0)[:, :, None, None]
        codes = s[name].view(torch.uint8)
        was = codes[at]
        again = (was.view(F8).float() * (before[:, :, None, None] * inv)).to(F8).view(torch.uint8)
        mixed = torch.where(fresh[:, None, :, None], (x * inv).to(F8).view(torch.uint8),
                            torch.where(old[:, None, :, None], again, was))
        codes[at] = mixed
        s[name + "s"][at] = scale
    return s["k"], s["v"], s["ks"], s["vs"]


def _plain_attend(s):
    case = s["case"]
    page, hq, hkv, hd = case["page"], case["q_heads"], case["kv_heads"], case["hd"]
    group, total, batch = hq // hkv, s["qkv"].shape[0], case["batch"]
    table = s["table"][:, : -(-s["max_kv"] // page)].long()

    def cached(name):
        v = s[name].view(torch.uint8)[table].view(F8).float()  # [batch, pages, heads, page, hd]
        v *= s[name + "s"][table][..., None, None]
        return v.permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, hd)

    cu, past = s["cu"].long(), s["past_lens"].long()
    length = cu[1:] - cu[:-1]
    i = torch.arange(s["max_new"], device=table.device)
    token = (cu[:-1, None] + i).clamp_max(total - 1)
    q = s["qkv"].view(total, -1, hd)[:, :hq][token].float()  # [batch, new, hq, hd]
    q = q.view(batch, -1, hkv, group, hd).permute(0, 2, 3, 1, 4).reshape(batch, hkv, -1, hd)
    scores = (q @ cached("k").transpose(-1, -2)).mul_(hd ** -0.5)
    last = past[:, None] + i if case["causal"] else (past + length - 1)[:, None].expand(-1, s["max_new"])
    keep = torch.arange(scores.shape[-1], device=table.device) <= last[:, :, None]
    scores = scores.view(batch, hkv, group, s["max_new"], -1)
    scores = scores.masked_fill_(~keep[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    p = scores.sub_(top).exp_()
    out = p.view(batch, hkv, group * s["max_new"], -1) @ cached("v")
    out = out / p.sum(-1).view(batch, hkv, -1, 1).clamp_min(1e-38)
    out = out.view(batch, hkv, group, s["max_new"], hd).permute(0, 3, 1, 2, 4).reshape(batch, s["max_new"], hq * hd)
    seq = torch.searchsorted(cu[1:], torch.arange(total, device=table.device), right=True)
    return out[seq, torch.arange(total, device=table.device) - cu[seq]].to(torch.bfloat16)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from fastembed_b200 import ops
        if op == "norm":
            q, scale = ops.add_rmsnorm_e4m3(state["y"], state["h"], state["w"], EPS)
            return state["h"], q, scale
        if op == "quant":
            return ops.quantize_rows_e4m3(state["x"])
        if op == "linear":
            return ops.linear_e4m3(state["x"], state["xs"], state["w"], state["ws"], state["bias"], state["residual"],
                                   case["epilogue"], case["out"])
        cache = ops.KvCacheE4m3(state["k"], state["v"], state["ks"], state["vs"])
        if op == "append":
            ops.kv_cache_append_e4m3(state["qkv"], state["cu"], state["max_new"], state["past_lens"], state["table"],
                                     cache, case["q_heads"])
            return cache.k, cache.v, cache.k_scale, cache.v_scale
        return ops.attention_cache_e4m3(state["qkv"], state["cu"], state["max_new"], state["past_lens"], state["max_kv"],
                                        state["table"], cache, case["q_heads"], case["causal"])
    if op == "norm":
        return _plain_norm(state)
    if op == "quant":
        return _quantize(state["x"].float())
    if op == "linear":
        return _plain_linear(state)
    return _plain_append(state) if op == "append" else _plain_attend(state)


# ------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op in ("norm", "quant"):
        rows, dim = case["rows"], case["dim"]
        size = {"bf16": 2, "f32": 4}[case["y" if op == "norm" else "x"]]
        if op == "norm":  # y and h in, h and codes out
            return {"bytes": rows * dim * (size + 4 + 4 + 1) + 4 * rows + 4 * dim, "flops": 8 * rows * dim}
        return {"bytes": rows * dim * (size + 1) + 4 * rows, "flops": 3 * rows * dim}
    if op == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        cols = n // 2 if case["epilogue"] in ("swiglu", "geglu") else n
        out = m * cols * (2 if case["out"] == "bf16" else 4)
        extra = 4 * n if case["epilogue"].startswith("bias") else 0
        extra += 4 * m * n if case["epilogue"] == "bias_residual" else 0
        return {"bytes": m * k + n * k + 4 * (m + n) + out + extra, "flops": 2 * m * n * k}
    new, past = _lengths(case)
    row = case["kv_heads"] * case["hd"]
    page = case["page"]
    if op == "append":
        pages = sum((p + n - 1) // page - p // page + 1 for n, p in zip(new, past))
        return {"bytes": sum(new) * 2 * row * 3 + pages * case["kv_heads"] * 16, "flops": 2 * sum(new) * 2 * row}
    pages = sum(-(-(n + p) // page) for n, p in zip(new, past))
    if case["causal"]:
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    else:
        pairs = sum(n * (n + p) for n, p in zip(new, past))
    tokens = sum(n + p for n, p in zip(new, past))
    q = sum(new) * case["q_heads"] * case["hd"]
    return {"bytes": 4 * q + 2 * row * tokens + pages * case["kv_heads"] * 8, "flops": 4 * case["q_heads"] * case["hd"] * pairs}


# ------------------------------------------------------------------------ exact
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = s["h"].double() + s["y"].double()
        n = s["w"].double() * h / (h.pow(2).sum(-1, keepdim=True) / case["dim"] + EPS).sqrt()
        scale = n.abs().max(-1).values / E4M3_MAX
        return h, n / scale.unsqueeze(-1), scale
    if op == "quant":
        x = s["x"].double()
        scale = x.abs().max(-1).values / E4M3_MAX
        return x / scale.unsqueeze(-1), scale
    if op == "linear":
        # sum over the codes first, scales last
        z = torch.nn.functional.linear(s["x"].double(), s["w"].double()) * torch.outer(s["xs"].double(), s["ws"].double())
        if s["bias"] is not None:
            z += s["bias"].double()
        epi = case["epilogue"]
        if s["residual"] is not None:
            z += s["residual"].double()
        if epi in ("swiglu", "geglu"):
            blocks = z.split(32, dim=1)
            gate, value = torch.cat(blocks[0::2], 1), torch.cat(blocks[1::2], 1)
            z = (torch.sigmoid(gate) * gate if epi == "swiglu" else torch.nn.functional.gelu(gate, approximate="tanh")) * value
        elif epi == "bias_gelu":
            z = torch.nn.functional.gelu(z, approximate="tanh")
        elif epi == "bias_relu":
            z = torch.relu(z)
        elif epi == "bias_swish":
            z = torch.sigmoid(z) * z
        return z
    hq, hkv, hd, page = case["q_heads"], case["kv_heads"], case["hd"], case["page"]
    x = s["qkv"].view(-1, hq + 2 * hkv, hd)
    if op == "append":
        if max(s["new"]) * case["batch"] > 200_000:
            return None
        pools, scales = [], []
        for i, name in enumerate("kv"):
            values, scale = s[name].double(), s[name + "s"].double().clone()
            t0 = 0
            for b, (n, p) in enumerate(zip(s["new"], s["past"])):
                rows = x[t0:t0 + n, hq + i * hkv:hq + (i + 1) * hkv].double()
                t0 += n
                pages = s["table"][b].tolist()
                for ordinal in range(p // page, (p + n - 1) // page + 1):
                    lo, hi = max(p, ordinal * page), min(p + n, (ordinal + 1) * page)
                    block = rows[lo - p:hi - p].transpose(0, 1)
                    used = lo - ordinal * page
                    at = pages[ordinal]
                    m, e = torch.frexp(block.abs().amax((-1, -2)) / E4M3_MAX)  # 2^ceil(log2 .)
                    need = torch.where(m == 0.5, 2.0 ** (e - 1.0), 2.0 ** e.double())
                    if used:
                        grown = torch.maximum(need, scale[at])
                        values[at, :, :used] *= (scale[at] / grown)[:, None, None]
                        need = grown
                    values[at, :, used:used + hi - lo] = block / need[:, None, None]
                    scale[at] = need
            pools.append(values)
            scales.append(scale)
        return pools[0], pools[1], scales[0], scales[1]
    out = torch.empty(x.shape[0], hq * hd, dtype=torch.float64, device=x.device)
    t0 = 0
    for b, (n, p) in enumerate(zip(s["new"], s["past"])):
        at = s["table"][b, : -(-(n + p) // page)].long()
        keep = torch.ones(n, n + p, dtype=torch.bool, device=x.device)
        if case["causal"]:
            keep = keep.tril(p)
        for head in range(hkv):
            k, v = ((s[name].view(torch.uint8)[at, head].view(F8).double() * s[name + "s"][at, head].double()[:, None, None])
                    .reshape(-1, hd)[: n + p] for name in "kv")
            q = x[t0:t0 + n, head * (hq // hkv):(head + 1) * (hq // hkv)].double().transpose(0, 1)
            a = torch.softmax((q @ k.T / math.sqrt(hd)).masked_fill(~keep, -math.inf), -1) @ v
            out.view(-1, hq, hd)[t0:t0 + n, head * (hq // hkv):(head + 1) * (hq // hkv)] = a.transpose(0, 1)
        t0 += n
    return out
