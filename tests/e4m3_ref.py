"""Plain 64-bit forms of the 8-bit (e4m3) operators, and batches to run them on."""
import math

import numpy as np
import torch

F8 = torch.float8_e4m3fn
TINY = 2.0 ** -110


def values(codes, scale):
    """codes * scale in 64 bits, the scale spread over the codes' trailing dimensions."""
    s = scale.double()
    return codes.to(torch.float32).double() * s.view(s.shape + (1,) * (codes.dim() - s.dim()))


def row_scale(v):
    """max over the finite values of each row / 448 (v in 64 bits)."""
    a = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v))
    return a.amax(-1).clamp_min(TINY) / 448.0


def rmsnorm(h, w, eps, one_plus):
    g = w.double() + (1.0 if one_plus else 0.0)
    return h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + eps) * g


def linear(x, xs, w, ws, bias, residual, epilogue):
    """(z, absolute sum): the epilogue's result and sum_k |x w| of each output (after the scales)."""
    xv, wv = values(x, xs), values(w, ws)
    z, mag = xv @ wv.T, xv.abs() @ wv.abs().T
    if bias is not None and epilogue not in ("none", "swiglu", "geglu"):
        z = z + bias.double()
    act = {"bias_gelu": lambda t: 0.5 * t * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3))),
           "bias_relu": lambda t: t.clamp_min(0), "bias_swish": lambda t: t * torch.sigmoid(t)}
    if epilogue in act:
        return act[epilogue](z), z, mag
    if epilogue == "bias_residual":
        return z + residual.double(), z, mag
    if epilogue in ("swiglu", "geglu"):
        zz, mm = z.view(z.shape[0], -1, 2, 32), mag.view(z.shape[0], -1, 2, 32)
        gate, up = zz[:, :, 0], zz[:, :, 1]
        f = act["bias_swish"](gate) if epilogue == "swiglu" else act["bias_gelu"](gate)
        # |d(f u)| <= 1.13 |u| dg + |f| du, returned as the magnitude that the accumulation error multiplies
        flat = lambda t: t.reshape(z.shape[0], -1)
        return flat(f * up), flat(f * up), flat(1.13 * up.abs() * mm[:, :, 0] + f.abs() * mm[:, :, 1])
    return z, z, mag


def pow2_scale(amax):
    """Smallest 2^e >= amax / 448, e >= -80; 0 for 0."""
    m, e = torch.frexp(amax.double() / 448.0)
    e = torch.where(m == 0.5, e - 1, e).clamp_min(-80)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(m), e), torch.zeros_like(m))


def append(cache, qkv, new, past, table, q_heads):
    """The cache after the append: (k codes as uint8, v, k scales, v scales), one token block at a time."""
    kc, vc = cache.k.view(torch.uint8).clone(), cache.v.view(torch.uint8).clone()
    ks, vs = cache.k_scale.double().clone(), cache.v_scale.double().clone()
    pages, hkv, page, hd = kc.shape
    x = qkv.view(qkv.shape[0], -1, hd).double()
    t0 = 0
    for b, (n, p) in enumerate(zip(new, past)):
        k, v = x[t0:t0 + n, q_heads:q_heads + hkv], x[t0:t0 + n, q_heads + hkv:]
        t0 += n
        if n == 0:
            continue
        bad = ~(torch.isfinite(k).all(-1) & torch.isfinite(v).all(-1))  # [n, hkv]
        k = torch.where(bad[..., None], torch.zeros_like(k), k)
        v = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
        for o in range(p // page, (p + n - 1) // page + 1):
            at, lo, hi = int(table[b, o]), max(p, o * page), min(p + n, (o + 1) * page)
            used = lo - o * page
            for codes, scales, src, nan in ((kc, ks, k, bad), (vc, vs, v, None)):
                blk = src[lo - p:hi - p].transpose(0, 1)  # [hkv, m, hd]
                need = pow2_scale(blk.abs().amax((-1, -2)))
                if used:
                    old = scales[at].clone()
                    need = torch.maximum(need, old)
                    ratio = torch.where(need > 0, old / need.clamp_min(1e-300), torch.zeros_like(need))
                    was = codes[at, :, :used].view(F8).float().double() * ratio[:, None, None]
                    grown = need > old
                    codes[at, :, :used] = torch.where(grown[:, None, None], was.float().to(F8).view(torch.uint8),
                                                      codes[at, :, :used])
                inv = torch.where(need > 0, 1.0 / need.clamp_min(1e-300), torch.zeros_like(need))
                c = (blk * inv[:, None, None]).float().to(F8).view(torch.uint8)
                if nan is not None:
                    m = nan[lo - p:hi - p].transpose(0, 1)
                    c = torch.where(m[..., None], torch.full_like(c, 0x7F), c)
                codes[at, :, used:used + hi - lo] = c
                scales[at] = need
    return kc, vc, ks, vs


def attention(cache, qkv, new, past, table, q_heads, causal, scale):
    """(out, sum_j p |v|, largest scale * sum_d |q k|, floor) per (token, head) in 64 bits; floor: the
    row's largest weight as it meets the codes (p times the page's value scale) times sum_j |codes|."""
    pages, hkv, page, hd = cache.k.shape
    group = q_heads // hkv
    x = qkv.view(qkv.shape[0], -1, hd)[:, :q_heads].double()
    T = sum(new)
    out = torch.zeros(T, q_heads, hd, dtype=torch.float64, device=qkv.device)
    mag, floor = torch.zeros_like(out), torch.zeros_like(out)
    dot = torch.zeros(T, q_heads, dtype=torch.float64, device=qkv.device)
    t0 = 0
    for b, (n, p) in enumerate(zip(new, past)):
        if n == 0:
            continue
        at = table[b, : -(-(n + p) // page)].long()
        k = values(cache.k.view(torch.uint8)[at].view(F8), cache.k_scale[at]).transpose(0, 1).reshape(hkv, -1, hd)[:, :n + p]
        v = values(cache.v.view(torch.uint8)[at].view(F8), cache.v_scale[at]).transpose(0, 1).reshape(hkv, -1, hd)[:, :n + p]
        k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
        sv = cache.v_scale[at].double().t().repeat_interleave(page, 1)[:, :n + p].repeat_interleave(group, 0)
        codes = torch.where(sv[..., None] > 0, v.abs() / sv.clamp_min(1e-300)[..., None], torch.zeros_like(v))
        q = x[t0:t0 + n].transpose(0, 1)
        keep = torch.ones(n, n + p, dtype=torch.bool, device=q.device)
        if causal:
            keep = keep.tril(p)
        s = (q @ k.transpose(1, 2) * scale).masked_fill(~keep, -math.inf)
        pr = torch.softmax(s, -1)
        out[t0:t0 + n] = (pr @ v).transpose(0, 1)
        mag[t0:t0 + n] = (pr @ v.abs()).transpose(0, 1)
        floor[t0:t0 + n] = ((pr * torch.where(sv > 0, sv, torch.ones_like(sv))[:, None]).amax(-1, keepdim=True) *
                            (keep.double() @ codes)).transpose(0, 1)
        dot[t0:t0 + n] = ((q.abs() @ k.abs().transpose(1, 2)).amax(-1) * abs(scale)).transpose(0, 1)
        t0 += n
    return tuple(t.reshape(T, -1) for t in (out, mag, dot.repeat_interleave(hd, -1), floor))


def attention_bound(out, mag, dot, floor, hd):
    """How far the bf16 output of an fp32 kernel may be from `out`: half a bf16 step of the
    result; weights off by 2^-11 (f16) + 2^-20 (exponential, running sums of them) and by what
    the logits are off, hd + 8 fp32 operations of half a step each on sum |q k| (counted whole
    steps: the tensor cores may truncate), in numerator and denominator alike.  f16 has no step
    below 2^-24: a weight is held at 2^7 or more where the row's largest is, so it is off by at most
    half of 2^-24 / 2^7 = 2^-32 of the largest, whatever its own size (a row whose largest weights
    fall on a page of zero values shows it)."""
    ds = (hd + 8) * 2.0 ** -23 * dot
    return 2.0 ** -8 * out.abs() + (2.0 ** -11 + 2.0 ** -19 + 2.0 * ds) * mag * 1.01 + 2.0 ** -32 * floor + 1e-30


class Batch:
    """A packed batch with its page table: every sequence has pages of its own, in random order."""

    def __init__(self, new, past, page, q_heads, kv_heads, hd, device, seed=0, spare=2, extra_rows=0):
        self.new, self.past, self.page, self.q_heads, self.kv_heads, self.hd = new, past, page, q_heads, kv_heads, hd
        self.g = torch.Generator(device=device).manual_seed(seed)
        T = sum(new) + extra_rows
        spread = torch.exp(0.3 * torch.randn(q_heads + 2 * kv_heads, hd, device=device, generator=self.g))
        self.qkv = (torch.randn(T, q_heads + 2 * kv_heads, hd, device=device, generator=self.g) * spread).to(
            torch.bfloat16).view(T, -1)
        need = [-(-(n + p) // page) for n, p in zip(new, past)]
        self.pages = sum(need) + spare
        width = max(need + [1]) + 1
        order = torch.randperm(self.pages, device=device, generator=self.g).tolist()
        table = np.zeros((len(new), width), np.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
        self.table = i32(table)
        self.cu = i32(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
        self.past_lens = i32(past)
        self.max_new, self.max_kv = max(new + [0]), max([n + p for n, p in zip(new, past)] + [0])

    def random_cache(self, ops):
        """A cache full of codes in every page (what earlier calls left there), scales 2^-9 .. 2^-6."""
        dev = self.qkv.device
        c = ops.kv_cache_e4m3(self.pages, self.page, self.kv_heads, self.hd, dev)
        for codes in (c.k, c.v):
            codes.copy_((torch.randn(codes.shape, device=dev, generator=self.g) * 80).clamp(-448, 448).to(F8))
        for s in (c.k_scale, c.v_scale):
            s.copy_(2.0 ** torch.randint(-9, -5, s.shape, device=dev, generator=self.g).float())
        return c
