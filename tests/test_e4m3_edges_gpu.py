"""The 8-bit operators at the edges of their contracts, against their plain 64-bit forms: codes that lie on a
border, value scales of any size, pages that are not there, offsets that run backwards."""
import math

import pytest
import torch

from tests import e4m3_ref as ref
from tests.e4m3_ref import F8, Batch

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------ codes are those of v / scale
def _divided(v):
    """(codes, scales) of fp32 rows by the formula as it is written: scale = max / 448, v / scale rounded
    to fp32, then to e4m3.  (448 as a tensor: torch multiplies by the reciprocal of a plain number.)"""
    top = v.abs().amax(-1).clamp_min(2.0 ** -110)
    s = top / torch.full_like(top, 448.0)
    return (v / s[:, None]).to(F8), s


def _same(got, want):
    assert torch.equal(got[1], want[1])
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8))


def _bf16_pairs(dev):
    """For each of the 128 mantissas of a row's maximum, in [1, 2): every bf16 of both signs from 2^-13 (below
    half of the smallest code) up to that maximum.  Powers of two change nothing about v / scale."""
    bits = torch.arange((127 - 13) << 7, 128 << 7, dtype=torch.int32, device=dev).to(torch.int16)
    v = bits.view(torch.bfloat16)  # 14 binades of 128
    rows = []
    for i in range(128):
        top = 1.0 + i / 128
        row = v.clone()
        row[v.float() > top] = top
        row[1::2] *= -1
        rows.append(row)
        rows.append(-row)
    return torch.stack(rows)  # [256, 1792]


@pytest.mark.parametrize("width", [64, 256, 512, 1792, 1791, 7])
def test_bf16_codes_are_the_division(cuda_dev, width):
    """Codes of bf16 rows equal those of x / scale bit for bit, values on a border between two codes
    included: all pairs of a row's maximum and an element, through every kernel that a width selects."""
    from fastembed_b200 import ops
    full = _bf16_pairs(cuda_dev)
    top = full.abs().amax(-1, keepdim=True)
    parts = []
    for c0 in range(0, full.shape[1], width - 1):
        cut = full[:, c0:c0 + width - 1]
        cut = torch.nn.functional.pad(cut, (0, width - 1 - cut.shape[1]))
        parts.append(torch.cat([top, cut], 1))
    x = torch.cat(parts).contiguous()
    x[1::2, -1] = -0.0
    _same(ops.quantize_rows_e4m3(x), _divided(x.float()))
    for r0 in range(0, min(x.shape[0], 700), 100):  # few rows: a block each
        _same(ops.quantize_rows_e4m3(x[r0:r0 + 100].contiguous()), _divided(x[r0:r0 + 100].float()))
    _same(ops.quantize_rows_e4m3(x.float()), _divided(x.float()))


def test_tiny_and_huge_codes_are_the_division(cuda_dev):
    """Rows below the smallest maximum, subnormal elements, rows up to the largest bf16 and fp32."""
    from fastembed_b200 import ops
    every = torch.arange(1, 0x7f80, dtype=torch.int32, device=cuda_dev).to(torch.int16).view(torch.bfloat16)
    small = every[every.float() < 2.0 ** -108]
    for top in (2.0 ** -120, 1.5 * 2.0 ** -111, 2.0 ** -110, 1.2 * 2.0 ** -110, 1.9 * 2.0 ** -109):
        row = small[small.float() <= top]
        row = torch.nn.functional.pad(row, (0, -row.numel() % 1024)).view(-1, 1024).clone()
        row[:, 0] = top
        row[:, 1::2] *= -1
        _same(ops.quantize_rows_e4m3(row), _divided(row.float()))
        _same(ops.quantize_rows_e4m3(row.float()), _divided(row.float()))
    big = every[every.float() > 2.0 ** 110]
    for top in (float(every[-1]), 1.5 * 2.0 ** 126):
        row = big[big.float() <= top]
        row = torch.nn.functional.pad(row, (0, -row.numel() % 512)).view(-1, 512).clone()
        row[:, 0] = top
        _same(ops.quantize_rows_e4m3(row), _divided(row.float()))
    wide = torch.tensor([[3.4028234663852886e38, 1e38, -3.3e38, 0.0, 1e-38, 2.5e37, 1.0, -7e36]], device=cuda_dev)
    _same(ops.quantize_rows_e4m3(wide), _divided(wide))


@pytest.mark.parametrize("rows,dim", [(300, 1024), (40, 1024), (900, 256), (3, 8192), (2, 16392), (500, 999)])
def test_f32_codes_are_the_division(cuda_dev, rows, dim):
    """fp32 rows, most of their elements within a few steps of a border between two codes."""
    from fastembed_b200 import ops
    g = torch.Generator(device=cuda_dev).manual_seed(rows + dim)
    top = 1.0 + torch.rand(rows, 1, device=cuda_dev, generator=g)
    s = top / 448
    codes = torch.randint(0, 126, (rows, dim), device=cuda_dev, generator=g, dtype=torch.int32).to(torch.uint8)
    a = codes.view(F8).float()
    b = (codes + 1).view(F8).float()
    x = (a + b) / 2 * s
    x = (x.view(torch.int32) + torch.randint(-3, 4, x.shape, device=cuda_dev, generator=g, dtype=torch.int32)).view(torch.float32)
    x = torch.minimum(x, top) * (torch.randint(0, 2, x.shape, device=cuda_dev, generator=g) * 2 - 1)
    x[:, 0] = top[:, 0]
    _same(ops.quantize_rows_e4m3(x.contiguous()), _divided(x))


@pytest.mark.parametrize("rows,dim", [(300, 1024), (40, 1024), (900, 256), (3, 8192), (2, 16392), (500, 1000), (30, 999)])
@pytest.mark.parametrize("ydt", [torch.float32, torch.bfloat16, None])
def test_norm_codes_are_the_division(cuda_dev, rows, dim, ydt):
    """Rows of +-1: their root mean square is 1 exactly and what is quantised is +-w, here bf16 numbers
    whose quotients fall on borders between codes.  (A zero added through y changes nothing.)"""
    from fastembed_b200 import ops
    g = torch.Generator(device=cuda_dev).manual_seed(dim)
    w = (torch.randn(dim, device=cuda_dev, generator=g) * 0.3).to(torch.bfloat16).float()
    w[: dim // 2] = w[0].abs() * torch.randint(1, 120, (dim // 2,), device=cuda_dev, generator=g) / 64
    h = (torch.randint(0, 2, (rows, dim), device=cuda_dev, generator=g) * 2 - 1).float()
    y = None if ydt is None else torch.zeros(rows, dim, dtype=ydt, device=cuda_dev)
    for top in (1.0, 1.0546875, 1.3125, 1.75, 1.9921875):
        w[1] = top * 4
        _same(ops.add_rmsnorm_e4m3(y, h.clone(), w, 0.0), _divided(h * w))


def test_norm_of_a_row_whose_sum_of_squares_overflows(cuda_dev):
    """Squares past fp32: the row's norm is infinite and its codes are 0, at the smallest scale; the next
    row does not notice."""
    from fastembed_b200 import ops
    for dim in (1024, 1001):
        h = torch.ones(3, dim, device=cuda_dev)
        h[1] = 1e20
        w = torch.ones(dim, device=cuda_dev)
        q, s = ops.add_rmsnorm_e4m3(None, h, w, 1e-6)
        assert torch.all(q[1].float() == 0) and float(s[1]) == float(torch.tensor(2.0 ** -110) / torch.tensor(448.0))
        assert torch.all(q[0].float() == 448) and torch.all(q[2].float() == 448)
        h[1] = 1e-30
        q, s = ops.add_rmsnorm_e4m3(None, h, w, 0.0)  # without eps, squares that vanish leave nothing to divide by
        assert torch.isnan(q[1].float()).all() and torch.all(q[0].float() == 448) and torch.all(q[2].float() == 448)


# ------------------------------------------------------------ value scales of pages
def _strict(b, cache, want, mag, dot, causal, scale):
    """How far attention may be off when nothing is granted for pages of zero values or for the size of the
    scales.  As ref.attention_bound, with these changes: a page whose value scale is 0 adds nothing to the
    row's largest weight as it meets the codes; the exponents that carry a scale (logit + log2 sv, minus
    the reference, plus the reference's difference from the sum's own) are numbers of at most E = |log2 sv|
    + 3 |logit| + 20 in base 2, and eight roundings of half a step each on them pass on ln 2 * 8 * 2^-24 E;
    results below 2^-126 keep bf16's absolute step of 2^-133, half of it and half of fp32's 2^-149 thrice."""
    out = torch.zeros_like(want)
    q = b.qkv.view(b.qkv.shape[0], -1, b.hd)[:, :b.q_heads].double()
    group, t0, floor = b.q_heads // b.kv_heads, 0, torch.zeros_like(want).view(-1, b.q_heads, b.hd)
    e_max = torch.where(cache.v_scale > 0, cache.v_scale.double().log2().abs(), 0.0).max()
    for s, (n, p) in enumerate(zip(b.new, b.past)):
        at = b.table[s, : -(-(n + p) // b.page)].long()
        k = ref.values(cache.k.view(torch.uint8)[at].view(F8), cache.k_scale[at]).transpose(0, 1).reshape(b.kv_heads, -1, b.hd)
        k = k[:, :n + p].repeat_interleave(group, 0)
        sv = cache.v_scale[at].double().t().repeat_interleave(b.page, 1)[:, :n + p].repeat_interleave(group, 0)
        codes = cache.v.view(torch.uint8)[at].view(F8).float().double().abs().transpose(0, 1).reshape(b.kv_heads, -1, b.hd)
        codes = codes[:, :n + p].repeat_interleave(group, 0)
        keep = torch.ones(n, n + p, dtype=torch.bool, device=k.device)
        if causal:
            keep = keep.tril(p)
        logits = (q[t0:t0 + n].transpose(0, 1) @ k.transpose(1, 2) * scale).masked_fill(~keep, -math.inf)
        w = torch.softmax(logits, -1) * sv[:, None]
        codes = torch.where(sv[..., None] > 0, codes, 0.0)
        floor[t0:t0 + n] = (w.amax(-1, keepdim=True) * (keep.double() @ codes)).transpose(0, 1)
        t0 += n
    ds = (b.hd + 8) * 2.0 ** -23 * dot + math.log(2) * 8 * 2.0 ** -24 * (e_max + 3 * 1.45 * dot + 20)
    rel = 2.0 ** -11 + 2.0 ** -19 + 2.0 * ds
    return 2.0 ** -8 * want.abs() + rel * mag * 1.01 + 2.0 ** -32 * floor.reshape(want.shape) + 2.0 ** -133


FORMS = [([1, 1], None), ([1, 1], 1 << 20), ([5, 2], None), ([5, 2], 1 << 20), ([80, 3], None), ([300, 90], 1 << 20)]


def _check(b, ops, cache, bound=None, causal=True, scale=None):
    scale = b.hd ** -0.5 if scale is None else scale
    out = ops.attention_cache_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, bound or b.max_kv, b.table, cache, b.q_heads, causal, scale)
    want, mag, dot, _ = ref.attention(cache, b.qkv, b.new, b.past, b.table, b.q_heads, causal, scale)
    err, most = (out.double() - want).abs(), _strict(b, cache, want, mag, dot, causal, scale)
    assert torch.all(err <= most), (float((err / most).max()), float(out.double().abs().max()), float(want.abs().max()))
    ops.device_status(0)
    return out


def _zero_pages(b, cache, seq, ordinals):
    for o in ordinals:
        at = int(b.table[seq, o])
        cache.v_scale[at] = 0
        cache.v.view(torch.uint8)[at] = 0


@pytest.mark.parametrize("new,bound", FORMS)
@pytest.mark.parametrize("hd,heads", [(64, (4, 4)), (128, (4, 2)), (256, (3, 1))])
def test_zero_value_pages_leave_the_others_their_weights(cuda_dev, new, bound, hd, heads):
    """A page of zero values beside pages of small ones (2^-40, 2^-100) and of ordinary ones, at equal logits and
    with the zero page's tokens far ahead: its weight counts in the sum and takes nothing from the others'."""
    from fastembed_b200 import ops
    b = Batch(new, [500, 333], 16, *heads, hd, cuda_dev, seed=hd)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    keys = cache.k.view(torch.uint8).clone()
    for zero in ([0], [3, 4, 9], [8, 12, 13, 14, 15, 16, 17, 18, 19, 20]):
        for exponent in (-40, -100, -9):
            cache.k.view(torch.uint8).copy_(keys)
            cache.v.copy_(torch.where(cache.v.float().abs() < 2.0, 2.0, cache.v.float()).to(F8))
            cache.v_scale.fill_(2.0 ** exponent)
            for s in range(2):
                _zero_pages(b, cache, s, zero)
            _check(b, ops, cache, bound, scale=0.0)  # equal logits
            _check(b, ops, cache, bound)
            # the first zero page's keys along the query of token 0: some 25 to 35 in base 2 above the rest
            q0 = b.qkv.view(b.qkv.shape[0], -1, hd)[0, : b.q_heads].float()
            at = int(b.table[0, zero[0]])
            for h in range(b.kv_heads):
                unit = q0[h * (b.q_heads // b.kv_heads)]
                cache.k[at, h] = (unit / unit.abs().max() * 400).to(F8)
            cache.k_scale[at] = 2.0 ** -6
            _check(b, ops, cache, bound)


@pytest.mark.parametrize("new,bound", FORMS)
def test_only_zero_value_pages(cuda_dev, new, bound):
    """Nothing but pages of zero values: zeros, causal and not.  Then one page of ordinary values at the end."""
    from fastembed_b200 import ops
    b = Batch(new, [300, 150], 32, 4, 2, 128, cuda_dev)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    scales, codes = cache.v_scale.clone(), cache.v.view(torch.uint8).clone()
    cache.v_scale.zero_()
    cache.v.view(torch.uint8).zero_()
    for causal in (True, False):
        assert torch.all(_check(b, ops, cache, bound, causal) == 0)
    at = int(b.table[0, 300 // 32])
    cache.v_scale[at] = scales[at]
    cache.v.view(torch.uint8)[at] = codes[at]
    _check(b, ops, cache, bound)


@pytest.mark.parametrize("new,bound", FORMS)
@pytest.mark.parametrize("hd,heads", [(64, (4, 4)), (128, (4, 2)), (256, (3, 1))])
def test_value_scales_of_any_size(cuda_dev, new, bound, hd, heads):
    """Scales from 2^-130 to 2^117, one size in all pages and sizes far apart in either order, at equal logits too: neither
    the sum nor a row's weights overflow or vanish."""
    from fastembed_b200 import ops
    b = Batch(new, [500, 333], 16, *heads, hd, cuda_dev, seed=hd + 1)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    for exps in ([-113], [-122], [-130], [117], [-80, 100], [100, -80], [-126, 0, 0, 110], [3, 2, 1, 0, -1, -2, -50, -120]):
        e = torch.zeros(b.pages, device=cuda_dev, dtype=torch.float64)
        for s in range(2):
            at = b.table[s].long()
            count = -(-(b.new[s] + b.past[s]) // 16)
            e[at[:count]] = torch.tensor(exps, device=cuda_dev, dtype=torch.float64).repeat(count)[:count]
        factor = 1.37 if len(exps) % 2 == 0 else 1.0  # not only powers of two
        cache.v_scale.copy_((2.0 ** e * factor).float()[:, None].expand(-1, b.kv_heads))
        _check(b, ops, cache, bound, scale=0.0)
        _check(b, ops, cache, bound)


# ------------------------------------------------------------ pages that are not there
@pytest.mark.parametrize("new,bound", [([3, 2], None), ([3, 2], 1 << 20), ([60, 40], None), ([90, 200], 1 << 20)])
@pytest.mark.parametrize("hd,heads", [(64, (4, 4)), (128, (4, 2)), (256, (3, 1))])
def test_non_finite_queries_over_absent_pages(cuda_dev, new, bound, hd, heads):
    """A query with a NaN or an infinity that sees no token (its pages are all out of the pool) is zero like any other;
    one that sees some page is NaN; finite rows see what is there."""
    from fastembed_b200 import ops
    from fastembed_b200.capi import FeError
    b = Batch(new, [200, 300], 32, *heads, hd, cuda_dev)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    q = b.qkv.view(-1, heads[0] + 2 * heads[1], hd)
    T, a = sum(new), new[0]
    run = lambda t: ops.attention_cache_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, bound or b.max_kv, t, cache,
                                             heads[0]).view(T, heads[0], hd)
    gone, part = b.table.clone(), b.table.clone()
    gone[0] = -5
    part[0, ::2] = b.pages
    finite = {"gone": run(gone).clone(), "part": run(part).clone()}
    with pytest.raises(FeError):
        ops.device_status(0)
    bad = torch.zeros(T, heads[0], dtype=torch.bool, device=cuda_dev)
    for t, h, x in ((0, 0, math.nan), (1, 2, math.inf), (2, 1, -math.inf), (a, 0, math.nan), (a + 1, 2, math.inf)):
        q[t, h, 3] = x
        bad[t, h] = True
    got = run(gone).clone()
    assert torch.all(got[:a] == 0)
    assert torch.isnan(got[a:][bad[a:]]).all() and torch.equal(got[a:][~bad[a:]], finite["gone"][a:][~bad[a:]])
    got = run(part).clone()
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], finite["part"][~bad])
    with pytest.raises(FeError):
        ops.device_status(0)
    ops.device_status(0)


def test_finite_queries_over_some_absent_pages(cuda_dev):
    """What is left of a sequence when pages are missing: the softmax over the tokens of the others."""
    from fastembed_b200 import ops
    from fastembed_b200.capi import FeError
    for new, bound in (([1, 1], 1 << 20), ([4, 2], 400), ([70, 40], 400), ([130, 40], 1 << 20)):
        b = Batch(new, [256, 128], 16, 4, 2, 128, cuda_dev, seed=3)
        cache = b.random_cache(ops)
        ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
        table = b.table.clone()
        gone = [1, 2, 6]
        for o in gone:
            table[:, o] = -1
        out = ops.attention_cache_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, bound, table, cache, 4)
        with pytest.raises(FeError):
            ops.device_status(0)
        # the same tokens without those pages: positions move up by their 48 tokens
        left = [o for o in range(b.table.shape[1]) if o not in gone]
        short = b.table[:, left].contiguous()
        past = [p - 16 * len(gone) for p in b.past]
        want, mag, dot, floor = ref.attention(cache, b.qkv, b.new, past, short, 4, True, 128 ** -0.5)
        assert torch.all((out.double() - want).abs() <= ref.attention_bound(want, mag, dot, floor, 128))


# ------------------------------------------------------------ gated linear layers have no bias
@pytest.mark.parametrize("m,n,k", [(3, 256, 64), (130, 512, 256), (700, 1024, 256), (2000, 2304, 128)])
@pytest.mark.parametrize("epi", ["swiglu", "geglu"])
def test_gated_linear_takes_no_bias(cuda_dev, m, n, k, epi):
    """The gated epilogues and "none" are without a bias, as in the bf16 linear layer: one that is passed all the same is
    not read."""
    from fastembed_b200 import ops
    g = torch.Generator(device=cuda_dev).manual_seed(m)
    x, xs = ops.quantize_rows_e4m3(torch.randn(m, k, device=cuda_dev, generator=g))
    w, ws = ops.quantize_rows_e4m3(torch.randn(n, k, device=cuda_dev, generator=g))
    bias = torch.randn(n, device=cuda_dev, generator=g)
    for e in (epi, "none"):
        assert torch.equal(ops.linear_e4m3(x, xs, w, ws, bias, None, e), ops.linear_e4m3(x, xs, w, ws, None, None, e))
    ops.device_status(0)


# ------------------------------------------------------------ offsets that run backwards
@pytest.mark.parametrize("new,bound", [([4, 3, 2], 300), ([90, 40, 20], 300), ([90, 40, 20], 1 << 20)])
def test_offsets_that_run_backwards_are_reported(cuda_dev, new, bound):
    """A sequence whose end lies before its start does not fit: left out by both calls, and reported.  (Equal offsets are an
    empty sequence, which is nothing to report.)"""
    from fastembed_b200 import ops
    from fastembed_b200.capi import FeError
    b = Batch(new, [40, 33, 50], 32, 8, 2, 128, cuda_dev)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, 8)
    T = sum(new)
    run = lambda cu, past: ops.attention_cache_e4m3(b.qkv, cu, b.max_new, past, bound, b.table, cache, 8,
                                                    out=torch.full((T, 8 * 128), 9.0, dtype=torch.bfloat16, device=cuda_dev))
    want = run(b.cu, b.past_lens)
    ops.device_status(0)
    state = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_dev)
    a = new[0]
    for back in ([0, a, a - 2, a - 2], [0, a, -2147483647, -2147483647]):
        got = run(i32(back), b.past_lens)
        with pytest.raises(FeError):
            ops.device_status(0)
        assert torch.equal(got[:a], want[:a]) and torch.all(got[a:] == 9.0)
        b.qkv[a:].neg_()
        ops.kv_cache_append_e4m3(b.qkv, i32(back), b.max_new, b.past_lens, b.table, cache, 8)
        b.qkv[a:].neg_()
        with pytest.raises(FeError):
            ops.device_status(0)
        for was, now in zip(state, (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)):
            assert torch.equal(was, now)
    got = run(i32([0, a, a, a]), i32([40, -1, 50]))  # empty ones, whatever else stands there
    assert torch.equal(got[:a], want[:a]) and torch.all(got[a:] == 9.0)
    ops.device_status(0)


# ------------------------------------------------------------ queries of any size
@pytest.mark.parametrize("hd,heads", [(64, (4, 4)), (128, (4, 2)), (256, (3, 1))])
@pytest.mark.parametrize("new,bound", [([3, 1], None), ([3, 1], 1 << 20), ([90, 40], None), ([200, 40], 1 << 20)])
def test_queries_of_any_size(cuda_dev, hd, heads, new, bound):
    """Queries from 1e-38 to 1e36 with a softmax scale that brings their logits back to ordinary size."""
    from fastembed_b200 import ops
    b = Batch(new, [150, 333], 32, *heads, hd, cuda_dev, seed=hd + 5)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    x = b.qkv.view(sum(new), -1, hd)
    q1 = x[:, :heads[0]].clone()
    for size in (1e-38, 1e-36, 1e-34, 1e-30, 1e-25, 1.0, 1e20, 1e36):
        x[:, :heads[0]] = (q1.double() * size).to(torch.bfloat16)
        scale = hd ** -0.5 / size
        if scale * math.log2(math.e) > 3.4e38:
            x[:, :heads[0]], scale = x[:, :heads[0]] * 64, scale / 64
        out = ops.attention_cache_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, bound or b.max_kv, b.table, cache, heads[0], True, scale)
        want, mag, dot, floor = ref.attention(cache, b.qkv, b.new, b.past, b.table, heads[0], True, scale)
        # elements are off by 2^-16 of the row's largest, or 2^-135: times the largest sum of |k|, in numerator and
        # denominator; the softmax scale in base 2 by two roundings
        top = x[:, :heads[0]].abs().amax(-1).double()
        kv = torch.cat([ref.values(cache.k.view(torch.uint8)[b.table[s, : -(-(n + p) // 32)].long()].view(F8),
                                   cache.k_scale[b.table[s, : -(-(n + p) // 32)].long()]).abs().sum(-1).amax(-1)
                        for s, (n, p) in enumerate(zip(b.new, b.past))]).amax(0)
        off = torch.maximum(2.0 ** -16 * top, torch.tensor(2.0 ** -135, device=cuda_dev, dtype=torch.float64)) * abs(scale)
        off = off * kv.repeat_interleave(heads[0] // heads[1])[None] + 2.0 ** -23 * dot.view(sum(new), heads[0], hd)[..., 0]
        bound_ = ref.attention_bound(want, mag, dot, floor, hd) + (torch.expm1(2 * off)[..., None] * mag.view(-1, heads[0], hd)).reshape(
            want.shape)
        err = (out.double() - want).abs()
        assert torch.all(err <= bound_), (size, float((err / bound_).max()))
        ops.device_status(0)
