"""The 8-bit operators on a B200, through the C ABI, against their plain 64-bit forms."""
import math

import pytest
import torch

from tests import e4m3_ref as ref
from tests.e4m3_ref import F8, Batch

pytestmark = pytest.mark.gpu


def _check_codes(q, scale, v, exact_scale):
    """Row scales within four fp32 roundings; codes within half an e4m3 step of v / scale (2^-4
    of it, 2^-10 where subnormal) plus 2^-20 of it for the fp32 arithmetic before."""
    assert torch.all((scale.double() - exact_scale).abs() <= 2.0 ** -22 * exact_scale)
    x = v / scale.double()[:, None]
    got = q.float().double()
    fin = torch.isfinite(v)
    assert torch.equal(torch.isnan(got), ~fin)
    err = (got - x).abs()[fin]
    a = x.abs()[fin]
    assert torch.all(err <= a * (2.0 ** -4 + 2.0 ** -20) + 2.0 ** -10)


# ------------------------------------------------------------ rows to e4m3
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 8), (3, 7), (5, 250), (2, 256), (7, 264), (33, 384), (200, 512), (9, 1000),
                                      (149, 1024), (1, 2048), (300, 2048), (5, 2056), (3, 4096), (2, 8192), (2, 16384),
                                      (2, 16392), (3, 5001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_rows(cuda_dev, rows, dim, dtype):
    from fastembed_b200 import ops
    g = torch.Generator(device=cuda_dev).manual_seed(rows * 31 + dim)
    x = torch.randn(rows, dim, device=cuda_dev, generator=g) * torch.exp(3 * torch.randn(rows, 1, device=cuda_dev, generator=g))
    x = x.to(dtype)
    q, s = ops.quantize_rows_e4m3(x)
    assert q.dtype == F8 and q.shape == x.shape
    _check_codes(q, s, x.double(), ref.row_scale(x.double()))


def test_quantize_rows_special_values(cuda_dev):
    """Zero rows, tiny and huge rows, infinities and NaN: the others of the row as without them."""
    from fastembed_b200 import ops
    g = torch.Generator(device=cuda_dev).manual_seed(5)
    for dim in (64, 63):
        x = torch.randn(9, dim, device=cuda_dev, generator=g)
        x[0] = 0
        x[1] *= 1e-38
        x[2] *= 1e37
        x[3, 5], x[3, 6], x[4, 0] = math.inf, -math.inf, math.nan
        x[5] = math.nan
        x[6] = torch.finfo(torch.float32).min
        q, s = ops.quantize_rows_e4m3(x)
        v = x.double()
        _check_codes(q, s, v, ref.row_scale(v))
        assert torch.all(q[0].float() == 0) and torch.all(q[6].float() == -448)


@pytest.mark.parametrize("rows,dim", [(1, 8), (1, 1024), (4, 100), (17, 768), (200, 1024), (1100, 1024), (6, 2048), (3, 4096),
                                      (2, 16400), (2, 12000)])
@pytest.mark.parametrize("ydt", [torch.float32, torch.bfloat16, None])
@pytest.mark.parametrize("one_plus", [False, True])
def test_add_rmsnorm(cuda_dev, rows, dim, ydt, one_plus):
    from fastembed_b200 import ops
    g = torch.Generator(device=cuda_dev).manual_seed(rows + dim)
    h = torch.randn(rows, dim, device=cuda_dev, generator=g) * 3
    w = 0.3 * torch.randn(dim, device=cuda_dev, generator=g) + (0.0 if one_plus else 1.0)
    y = None if ydt is None else torch.randn(rows, dim, device=cuda_dev, generator=g).to(ydt)
    want_h = h if y is None else h + y.float()  # one fp32 addition: bit for bit
    got_h = h.clone()
    q, s = ops.add_rmsnorm_e4m3(y, got_h, w, 1e-6, one_plus)
    assert torch.equal(got_h, want_h)
    # sums of squares: dim terms in fp32, at most (dim / 32 + 5) additions deep, all of one sign; then a
    # handful of roundings (root, division, two products): relative 2^-24 (dim / 32 + 16) of the normalised row
    v = ref.rmsnorm(want_h.double(), w, 1e-6, one_plus)
    exact = ref.row_scale(v)
    tol = 2.0 ** -24 * (dim / 32 + 16)
    assert torch.all((s.double() - exact).abs() <= tol * exact)
    x = v / s.double()[:, None]
    assert torch.all((q.float().double() - x).abs() <= x.abs() * (2.0 ** -4 + 2 * tol) + 2.0 ** -10)


def test_add_rmsnorm_poisoned_row_stays_alone(cuda_dev):
    from fastembed_b200 import ops
    for dim in (1024, 1001):
        h = torch.ones(4, dim, device=cuda_dev)
        h[1, 3], h[2, 0] = math.nan, math.inf
        w = torch.ones(dim, device=cuda_dev)
        q, s = ops.add_rmsnorm_e4m3(None, h, w, 1e-6)
        assert torch.all(q[0].float() == 448) and torch.all(q[3].float() == 448)
        assert torch.all(torch.isnan(q[1].float()))
        assert torch.isnan(q[2, 0].float()) and torch.isfinite(s).all()


# ------------------------------------------------------------ linear
LINEAR_SHAPES = [(1, 8, 16), (1, 128, 64), (8, 4096, 1024), (5, 200, 48), (130, 256, 128), (129, 1000, 144), (300, 384, 2048),
                 (512, 256, 128), (513, 1152, 768), (700, 264, 272), (1025, 1024, 4096), (2500, 2304, 768)]


def _e4m3_rows(rows, cols, dev, g):
    x = torch.randn(rows, cols, device=dev, generator=g)
    s = x.abs().amax(-1) / 448
    return (x / s[:, None]).to(F8), s


@pytest.mark.parametrize("m,n,k", LINEAR_SHAPES)
@pytest.mark.parametrize("epi,out", [("none", "bf16"), ("none", "f32"), ("bias", "bf16"), ("bias", "f32"),
                                     ("bias_gelu", "bf16"), ("bias_relu", "bf16"), ("bias_swish", "bf16"),
                                     ("bias_residual", "f32")])
def test_linear(cuda_dev, m, n, k, epi, out):
    from fastembed_b200 import ops
    g = torch.Generator(device=cuda_dev).manual_seed(m + 3 * n + 7 * k)
    x, xs = _e4m3_rows(m, k, cuda_dev, g)
    w, ws = _e4m3_rows(n, k, cuda_dev, g)
    ws = ws / math.sqrt(k)
    bias = torch.randn(n, device=cuda_dev, generator=g) * 0.3
    res = torch.randn(m, n, device=cuda_dev, generator=g)
    y = ops.linear_e4m3(x, xs, w, ws, None if epi == "none" else bias, res if epi == "bias_residual" else None, epi, out)
    want, z, mag = ref.linear(x, xs, w, ws, bias, res, epi)
    assert torch.all((y.double() - want).abs() <= _linear_bound(want, z, mag, k, epi, out, bias, res))
    ops.device_status(0)


def _linear_bound(want, z, mag, k, epi, out, bias=None, res=None):
    """k fp32 accumulations of at most a whole step (2^-23) of the running sum, itself at most
    mag, and four roundings of the result's parts; an activation passes that on by a slope of at
    most 1.13; tanh.approx is off by 2^-10.98 (gelu: |z| / 2 of it), ex2 / rcp.approx by 2^-21;
    bf16 output rounds by half a step."""
    parts = mag + (0 if bias is None else bias.double().abs()) + (res.double().abs() if epi == "bias_residual" else 0)
    b = 1.13 * (k * 2.0 ** -23 * mag + 2.0 ** -22 * parts) + 2.0 ** -20 * want.abs()
    if epi in ("bias_gelu", "geglu"):
        b = b + 2.0 ** -10.9 * (z.abs() / 2 if epi == "bias_gelu" else 0)
    return b + (2.0 ** -8 * want.abs() if out == "bf16" else 0) + 1e-30


@pytest.mark.parametrize("m,n,k", [(1, 128, 32), (65, 256, 512), (600, 2304, 768), (530, 384, 1024)])
@pytest.mark.parametrize("epi", ["swiglu", "geglu"])
def test_linear_gated(cuda_dev, m, n, k, epi):
    from fastembed_b200 import ops
    g = torch.Generator(device=cuda_dev).manual_seed(m + n + k)
    x, xs = _e4m3_rows(m, k, cuda_dev, g)
    w, ws = _e4m3_rows(n, k, cuda_dev, g)
    ws = ws / math.sqrt(k)
    y = ops.linear_e4m3(x, xs, w, ws, epilogue=epi)
    want, z, mag = ref.linear(x, xs, w, ws, None, None, epi)
    # geglu: the gate's tanh error reaches the product as |gate up| / 2 * 2^-10.9, and |gate up| is at
    # most what the magnitudes of the two accumulators give
    lin = ref.linear(x, xs, w, ws, None, None, "none")[0].view(m, -1, 2, 32)
    extra = 2.0 ** -10.9 * (lin[:, :, 0] * lin[:, :, 1]).abs().reshape(m, -1) / 2 if epi == "geglu" else 0
    assert y.shape == (m, n // 2)
    assert torch.all((y.double() - want).abs() <= _linear_bound(want, z, mag, k, epi, "bf16") + extra)


def test_linear_residual_in_place_and_repeatable(cuda_dev):
    """y may be the residual; a repeat is bit-identical, and a block of rows alone gives the same
    bits (each row depends on its own codes only, whichever kernel runs)."""
    from fastembed_b200 import capi, ops
    g = torch.Generator(device=cuda_dev).manual_seed(2)
    x, xs = _e4m3_rows(900, 1024, cuda_dev, g)
    w, ws = _e4m3_rows(512, 1024, cuda_dev, g)
    b = torch.randn(512, device=cuda_dev, generator=g)
    r = torch.randn(900, 512, device=cuda_dev, generator=g)
    y1 = ops.linear_e4m3(x, xs, w, ws, b, r, "bias_residual", "f32")
    y2 = ops.linear_e4m3(x, xs, w, ws, b, r, "bias_residual", "f32")
    y3 = ops.linear_e4m3(x[100:231].contiguous(), xs[100:231].contiguous(), w, ws, b, r[100:231].contiguous(),
                         "bias_residual", "f32")
    assert torch.equal(y1, y2) and torch.equal(y1[100:231], y3)
    capi.call("fe_linear_e4m3", x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), b.data_ptr(), r.data_ptr(),
              r.data_ptr(), 900, 512, 1024, capi.EPI["bias_residual"], capi.DTYPE["f32"],
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(r, y1)


def test_linear_nan_row_stays_alone(cuda_dev):
    from fastembed_b200 import ops
    x = torch.ones(600, 256, device=cuda_dev)
    x[7, 9] = math.nan
    q, s = ops.quantize_rows_e4m3(x)
    w, ws = ops.quantize_rows_e4m3(torch.ones(256, 256, device=cuda_dev))
    y = ops.linear_e4m3(q, s, w, ws, out_dtype="f32")
    assert torch.isnan(y[7]).all()
    keep = torch.arange(600, device=cuda_dev) != 7
    assert torch.all((y[keep] - 256).abs() <= 256 * 2.0 ** -20)


# ------------------------------------------------------------ cache append
def _append_both(b, ops, cache):
    kc, vc, ks, vs = ref.append(cache, b.qkv, b.new, b.past, b.table.cpu(), b.q_heads)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    # a power of two moves no rounding: everything is exact
    assert torch.equal(cache.k_scale.double(), ks) and torch.equal(cache.v_scale.double(), vs)
    for got, want in ((cache.k, kc), (cache.v, vc)):
        got = got.view(torch.uint8)
        nan = (got & 0x7F) == 0x7F
        assert torch.equal(nan, (want & 0x7F) == 0x7F)
        assert torch.equal(got[~nan], want[~nan])
    ops.device_status(0)


APPENDS = [([1], [0]), ([1], [63]), ([1, 1, 1], [5, 64, 1000]), ([0, 7, 0, 1], [3, 60, 0, 15]), ([300, 1, 129], [0, 500, 77]),
           ([17, 33, 65, 128], [15, 31, 63, 127])]


@pytest.mark.parametrize("new,past", APPENDS)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("hd,heads", [(64, (4, 4)), (128, (16, 8)), (256, (3, 1))])
def test_append(cuda_dev, new, past, page, hd, heads):
    from fastembed_b200 import ops
    b = Batch(new, past, page, *heads, hd, cuda_dev, seed=page + hd)
    _append_both(b, ops, b.random_cache(ops))


def test_append_scale_grows_and_starts_afresh(cuda_dev):
    """Token by token: small, then larger keys re-encode the page; a zero page; a reused page."""
    from fastembed_b200 import ops
    b = Batch([1], [0], 16, 2, 1, 64, cuda_dev)
    cache = b.random_cache(ops)  # stale scales in every page: slot 0 must not look at them
    for i, mag in enumerate([0.0, 0.0, 1e-20, 1e-3, 1.0, 0.5, 3e4, 1e30, 7.0]):
        b.past, b.past_lens = [i], torch.tensor([i], dtype=torch.int32, device=cuda_dev)
        b.qkv.copy_(torch.randn(b.qkv.shape, device=cuda_dev, generator=b.g) * mag)
        _append_both(b, ops, cache)


@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64), (256, 128)])
def test_append_non_finite_tokens(cuda_dev, hd, page):
    from fastembed_b200 import ops
    b = Batch([40, 3], [9, 100], page, 4, 2, hd, cuda_dev)
    x = b.qkv.view(-1, 8, hd)
    x[3, 4, 5] = math.nan     # key, head 0
    x[8, 7, hd - 1] = math.inf  # value, head 1
    x[9, 6, 0] = -math.inf    # value, head 0
    x[41, 5, 1] = math.nan
    x[20, 0] = math.nan       # a query: not the cache's business
    _append_both(b, ops, b.random_cache(ops))


def test_append_leaves_other_bytes_alone_and_reports_bad_input(cuda_dev):
    from fastembed_b200 import ops
    from fastembed_b200.capi import FeError
    b = Batch([5, 6, 4], [30, 2, 0], 16, 4, 2, 64, cuda_dev, spare=3)

    def run(cu=None, past=None, table=None, max_new=None):
        cache = b.random_cache(ops)
        before = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
        ops.kv_cache_append_e4m3(b.qkv, b.cu if cu is None else cu, max_new or b.max_new,
                                 b.past_lens if past is None else past, b.table if table is None else table, cache, 4)
        after = (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)
        return [p for p in range(b.pages) if any(not torch.equal(x[p], y[p]) for x, y in zip(before, after))]

    t = b.table.cpu()
    own = [sorted({int(t[0, 1]), int(t[0, 2])}), [int(t[1, 0])], [int(t[2, 0])]]
    assert run() == sorted(sum(own, []))
    ops.device_status(0)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_dev)
    bad = b.table.clone()
    bad[1, 0], bad[0, 1] = b.pages, -1
    cases = [(dict(table=bad), sorted([int(t[0, 2])] + own[2])),               # page ids outside the pool
             (dict(past=i32([30, -4, 0])), sorted(own[0] + own[2])),           # a negative past
             (dict(cu=i32([0, 5, 11, 16])), sorted(own[0] + own[1])),          # rows past the batch
             (dict(past=i32([30, 100, 0])), sorted(own[0] + own[2]))]          # past the table's width
    for kw, want in cases:
        assert run(**kw) == want, kw
        with pytest.raises(FeError):
            ops.device_status(0)
        ops.device_status(0)


# ------------------------------------------------------------ attention over the cache
def _attend(b, ops, cache, causal=True, scale=None, check=None):
    out = ops.attention_cache_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.max_kv, b.table, cache, b.q_heads, causal, scale)
    want, mag, dot, floor = ref.attention(cache, b.qkv, b.new, b.past, b.table, b.q_heads, causal,
                                          b.hd ** -0.5 if scale is None else scale)
    T = sum(b.new)
    err, bound = (out[:T].double() - want).abs(), ref.attention_bound(want, mag, dot, floor, b.hd)
    assert torch.all(err <= bound), float((err / bound).max())
    ops.device_status(0)
    return out


ATTENDS = [([1], [0]), ([1], [1]), ([1], [700]), ([1], [9000]), ([2], [40000]), ([1, 1, 1], [5, 64, 2500]), ([0, 7, 0, 1], [3, 60, 0, 15]), ([3, 1], [13, 0]),
           ([130, 1, 64], [0, 500, 77]), ([17, 33, 65, 128], [15, 31, 63, 127]), ([300], [0]), ([257, 129], [1000, 3])]


@pytest.mark.parametrize("new,past", ATTENDS)
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("hd,heads", [(64, (4, 4)), (128, (16, 8)), (128, (10, 2)), (256, (3, 1))])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_cache(cuda_dev, new, past, page, hd, heads, causal):
    from fastembed_b200 import ops
    b = Batch(new, past, page, *heads, hd, cuda_dev, seed=sum(new) + hd)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    _attend(b, ops, cache, causal)


@pytest.mark.parametrize("heads", [(1, 1), (8, 1), (32, 2), (12, 4)])
def test_attention_cache_groups_and_scale(cuda_dev, heads):
    from fastembed_b200 import ops
    b = Batch([1, 5, 40], [90, 33, 7], 32, *heads, 128, cuda_dev, seed=heads[0])
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    for scale in (0.0, 0.02, 0.3, -0.1):
        _attend(b, ops, cache, True, scale)


@pytest.mark.parametrize("new", [[1, 1], [80, 3]])
def test_attention_cache_scales_far_apart(cuda_dev, new):
    """Value scales of pages from 2^-60 to 2^60, a page of zeros, large queries: the weights meet
    the codes at the right size, and the softmax sums do not lose the pages with small values."""
    from fastembed_b200 import ops
    b = Batch(new, [200, 150], 16, 4, 2, 128, cuda_dev)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    for exps in ([-20, 0, 20, -3], [-60, 60, 0, -8], [-8, -8, 0, -40]):
        e = torch.tensor(exps, device=cuda_dev).repeat(b.pages)[:b.pages].float()
        cache.v_scale.copy_((2.0 ** e)[:, None].expand(-1, 2))
        zero = int(b.table[0, 2])
        cache.v_scale[zero] = 0
        cache.v.view(torch.uint8)[zero] = 0
        _attend(b, ops, cache)
    cache.v_scale.fill_(2.0 ** -7)
    b.qkv *= 1e30  # past f16; logits of one token swamp the rest
    _attend(b, ops, cache, True, 1e-30)


def test_attention_cache_ignores_what_lies_behind(cuda_dev):
    """NaN codes in slots past a sequence's end and in other pages, rows of out behind the last
    sequence, and a later token that is NaN for the queries that do not see it."""
    from fastembed_b200 import ops
    for hd, new in ((64, [3, 20]), (128, [3, 20]), (128, [1, 1]), (256, [2, 9]), (128, [150, 70])):
        b = Batch(new, [21, 100], 64, 4, 2, hd, cuda_dev, extra_rows=3)
        cache = b.random_cache(ops)
        ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
        want = _attend(b, ops, cache)
        used = torch.zeros(b.pages, 64, dtype=torch.bool, device=cuda_dev)
        for s, (n, p) in enumerate(zip(b.new, b.past)):
            for t in range(0, n + p):
                used[int(b.table[s, t // 64]), t % 64] = True
        for codes in (cache.k, cache.v):
            raw = codes.view(torch.uint8)
            raw.copy_(torch.where(used[:, None, :, None], raw, torch.full_like(raw, 0x7F)))
        out = torch.full_like(want, 7.0)
        ops.attention_cache_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.max_kv, b.table, cache, b.q_heads, out=out)
        T = sum(new)
        assert torch.equal(out[:T], want[:T]) and torch.all(out[T:] == 7.0)
        if new[0] > 1:  # the last new token of sequence 0 is poisoned
            x = b.qkv.view(b.qkv.shape[0], -1, hd)
            x[new[0] - 1, 4 + 2, 0] = math.inf  # its value, head 0
            ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
            out = ops.attention_cache_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.max_kv, b.table, cache, b.q_heads)
            rows = out[:T].view(T, 4, hd)
            assert torch.isnan(rows[new[0] - 1, :2]).all()  # the heads of key-value head 0
            rows[new[0] - 1, :2] = 0
            assert torch.isfinite(rows).all()
        ops.device_status(0)


def test_attention_cache_bad_pages_and_offsets(cuda_dev):
    """Pages outside the pool are left out (a row that sees none is zero) and reported; a sequence
    whose offsets do not fit leaves its rows as they are."""
    from fastembed_b200 import ops
    from fastembed_b200.capi import FeError
    for new in ([1, 1, 1], [40, 30, 20]):
        b = Batch(new, [100, 90, 40], 32, 4, 2, 128, cuda_dev)
        cache = b.random_cache(ops)
        ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
        want = _attend(b, ops, cache)
        table = b.table.clone()
        table[1] = b.pages + 7
        out = torch.full_like(want, 5.0)
        run = lambda **kw: ops.attention_cache_e4m3(b.qkv, kw.get("cu", b.cu), kw.get("max_new", b.max_new),
                                                    kw.get("past", b.past_lens), b.max_kv, kw.get("table", b.table), cache,
                                                    b.q_heads, out=out)
        run(table=table)
        with pytest.raises(FeError):
            ops.device_status(0)
        a, c = new[0], new[0] + new[1]
        assert torch.equal(out[:a], want[:a]) and torch.equal(out[c:], want[c:]) and torch.all(out[a:c] == 0)
        out.fill_(5.0)
        past = b.past_lens.clone()
        past[1] = -1
        run(past=past)
        with pytest.raises(FeError):
            ops.device_status(0)
        assert torch.equal(out[:a], want[:a]) and torch.equal(out[c:], want[c:]) and torch.all(out[a:c] == 5.0)
        ops.device_status(0)


def test_attention_cache_shared_prefix_and_repeat(cuda_dev):
    """Two sequences over the same prefix pages; repeats are bit-identical."""
    from fastembed_b200 import ops
    b = Batch([20, 20], [64, 64], 32, 8, 2, 128, cuda_dev)
    cache = b.random_cache(ops)
    b.table[1, :2] = b.table[0, :2]
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    one = _attend(b, ops, cache)
    assert torch.equal(one, _attend(b, ops, cache))


def test_cache_offsets_past_32_bits(cuda_dev):
    """A pool of more than 2^32 bytes of keys: the last pages are written and read in place."""
    from fastembed_b200 import ops
    pages = (1 << 32) // (8 * 64 * 128) + 40
    b = Batch([70, 1], [10, 130], 64, 16, 8, 128, cuda_dev)
    small = b.random_cache(ops)
    raw = [torch.empty(pages, 8, 64, 128, dtype=torch.uint8, device=cuda_dev) for _ in range(2)]
    scales = [torch.empty(pages, 8, device=cuda_dev) for _ in range(2)]
    for big, src in zip(raw + scales, (small.k.view(torch.uint8), small.v.view(torch.uint8), small.k_scale, small.v_scale)):
        big[pages - b.pages:] = src
    big = ops.KvCacheE4m3(raw[0].view(F8), raw[1].view(F8), *scales)
    table = b.table + (pages - b.pages)
    for cache, tab in ((small, b.table), (big, table)):
        ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, tab, cache, b.q_heads)
    assert torch.equal(raw[0][pages - b.pages:], small.k.view(torch.uint8))
    assert torch.equal(raw[1][pages - b.pages:], small.v.view(torch.uint8))
    want = _attend(b, ops, small)
    got = ops.attention_cache_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.max_kv, table, big, b.q_heads)
    assert torch.equal(got, want)
    ops.device_status(0)


# ------------------------------------------------------------ together
def _layer(ops, st, h, y, past, cache, table, cu, max_new, max_kv):
    """One pre-norm attention step as an 8-bit serving program runs it; returns (h, y of the out-projection)."""
    q, s = ops.add_rmsnorm_e4m3(y, h, st["norm"], 1e-6)
    qkv = ops.linear_e4m3(q, s, *st["wqkv"])
    ops.kv_cache_append_e4m3(qkv, cu, max_new, past, table, cache, st["hq"])
    a = ops.attention_cache_e4m3(qkv, cu, max_new, past, max_kv, table, cache, st["hq"])
    q, s = ops.quantize_rows_e4m3(a)
    return ops.linear_e4m3(q, s, *st["wo"], st["zero"], h, "bias_residual", "f32")


def _layer_state(ops, dev, hidden=512, hq=4, hkv=2, hd=128):
    g = torch.Generator(device=dev).manual_seed(11)
    mk = lambda n, k: ops.quantize_rows_e4m3(torch.randn(n, k, device=dev, generator=g) / math.sqrt(k))
    return {"norm": 1 + 0.1 * torch.randn(hidden, device=dev, generator=g), "wqkv": mk((hq + 2 * hkv) * hd, hidden),
            "wo": mk(hidden, hq * hd), "zero": torch.zeros(hidden, device=dev), "hq": hq, "hkv": hkv, "hd": hd, "hidden": hidden}


def test_prefix_then_rest_equals_all_at_once(cuda_dev):
    """A step over a cached prefix, then over the rest (as a chunk and token by token), against the
    64-bit step over the whole sequence: every element within what 8-bit operands leave."""
    from fastembed_b200 import ops
    st = _layer_state(ops, cuda_dev)
    T, page = 100, 32
    g = torch.Generator(device=cuda_dev).manual_seed(12)
    h = torch.randn(T, st["hidden"], device=cuda_dev, generator=g)
    table = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32, device=cuda_dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_dev)

    def run(cuts):
        cache = ops.kv_cache_e4m3(4, page, st["hkv"], st["hd"], cuda_dev)
        outs, at = [], 0
        for n in cuts:
            outs.append(_layer(ops, st, h[at:at + n].clone(), None, i32(at), cache, table, i32(0, n), n, at + n))
            at += n
        return torch.cat(outs)

    whole = run([T])
    for cuts in ([64, 36], [50, 50], [40] + [1] * 60):
        # what differs is the scale of a page while it fills and the kernel that runs: a key's code is
        # within 2^-4 of its value either way, most of it common to both runs
        assert float((run(cuts) - whole).norm() / (whole - h).norm()) < 2.0 ** -4
    # against 64 bits from the same quantised operands up to the cache: the attention and out-projection alone
    hv = h.double()
    nrm = ref.rmsnorm(hv, st["norm"], 1e-6, False)
    wq, wo = ref.values(*st["wqkv"]), ref.values(*st["wo"])
    qkv = (nrm @ wq.T).view(T, -1, st["hd"])
    q, k, v = qkv[:, :4], qkv[:, 4:6].repeat_interleave(2, 1), qkv[:, 6:].repeat_interleave(2, 1)
    sc = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(st["hd"])
    sc = sc.masked_fill(~torch.ones(T, T, dtype=torch.bool, device=cuda_dev).tril(), -math.inf)
    exact = torch.einsum("hij,jhd->ihd", sc.softmax(-1), v).reshape(T, -1) @ wo.T
    got = (whole - h).double()
    # four e4m3 roundings lie on the way (norm, keys, values, attention rows), each at most 2^-4 of its
    # operand and of random sign: together below their sum in norm
    assert float((got - exact).norm() / exact.norm()) < 4 * 2.0 ** -4
    ops.device_status(0)


def test_steps_captured_in_a_graph_and_on_a_side_stream(cuda_dev):
    """The whole step captured once and replayed with other inputs, positions and pages, and the
    same on a stream that is not the default one: equal to eager calls."""
    from fastembed_b200 import ops
    ops.device_status(0)
    st = _layer_state(ops, cuda_dev)
    page, B = 32, 3
    g = torch.Generator(device=cuda_dev).manual_seed(13)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_dev)
    table = i32([[1, 4, 7], [0, 3, 6], [8, 5, 2]])
    cu = i32([0, 1, 2, 3])
    hs = [torch.randn(B, st["hidden"], device=cuda_dev, generator=g) for _ in range(4)]
    pasts = [[0, 30, 64], [1, 31, 65], [2, 32, 66], [3, 33, 67]]

    def eager():
        cache = ops.kv_cache_e4m3(9, page, st["hkv"], st["hd"], cuda_dev)
        return [_layer(ops, st, h.clone(), None, i32(p), cache, table, cu, 1, 96) for h, p in zip(hs, pasts)], cache

    want, wcache = eager()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = eager()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    cache = ops.kv_cache_e4m3(9, page, st["hkv"], st["hd"], cuda_dev)
    h, past = hs[0].clone(), i32(pasts[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _layer(ops, st, h, None, past, cache, table, cu, 1, 96)
    for src, p, w in zip(hs, pasts, want):
        h.copy_(src)
        past.copy_(i32(p))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, w)
    assert torch.equal(cache.k.view(torch.uint8), wcache.k.view(torch.uint8))
    ops.device_status(0)


# ------------------------------------------------------------ both attention kernels at every size
@pytest.mark.parametrize("new,past", ATTENDS)
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("hd,heads", [(64, (4, 4)), (128, (16, 8)), (128, (10, 2)), (256, (3, 1))])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_cache_loose_bound(cuda_dev, new, past, page, hd, heads, causal):
    """max_kv_len is a bound: one far above the lengths gives sequences parts of which most are
    empty, and turns rows that few tokens are read for over to the tile kernel."""
    from fastembed_b200 import ops
    b = Batch(new, past, page, *heads, hd, cuda_dev, seed=sum(new) + hd)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    b.max_kv = 1 << 20
    _attend(b, ops, cache, causal)


MANY = [65, 0, 17, 128, 1, 33, 64, 300, 129, 2, 96, 256]


@pytest.mark.parametrize("hd,heads", [(64, (8, 8)), (64, (6, 2)), (128, (16, 8)), (128, (10, 2)), (256, (6, 2)), (256, (4, 4))])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_cache_many_prompts(cuda_dev, hd, heads, page, causal):
    """Enough row tiles that no sequence is split."""
    from fastembed_b200 import ops
    b = Batch(MANY, [(37 * i * i) % 400 for i in range(len(MANY))], page, *heads, hd, cuda_dev, seed=hd + page, extra_rows=2)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    _attend(b, ops, cache, causal)


@pytest.mark.parametrize("hd,heads,batch", [(128, (4, 2), 150), (64, (2, 2), 250), (256, (2, 1), 300), (128, (8, 1), 160)])
@pytest.mark.parametrize("top", [1, 5])
def test_attention_cache_many_sequences(cuda_dev, hd, heads, batch, top):
    """Few rows each in more sequences than there are multiprocessors: one part each, or two."""
    from fastembed_b200 import ops
    b = Batch([(7 * i) % top + 1 for i in range(batch)], [(53 * i) % 700 for i in range(batch)], 32, *heads, hd, cuda_dev)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    _attend(b, ops, cache)


# ------------------------------------------------------------ lengths that do not fit, graphs, waits
@pytest.mark.parametrize("new,bound", [([1, 6, 2], 300), ([1, 90, 2], 1 << 20), ([1, 6, 2], 1 << 20)])
def test_longer_than_max_len_is_reported(cuda_dev, new, bound):
    """A sequence with more new tokens than max_len: neither written, nor answered, nor read past; the
    others as without it."""
    from fastembed_b200 import ops
    from fastembed_b200.capi import FeError
    b = Batch(new, [20, 33, 40], 32, 8, 2, 128, cuda_dev)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    ops.device_status(0)
    short = new[1] - 1
    state = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
    out = torch.full((sum(new), 8 * 128), 3.0, dtype=torch.bfloat16, device=cuda_dev)
    ops.attention_cache_e4m3(b.qkv, b.cu, short, b.past_lens, bound, b.table, cache, 8, out=out)
    with pytest.raises(FeError):
        ops.device_status(0)
    want, mag, dot, floor = ref.attention(cache, b.qkv, b.new, b.past, b.table, 8, True, 128 ** -0.5)
    fits = (out.double() - want).abs() <= ref.attention_bound(want, mag, dot, floor, 128)
    a, c = new[0], new[0] + new[1]
    assert torch.all(out[a:c] == 3.0) and torch.all(fits[:a]) and torch.all(fits[c:])
    b.qkv.neg_()
    ops.kv_cache_append_e4m3(b.qkv, b.cu, short, b.past_lens, b.table, cache, 8)
    with pytest.raises(FeError):
        ops.device_status(0)
    t = b.table.cpu()
    mine = {int(t[1, o]) for o in range(33 // 32, (33 + new[1] - 1) // 32 + 1)}
    for was, now in zip(state, (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)):
        for p in mine:
            assert torch.equal(was[p], now[p])
    ops.device_status(0)


@pytest.mark.parametrize("new,past,bound", [([1, 1], [900, 300], 901), ([1, 1], [900, 300], 1 << 20),
                                            ([70, 40], [600, 10], 1 << 20), (MANY, [5] * len(MANY), 400)])
def test_attention_cache_captured(cuda_dev, new, past, bound):
    """Each form of the attention (parts in a cluster, parts in a workspace, tiles in parts, tiles)
    captured and replayed over changed queries and pages: the bits of eager calls.  Two graphs of one
    stream with a workspace each."""
    from fastembed_b200 import ops
    b = Batch(new, past, 32, 16, 8, 128, cuda_dev, seed=5)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, 16)
    run = lambda q: ops.attention_cache_e4m3(q, b.cu, b.max_new, b.past_lens, bound, b.table, cache, 16)
    q1, q2 = b.qkv.clone(), (b.qkv.float() * -0.5).to(torch.bfloat16)
    w1, w2 = run(q1), run(q2)
    a1, a2 = torch.zeros_like(q1), torch.zeros_like(q2)
    graphs, outs = [], []
    for a in (a1, a2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(a))
        graphs.append(g)
    for src, dst in ((q1, a1), (q2, a2)):
        dst.copy_(src)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], w1) and torch.equal(outs[1], w2)
    a1.copy_(q2)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], w2)
    ops.device_status(0)


def _short_waits(call):
    """The call under a wait limit of a microsecond, then under the default again: the status of the first, which
    has the bits of a call before it unless it reports that a wait ran out, as the second has in any case."""
    from fastembed_b200 import capi
    L = capi.lib()
    before = call().clone()
    torch.cuda.synchronize()
    assert L.fe_device_status(0) == 0
    assert L.fe_set_wait_limit(0, 1000) == 0
    try:
        got = call()
        st = L.fe_device_status(0)
    finally:
        assert L.fe_set_wait_limit(0, 2_000_000_000) == 0
    assert st == 5 or (st == 0 and torch.equal(got, before)), st  # FE_ERR_DEVICE_TIMEOUT
    assert torch.equal(call(), before)
    torch.cuda.synchronize()
    assert L.fe_device_status(0) == 0
    return st


@pytest.mark.parametrize("epi", ["none", "bias_residual"])
def test_linear_wait_runs_out_then_recovers(cuda_dev, epi):
    """One tile whose 64-block main loop takes tens of microseconds: the epilogue's wait for it runs out."""
    from fastembed_b200 import ops
    g = torch.Generator(device=cuda_dev).manual_seed(3)
    x = ops.quantize_rows_e4m3(torch.randn(128, 8192, device=cuda_dev, generator=g))
    w = ops.quantize_rows_e4m3(torch.randn(64, 8192, device=cuda_dev, generator=g))
    bias, res = torch.randn(64, device=cuda_dev, generator=g), torch.randn(128, 64, device=cuda_dev, generator=g)
    if epi == "none":
        assert _short_waits(lambda: ops.linear_e4m3(*x, *w, None, None, "none", "f32")) == 5
    else:
        assert _short_waits(lambda: ops.linear_e4m3(*x, *w, bias, res, "bias_residual", "f32")) == 5


@pytest.mark.parametrize("hd,heads", [(64, (8, 4)), (128, (16, 8)), (256, (6, 2))])
def test_attention_cache_short_waits(cuda_dev, hd, heads):
    """The tile kernel's waits are for a load, a product or a softmax step, a microsecond or two: they may run
    out or not (the limit is looked at every 256 tries), and the call stays sound either way."""
    from fastembed_b200 import ops
    b = Batch([300, 17, 129, 64], [700, 0, 3000, 10], 64, *heads, hd, cuda_dev)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    _short_waits(lambda: ops.attention_cache_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.max_kv, b.table, cache, b.q_heads))


@pytest.mark.parametrize("m,n", [(64, 64), (300, 520), (511, 256), (700, 512)])
def test_linear_residual_in_place_every_kernel(cuda_dev, m, n):
    from fastembed_b200 import capi, ops
    g = torch.Generator(device=cuda_dev).manual_seed(m)
    x = ops.quantize_rows_e4m3(torch.randn(m, 256, device=cuda_dev, generator=g))
    w = ops.quantize_rows_e4m3(torch.randn(n, 256, device=cuda_dev, generator=g))
    bias, res = torch.randn(n, device=cuda_dev, generator=g), torch.randn(m, n, device=cuda_dev, generator=g)
    want = ops.linear_e4m3(*x, *w, bias, res, "bias_residual", "f32")
    y = res.clone()
    capi.call("fe_linear_e4m3", x[0].data_ptr(), x[1].data_ptr(), w[0].data_ptr(), w[1].data_ptr(), bias.data_ptr(),
              y.data_ptr(), y.data_ptr(), m, n, 256, capi.EPI["bias_residual"], capi.DTYPE["f32"],
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(y, want)


@pytest.mark.parametrize("hd,heads", [(64, (4, 4)), (128, (4, 2)), (256, (3, 1))])
@pytest.mark.parametrize("bound", [200, 1 << 20])
def test_attention_cache_non_finite_queries(cuda_dev, hd, heads, bound):
    """An infinity or NaN among a query's elements: that head's row is NaN whatever the keys' signs
    are, the others as without it.  By streaming and (300 new tokens, loose bound) by tiles."""
    from fastembed_b200 import ops
    b = Batch([3, 300 if bound > 1000 else 12], [90, 33], 32, *heads, hd, cuda_dev)
    b.qkv.view(-1, heads[0] + 2 * heads[1], hd)[:, heads[0]:, 1] = 1.0  # keys (and values) of one sign there
    cache = b.random_cache(ops)
    cache.k[..., 1] = torch.tensor(200.0, device=cuda_dev).to(F8)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    run = lambda: ops.attention_cache_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, bound, b.table, cache, b.q_heads)
    want = run().view(-1, heads[0], hd).clone()
    q = b.qkv.view(-1, heads[0] + 2 * heads[1], hd)
    spots = [(0, 0, math.inf), (2, 1, -math.inf), (4, 0, -math.inf), (7, 2, math.nan), (14, 1, math.inf)]
    for t, h, x in spots:
        q[t, h, 1] = x
    got = run().view(-1, heads[0], hd)
    for t, h, x in spots:
        assert torch.isnan(got[t, h]).all(), (t, h, x)
        got[t, h] = want[t, h]
    assert torch.equal(got, want)
    ops.device_status(0)


def test_front_end_refuses(cuda_dev):
    """What the front end turns away before a launch, and what the library does."""
    from fastembed_b200 import ops
    from fastembed_b200.capi import FeError
    b = Batch([2, 1], [5, 9], 16, 4, 2, 64, cuda_dev)
    cache = b.random_cache(ops)
    calls = {"append": lambda **k: ops.kv_cache_append_e4m3(*[k.get(n, v) for n, v in base.items()]),
             "attend": lambda **k: ops.attention_cache_e4m3(
                 *[k.get(n, v) for n, v in list(base.items())[:4]], 20, *[k.get(n, v) for n, v in list(base.items())[4:]],
                 out=k.get("out"))}
    base = dict(qkv=b.qkv, cu=b.cu, max_len=2, past=b.past_lens, table=b.table, cache=cache, q_heads=4)
    bad = [dict(qkv=b.qkv.float()), dict(qkv=b.qkv[:, :-64]), dict(qkv=b.qkv.cpu()), dict(qkv=b.qkv.t()), dict(cu=b.cu.long()),
           dict(cu=b.cu[:2]), dict(past=b.past_lens[:1]), dict(past=b.past_lens.cpu()), dict(table=b.table[:1]),
           dict(table=b.table.float()), dict(cache=cache._replace(v=cache.v[1:])), dict(cache=cache._replace(k=cache.k[0])),
           dict(cache=cache._replace(k_scale=cache.k_scale.half())), dict(cache=cache._replace(v=cache.v.view(torch.uint8)))]
    for name, call in calls.items():
        for kw in bad:
            with pytest.raises(ValueError):
                call(**kw)
        with pytest.raises((ValueError, FeError)):
            call(q_heads=3)
        with pytest.raises(FeError):
            call(max_len=-1)
        odd = torch.zeros(b.qkv.numel() + 1, dtype=torch.bfloat16, device=cuda_dev)[1:].view(b.qkv.shape)
        with pytest.raises(FeError):
            call(qkv=odd)
    with pytest.raises(ValueError):
        calls["attend"](out=torch.zeros(3, 256, device=cuda_dev))
    x, s = ops.quantize_rows_e4m3(torch.randn(4, 64, device=cuda_dev))
    w, ws = ops.quantize_rows_e4m3(torch.randn(64, 64, device=cuda_dev))
    one = torch.ones(64, device=cuda_dev)
    for args in ((x, s[:3], w, ws), (x, s, w[:, :32], ws), (x, s, w, ws[:5]), (x.view(torch.uint8), s, w, ws), (x, s, w, ws, one[:8]),
                 (x, s, w, ws, one, torch.zeros(4, 32, device=cuda_dev)), (x.t(), s, w, ws), (x[0], s, w, ws)):
        with pytest.raises(ValueError):
            ops.linear_e4m3(*args)
    for kw in (dict(epilogue="bias"), dict(epilogue="swiglu"), dict(epilogue="bias_residual", out_dtype="f32", bias=one),
               dict(epilogue="bias_gelu", bias=one, out_dtype="f32")):
        with pytest.raises(FeError):
            ops.linear_e4m3(x, s, w, ws, **kw)
    for call in (lambda: ops.quantize_rows_e4m3(one.half()[None]), lambda: ops.quantize_rows_e4m3(one),
                 lambda: ops.quantize_rows_e4m3(torch.ones(8, 8, device=cuda_dev).t()[1:]),
                 lambda: ops.add_rmsnorm_e4m3(None, one[None], one[:8], 1e-6),
                 lambda: ops.add_rmsnorm_e4m3(one.half()[None], one[None], one, 1e-6)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(FeError):
        ops.add_rmsnorm_e4m3(None, one[None], one, -1.0)
    ops.device_status(0)


# ------------------------------------------------------------ linear layers past one round of tiles
@pytest.mark.parametrize("m,n,k", [(1030, 2312, 272), (2600, 1000, 48), (20000, 264, 128), (513, 5000, 400), (700, 4104, 1024),
                                   (300, 16384, 144), (511, 8200, 160), (130, 30000, 80)])
@pytest.mark.parametrize("epi,out", [("none", "bf16"), ("bias", "f32"), ("bias_residual", "f32"), ("bias_gelu", "bf16")])
def test_linear_large(cuda_dev, m, n, k, epi, out):
    """Pairs of CTAs, and tiles of 128 and 256 columns in several rounds, at ragged edges."""
    test_linear(cuda_dev, m, n, k, epi, out)


@pytest.mark.parametrize("m,n,k", [(1100, 2304, 272), (3000, 768, 768), (300, 16384, 144), (511, 8192, 160)])
@pytest.mark.parametrize("epi", ["swiglu", "geglu"])
def test_linear_gated_large(cuda_dev, m, n, k, epi):
    test_linear_gated(cuda_dev, m, n, k, epi)


def test_linear_rows_alone_across_kernels(cuda_dev):
    """Rows of a call that pairs of CTAs compute, alone: the same bits from every tile size; in place too."""
    from fastembed_b200 import capi, ops
    g = torch.Generator(device=cuda_dev).manual_seed(8)
    x, xs = _e4m3_rows(3001, 640, cuda_dev, g)
    w, ws = _e4m3_rows(1032, 640, cuda_dev, g)
    b = torch.randn(1032, device=cuda_dev, generator=g)
    r = torch.randn(3001, 1032, device=cuda_dev, generator=g)
    run = lambda lo, hi: ops.linear_e4m3(x[lo:hi].contiguous(), xs[lo:hi].contiguous(), w, ws, b, r[lo:hi].contiguous(),
                                         "bias_residual", "f32")
    whole = run(0, 3001)
    for lo, hi in ((0, 1), (100, 1000), (5, 2100), (2999, 3001)):
        assert torch.equal(run(lo, hi), whole[lo:hi])
    capi.call("fe_linear_e4m3", x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), b.data_ptr(), r.data_ptr(),
              r.data_ptr(), 3001, 1032, 640, capi.EPI["bias_residual"], capi.DTYPE["f32"],
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(r, whole)


# ------------------------------------------------------------ the ends of the ranges
def test_nothing_to_do(cuda_dev):
    """No rows, no sequences, no tokens: empty results, nothing launched or touched."""
    from fastembed_b200 import ops
    z = lambda *s: torch.zeros(*s, device=cuda_dev)
    q, s = ops.quantize_rows_e4m3(z(0, 64))
    assert q.shape == (0, 64) and s.shape == (0,)
    q, s = ops.add_rmsnorm_e4m3(None, z(0, 64), z(64), 1e-6)
    assert q.shape == (0, 64)
    w, ws = ops.quantize_rows_e4m3(torch.randn(128, 64, device=cuda_dev))
    assert ops.linear_e4m3(q, s, w, ws).shape == (0, 128)
    assert ops.linear_e4m3(q, s, w, ws, epilogue="swiglu").shape == (0, 64)
    b = Batch([0, 0], [3, 0], 16, 4, 2, 64, cuda_dev, extra_rows=3)
    cache = b.random_cache(ops)
    before = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
    rows = b.qkv  # of no sequence
    for qkv, max_len in ((rows[:0], 0), (rows[:0], 2), (rows, 0), (rows, 2)):
        ops.kv_cache_append_e4m3(qkv, b.cu, max_len, b.past_lens, b.table, cache, 4)
        out = torch.full((qkv.shape[0], 4 * 64), 2.0, dtype=torch.bfloat16, device=cuda_dev)
        ops.attention_cache_e4m3(qkv, b.cu, max_len, b.past_lens, 3, b.table, cache, 4, out=out)
        assert torch.all(out == 2.0)
    none = torch.zeros(0, dtype=torch.int32, device=cuda_dev)
    ops.kv_cache_append_e4m3(rows, b.cu[:1], 2, none, b.table[:0], cache, 4)
    ops.attention_cache_e4m3(rows, b.cu[:1], 2, none, 3, b.table[:0], cache, 4)
    after = (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)
    assert all(torch.equal(x, y) for x, y in zip(before, after))
    ops.device_status(0)


@pytest.mark.parametrize("hd,heads", [(64, (96, 1)), (128, (128, 1)), (128, (60, 4)), (256, (40, 1))])
@pytest.mark.parametrize("new,past,bound", [([1, 1, 2], [40, 0, 700], None), ([3, 9], [500, 20], 1 << 20), ([40], [90], 1 << 20)])
def test_attention_cache_wide_groups(cuda_dev, hd, heads, new, past, bound):
    """More query heads to a key-value head than a tile loads in a round, powers of two and not."""
    from fastembed_b200 import ops
    b = Batch(new, past, 16, *heads, hd, cuda_dev, seed=heads[0])
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    b.max_kv = bound or b.max_kv
    _attend(b, ops, cache)
    _attend(b, ops, cache, False)


def test_calls_on_two_streams_at_once(cuda_dev):
    """The same cache read on two streams side by side, each call with its own workspace."""
    from fastembed_b200 import ops
    b = Batch([1, 2, 60], [3000, 40, 900], 32, 16, 8, 128, cuda_dev)
    cache = b.random_cache(ops)
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, 16)
    other = (b.qkv.float() * 0.25).to(torch.bfloat16)
    run = lambda q: ops.attention_cache_e4m3(q, b.cu, b.max_new, b.past_lens, 1 << 20, b.table, cache, 16)
    want = run(b.qkv), run(other)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (st, q) in enumerate(zip(streams, (b.qkv, other))):
            with torch.cuda.stream(st):
                got[i].append(run(q))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)
    ops.device_status(0)


@pytest.mark.parametrize("hd,heads", [(64, (4, 4)), (128, (4, 2)), (256, (3, 1))])
@pytest.mark.parametrize("new,bound", [([3, 1], None), ([90, 40], 1 << 20)])
def test_attention_cache_query_outliers(cuda_dev, hd, heads, new, bound):
    """One element of each query thousands of times the others (and the keys small there): the others count
    to 2^-16 of it, by streaming and by tiles."""
    from fastembed_b200 import ops
    b = Batch(new, [200, 77], 32, *heads, hd, cuda_dev)
    x = b.qkv.view(-1, heads[0] + 2 * heads[1], hd)
    x[:, :heads[0], 5] = 4096.0
    x[:, heads[0]:heads[0] + heads[1], 5] *= 2.0 ** -12
    cache = ops.kv_cache_e4m3(b.pages, 32, heads[1], hd, cuda_dev)
    for s, p in enumerate(b.past):  # the prefix, from the same distribution
        k = torch.randn(b.pages, heads[1], 32, hd, device=cuda_dev, generator=b.g) * 40
        cache.k.copy_(k.to(F8))
        cache.v.copy_(torch.randn(k.shape, device=cuda_dev, generator=b.g).mul(40).to(F8))
    cache.k_scale.fill_(2.0 ** -9)
    cache.v_scale.fill_(2.0 ** -6)
    cache.k.view(torch.uint8)[..., 5] = 0
    ops.kv_cache_append_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, b.table, cache, b.q_heads)
    out = ops.attention_cache_e4m3(b.qkv, b.cu, b.max_new, b.past_lens, bound or b.max_kv, b.table, cache, b.q_heads)
    scale = hd ** -0.5
    want, mag, dot, floor = ref.attention(cache, b.qkv, b.new, b.past, b.table, b.q_heads, True, scale)
    ones = torch.ones_like(b.qkv)  # sum_d |k| at its largest, as the magnitudes of a query of ones
    dot1 = ref.attention(cache, ones, b.new, b.past, b.table, b.q_heads, True, scale)[2]
    top = x[:sum(new), :heads[0]].double().abs().amax(-1).repeat_interleave(hd, -1).view(sum(new), -1)
    # each element of a query is off by at most 2^-16 of its row's largest, and a logit by that times
    # scale sum_d |k|; weights pass it on in numerator and denominator
    extra = 2.0 * (2.0 ** -16 * top * dot1) * mag * 1.1
    err = (out[:sum(new)].double() - want).abs()
    assert torch.all(err <= ref.attention_bound(want, mag, dot, floor, hd) + extra)
    ops.device_status(0)
