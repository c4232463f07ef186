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
