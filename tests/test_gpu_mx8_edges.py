"""GPU: 8-bit activation checkpoints at the ends of their types' ranges and at the row counts of a training batch.

Tolerance of a weight gradient, as in tests/test_gpu_mx8.py: products are exact, each fp32 addition is off by at most 2^-23 of the running
magnitude, which is at most S = sum |dY| |x|; a result is made of at most `rows of a slice + partial results / 16 + 16` additions."""
import pytest
import torch

from tests import mx8_oracle as Q
from tests.test_gpu_mx8 import act

pytestmark = pytest.mark.gpu
D_ = 'cuda:0'
SMALL = 112 * 2.0 ** -23               # up to 256 slices of 64 rows


@pytest.mark.parametrize('shape', [(64, 256), (256, 64), (32, 32), (128, 64)], ids=lambda s: f'{s[0]}-{s[1]}')
def test_linear_wgrad_of_finite_gradients_at_the_top(shape):
    """fp32 dY whose first eight bits round past the largest bf16 (3.3953e38 to 3.4028e38) is finite, and so is its weight gradient: with a small
    x and with x = 0 (a padded pair).  One such element a column, so that the column sums stay finite too."""
    from diffalign_amd import mx8
    i, o = shape
    R = 150
    codes, scales, x = Q.quantize(act(R, i, torch.float32, 3) * 2.0 ** -60)
    assert bool((x == 0).all(1).any()) and bool((x != 0).any(1).any())
    g = torch.Generator().manual_seed(4)
    dy = act(R, o, torch.float32, 5)
    top = torch.finfo(torch.float32).max
    big = (3.39e38 + torch.rand(o, generator=g, dtype=torch.float64) * (top - 3.39e38)).float().clamp_max(top)
    big[0], big[1], big[2] = top, torch.tensor(0x7f7f8000, dtype=torch.int32).view(torch.float32), torch.tensor(0x7f7f7fff, dtype=torch.int32).view(torch.float32)
    dy[torch.randint(0, R, (o,), generator=g), torch.arange(o)] = big * (torch.randint(0, 2, (o,), generator=g) * 2 - 1)
    dW, db = mx8.linear_wgrad(mx8.Mx8(codes.to(D_), scales.to(D_)), dy.to(D_))
    d = dy.double()
    assert bool(((dW.cpu().double() - d.t() @ x).abs() <= SMALL * (d.abs().t() @ x.abs())).all())
    assert bool(((db.cpu().double() - d.sum(0)).abs() <= SMALL * d.abs().sum(0)).all())


def test_linear_wgrad_of_infinite_and_nan_gradients():
    """They reach exactly their own row of dW and element of db: infinite times a positive x is infinite, NaN is NaN whatever its payload."""
    from diffalign_amd import mx8
    codes, scales, x = Q.quantize(torch.rand(40, 64, generator=torch.Generator().manual_seed(1)) + 1)
    dy = act(40, 64, torch.float32, 2)
    dy[7, 3], dy[9, 4], dy[11, 5] = float('inf'), float('-inf'), float('nan')
    dy[39, 6] = torch.tensor(0x7f800001, dtype=torch.int32).view(torch.float32)              # a NaN whose upper half reads as an infinity
    dW, db = (t.cpu() for t in mx8.linear_wgrad(mx8.Mx8(codes.to(D_), scales.to(D_)), dy.to(D_)))
    assert bool((dW[3] == float('inf')).all()) and bool((dW[4] == float('-inf')).all()) and bool(dW[5:7].isnan().all())
    assert float(db[3]) == float('inf') and float(db[4]) == float('-inf') and bool(db[5:7].isnan().all())
    ok = [k for k in range(64) if k not in (3, 4, 5, 6)]
    assert bool(torch.isfinite(dW[ok]).all()) and bool(torch.isfinite(db[ok]).all())


def test_linear_wgrad_of_tiny_gradients():
    """fp32 dY down to the smallest normal beside a large x.  A part of dY below 2^-126 is a subnormal bf16, which the matrix instruction takes as
    it is, and what no bf16 holds is lost: less than 2^-133 |x| a product."""
    from diffalign_amd import mx8
    g = torch.Generator().manual_seed(8)
    R = 200
    codes, scales, x = Q.quantize(act(R, 64, torch.float32, 6) * 2.0 ** 100)
    dy = torch.randn(R, 64, generator=g) * torch.exp2(-126 + 30 * torch.rand(R, 1, generator=g))
    dW, db = mx8.linear_wgrad(mx8.Mx8(codes.to(D_), scales.to(D_)), dy.to(D_))
    d = dy.double()
    assert bool(((dW.cpu().double() - d.t() @ x).abs() <= SMALL * (d.abs().t() @ x.abs()) + 2.0 ** -133 * x.abs().sum(0)).all())


def small_scales(rows, D, seed, most=31):
    """Codes with every scale byte a caller's own 8-bit data may have: 0 to 26 are not written by quantize."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-127, 128, (rows, D), generator=g).to(torch.int8)
    G = -(-D // 32)
    scales = (torch.arange(rows * G) % most).reshape(rows, G).to(torch.uint8)
    vals = codes.double() * torch.exp2(scales.double() - 133).repeat_interleave(32, 1)[:, :D]
    return codes, scales, vals


@pytest.mark.parametrize('rows,D', [(37, 64), (19, 33), (40, 256)])
def test_scale_bytes_from_zero(rows, D):
    """The scale byte b stands for 2^(b - 127) from 0 on, 255 for NaN; the values, subnormal or not, are exact in fp32 and bf16."""
    from diffalign_amd import mx8
    codes, scales, vals = small_scales(rows, D, 1)
    q = mx8.Mx8(codes.to(D_), scales.to(D_))
    for out in (torch.float32, torch.bfloat16):
        assert torch.equal(mx8.dequantize(q, out).cpu().double(), vals)
    scales[3] = 255
    got = mx8.dequantize(mx8.Mx8(codes.to(D_), scales.to(D_))).cpu()
    assert bool(got[3].isnan().all()) and torch.equal(torch.cat((got[:3], got[4:])).double(), torch.cat((vals[:3], vals[4:])))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('most', [5, 31])
def test_linear_wgrad_of_scale_bytes_from_zero(most, dtype):
    """Small x (up to byte 4: subnormal throughout) beside a dY that makes up for it."""
    from diffalign_amd import mx8
    codes, scales, x = small_scales(200, 64, 2, most)
    dy = (act(200, 128, torch.float32, 7) * 2.0 ** 90).to(dtype)
    dW, db = mx8.linear_wgrad(mx8.Mx8(codes.to(D_), scales.to(D_)), dy.to(D_))
    d = dy.double()
    assert bool(((dW.cpu().double() - d.t() @ x).abs() <= SMALL * (d.abs().t() @ x.abs())).all())
    assert bool(((db.cpu().double() - d.sum(0)).abs() <= SMALL * d.abs().sum(0)).all())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('shape', [(64, 256), (256, 64), (32, 32), (128, 64)], ids=lambda s: f'{s[0]}-{s[1]}')
@pytest.mark.parametrize('R', [60_001, 140_001])
def test_linear_wgrad_rows_of_a_training_batch(R, shape, dtype):
    """Slices of several tiles with data in every row, on both sides of the change of the number of slices, the last slice ragged."""
    from diffalign_amd import mx8
    i, o = shape
    g = torch.Generator(device=D_).manual_seed(R + i)
    q = mx8.quantize(torch.randn(R, i, device=D_, generator=g) * torch.exp(torch.randn(R, 1, device=D_, generator=g)))
    dy = torch.randn(R, o, device=D_, generator=g).to(dtype)
    dW, db = mx8.linear_wgrad(q, dy)
    x, d = mx8.dequantize(q).double(), dy.double()
    slice_rows = 256 if R == 60_001 else 320
    parts = -(-R // slice_rows) * (4 if i * o == 1024 else 1)                                 # 32 -> 32: four waves over a slice's rows
    tol = (slice_rows + -(-parts // 16) + 16) * 2.0 ** -23
    assert bool(((dW.double() - d.t() @ x).abs() <= tol * (d.abs().t() @ x.abs())).all())
    assert bool(((db.double() - d.sum(0)).abs() <= tol * d.abs().sum(0)).all())
    again = mx8.linear_wgrad(q, dy)
    assert torch.equal(dW, again[0]) and torch.equal(db, again[1])
