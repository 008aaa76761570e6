"""GPU: 8-bit activation checkpoints (csrc/k_mx8.hip) against the format's definition in 64 bits and the gradients' formulas.

Tolerances.  Codes, scales and restored values: equal, bit for bit.  Weight gradient: every product of an 8-bit x and a bf16 dY (or a
third of an fp32 dY; what the three parts leave of it is below 2^-26 relative) is exact in fp32, so only the fp32 sums round: a slice
adds at most 64 rows here (R <= 256 * 64), the fold at most 32 + 16 partial results; each addition is off by at most 2^-23 of the
running magnitude (the matrix unit may truncate instead of rounding), which is at most S = sum |dY| |x|: 112 * 2^-23 S.
Column sums likewise, with S = sum |dY|."""
import pytest
import torch

from tests import mx8_oracle as Q

pytestmark = pytest.mark.gpu
D_ = 'cuda:0'


def act(rows, D, dtype, seed, relu=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, D, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g)) * torch.exp(torch.randn(D, generator=g))
    x *= torch.rand(rows, 1, generator=g) < 0.8
    return (x.relu() if relu else x).to(dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('keep', [False, True])
@pytest.mark.parametrize('rows,D', [(1, 1), (1, 32), (3, 64), (5, 31), (7, 33), (257, 100), (64, 256), (1001, 96), (2, 300)])
def test_quantize_roundtrip(rows, D, keep, dtype):
    from diffalign_amd import mx8
    x = act(rows, D, dtype, rows + D, relu=keep)
    codes, scales, vals = Q.quantize(x, keep)
    q = mx8.quantize(x.to(D_), keep_nonzero=keep)
    assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)
    for out in (torch.float32, torch.bfloat16):
        assert torch.equal(mx8.dequantize(q, out).cpu().double(), vals)


def test_quantize_edge_values():
    """Zeros, the borders of a scale step, ties, the smallest and largest values, infinities and NaN, in every place of a group."""
    from diffalign_amd import mx8
    rows = [torch.zeros(32)]
    for top in (127.0, 127.25, 127.49, 127.5, 127.75, 128.0, 1.0, 63.5):
        r = torch.linspace(-126.5, 126.5, 32); r[7] = top
        rows += [r, r * 2.0 ** -40, r * 2.0 ** 60]
    rows += [torch.full((32,), 3.4e38), torch.full((32,), 2.0 ** -140), torch.full((32,), 2.0 ** -100 * 0.4), torch.full((32,), 2.0 ** -106)]
    for k, bad in enumerate((float('inf'), float('-inf'), float('nan'))):
        r = torch.randn(32, generator=torch.Generator().manual_seed(k)); r[11 * k] = bad
        rows.append(r)
    x = torch.stack(rows)
    for D in (32, 31):                                                     # the wide and the general path
        for keep in (False, True):
            codes, scales, vals = Q.quantize(x[:, :D].contiguous(), keep)
            q = mx8.quantize(x[:, :D].contiguous().to(D_), keep)
            fine = scales[:, 0] != 255                                      # (codes of a NaN group with keep_nonzero: any, its values are NaN)
            assert torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu()[fine], codes[fine])
            assert torch.equal(torch.nan_to_num(mx8.dequantize(q).cpu().double(), nan=7.0), torch.nan_to_num(vals, nan=7.0))


def test_quantize_unaligned_strided_and_empty():
    from diffalign_amd import mx8
    x = act(33, 64, torch.float32, 3)
    base = torch.zeros(33 * 64 + 3, device=D_)
    for off in (1, 2, 3):                                                  # addresses off the 16-byte grid
        v = base[off:off + 33 * 64].view(33, 64)
        v.copy_(x)
        assert torch.equal(mx8.quantize(v).codes.cpu(), Q.quantize(x)[0])
    assert torch.equal(mx8.quantize(x.to(D_).t()).codes.cpu(), Q.quantize(x.t().contiguous())[0])
    e = mx8.quantize(torch.empty(0, 5, 64, device=D_))
    assert e.codes.shape == (0, 5, 64) and e.scales.shape == (0, 5, 2) and mx8.dequantize(e).shape == (0, 5, 64)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('p', [0.0, 0.25])
def test_relu_dropout_bwd(dtype, p):
    """dy scaled by the dropout's factor where the forward result was not zero, however small it was."""
    from diffalign_amd import mx8, _lib as L
    for shape in ((17, 64), (5, 33)):
        h = act(*shape, dtype, 5, relu=True)
        h[3, 4] = 1e-20                                                     # far below its group's step
        dy = act(*shape, dtype, 6)
        q = mx8.quantize(h.to(D_), keep_nonzero=True)
        got = mx8.relu_dropout_bwd(q, dy.to(D_), p)
        if dy.numel() % 4 == 0:
            want = torch.empty_like(dy, device=D_)
            hd, dyd = h.to(D_), dy.to(D_)
            L.check(L.lib().da_relu_dropout_bwd(L.ptr(hd), L.ptr(dyd), L.ptr(want), int(dtype == torch.bfloat16), dy.numel(), p, L.stream()), 'bwd')
            assert torch.equal(got, want)
        scale = 65536 / (65536 - int(p * 65536 + 0.5))
        want = torch.where(h != 0, dy.double() * scale, 0.0)
        # three roundings: the factor 65536 / (65536 - t) to fp32 (2^-24), its product with dy (2^-24), the result to its type (eps / 2)
        bound = torch.finfo(dtype).eps / 2 + 2.01 * 2.0 ** -24
        assert bool(((got.cpu().double() - want).abs() <= bound * want.abs()).all())


SHAPES = [(i, o) for i in (32, 64, 128, 256) for o in (32, 64, 128, 256) if i * o <= 64 * 256]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: f'{s[0]}-{s[1]}')
def test_linear_wgrad(shape, dtype):
    from diffalign_amd import mx8
    i, o = shape
    for R in (1, 2, 31, 33, 64, 200, 3001):
        codes, scales, x = Q.quantize(act(R, i, torch.float32, R))
        dy = act(R, o, dtype, R + 1)
        q = mx8.Mx8(codes.to(D_), scales.to(D_))
        dW, db = mx8.linear_wgrad(q, dy.to(D_))
        dyd = dy.double()
        tol = 112 * 2.0 ** -23
        want, S = dyd.t() @ x, dyd.abs().t() @ x.abs()
        assert ((dW.cpu().double() - want).abs() <= tol * S).all(), (R, float(((dW.cpu().double() - want).abs() / (S + 1e-300)).max()))
        assert ((db.cpu().double() - dyd.sum(0)).abs() <= tol * dyd.abs().sum(0)).all(), R
        again = mx8.linear_wgrad(q, dy.to(D_))
        assert torch.equal(dW, again[0]) and torch.equal(db, again[1])       # no order-dependent sums


def test_linear_wgrad_many_rows_and_nonfinite():
    """Slices of several tiles; an infinite and a NaN gradient reach exactly their own row of dW and element of db."""
    from diffalign_amd import mx8
    R, i, o = 70_001, 64, 64
    codes, scales, x = Q.quantize(act(R, i, torch.float32, 1))
    dy = act(R, o, torch.float32, 2)
    dW, db = mx8.linear_wgrad(mx8.Mx8(codes.to(D_), scales.to(D_)), dy.to(D_))
    S = dy.double().abs().t() @ x.abs()
    assert ((dW.cpu().double() - dy.double().t() @ x).abs() <= (320 + 48) * 2.0 ** -23 * S).all()      # slices of 320 rows
    dy[40_000, 3], dy[5, 7] = float('inf'), float('nan')
    dW, db = mx8.linear_wgrad(mx8.Mx8(codes.to(D_), scales.to(D_)), dy.to(D_))
    ok = torch.ones(o, dtype=torch.bool); ok[3] = ok[7] = False
    assert torch.isfinite(dW.cpu()[ok]).all() and torch.isfinite(db.cpu()[ok]).all()
    assert torch.isinf(db[3]) and torch.isnan(db[7]) and torch.isnan(dW[7]).all() and not torch.isfinite(dW[3]).any()


def test_offsets_past_32_bits():
    """2.1e9 elements: the last rows of a large tensor through every kernel equal the same rows alone."""
    from diffalign_amd import mx8
    R, D = (1 << 23) + 5, 256
    x = torch.zeros(R, D, dtype=torch.bfloat16, device=D_)
    tail = act(9, D, torch.bfloat16, 1).to(D_)
    x[-9:] = tail
    q = mx8.quantize(x)
    one = mx8.quantize(tail)
    assert torch.equal(q.codes[-9:], one.codes) and torch.equal(q.scales[-9:], one.scales) and int(q.scales[:-9].max()) == 27
    del x
    assert torch.equal(mx8.dequantize(q, torch.bfloat16)[-9:], mx8.dequantize(one, torch.bfloat16))
    dy = torch.zeros(R, 64, dtype=torch.bfloat16, device=D_)
    dt = act(9, 64, torch.bfloat16, 2).to(D_)
    dy[-9:] = dt
    got, want = mx8.linear_wgrad(q, dy), mx8.linear_wgrad(one, dt)
    # nine rows in one 16-row step of the matrix instruction, or in two: the same nine products in another order
    S = dt.double().abs().t() @ mx8.dequantize(one).double().abs()
    assert bool(((got[0] - want[0]).abs().double() <= 16 * 2.0 ** -23 * S).all())
    h = mx8.relu_dropout_bwd(mx8.Mx8(q.codes[:, :64].contiguous(), q.scales[:, :2].contiguous()), dy, 0.0)
    assert torch.equal(h[-9:], torch.where(one.codes[:, :64] != 0, dt, torch.zeros_like(dt)))


def test_other_stream_and_captured_graphs():
    """Two captured passes (quantise, weight gradient, restore) replayed in turn and side by side, with eager work between."""
    from diffalign_amd import mx8
    sets = []
    for seed in (1, 2):
        x, dy = act(3000, 64, torch.bfloat16, seed).to(D_), act(3000, 128, torch.bfloat16, seed + 5).to(D_)

        def step(x, dy):
            q = mx8.quantize(x)
            return (mx8.dequantize(q),) + mx8.linear_wgrad(q, dy)
        want = step(x, dy)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = step(x, dy)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step(x, dy)
        sets.append((graph, out, want, s, x, dy))
    for k in range(3):
        for graph, out, *_ in sets:
            for o in out: o.zero_()
        torch.cuda.synchronize()
        for graph, out, want, s, *_ in sets:
            with torch.cuda.stream(s): graph.replay()
        torch.cuda.synchronize()
        for graph, out, want, *_ in sets:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        torch.randn(1 << 20, device=D_).sum()
        torch.cuda.synchronize()
