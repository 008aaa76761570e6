"""GPU: the training step with 8-bit activations (module.train_checkpoint = 'mx8') and the per-head attention (improved=True) as the model
runs them: the Linears, the feed-forward branch, whole models against the same step with the rounding written out in torch, replayed from a
HIP graph, the bytes that are kept, and the attention's scope and cap."""
import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from tests import mx8_oracle as Q8
from tests.test_gpu_denoiser import FULL, TINY, IN_DIMS, OUT_DIMS, inputs

pytestmark = pytest.mark.gpu
D_ = 'cuda:0'
SUM = 112 * 2.0 ** -23               # tests/test_gpu_mx8.py: sums of a weight gradient at these row counts


def held(x, keep=False):
    return Q8.quantize(x.reshape(-1, x.shape[-1]), keep)[2]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('p', [0.0, 0.25])
def test_linear_and_feed_forward(dtype, p):
    """Outputs are those of the full-width form, bit for bit; the gradients are the formulas' with x and h as 8 bits hold them."""
    from diffalign_amd import autograd_ops as A, mx8
    g = torch.Generator().manual_seed(3)
    lin1, lin2 = nn.Linear(64, 128).to(D_), nn.Linear(128, 64).to(D_)
    x = torch.randn(2, 11, 11, 64, generator=g).to(dtype).to(D_)
    gy = torch.randn(2, 11, 11, 64, generator=g).to(dtype).to(D_)
    gz = torch.randn(2, 11, 11, 128, generator=g).to(dtype).to(D_)
    seed = torch.tensor([77], dtype=torch.int64, device=D_)
    # one Linear
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    out = A.wide_linear(lin1, a, held=mx8.quantize(a))
    ref = A.wide_linear(lin1, b)
    assert torch.equal(out, ref)
    dx, dW, db = torch.autograd.grad(out, (a, lin1.weight, lin1.bias), gz)
    rx, _, _ = torch.autograd.grad(ref, (b, lin1.weight, lin1.bias), gz)
    assert torch.equal(dx, rx)
    dy, xh = gz.reshape(-1, 128).cpu().double(), held(x)
    assert bool(((dW.cpu().double() - dy.t() @ xh).abs() <= SUM * (dy.abs().t() @ xh.abs())).all())
    assert bool(((db.cpu().double() - dy.sum(0)).abs() <= SUM * dy.abs().sum(0)).all())
    # the branch
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    act = (seed if p else None, 5, p)
    out = A.feed_forward(lin1, lin2, a, act, 'mx8')
    ref = A.feed_forward(lin1, lin2, b, act, 'none')
    assert torch.equal(out, ref)
    params = (lin1.weight, lin1.bias, lin2.weight, lin2.bias)
    got = torch.autograd.grad(out, (a,) + params, gy)
    want = torch.autograd.grad(ref, (b,) + params, gy)
    assert torch.equal(got[0], want[0])                                    # the mask is exact, dX sees no rounding
    with torch.no_grad():
        w2 = lin2.weight.to(dtype)
        h = A._relu_dropout_(F.linear(x, lin1.weight.to(dtype), lin1.bias.to(dtype)), *act)
        dh = mx8.relu_dropout_bwd(mx8.quantize(h, True), gy @ w2, p)
    y2, hh = gy.reshape(-1, 64).cpu().double(), Q8.quantize(h.reshape(-1, 128), True)[2]
    y1 = dh.reshape(-1, 128).cpu().double()
    for d, u, v in ((got[3], y2, hh), (got[1], y1, xh)):
        assert bool(((d.cpu().double() - u.t() @ v).abs() <= SUM * (u.abs().t() @ v.abs())).all())
    for d, u in ((got[4], y2), (got[2], y1)):
        assert bool(((d.cpu().double() - u.sum(0)).abs() <= SUM * u.abs().sum(0)).all())


@pytest.mark.parametrize('cast', [torch.float16, torch.bfloat16], ids=['fp16', 'bf16'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
def test_callers_autocast_changes_nothing(dtype, cast):
    """Forward and backward inside a caller's autocast: the operands' own types, bit for bit what they are outside."""
    from diffalign_amd import autograd_ops as A, mx8
    torch.manual_seed(3)
    lin1, lin2 = nn.Linear(64, 128).to(D_), nn.Linear(128, 64).to(D_)
    x = torch.randn(2, 9, 9, 64, device=D_).to(dtype)
    gy, gz = torch.randn(2, 9, 9, 64, device=D_).to(dtype), torch.randn(2, 9, 9, 128, device=D_).to(dtype)

    def run():
        a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
        z = A.wide_linear(lin1, a, held=mx8.quantize(a.detach()))
        out = A.feed_forward(lin1, lin2, b, (None, 5, 0.0), 'mx8')
        assert z.dtype == out.dtype == dtype
        return (z, out) + torch.autograd.grad(z, (a, lin1.weight, lin1.bias), gz) + torch.autograd.grad(out, (b, *lin1.parameters(), *lin2.parameters()), gy)
    want = run()
    with torch.autocast('cuda', dtype=cast):
        got = run()
    assert all(torch.equal(p, q) and p.dtype == q.dtype for p, q in zip(got, want))


def build(dims, improved, n_layers=2, **kw):
    from diffalign_amd.transformer_model_with_y import GraphTransformerWithYAtomMapPosEmb
    torch.manual_seed(5)
    return GraphTransformerWithYAtomMapPosEmb(n_layers, IN_DIMS, dims['hidden_mlp_dims'], dims['hidden_dims'], OUT_DIMS, nn.ReLU(), nn.ReLU(), dropout=0.0,
                                              p_to_r_skip_connection=True, p_to_r_init=1.0, alignment_type='correct', improved=improved, **kw).to(D_).train()


def step(m, ins, gX, gE):
    Xo, Eo, _, _ = m(*ins)
    ps = [q for q in m.parameters()]
    return Xo, Eo, torch.autograd.grad((Xo, Eo), ps, (gX, gE), allow_unused=True)


def case(dims, seed=9, B=3, n=19):
    X, E, y, nm, am, pos, mol = inputs(B, n, seed=seed, dx=dims['hidden_dims']['dx'])
    g = torch.Generator().manual_seed(seed + 1)
    gX, gE = torch.randn(B, n, OUT_DIMS['X'], generator=g), torch.randn(B, n, n, OUT_DIMS['E'], generator=g)
    return [t.to(D_) for t in (X, E, y, nm, am, pos, mol)], gX.to(D_), gE.to(D_)


class _RefLinear(torch.autograd.Function):
    """A Linear whose weight gradient takes the given values for x, in torch."""

    @staticmethod
    def forward(ctx, x, w, b, xh):
        ctx.save_for_backward(xh, w)
        return F.linear(x, w, b)

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        d2 = dy.reshape(-1, dy.shape[-1])
        return dy @ w, d2.t() @ x.reshape(-1, x.shape[-1]), d2.sum(0), None


class _RefHead(torch.autograd.Function):
    """Per-head attention whose dQ and dK take E1 as 8 bits hold it: oracle of tests/attn_head_oracle.py on the host."""

    @staticmethod
    def forward(ctx, Q, K, V, E1, E2, nm, H, cap, groups):
        from tests import attn_head_oracle as O
        d = [t.detach().cpu().double() for t in (Q, K, V, E1, E2)]
        gr = None if groups is None else groups.cpu()
        Y, wV, _, _ = O.forward(*d, nm.cpu().bool(), H, cap, gr)
        ctx.save_for_backward(*d, nm.cpu().bool(), gr)
        ctx.meta = (H, cap)
        return Y.float().to(D_), wV.float().to(D_)

    @staticmethod
    def backward(ctx, dY, dwV):
        from tests import attn_head_oracle as O
        *d, nm, gr = ctx.saved_tensors
        H, cap = ctx.meta
        with torch.enable_grad():
            g = O.gradients(*d, nm, H, dY.cpu().double(), dwV.cpu().double(), cap, gr, e1_held=O.held(d[3]))
        return tuple(t.float().to(D_) for t in g) + (None,) * 4


@pytest.mark.parametrize('improved,kw', [(False, {}), (True, {}), (True, dict(score_cap=6.0, attn_scope='side'))], ids=['plain', 'improved', 'improved-cap-side'])
@pytest.mark.parametrize('dims', [TINY, FULL], ids=['tiny', 'full'])
def test_model_gradients(dims, improved, kw, monkeypatch):
    """fp32: logits and every parameter gradient against the same model with the 8-bit rounding of the backward written out in torch: the
    Linears' inputs as the step itself had quantised them, in the order of its calls.  1e-4 relative for a whole gradient, as for the fp32
    training forward against its oracle (tests/test_gpu_backward.py).  improved: 3e-4 -- the oracle quantises its own E1, which in the second
    layer is off by up to 1e-6 of a group's maximum; that moves one code in 1 / (127 * 1e-6) = 8,000 by a step of up to 1 / 63.5 of the maximum, and
    sqrt(1 / 8,000) / 63.5 = 1.8e-4 of what dQ, dK and everything before them is made of, in quadrature."""
    from diffalign_amd import mx8, train_forward as TF
    m = build(dims, improved, **kw)
    ins, gX, gE = case(dims)
    m.train_checkpoint = 'mx8'
    quantize, made = mx8.quantize, []

    def record(x, keep_nonzero=False):
        made.append(quantize(x, keep_nonzero))
        return made[-1]
    monkeypatch.setattr(mx8, 'quantize', record)
    got = step(m, ins, gX, gE)
    assert len(made) == 4 * len(m.tf_layers)

    def lin(l, x, act=None, held=None):
        assert act is None
        return F.linear(x, l.weight, l.bias) if held is None else _RefLinear.apply(x, l.weight, l.bias, mx8.dequantize(held))

    def ffn(l1, l2, x, act, ck):
        xh, hh = (mx8.dequantize(made.pop(0)) for _ in range(2))
        return _RefLinear.apply(F.relu(_RefLinear.apply(x, l1.weight, l1.bias, xh)), l2.weight, l2.bias, hh)
    monkeypatch.setattr(mx8, 'quantize', lambda x, keep_nonzero=False: made.pop(0))
    monkeypatch.setattr(TF, 'wide_linear', lin)
    monkeypatch.setattr(TF, 'feed_forward', ffn)
    monkeypatch.setattr(TF, 'head_attention', lambda Q, K, V, E1, E2, nm, H, cap=0.0, groups=None, checkpoint='none': _RefHead.apply(Q, K, V, E1, E2, nm, H, cap, groups))
    want = step(m, ins, gX, gE)
    assert not made
    for a, b in zip(got[:2], want[:2]):
        assert float((a - b).detach().abs().max()) <= 1e-4 * max(1.0, float(b.detach().abs().max()))
    seen, tol = 0, 3e-4 if improved else 1e-4
    for (name, _), a, b in zip(m.named_parameters(), got[2], want[2]):
        assert (a is None) == (b is None), name
        if a is not None:
            seen += 1
            assert float((a - b).norm()) <= tol * float(b.norm()) + 1e-6, (name, float((a - b).norm() / b.norm()))
    assert seen > 30


@pytest.mark.parametrize('precision', ['fp32', 'bf16'])
def test_plain_block_forward_is_unchanged(precision):
    """The forward of the plain block, and every gradient that no weight of a per-pair Linear is, are those of the full-width form."""
    m = build(FULL, False)
    ins, gX, gE = case(FULL)
    m.train_precision = precision
    from diffalign_amd import autograd_ops
    old, autograd_ops.WIDE_MIN_ROWS = autograd_ops.WIDE_MIN_ROWS, 1
    try:
        m.train_checkpoint = 'none'
        want = step(m, ins, gX, gE)
        m.train_checkpoint = 'mx8'
        got = step(m, ins, gX, gE)
    finally:
        autograd_ops.WIDE_MIN_ROWS = old
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for (name, _), a, b in zip(m.named_parameters(), got[2], want[2]):
        if a is None or any(k in name for k in ('e_mul', 'e_add', 'e_out', 'linE1', 'linE2')):
            continue
        assert float((a - b).norm()) <= 1e-5 * float(b.norm()) + 1e-7, name           # (sums by atomics differ in the last bits)


def test_bf16_improved_close_to_fp32():
    """improved, mixed precision, 8 bits: against its own fp32 form without them, at the tolerance of the mixed-precision step (1.5e-1 of
    a whole gradient, tests/test_gpu_backward.py)."""
    m = build(FULL, True)
    ins, gX, gE = case(FULL)
    want = step(m, ins, gX, gE)
    m.train_precision, m.train_checkpoint = 'bf16', 'mx8'
    got = step(m, ins, gX, gE)
    assert float((got[1] - want[1]).detach().abs().max()) <= 3e-2 * float(want[1].detach().abs().max())
    for (name, _), a, b in zip(m.named_parameters(), got[2], want[2]):
        if a is not None and float(b.norm()) > 0:
            assert float((a - b).norm()) <= 1.5e-1 * float(b.norm()) + 1e-6, (name, float((a - b).norm() / b.norm()))


@pytest.mark.parametrize('improved', [False, True])
def test_captured_training_pass(improved):
    """Forward and backward with dropout off, replayed four times with eager passes and a synchronisation between: the eager gradients."""
    m = build(TINY, improved, score_cap=8.0 if improved else 0.0)
    m.train_checkpoint, m.train_precision = 'mx8', 'bf16'
    ins, gX, gE = case(TINY)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            want = [None if t is None else t.detach().clone() for t in step(m, ins, gX, gE)[2]]
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = step(m, ins, gX, gE)[2]
    for k in range(4):
        for t in out:
            if t is not None: t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for (name, _), a, b in zip(m.named_parameters(), out, want):
            assert (a is None) == (b is None)
            if a is not None:
                assert float((a - b).norm()) <= 1e-5 * float(b.norm()) + 1e-7, (k, name)
        if k == 1:
            with torch.no_grad():
                m(*ins)
            torch.cuda.synchronize()


def test_bytes_kept_for_the_backward():
    """What the backward keeps per pair and layer: the inputs of the projections, of e_out and of the feed-forward's two Linears go from two
    bytes (bf16) to 33 / 32."""
    m = build(FULL, False)
    m.train_precision = 'bf16'
    ins, gX, gE = case(FULL, B=2, n=40)
    kept = {}
    for ck in ('none', 'mx8'):
        m.train_checkpoint = ck
        seen = {}

        def pack(t):
            if t.is_cuda: seen[t.untyped_storage().data_ptr()] = t.untyped_storage().nbytes()
            return t
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            out = m(*ins)
        kept[ck] = sum(seen.values())
        del out
    hd = FULL['hidden_dims']
    pairs, per = 2 * 40 * 40, hd['de'] + hd['dx'] + hd['de'] + hd['dim_ffE']
    expect = len(m.tf_layers) * pairs * per * (2 - 33 / 32)
    assert abs(kept['none'] - kept['mx8'] - expect) <= 0.02 * expect, (kept, expect)


@pytest.mark.parametrize('scope', ['all', 'nodes', 'side'])
def test_scope_and_cap_kernel_equals_torch_form(scope, monkeypatch):
    """improved with a scope and a cap: the kernels against the same block in torch operations, evaluation and gradients (fp32, 1e-4)."""
    from diffalign_amd import train_forward as TF
    m = build(TINY, True, score_cap=4.0, attn_scope=scope)
    ins, gX, gE = case(TINY)
    assert not bool(ins[3].all())                                          # padded nodes are there
    res = []
    for built in (TF.head_attention_built, lambda dx, H: False):
        monkeypatch.setattr(TF, 'head_attention_built', built)
        m.eval()
        with torch.no_grad():
            e = m(*ins)[:2]
        m.train()
        res.append(tuple(e) + step(m, ins, gX, gE)[2])
    for a, b in zip(*res):
        if a is not None:
            assert float((a - b).norm()) <= 1e-4 * float(b.norm()) + 1e-6
    if scope != 'all':                                                     # the scope does something
        other = build(TINY, True, score_cap=4.0)
        other.load_state_dict(m.state_dict())
        with torch.no_grad():
            assert float((other.eval()(*ins)[0] - res[0][0]).abs().max()) > 1e-3


def test_refused_settings():
    m = build(TINY, False)
    ins, gX, gE = case(TINY)
    m.train_checkpoint = '8bit'
    with pytest.raises(ValueError):
        m(*ins)
    m.train_checkpoint, m.train_fused = 'mx8', False
    with pytest.raises(ValueError):
        m(*ins)
    m.train_fused = True
    m.eval()
    with torch.no_grad():
        m(*ins)                                                            # inference keeps nothing: the setting is without meaning there
