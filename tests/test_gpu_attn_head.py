"""GPU: per-head edge attention (csrc/k_attn_head.hip), forward and gradients, against its definition in 64 bits within the elementwise
bounds that attn_head_oracle.bounds derives from the roundings."""
import math

import pytest
import torch

from tests import attn_head_oracle as O

pytestmark = pytest.mark.gpu
D_ = 'cuda:0'
NAMES = ('Y', 'wV', 'dQ', 'dK', 'dV', 'dE1', 'dE2')


def inputs(B, n, dx, dtype, seed, groups, real=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    nm = torch.rand(B, n, generator=g) < 0.8 if real is None else torch.arange(n)[None] < torch.tensor(real)[:, None]
    gr = torch.randint(-1, 3, (B, n), generator=g) if groups else None
    t = [r(B, n, dx), r(B, n, dx), r(B, n, dx), (r(B, n, n, dx) * 0.5).to(dtype), (r(B, n, n, dx) * 0.5).to(dtype)]
    return t, nm, gr, (r(B, n, n, dx) * 0.3).to(dtype), r(B, n, dx)


def run(t, nm, gr, dY, dwV, H, cap, ckpt):
    from diffalign_amd.autograd_ops import head_attention
    leaves = [x.to(D_).requires_grad_(True) for x in t]
    Y, wV = head_attention(*leaves, nm.to(D_), H, cap=cap, groups=None if gr is None else gr.to(D_), checkpoint=ckpt)
    return (Y, wV) + torch.autograd.grad((Y, wV), leaves, (dY.to(D_), dwV.to(D_)))


def check(t, nm, gr, dY, dwV, H, cap, ckpt, tag=''):
    got = run(t, nm, gr, dY, dwV, H, cap, ckpt)
    d = [x.double() for x in t]
    held = O.held(t[3]) if ckpt == 'mx8' else None
    Y, wV, _, _ = O.forward(*d, nm, H, cap, gr)
    want = [Y, wV] + O.gradients(*d, nm, H, dY.double(), dwV.double(), cap, gr, held)
    out_eps = torch.finfo(t[3].dtype).eps / 2
    for name, a, b, tol in zip(NAMES, got, want, O.bounds(*d, nm, H, dY.double(), dwV.double(), out_eps, cap, gr, held)):
        err = (a.detach().cpu().double() - b).abs()
        assert bool((err <= tol + 1e-30).all()), (tag, name, float((err / (tol + 1e-30)).max()))
    return got


SHAPES = [(256, 8), (64, 4), (32, 8), (96, 3), (192, 6), (40, 5), (128, 1), (512, 8), (512, 4), (8, 1), (4, 1), (256, 64)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('dx,H', SHAPES)
def test_forward_and_gradients(dx, H, dtype):
    """Head widths 4 to 128, one node to more than the row and key tiles, with and without groups (rows that no key is left for), a cap and
    the 8-bit copy of E1."""
    seed = 0
    for B, n in ((1, 1), (2, 3), (3, 17), (1, 66)):
        for gr, cap, ckpt in ((False, 0.0, 'none'), (True, 6.5, 'none'), (True, 0.0, 'mx8' if dx % 32 == 0 else 'none')):
            seed += 1
            check(*inputs(B, n, dx, dtype, seed, gr), H, cap, ckpt, (B, n, gr, cap, ckpt))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('B,n', [(16, 140), (2, 300), (40, 53)])
def test_sizes_of_use(B, n, dtype):
    """Batches that take the wide row tiles, several row blocks and key chunks.  The oracle runs on three of the graphs."""
    from diffalign_amd.autograd_ops import head_attention
    dx, H, ckpt = 256, 8, 'mx8' if n != 53 else 'none'
    t, nm, gr, dY, dwV = inputs(B, n, dx, dtype, n, n == 300, real=[n - 3 * b % (n // 2) for b in range(B)])
    got = run(t, nm, gr, dY, dwV, H, 30.0, ckpt)
    with torch.no_grad():
        Y, wV = head_attention(*[x.to(D_) for x in t], nm.to(D_), H, cap=30.0, groups=None if gr is None else gr.to(D_))
    assert torch.equal(Y, got[0]) and torch.equal(wV, got[1])              # the same forward without a backward
    for b in sorted({0, B // 2, B - 1})[:1 if n == 300 else 3]:
        s = slice(b, b + 1)
        d = [x[s].double() for x in t]
        g1 = None if gr is None else gr[s]
        held = O.held(t[3][s]) if ckpt == 'mx8' else None
        Y, wV, _, _ = O.forward(*d, nm[s], H, 30.0, g1)
        want = [Y, wV] + O.gradients(*d, nm[s], H, dY[s].double(), dwV[s].double(), 30.0, g1, held)
        tol = O.bounds(*d, nm[s], H, dY[s].double(), dwV[s].double(), torch.finfo(dtype).eps / 2, 30.0, g1, held)
        for name, a, w, x in zip(NAMES, got, want, tol):
            err = (a[s].detach().cpu().double() - w).abs()
            assert bool((err <= x + 1e-30).all()), (b, name, float((err / (x + 1e-30)).max()))
    again = run(t, nm, gr, dY, dwV, H, 30.0, ckpt)
    assert all(torch.equal(a, b) for a, b in zip(got, again))              # no order-dependent sums


def test_what_is_masked_is_not_looked_at():
    """NaN and infinities in E1, E2 of masked pairs, in V of keys outside the group, and everywhere in rows without a key."""
    t, nm, gr, dY, dwV = inputs(2, 21, 64, torch.float32, 3, True)
    want = check(t, nm, gr, dY, dwV, 4, 0.0, 'none')
    bad = [x.clone() for x in t]
    pm = nm[:, :, None] & nm[:, None, :]
    bad[3][~pm] = float('nan'); bad[4][~pm] = float('inf')
    bad[2][gr < 0] = float('nan')
    for ckpt in ('none', 'mx8'):
        got = run(bad, nm, gr, dY, dwV, 4, 0.0, ckpt)
        for name, a, b in zip(NAMES, got, want):
            if ckpt == 'none' or name not in ('dQ', 'dK'):
                assert torch.equal(a, b), (ckpt, name)
            else:
                assert torch.isfinite(a).all()
    empty = run(t, nm, torch.full_like(gr, -1), dY, dwV, 4, 5.0, 'none')   # no row has a key
    assert (empty[1] == 0).all() and (empty[4] == 0).all() and torch.isfinite(empty[2]).all()
    assert torch.equal(empty[6], torch.where(pm.to(D_)[..., None], dY.to(D_), torch.zeros((), device=D_)))


def test_bias_of_lowest_value_and_minus_infinity():
    """A bias that shuts keys out: -inf, and the type's lowest value, whose sum over a head overflows to -inf; a row with no key left gets 0."""
    for dtype in (torch.float32, torch.bfloat16):
        for shut in (float('-inf'), torch.finfo(dtype).min):
            t, nm, _, dY, dwV = inputs(1, 9, 64, dtype, 5, False)
            nm[:] = True
            t[4][0, :, 4] = shut                                            # nobody sees key 4
            t[4][0, 2] = shut                                               # row 2 sees nothing
            dY[0, :, 4] = 0; dY[0, 2] = 0
            got = run(t, nm, None, dY, dwV, 4, 0.0, 'none')
            nan = [x.clone() for x in t]
            nan[2][0, 4] = float('nan')                                     # what a shut key's V holds has no effect
            assert all(torch.equal(a, b) for a, b in zip(run(nan, nm, None, dY, dwV, 4, 0.0, 'none'), got))
            assert (got[1][0, 2] == 0).all() and torch.isfinite(got[1]).all()
            assert all(torch.isfinite(x).all() for x in got[2:]) and (got[4][0, 4] == 0).all()
            keep = [j for j in range(9) if j != 4]
            rows = [i for i in range(9) if i not in (2, 4)]
            sub = [t[0][:, rows], t[1][:, keep], t[2][:, keep]]
            q, k, v = (x.double().reshape(x.shape[1], 4, 16) for x in sub)
            e1, e2 = (x[0][rows][:, keep].double().reshape(len(rows), 8, 4, 16) for x in t[3:])
            S = (torch.einsum('ihc,jhc->ijhc', q, k) / 4 * (1 + e1) + e2).sum(-1)
            w = torch.einsum('ijh,jhc->ihc', torch.softmax(S, 1), v).reshape(len(rows), 64)
            assert (got[1][0, rows].cpu().double() - w).abs().max() <= 1e-5 * w.abs().max()


def test_strides_alignment_and_types_of_masks():
    from diffalign_amd.autograd_ops import head_attention
    t, nm, gr, dY, dwV = inputs(2, 13, 64, torch.bfloat16, 8, True)
    want = run(t, nm, gr, dY, dwV, 4, 0.0, 'none')
    dev = [x.to(D_) for x in t]
    odd = []
    for x in dev:                                                           # addresses off the 16-byte grid
        base = torch.empty(x.numel() + 1, dtype=x.dtype, device=D_)
        v = base[1:].view(x.shape)
        v.copy_(x)
        odd.append(v.requires_grad_(True))
    odd[1] = dev[1].transpose(1, 2).contiguous().transpose(1, 2).requires_grad_(True)
    odd[3] = dev[3].transpose(1, 2).contiguous().transpose(1, 2).requires_grad_(True)
    Y, wV = head_attention(*odd, nm.to(D_).to(torch.uint8), 4, groups=gr.to(D_).to(torch.int64))
    grads = torch.autograd.grad((Y, wV), odd, (dY.to(D_).transpose(1, 2).contiguous().transpose(1, 2), dwV.to(D_)))
    assert all(torch.equal(a, b) for a, b in zip((Y, wV) + grads, want))
    # one vector for all: a gradient of stride 0; shared inputs get the sum of their gradients
    leaves = [x.clone().requires_grad_(True) for x in dev]
    Y, wV = head_attention(*leaves, nm.to(D_), 4, groups=gr.to(D_))
    one = torch.autograd.grad((Y.float().sum() + wV.sum()), leaves)
    two = run(t, nm, gr, torch.ones_like(dY), torch.ones_like(dwV), 4, 0.0, 'none')[2:]
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    x = dev[0].clone().requires_grad_(True)
    e = dev[3].clone().requires_grad_(True)
    Y, wV = head_attention(x, x, x, e, e, nm.to(D_), 4)
    gx, ge = torch.autograd.grad((Y, wV), (x, e), (dY.to(D_), dwV.to(D_)))
    p = [dev[0].clone().requires_grad_(True) for _ in range(3)] + [dev[3].clone().requires_grad_(True) for _ in range(2)]
    Y, wV = head_attention(*p, nm.to(D_), 4)
    g = torch.autograd.grad((Y, wV), p, (dY.to(D_), dwV.to(D_)))
    assert torch.allclose(gx, g[0] + g[1] + g[2], rtol=1e-6, atol=1e-6) and torch.allclose(ge.float(), (g[3].float() + g[4].float()), rtol=2e-2, atol=1e-2)
    empty = head_attention(*[x[:0] for x in dev], nm.to(D_)[:0], 4)
    assert empty[0].shape == (0, 13, 13, 64) and empty[1].shape == (0, 13, 64)
    none = head_attention(dev[0][:, :0], dev[1][:, :0], dev[2][:, :0], dev[3][:, :0, :0], dev[4][:, :0, :0], nm.to(D_)[:, :0], 4)
    assert none[0].shape == (2, 0, 0, 64)


def test_other_stream_and_captured_graphs():
    """A call on a side stream; two captured training passes replayed in turn and on two streams at once, with eager work in between."""
    from diffalign_amd.autograd_ops import head_attention
    sets = []
    for seed in (1, 2):
        t, nm, gr, dY, dwV = inputs(3, 45, 64, torch.bfloat16, seed, True)
        want = run(t, nm, gr, dY, dwV, 4, 20.0, 'mx8')
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = run(t, nm, gr, dY, dwV, 4, 20.0, 'mx8')
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        st = [x.to(D_).requires_grad_(True) for x in t]
        aux = (nm.to(D_), gr.to(D_).to(torch.int32), dY.to(D_), dwV.to(D_))

        def step():
            Y, wV = head_attention(*st, aux[0], 4, cap=20.0, groups=aux[1], checkpoint='mx8')
            return (Y, wV) + torch.autograd.grad((Y, wV), st, (aux[2], aux[3]))
        with torch.cuda.stream(s):
            for _ in range(2):
                del got
                got = step()
            del got
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step()
        sets.append((graph, out, want, (st, aux), s))                       # (a graph reads its inputs where they were: they are kept)
    for k in range(3):
        for graph, out, want, st, s in sets:
            for o in out: o.detach().zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        eager = torch.randn(1 << 20, device=D_).sum()
        torch.cuda.synchronize()
        for graph, out, want, st, s in sets:
            for o in out: o.detach().zero_()
        torch.cuda.synchronize()
        for graph, out, want, st, s in sets:
            with torch.cuda.stream(s): graph.replay()
        torch.cuda.synchronize()
        for graph, out, want, st, s in sets:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        del eager


def test_offsets_past_32_bits():
    """2.6e9 pair-channels: the last graph of a large batch equals the same graph alone."""
    from diffalign_amd.autograd_ops import head_attention
    B, n, dx, H = 64, 400, 256, 8
    g = torch.Generator(device=D_).manual_seed(0)
    Q, K, V = (torch.randn(B, n, dx, device=D_, generator=g) for _ in range(3))
    E1 = torch.empty(B, n, n, dx, dtype=torch.bfloat16, device=D_).normal_(generator=g)
    E2 = torch.empty_like(E1).normal_(generator=g)
    nm = torch.ones(B, n, dtype=torch.bool, device=D_)
    dY, dwV = torch.empty_like(E1).normal_(generator=g), torch.randn(B, n, dx, device=D_, generator=g)
    leaves = [x.requires_grad_(True) for x in (Q, K, V, E1, E2)]
    Y, wV = head_attention(*leaves, nm, H, cap=30.0, checkpoint='mx8')
    big = (Y, wV) + torch.autograd.grad((Y, wV), leaves, (dY, dwV))
    one = [x.detach()[-1:].clone().requires_grad_(True) for x in leaves]
    y1, w1 = head_attention(*one, nm[-1:], H, cap=30.0, checkpoint='mx8')
    small = (y1, w1) + torch.autograd.grad((y1, w1), one, (dY[-1:], dwV[-1:]))
    for name, a, b in zip(NAMES, big, small):
        a, b = a.detach()[-1].float(), b.detach()[0].float()
        # another batch size takes other tiles: Y is the same expression, the sums over keys round differently.  Each of the two is within
        # eps = (n + 32 + 4 spread) U = 3.5e-5 (spread of the scores under 40) of sum P |V|, which is at most about 10 times the result's norm
        # here: 1e-3 covers both; dE1, dE2 differ where that moves a rounding to bf16, by one step of 2^-7
        if name == 'Y':
            assert torch.equal(a, b)
        else:
            assert bool((a - b).norm() <= (2.0 ** -7 if name in ('dE1', 'dE2') else 1e-3) * b.norm()), (name, float((a - b).norm() / b.norm()))


def test_second_derivative_is_refused():
    """Differentiable once: under create_graph the gradients come out as ever, and refuse to be differentiated again."""
    from diffalign_amd.autograd_ops import head_attention
    t, nm, gr, dY, dwV = inputs(1, 7, 64, torch.float32, 4, False)
    want = run(t, nm, None, dY, dwV, 4, 0.0, 'none')
    leaves = [x.to(D_).requires_grad_(True) for x in t]
    Y, wV = head_attention(*leaves, nm.to(D_), 4)
    grads = torch.autograd.grad((Y, wV), leaves, (dY.to(D_), dwV.to(D_)), create_graph=True)
    assert all(torch.equal(a.detach(), b) for a, b in zip(grads, want[2:]))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grads[0].sum(), leaves[3])
