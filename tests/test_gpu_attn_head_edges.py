"""GPU: per-head edge attention where several of its forms meet, and what non-finite values may reach; bounds as in test_gpu_attn_head.py."""
import pytest
import torch

from tests import attn_head_oracle as O
from tests.test_gpu_attn_head import NAMES, inputs, run

pytestmark = pytest.mark.gpu
D_ = 'cuda:0'


def check_graphs(t, nm, gr, dY, dwV, H, cap, ckpt, graphs):
    got = run(t, nm, gr, dY, dwV, H, cap, ckpt)
    for b in graphs:
        s = slice(b, b + 1)
        d = [x[s].double() for x in t]
        g1 = None if gr is None else gr[s]
        held = O.held(t[3][s]) if ckpt == 'mx8' else None
        Y, wV, _, _ = O.forward(*d, nm[s], H, cap, g1)
        want = [Y, wV] + O.gradients(*d, nm[s], H, dY[s].double(), dwV[s].double(), cap, g1, held)
        tol = O.bounds(*d, nm[s], H, dY[s].double(), dwV[s].double(), torch.finfo(t[3].dtype).eps / 2, cap, g1, held)
        for name, a, w, x in zip(NAMES, got, want, tol):
            err = (a[s].detach().cpu().double() - w).abs()
            assert bool((err <= x + 1e-30).all()), (b, name, float((err / (x + 1e-30)).max()))
    return got


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('cap,ckpt', [(0.0, 'none'), (6.5, 'mx8')])
@pytest.mark.parametrize('dx,H', [(64, 4), (96, 3), (256, 8), (512, 8), (256, 64)])
def test_two_rows_a_workgroup_with_groups(dx, H, cap, ckpt, dtype):
    """B ceil(n / 2) >= 512 takes the forward's two-row form; odd n, groups that leave rows without a key, cap and 8-bit E1 in it."""
    from diffalign_amd.autograd_ops import head_attention
    B, n = 40, 27
    assert B * ((n + 1) // 2) >= 512
    t, nm, gr, dY, dwV = inputs(B, n, dx, dtype, dx + H, True)
    gr[0] = -1                                                             # a graph without any key
    gr[1, :-1], gr[1, -1] = -1, 2                                          # one node alone
    got = check_graphs(t, nm, gr, dY, dwV, H, cap, ckpt, (0, 1, 21, B - 1))
    assert bool((got[1][0] == 0).all()) and torch.equal(got[1][1, -1].cpu(), t[2][1, -1])      # a single key: its V
    with torch.no_grad():
        Y, wV = head_attention(*[x.to(D_) for x in t], nm.to(D_), H, cap=cap, groups=gr.to(D_))
    assert torch.equal(Y, got[0]) and torch.equal(wV, got[1])


def test_gradients_of_rows_that_see_nothing():
    """wV of a row without a key is 0 whatever the inputs: what its gradient holds has no effect.  Of a row with keys it has none on the V of
    keys that the row does not see."""
    for dx, H, dtype in ((64, 4, torch.float32), (64, 4, torch.bfloat16), (512, 8, torch.float32)):
        t, nm, gr, dY, dwV = inputs(2, 21, dx, dtype, 3, True)
        assert bool((gr < 0).any()) and bool((gr == 0).any()) and bool((gr == 1).any())
        for ckpt in ('none', 'mx8'):
            dwV[gr < 0] = 0
            want = run(t, nm, gr, dY, dwV, H, 4.0, ckpt)
            for bad in (float('nan'), float('inf')):
                w = dwV.clone()
                w[gr < 0] = bad
                got = run(t, nm, gr, dY, w, H, 4.0, ckpt)
                assert all(torch.equal(a, b) for a, b in zip(got, want)), (ckpt, bad)
                w = dwV.clone()
                w[gr == 0] = bad
                got = run(t, nm, gr, dY, w, H, 4.0, ckpt)
                assert torch.equal(got[4][(gr != 0).to(D_)], want[4][(gr != 0).to(D_)]), (ckpt, bad)
                assert torch.equal(got[2][(gr != 0).to(D_)], want[2][(gr != 0).to(D_)])
                assert not torch.isfinite(got[4][(gr == 0).to(D_)]).all()


def test_non_finite_values_that_are_seen():
    """A NaN in E1 or E2 of an unmasked pair, or in V of a visible key, reaches what the formulas make of it and nothing else."""
    B, n, dx, H = 2, 13, 64, 4
    t, nm, _, dY, dwV = inputs(B, n, dx, torch.float32, 9, False)
    nm[:] = True
    clean = run(t, nm, None, dY, dwV, H, 0.0, 'none')
    for which, where in ((3, (0, 5, 7, 33)), (4, (0, 5, 7, 33)), (2, (0, 7, 33))):
        bad = [x.clone() for x in t]
        bad[which][where] = float('nan')
        got = run(bad, nm, None, dY, dwV, H, 0.0, 'none')
        d = [x.double() for x in bad]
        Y, wV, _, _ = O.forward(*d, nm, H)
        want = [Y, wV] + O.gradients(*d, nm, H, dY.double(), dwV.double())
        for name, a, c, w in zip(NAMES, got, clean, want):
            a, c, hit = a.detach().cpu(), c.detach().cpu(), w.isnan()
            assert torch.equal(a.isnan(), hit), (which, name)
            assert hit[1].sum() == 0 and torch.equal(a[1], c[1])          # the other graph: the same bits
            if name in ('Y', 'wV'):
                assert torch.equal(a[~hit], c[~hit]) and bool(hit.any()) == (name == 'wV' or which != 2)
    for top in (float('inf'), 3.0e38):                                     # an infinite score: NaN, as a softmax has it; 16 of 3e38 sum to one
        bad = [x.clone() for x in t]
        bad[4][0, 5, 7, 16:32] = top
        _, wV = run(bad, nm, None, dY, dwV, H, 0.0, 'none')[:2]
        hit = torch.zeros(B, n, dx, dtype=torch.bool)
        hit[0, 5, 16:32] = True
        assert torch.equal(wV.detach().cpu().isnan(), hit)


@pytest.mark.parametrize('grad', [True, False])
def test_forward_mode_is_refused_and_traces_run(grad):
    """Without requires_grad: a dual tensor's tangent is refused, not dropped, and torch.jit.trace records the call."""
    import torch.autograd.forward_ad as fwd
    from diffalign_amd.autograd_ops import head_attention
    t, nm, gr, _, _ = inputs(2, 9, 64, torch.float32, 6, True)
    t, nm, gr = [x.to(D_) for x in t], nm.to(D_), gr.to(D_)
    with torch.set_grad_enabled(grad):
        want = head_attention(*t, nm, 4, groups=gr)
        assert not want[0].requires_grad
        for k in range(5):
            with fwd.dual_level():
                dual = list(t)
                dual[k] = fwd.make_dual(t[k], torch.ones_like(t[k]))
                with pytest.raises(NotImplementedError):
                    head_attention(*dual, nm, 4, groups=gr)
                plain = head_attention(*t, nm, 4, groups=gr)               # no tangent: as ever
            assert all(torch.equal(a, b) for a, b in zip(plain, want))
        traced = torch.jit.trace(lambda *x: head_attention(*x, nm, 4, groups=gr), tuple(t), check_trace=False)
        other = [x + 1 for x in t]
        assert all(torch.equal(a, b) for a, b in zip(traced(*other), head_attention(*other, nm, 4, groups=gr)))
