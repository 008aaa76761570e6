"""GPU: per-head edge attention where several of its forms meet, and what non-finite values may reach; bounds as in test_gpu_attn_head.py."""
import pytest
import torch

from tests import attn_head_oracle as O
from tests.test_gpu_attn_head import NAMES, inputs, run

pytestmark = pytest.mark.gpu
D_ = 'cuda:0'


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
