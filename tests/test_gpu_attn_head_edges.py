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
