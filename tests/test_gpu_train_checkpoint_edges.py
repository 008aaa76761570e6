"""GPU: 8-bit activations and the per-head attention in models they were not drawn for: widths without the fused residual blocks, a caller's autocast."""
import pytest
import torch

from tests.test_gpu_denoiser import FULL, TINY
from tests.test_gpu_train_checkpoint import build, case, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('improved', [False, True], ids=['plain', 'improved'])
@pytest.mark.parametrize('change', [dict(dx=48), dict(de=24), dict(dim_ffE=30), dict(dim_ffX=66)], ids=lambda c: next(iter(c)))
def test_8_bit_activations_are_refused_where_the_blocks_are_not_built(change, improved):
    """Not left out in silence: the setting raises.  Training without it runs (of the widths that LayerNorm's backward has: 48 and 24 are none), and
    so does inference."""
    dims = dict(TINY, hidden_dims=dict(TINY['hidden_dims'], **change))
    m = build(dims, improved)
    ins, gX, gE = case(dims)
    m.train_checkpoint = 'mx8'
    with pytest.raises(ValueError, match='mx8'):
        m(*ins)
    m.train_checkpoint = 'none'
    if not {'dx', 'de'} & set(change):
        assert all(t is None or bool(torch.isfinite(t).all()) for t in step(m, ins, gX, gE)[2])
    if improved:                                                           # (the plain block's inference kernels have widths of their own)
        m.train_checkpoint = 'mx8'
        with torch.no_grad():
            assert bool(torch.isfinite(m.eval()(*ins)[1]).all())
