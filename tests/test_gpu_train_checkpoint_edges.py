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


@pytest.mark.parametrize('dims', [TINY, FULL], ids=['tiny', 'full'])
def test_improved_inference_under_a_callers_autocast(dims, monkeypatch):
    """bf16 autocast around the model: the per-head attention runs on bf16 E1 and E2 without 8 bits, and the logits are those of the fp32 forward at the
    tolerance of the mixed-precision step (3e-2 of the largest, tests/test_gpu_train_checkpoint.py); without autocast it stays fp32, also where
    training is set to bf16."""
    from diffalign_amd import train_forward as TF
    m = build(dims, True, score_cap=4.0, attn_scope='side')
    ins, gX, gE = case(dims)
    seen, head = [], TF.head_attention

    def watch(Q, K, V, E1, *a, **k):
        seen.append((E1.dtype, k.get('checkpoint')))
        return head(Q, K, V, E1, *a, **k)
    monkeypatch.setattr(TF, 'head_attention', watch)
    m.eval()
    with torch.no_grad():
        want = m(*ins)[:2]
        assert seen == [(torch.float32, 'none')] * len(m.tf_layers)
        del seen[:]
        with torch.autocast('cuda', dtype=torch.bfloat16):
            got = m(*ins)[:2]
    assert seen == [(torch.bfloat16, 'none')] * len(m.tf_layers)
    for a, b in zip(got, want):
        assert float((a.float() - b).abs().max()) <= 3e-2 * float(b.abs().max())
    # the same in a training step: forward and backward of the bf16 kernels, against the fp32 step (1.5e-1 of a whole gradient, same place)
    m.train()
    want = step(m, ins, gX, gE)[2]
    del seen[:]
    with torch.autocast('cuda', dtype=torch.bfloat16):
        Xo, Eo, _, _ = m(*ins)
    got = torch.autograd.grad((Xo, Eo), list(m.parameters()), (gX.to(Xo.dtype), gE.to(Eo.dtype)), allow_unused=True)
    assert seen == [(torch.bfloat16, 'none')] * len(m.tf_layers)
    for (name, _), a, b in zip(m.named_parameters(), got, want):
        if a is not None and float(b.norm()) > 0:
            assert float((a.float() - b).norm()) <= 1.5e-1 * float(b.norm()) + 1e-6, (name, float((a - b).norm() / b.norm()))
    del seen[:]
    m.train_precision = 'bf16'
    m(*ins)
    assert seen == [(torch.float32, 'none')] * len(m.tf_layers)
    del seen[:]
    m.train_checkpoint = 'mx8'
    m(*ins)
    assert seen == [(torch.bfloat16, 'mx8')] * len(m.tf_layers)
