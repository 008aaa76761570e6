"""CPU: the per-head attention of head widths that have no kernel (torch operations) against the 64-bit oracle, where masks, groups and scores
of -inf leave keys out."""
from types import SimpleNamespace as ns

import pytest
import torch

from diffalign_amd import train_forward as TF
from tests import attn_head_oracle as O
from tests.test_attn_head import inputs


def torch_form(t, nm, gr, H, cap):
    B, n, dx = t[0].shape
    em = (nm[:, :, None] & nm[:, None, :]).float()[..., None]
    return TF._head_attention_torch(ns(n_head=H, df=dx // H, score_cap=cap), *[x.float() for x in t], em, gr)


def grads(t, nm, gr, H, cap, dY, dwV):
    leaves = [x.float().requires_grad_(True) for x in t]
    Y, wV = torch_form(leaves, nm, gr, H, cap)
    return [Y.detach(), wV.detach(), *torch.autograd.grad((Y, wV), leaves, (dY.float(), dwV.float()))]


@pytest.mark.parametrize('cap', [0.0, 7.0])
@pytest.mark.parametrize('groups', [False, True])
def test_torch_form_against_the_oracle(groups, cap):
    t, nm, gr, dY, dwV = inputs(2, 9, 12, 2, 3, groups)
    t = [x.float().double() for x in t]
    dY, dwV = dY.float().double(), dwV.float().double()
    Y, wV, _, _ = O.forward(*t, nm, 2, cap, gr)
    want = [Y, wV] + O.gradients(*t, nm, 2, dY, dwV, cap, gr)
    for a, b, tol in zip(grads(t, nm, gr, 2, cap, dY, dwV), want, O.bounds(*t, nm, 2, dY, dwV, 2.0 ** -24, cap, gr)):
        assert bool(((a.double() - b).abs() <= tol + 1e-30).all())


def test_torch_form_does_not_look_at_what_is_left_out():
    """As head_attention: E1, E2 of masked pairs, V of keys outside the group, dwV of rows without a key."""
    t, nm, gr, dY, dwV = inputs(2, 9, 12, 2, 4, True)
    assert not bool(nm.all()) and bool((gr < 0).any())
    want = grads(t, nm, gr, 2, 0.0, dY, dwV)
    pm = nm[:, :, None] & nm[:, None, :]
    t[3][~pm], t[4][~pm], t[2][gr < 0], dwV[gr < 0] = float('nan'), float('inf'), float('nan'), float('inf')
    for a, b in zip(grads(t, nm, gr, 2, 0.0, dY, dwV), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize('groups', [False, True])
@pytest.mark.parametrize('shut', [float('-inf'), torch.finfo(torch.float32).min], ids=['-inf', 'lowest'])
def test_torch_form_shuts_out_scores_of_minus_infinity(shut, groups):
    """A key whose scores are -inf (the type's lowest value sums to it) counts as a key outside the group; a row with no other key gets 0."""
    t, nm, gr, dY, dwV = inputs(1, 7, 12, 2, 5, groups)
    nm[:] = True
    if groups:
        gr[:] = 0
    t[4][0, :, 4], t[4][0, 2] = shut, shut
    dY[0, :, 4], dY[0, 2] = 0, 0
    got = grads(t, nm, gr, 2, 0.0, dY, dwV)
    assert bool((got[1][0, 2] == 0).all()) and all(torch.isfinite(x).all() for x in got[1:])
    assert bool((got[4][0, 4] == 0).all())
    t[2][0, 4], dwV[0, 2] = float('nan'), float('nan')
    again = grads(t, nm, gr, 2, 0.0, dY, dwV)
    assert all(torch.equal(a, b) for a, b in zip(again, got))
    keep, rows = [0, 1, 2, 3, 5, 6], [0, 1, 3, 4, 5, 6]
    q, k, v = (x.double().reshape(x.shape[1], 2, 6) for x in (t[0][:, rows], t[1][:, keep], t[2][:, keep]))
    e1, e2 = (x[0][rows][:, keep].double().reshape(6, 6, 2, 6) for x in t[3:])
    P = torch.softmax((torch.einsum('ihc,jhc->ijhc', q, k) / 6 ** 0.5 * (1 + e1) + e2).sum(-1), 1)
    want = torch.einsum('ijh,jhc->ihc', P, v).reshape(6, 12)
    assert float((got[1][0, rows].double() - want).abs().max()) <= 1e-5 * float(want.abs().max())


def test_c_entries_refuse_more_than_a_launch_holds():
    """2^32 threads and more, which no launch takes: refused before anything is launched, with the sizes in the message."""
    from diffalign_amd import _lib as L
    lib, p = L.lib(), 16
    fwd = lambda B, n: lib.da_attn_head_fwd(p, p, p, p, p, 0, p, 0, 1.0, 0.0, p, p, 0, 0, 0, 0, B, n, 64, 4, 0)
    bwd = lambda B, n: lib.da_attn_head_bwd(p, p, p, p, 0, 0, p, 1.0, 0.0, p, p, p, p, 0, p, p, p, p, p, p, p, 1 << 60, B, n, 64, 4, 0)
    for call, B, n in ((fwd, 1 << 24, 1), (fwd, 1 << 23, 3), (bwd, 1 << 23, 1), (bwd, 1 << 21, 100)):
        assert call(B, n) == -1 and b'launch' in lib.da_last_error() and str(B).encode() in lib.da_last_error()


def test_a_module_pickled_without_the_attentions_options():
    """A whole module that torch.save wrote before the block had a cap and a scope: the reference's arithmetic."""
    import io
    import torch.nn as nn
    from diffalign_amd.transformer_model_with_y import GraphTransformerWithY
    dims = dict(X=16, E=16, y=16)
    m = GraphTransformerWithY(2, dims, dims, dict(dx=16, de=16, dy=16, n_head=2, dim_ffX=16, dim_ffE=16), dims, nn.ReLU(), nn.ReLU(), improved=True)
    for layer in m.tf_layers:
        del layer.self_attn.__dict__['score_cap'], layer.self_attn.__dict__['scope']
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    old = torch.load(f, weights_only=False)
    assert TF._attn_groups(old, torch.ones(2, 3, dtype=torch.bool), None) is None
    t, nm, gr, _, _ = inputs(2, 3, 16, 2, 1, False)
    em = (nm[:, :, None] & nm[:, None, :]).float()[..., None]
    Y, wV = TF._head_attention_torch(old.tf_layers[1].self_attn, *[x.float() for x in t], em, None)
    want = O.forward(*t, nm, 2)
    assert float((Y - want[0]).abs().max()) < 1e-4 and float((wV - want[1]).abs().max()) < 1e-4
