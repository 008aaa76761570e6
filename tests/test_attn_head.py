"""CPU: the per-head attention's 64-bit oracle against differences, and what the entry points refuse."""
import pytest
import torch

from tests import attn_head_oracle as O


def inputs(B, n, dx, H, seed, groups=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    nm = torch.rand(B, n, generator=g) < 0.8
    gr = torch.randint(-1, 2, (B, n), generator=g) if groups else None
    return [r(B, n, dx), r(B, n, dx), r(B, n, dx), r(B, n, n, dx) * 0.5, r(B, n, n, dx) * 0.5], nm, gr, r(B, n, n, dx), r(B, n, dx)


@pytest.mark.parametrize('cap', [0.0, 7.0])
@pytest.mark.parametrize('groups', [False, True])
def test_oracle_gradient_against_differences(cap, groups):
    t, nm, gr, dY, dwV = inputs(2, 5, 16, 2, 1, groups)
    grads = O.gradients(*t, nm, 2, dY, dwV, cap, gr)
    gen = torch.Generator().manual_seed(2)
    L = lambda x: ((lambda Y, wV, S, P: (Y * dY).sum() + (wV * dwV).sum())(*O.forward(*x, nm, 2, cap, gr)))
    for k in range(5):
        d = torch.randn(t[k].shape, generator=gen, dtype=torch.float64)
        h = 1e-6
        up, dn = [x.clone() for x in t], [x.clone() for x in t]
        up[k] += h * d; dn[k] -= h * d
        fd = (L(up) - L(dn)) / (2 * h)
        assert abs(float(fd - (grads[k] * d).sum())) <= 1e-7 * (1 + abs(float(fd)))
    same = O.gradients(*t, nm, 2, dY, dwV, cap, gr, e1_held=t[3])            # held at full width: the same gradients
    for a, b in zip(grads, same):
        assert torch.allclose(a, b, rtol=1e-10, atol=1e-12)


def test_refusals():
    from diffalign_amd import _lib as L
    from diffalign_amd.autograd_ops import head_attention
    z = torch.zeros
    ok = lambda: dict(Q=z(2, 3, 64), K=z(2, 3, 64), V=z(2, 3, 64), E1=z(2, 3, 3, 64), E2=z(2, 3, 3, 64), node_mask=z(2, 3, dtype=torch.bool), n_head=4)
    for bad in (dict(), dict(K=z(2, 4, 64)), dict(Q=z(3, 64)), dict(E1=z(2, 3, 3, 32)), dict(E2=z(2, 3, 3, 64, dtype=torch.bfloat16)),
                dict(E1=z(2, 3, 3, 64).half(), E2=z(2, 3, 3, 64).half()), dict(node_mask=z(2, 4, dtype=torch.bool)), dict(groups=z(2, 4, dtype=torch.int32)),
                dict(groups=z(2, 3)), dict(groups=z(2, 3, dtype=torch.bool)), dict(n_head=5), dict(n_head=64), dict(n_head=0)):
        with pytest.raises(L.DiffAlignHipError):                            # (the first: CPU tensors)
            head_attention(**{**ok(), **bad})
        L._held.clear()
    for bad in (dict(cap=-1.0), dict(cap=float('nan')), dict(cap=float('inf')), dict(cap=1e-38), dict(cap=1e38), dict(checkpoint='8bit')):
        with pytest.raises(ValueError):
            head_attention(**{**ok(), **bad})
    with pytest.raises(L.DiffAlignHipError):
        head_attention(Q=z(1, 2, 40), K=z(1, 2, 40), V=z(1, 2, 40), E1=z(1, 2, 2, 40), E2=z(1, 2, 2, 40), node_mask=z(1, 2), n_head=5, checkpoint='mx8')


def test_c_entries_refuse_before_any_launch():
    from diffalign_amd import _lib as L
    lib = L.lib()
    p = 16                                                                  # an aligned address that nothing reads
    fwd = lambda **k: lib.da_attn_head_fwd(*[{**dict(Q=p, K=p, V=p, E1=p, E2=p, bf=0, nm=p, gr=0, qs=1.0, cap=0.0, Y=p, wV=p, S=0, st=0, c=0, sc=0, B=1, n=3,
                                                      dx=64, H=4, s=0), **k}[x] for x in ('Q', 'K', 'V', 'E1', 'E2', 'bf', 'nm', 'gr', 'qs', 'cap', 'Y', 'wV', 'S',
                                                                                          'st', 'c', 'sc', 'B', 'n', 'dx', 'H', 's')])
    assert fwd(B=-1) == -1 and fwd(H=5) == -3 and fwd(dx=60, H=2) == -3 and fwd(dx=1024, H=32) == -3 and fwd(dx=512, H=128) == -3
    assert fwd(B=0) == 0 and fwd(n=0) == 0
    assert fwd(Q=0) == -1 and fwd(S=p) == -1 and fwd(c=p, sc=p) == -1 and fwd(S=p, st=p, c=p) == -1
    assert fwd(cap=-1.0) == -1 and fwd(cap=float('nan')) == -1 and fwd(cap=1e-38) == -1 and fwd(cap=1e38) == -1 and fwd(E1=24) == -1 and b'unaligned' in lib.da_last_error()
    assert fwd(n=1 << 22) == -1 and b'too large' in lib.da_last_error()
    assert fwd(S=p, st=p, c=p, sc=p, dx=40, H=5) == -1 and b'32' in lib.da_last_error()
    bwd = lambda **k: lib.da_attn_head_bwd(*[{**dict(Q=p, K=p, V=p, E1=p, c=0, sc=0, nm=p, qs=1.0, cap=0.0, wV=p, S=p, st=p, dY=p, bf=0, g=p, dQ=p, dK=p, dV=p, d1=p,
                                                      d2=p, ws=p, nb=0, B=1, n=300, dx=64, H=4, s=0), **k}[x] for x in ('Q', 'K', 'V', 'E1', 'c', 'sc', 'nm', 'qs', 'cap',
                                              'wV', 'S', 'st', 'dY', 'bf', 'g', 'dQ', 'dK', 'dV', 'd1', 'd2', 'ws', 'nb', 'B', 'n', 'dx', 'H', 's')])
    assert lib.da_attn_head_bwd_workspace(1, 300, 64, 4, 0) > 0 and lib.da_attn_head_bwd_workspace(1, 1, 64, 4, 0) == 0
    assert lib.da_attn_head_bwd_workspace(1, 300, 64, 5, 0) == -1 and lib.da_attn_head_bwd_workspace(0, 300, 64, 4, 0) == 0
    assert bwd() == -1 and b'workspace' in lib.da_last_error()
    assert bwd(E1=0) == -1 and bwd(c=p, sc=p) == -1 and bwd(E1=0, c=p) == -1 and bwd(dY=0) == -1 and bwd(H=5) == -3 and bwd(B=0) == 0
    assert bwd(dQ=8) == -1 and b'unaligned' in lib.da_last_error()


def test_model_options_are_checked():
    import torch.nn as nn
    from diffalign_amd.layers import NodeEdgeBlock
    from diffalign_amd.transformer_model_with_y import GraphTransformerWithY
    for kw in (dict(score_cap=3.0), dict(scope='nodes'), dict(improved=True, scope='molecule'), dict(improved=True, score_cap=-1.0),
               dict(improved=True, score_cap=float('inf')), dict(improved=True, score_cap=float('nan'))):
        with pytest.raises(ValueError):
            NodeEdgeBlock(64, 32, 32, 4, **kw)
    blk = NodeEdgeBlock(64, 32, 32, 4, improved=True, score_cap=3.0, scope='side')
    assert blk.score_cap == 3.0 and blk.scope == 'side' and set(blk.state_dict()) == set(NodeEdgeBlock(64, 32, 32, 4).state_dict())
    dims = dict(X=16, E=16, y=16)
    with pytest.raises(ValueError):
        GraphTransformerWithY(1, dims, dims, dict(dx=16, de=16, dy=16, n_head=2, dim_ffX=16, dim_ffE=16), dims, nn.ReLU(), nn.ReLU(), improved=True,
                              attn_scope='side')
