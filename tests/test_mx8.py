"""CPU: the 8-bit activation format's oracle keeps its promises, and the entry points refuse what they do not take."""
import pytest
import torch

from tests import mx8_oracle as Q


def test_oracle_half_step_and_exact_in_bf16():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 70, generator=g) * torch.exp(4 * torch.randn(50, 1, generator=g))
    codes, scales, vals = Q.quantize(x)
    step = torch.ldexp(torch.ones(50, 3, dtype=torch.float64), scales.int() - 133).repeat_interleave(32, 1)[:, :70]
    assert ((vals - x.double()).abs() <= step / 2).all()
    assert torch.equal(vals.to(torch.bfloat16).double(), vals)
    amax = torch.nn.functional.pad(codes.abs().float(), (0, 26)).reshape(50, 3, 32).amax(-1)
    assert (amax >= 63.5).all() and (amax <= 127).all()                   # the smallest scale that holds the group


def test_refusals():
    from diffalign_amd import mx8, _lib as L
    x = torch.zeros(4, 32)
    q = mx8.Mx8(torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8))
    for call in (lambda: mx8.quantize(x),                                  # no CPU fallback
                 lambda: mx8.quantize(x.double()), lambda: mx8.quantize(x.half()), lambda: mx8.quantize(torch.zeros(())),
                 lambda: mx8.quantize(torch.zeros(3, 0)),
                 lambda: mx8.dequantize(q), lambda: mx8.dequantize(q, torch.float16),
                 lambda: mx8.dequantize(mx8.Mx8(q.codes, torch.zeros(4, 2, dtype=torch.uint8))),
                 lambda: mx8.dequantize(mx8.Mx8(q.codes.int(), q.scales)),
                 lambda: mx8.linear_wgrad(q, torch.zeros(4, 64)),          # on the CPU
                 lambda: mx8.linear_wgrad(q, torch.zeros(5, 64)), lambda: mx8.linear_wgrad(q, torch.zeros(4, 48)),
                 lambda: mx8.linear_wgrad(q, torch.zeros(4, 64, dtype=torch.float64)),
                 lambda: mx8.relu_dropout_bwd(q, torch.zeros(4, 33), 0.1), lambda: mx8.relu_dropout_bwd(q, torch.zeros(4, 32), 0.1)):
        with pytest.raises(L.DiffAlignHipError):
            call()
        L._held.clear()


def test_relu_dropout_refuses_other_types():
    """fp16 (the result of a Linear under a caller's fp16 autocast) would be read and written as twice as many bytes."""
    from diffalign_amd import autograd_ops as A, _lib as L
    for dtype in (torch.float16, torch.float64):
        with pytest.raises(L.DiffAlignHipError, match='fp32 or bf16'):
            A._relu_dropout_(torch.zeros(4, 8, dtype=dtype), None, 0, 0.0)


def test_c_entries_refuse_before_any_launch():
    """Argument checks of the C entry points: they return before anything is launched, so they run without a GPU."""
    from diffalign_amd import _lib as L
    lib = L.lib()
    z = 0
    assert lib.da_mx8_quant(z, 0, z, z, -1, 32, 0, z) == -1 and lib.da_mx8_quant(z, 0, z, z, 1, 0, 0, z) == -1
    assert lib.da_mx8_quant(z, 0, z, z, 1, 32, 0, z) == -1 and b'null' in lib.da_last_error()
    assert lib.da_mx8_quant(18, 0, 16, 16, 1, 32, 0, z) == -1 and b'aligned' in lib.da_last_error()
    assert lib.da_mx8_quant(z, 0, z, z, 0, 32, 0, z) == 0                  # nothing to do
    assert lib.da_mx8_dequant(16, 16, 18, 0, 1, 32, z) == -1 and lib.da_mx8_dequant(z, z, z, 0, 0, 32, z) == 0
    assert lib.da_relu_dropout_bwd_mx8(16, 16, 16, 0, 8, 1.0, z) == -1 and lib.da_relu_dropout_bwd_mx8(z, z, z, 0, 8, 0.1, z) == -1
    assert lib.da_linear_wgrad_mx8_workspace(10, 48, 64) == -1 and lib.da_linear_wgrad_mx8_workspace(10, 256, 128) == -1
    need = lib.da_linear_wgrad_mx8_workspace(10, 64, 256)
    assert need == 4 * (64 * 256 + 256)
    assert lib.da_linear_wgrad_mx8(16, 16, 16, 0, 16, 16, 16, need - 1, 10, 64, 256, z) == -1 and b'workspace' in lib.da_last_error()
    assert lib.da_linear_wgrad_mx8(16, 16, 20, 0, 16, 16, 16, need, 10, 64, 256, z) == -1 and b'aligned' in lib.da_last_error()
    assert lib.da_linear_wgrad_mx8(16, 16, 16, 0, 16, 16, 16, need, 10, 64, 48, z) == -3
    assert lib.da_linear_wgrad_mx8(16, 16, 16, 0, 16, 16, 16, need, 0, 64, 256, z) == -1
