"""Activations held in 8 bits between the forward and the backward pass (csrc/k_mx8.hip).

Format: MXINT8 of the OCP microscaling specification.  32 consecutive channels of a row share a power-of-two scale 2^(b - 127), held as one
byte b; an element is an int8 q and stands for q / 64 * 2^(b - 127).  The scale is the smallest at which the group's largest magnitude
still rounds to 127, so a restored value is within half a step, 2^(b - 127) / 128, of the original (at most 1/127 of the group's
largest magnitude); restored values are exact in bfloat16.  Scales go down to 2^-100: smaller values round to zero at that step.  A
group that holds an infinity or NaN is restored as NaN.  D channels take D + ceil(D / 32) bytes.

The reference keeps every activation at full width for `loss.backward()` (training/helpers.py:139-142); the callers here are the training
forward's per-pair Linears and the per-head attention core (train_forward.py, `train_checkpoint = 'mx8'`)."""
from __future__ import annotations

import contextlib
from typing import NamedTuple, Tuple

import torch

from . import _lib as L

GROUP = 32
# (in, out) features da_linear_wgrad_mx8 is built for
WGRAD_SHAPES = frozenset((i, o) for i in (32, 64, 128, 256) for o in (32, 64, 128, 256) if i * o <= 64 * 256)
_DTYPES = (torch.float32, torch.bfloat16)


class Mx8(NamedTuple):
    codes: torch.Tensor       # int8 (..., D)
    scales: torch.Tensor      # uint8 (..., ceil(D / 32))


def on_device_of(t: torch.Tensor):
    """Launches go to the tensor's device, also where it is not the current one."""
    return contextlib.nullcontext() if not t.is_cuda or t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _check(q: Mx8) -> Mx8:
    codes, scales = q
    if codes.dtype != torch.int8 or scales.dtype != torch.uint8:
        raise L.DiffAlignHipError(f'mx8: codes int8 and scales uint8 expected, got {codes.dtype} and {scales.dtype}')
    if codes.dim() < 1 or scales.shape != codes.shape[:-1] + (-(-codes.shape[-1] // GROUP),):
        raise L.DiffAlignHipError(f'mx8: scales {tuple(scales.shape)} do not belong to codes {tuple(codes.shape)} (one byte for {GROUP} channels)')
    if scales.device != codes.device:
        raise L.DiffAlignHipError(f'mx8: codes on {codes.device}, scales on {scales.device}')
    return Mx8(codes.contiguous(), scales.contiguous())


def quantize(x: torch.Tensor, keep_nonzero: bool = False) -> Mx8:
    """x (..., D) fp32 or bf16 -> its 8-bit form.  keep_nonzero: an element other than zero keeps a code other than zero (+-1 where it
    would round to 0, an error of up to one step instead of half), so the codes still tell what a ReLU let through
    (relu_dropout_bwd)."""
    if x.dtype not in _DTYPES:
        raise L.DiffAlignHipError(f'mx8.quantize: fp32 or bf16 expected, got {x.dtype}')
    if x.dim() < 1 or x.shape[-1] < 1:
        raise L.DiffAlignHipError(f'mx8.quantize: x needs a channel axis, got shape {tuple(x.shape)}')
    x = x.detach().contiguous()
    D = x.shape[-1]
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty(x.shape[:-1] + (-(-D // GROUP),), dtype=torch.uint8, device=x.device)
    with on_device_of(x):
        L.check(L.lib().da_mx8_quant(L.ptr(x), int(x.dtype == torch.bfloat16), L.ptr(codes), L.ptr(scales), x.numel() // D, D, int(keep_nonzero),
                                     L.stream()), 'da_mx8_quant')
    return Mx8(codes, scales)


def dequantize(q: Mx8, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of an 8-bit activation, fp32 or bf16 (both exact)."""
    if dtype not in _DTYPES:
        raise L.DiffAlignHipError(f'mx8.dequantize: fp32 or bf16, not {dtype}')
    q = _check(q)
    D = q.codes.shape[-1]
    out = torch.empty(q.codes.shape, dtype=dtype, device=q.codes.device)
    if D == 0:
        return out
    with on_device_of(out):
        L.check(L.lib().da_mx8_dequant(L.ptr(q.codes), L.ptr(q.scales), L.ptr(out), int(dtype == torch.bfloat16), out.numel() // D, D, L.stream()),
                'da_mx8_dequant')
    return out


def _aligned(t: torch.Tensor, to: int = 16) -> torch.Tensor:
    t = t.contiguous()
    return t.clone() if t.data_ptr() % to else t


def linear_wgrad(q: Mx8, dy: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dW (out,in), db (out)) fp32 of an nn.Linear whose input x is held in 8 bits: dW = dY^T x, db = column sums of dY.  dy (..., out)
    fp32 or bf16 with q's leading axes; (in, out) of WGRAD_SHAPES."""
    q = _check(q)
    in_f, out_f = q.codes.shape[-1], dy.shape[-1]
    if dy.dtype not in _DTYPES:
        raise L.DiffAlignHipError(f'mx8.linear_wgrad: dy fp32 or bf16, got {dy.dtype}')
    if q.codes.shape[:-1] != dy.shape[:-1] or q.codes.device != dy.device:
        raise L.DiffAlignHipError(f'mx8.linear_wgrad: x {tuple(q.codes.shape)} on {q.codes.device} and dy {tuple(dy.shape)} on {dy.device} do not belong together')
    if (in_f, out_f) not in WGRAD_SHAPES:
        raise L.DiffAlignHipError(f'mx8.linear_wgrad: {in_f} -> {out_f} features not built')
    R = q.codes.numel() // in_f
    dW, db = torch.empty(out_f, in_f, device=dy.device), torch.empty(out_f, device=dy.device)
    if R == 0:
        return dW.zero_(), db.zero_()
    codes, dy = _aligned(q.codes, 8), _aligned(dy.detach())
    with on_device_of(dy):
        ws = torch.empty(L.lib().da_linear_wgrad_mx8_workspace(R, in_f, out_f), dtype=torch.uint8, device=dy.device)
        L.check(L.lib().da_linear_wgrad_mx8(L.ptr(codes), L.ptr(q.scales), L.ptr(dy), int(dy.dtype == torch.bfloat16), L.ptr(dW), L.ptr(db), L.ptr(ws),
                                            ws.numel(), R, in_f, out_f, L.stream()), 'da_linear_wgrad_mx8')
    return dW, db


def relu_dropout_bwd(q: Mx8, dy: torch.Tensor, p: float) -> torch.Tensor:
    """Gradient of h = dropout_p(relu(a)) with respect to a, from h held in 8 bits with keep_nonzero: dy / (1 - p) where h is not zero,
    else 0.  dy fp32 or bf16, of h's shape."""
    q = _check(q)
    if dy.dtype not in _DTYPES or dy.shape != q.codes.shape or dy.device != q.codes.device:
        raise L.DiffAlignHipError(f'mx8.relu_dropout_bwd: dy fp32 or bf16 of shape {tuple(q.codes.shape)} expected, got {dy.dtype} {tuple(dy.shape)} on {dy.device}')
    dy = dy.detach().contiguous()
    dx = torch.empty_like(dy)
    with on_device_of(dy):
        L.check(L.lib().da_relu_dropout_bwd_mx8(L.ptr(q.codes), L.ptr(dy), L.ptr(dx), int(dy.dtype == torch.bfloat16), dy.numel(), float(p), L.stream()),
                'da_relu_dropout_bwd_mx8')
    return dx
