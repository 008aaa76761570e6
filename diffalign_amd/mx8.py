"""Activations held in 8 bits between the forward and the backward pass (csrc/k_mx8.hip).

Format: MXINT8 of the OCP microscaling specification.  32 consecutive channels of a row share a power-of-two scale 2^(b - 127), held as one
byte b; an element is an int8 q and stands for q / 64 * 2^(b - 127).  The scale is the smallest at which the group's largest magnitude
still rounds to 127, so a restored value is within half a step, 2^(b - 127) / 128, of the original: at most 1/127 of the group's
largest magnitude.  With keep_nonzero what would round to zero gets a whole step instead, up to 1/63.5 of that magnitude and, after a
ReLU, always upward.  Restored values are exact in bfloat16.  Written scales go down to 2^-100, so a group whose largest magnitude is below
about 2^-100 is held in steps of 2^-106; read, any scale byte stands for its power of two, 255 for NaN.  A group that holds an infinity or
NaN is restored as NaN.  D channels take D + ceil(D / 32) bytes.

The reference keeps every activation at full width for `loss.backward()` (training/helpers.py:139-142); the callers here are the training
forward's per-pair Linears and the per-head attention core (train_forward.py, `train_checkpoint = 'mx8'`).  The functions here are what
those callers' forward and backward are made of and stand outside autograd: results carry no gradient and no tangent, and a
torch.jit.trace does not see them."""
from __future__ import annotations

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


# Host cost: on the small calls (a few thousand rows) the kernels take 3 us and the way to them three times that, so the arguments are checked
# once here and travel as plain addresses; every tensor behind one is a local of the caller until the entry point has returned.
def refuse_cpu(t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise L.DiffAlignHipError('diffalign_amd ops need tensors on a HIP device (no CPU fallback); got ' + str(t.device))


def elsewhere(t: torch.Tensor) -> bool:
    """Whether t is on another device than the current one: the caller then runs again with t's device current."""
    return t.is_cuda and t.get_device() != torch._C._cuda_getDevice()


def aligned(t: torch.Tensor, to: int = 16) -> torch.Tensor:
    """t, contiguous at an address divisible by `to`; itself where it is already."""
    if not t.is_contiguous():
        t = t.contiguous()
    return t.clone() if t.data_ptr() % to else t


def _check(q: Mx8) -> Mx8:
    codes, scales = q
    if codes.dtype != torch.int8 or scales.dtype != torch.uint8:
        raise L.DiffAlignHipError(f'mx8: codes int8 and scales uint8 expected, got {codes.dtype} and {scales.dtype}')
    shape = codes.shape
    if len(shape) < 1 or scales.shape != shape[:-1] + (-(-shape[-1] // GROUP),):
        raise L.DiffAlignHipError(f'mx8: scales {tuple(scales.shape)} do not belong to codes {tuple(shape)} (one byte for {GROUP} channels)')
    if scales.device != codes.device:
        raise L.DiffAlignHipError(f'mx8: codes on {codes.device}, scales on {scales.device}')
    refuse_cpu(codes)
    return q if codes.is_contiguous() and scales.is_contiguous() else Mx8(codes.contiguous(), scales.contiguous())


def quantize(x: torch.Tensor, keep_nonzero: bool = False) -> Mx8:
    """x (..., D) fp32 or bf16 -> its 8-bit form.  keep_nonzero: an element other than zero keeps a code other than zero (+-1 where it
    would round to 0, an error of up to one step instead of half), so the codes still tell what a ReLU let through
    (relu_dropout_bwd)."""
    if x.dtype not in _DTYPES:
        raise L.DiffAlignHipError(f'mx8.quantize: fp32 or bf16 expected, got {x.dtype}')
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise L.DiffAlignHipError(f'mx8.quantize: x needs a channel axis, got shape {tuple(shape)}')
    refuse_cpu(x)
    if elsewhere(x):
        with torch.cuda.device(x.device):
            return quantize(x, keep_nonzero)
    if not x.is_contiguous():
        x = x.contiguous()
    D = shape[-1]
    codes = torch.empty(shape, dtype=torch.int8, device=x.device)
    scales = torch.empty(shape[:-1] + (-(-D // GROUP),), dtype=torch.uint8, device=x.device)
    L.raise_on(L.lib().da_mx8_quant(x.data_ptr(), x.dtype is torch.bfloat16, codes.data_ptr(), scales.data_ptr(), x.numel() // D, D, keep_nonzero, L.stream()),
            'da_mx8_quant')
    return Mx8(codes, scales)


def dequantize(q: Mx8, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of an 8-bit activation, fp32 or bf16 (both exact)."""
    if dtype not in _DTYPES:
        raise L.DiffAlignHipError(f'mx8.dequantize: fp32 or bf16, not {dtype}')
    codes, scales = _check(q)
    if elsewhere(codes):
        with torch.cuda.device(codes.device):
            return dequantize(q, dtype)
    D = codes.shape[-1]
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    if D == 0:
        return out
    L.raise_on(L.lib().da_mx8_dequant(codes.data_ptr(), scales.data_ptr(), out.data_ptr(), dtype is torch.bfloat16, out.numel() // D, D, L.stream()),
            'da_mx8_dequant')
    return out


def linear_wgrad(q: Mx8, dy: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dW (out,in), db (out)) fp32 of an nn.Linear whose input x is held in 8 bits: dW = dY^T x, db = column sums of dY.  dy (..., out)
    fp32 or bf16 with q's leading axes; (in, out) of WGRAD_SHAPES."""
    codes, scales = _check(q)
    if dy.dtype not in _DTYPES:
        raise L.DiffAlignHipError(f'mx8.linear_wgrad: dy fp32 or bf16, got {dy.dtype}')
    if dy.dim() < 1 or codes.shape[:-1] != dy.shape[:-1] or codes.device != dy.device:
        raise L.DiffAlignHipError(f'mx8.linear_wgrad: x {tuple(codes.shape)} on {codes.device} and dy {tuple(dy.shape)} on {dy.device} do not belong together')
    in_f, out_f = codes.shape[-1], dy.shape[-1]
    if (in_f, out_f) not in WGRAD_SHAPES:
        raise L.DiffAlignHipError(f'mx8.linear_wgrad: {in_f} -> {out_f} features not built')
    if elsewhere(dy):
        with torch.cuda.device(dy.device):
            return linear_wgrad(q, dy)
    R, dev = codes.numel() // in_f, dy.device
    dW, db = torch.empty(out_f, in_f, device=dev), torch.empty(out_f, device=dev)
    if R == 0:
        return dW.zero_(), db.zero_()
    codes, dy = aligned(codes, 8), aligned(dy)
    lib = L.lib()
    nbytes = lib.da_linear_wgrad_mx8_workspace(R, in_f, out_f)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    L.raise_on(lib.da_linear_wgrad_mx8(codes.data_ptr(), scales.data_ptr(), dy.data_ptr(), dy.dtype is torch.bfloat16, dW.data_ptr(), db.data_ptr(),
                                    ws.data_ptr(), nbytes, R, in_f, out_f, L.stream()), 'da_linear_wgrad_mx8')
    return dW, db


def relu_dropout_bwd(q: Mx8, dy: torch.Tensor, p: float) -> torch.Tensor:
    """Gradient of h = dropout_p(relu(a)) with respect to a, from h held in 8 bits with keep_nonzero: dy / (1 - p) where h is not zero,
    else 0.  dy fp32 or bf16, of h's shape."""
    codes, _ = _check(q)
    if dy.dtype not in _DTYPES or dy.shape != codes.shape or dy.device != codes.device:
        raise L.DiffAlignHipError(f'mx8.relu_dropout_bwd: dy fp32 or bf16 of shape {tuple(codes.shape)} expected, got {dy.dtype} {tuple(dy.shape)} on {dy.device}')
    if elsewhere(dy):
        with torch.cuda.device(dy.device):
            return relu_dropout_bwd(q, dy, p)
    dy = dy.contiguous()
    dx = torch.empty_like(dy)
    L.raise_on(L.lib().da_relu_dropout_bwd_mx8(codes.data_ptr(), dy.data_ptr(), dx.data_ptr(), dy.dtype is torch.bfloat16, dy.numel(), float(p), L.stream()),
            'da_relu_dropout_bwd_mx8')
    return dx
