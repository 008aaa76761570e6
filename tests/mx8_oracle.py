"""The MXINT8 format in 64 bits, from its definition (numpy on the host)."""
import numpy as np
import torch


def quantize(x, keep_nonzero=False):
    """(codes int8 (rows, D), scales uint8 (rows, ceil(D / 32)), values float64) of x (rows, D)."""
    x = x.detach().cpu().double().numpy()
    rows, D = x.shape
    G = -(-D // 32)
    codes, scales, vals = np.zeros((rows, D), np.int8), np.zeros((rows, G), np.uint8), np.zeros((rows, D))
    for g in range(G):
        part = x[:, 32 * g:32 * g + 32]
        amax = np.abs(part).max(1)
        bad = ~np.isfinite(part).all(1)
        e = np.full(rows, -100)
        ok = ~bad & (amax > 0)
        # smallest exponent with rint(64 amax / 2^e) <= 127; ties of rint go to even, 127.5 rounds to 128
        m, k = np.frexp(amax[ok])                                          # amax = m 2^k, m in [1/2, 1)
        e[ok] = np.clip(k - 1 + (m >= 127.5 / 128), -100, 127)
        step = np.ldexp(1.0, e - 6)
        with np.errstate(invalid='ignore'):
            q = np.clip(np.rint(part / step[:, None]), -127, 127)
        q = np.where(bad[:, None], 0, q)
        if keep_nonzero:
            q = np.where((q == 0) & (part != 0), np.where(part > 0, 1, -1), q)
        codes[:, 32 * g:32 * g + 32] = q
        scales[:, g] = np.where(bad, 255, e + 127)
        vals[:, 32 * g:32 * g + 32] = np.where(bad[:, None], np.nan, q * step[:, None])
    return torch.from_numpy(codes), torch.from_numpy(scales), torch.from_numpy(vals)
