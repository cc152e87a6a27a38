"""MXFP4 by its definition, in 64 bits on the CPU: the oracle of the MXFP4 tests."""
import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """x [rows, cols] -> codes [rows, cols / 2] and scales [rows, cols / 32], uint8 numpy arrays."""
    v = x.detach().cpu().double().numpy()
    rows, cols = v.shape
    b = v.reshape(rows, cols // 32, 32)
    bad = ~np.isfinite(b).all(-1)
    top = np.abs(np.where(np.isfinite(b), b, 0)).max(-1)
    _, e = np.frexp(top)  # top = m 2^e, m in [0.5, 1): floor(log2 top) = e - 1
    ex = np.where(top > 0, np.maximum(e - 3, -127), -127)
    scale = np.where(bad, 255, ex + 127).astype(np.uint8)
    with np.errstate(invalid="ignore", over="ignore"):
        a = np.abs(b) / np.exp2(ex.astype(np.float64))[..., None]
        code = np.zeros(a.shape, np.uint8)
        for i in range(7):  # borders between neighbours; a tie goes to the even code
            border = (GRID[i] + GRID[i + 1]) / 2
            code += ((a > border) | ((a == border) & (i % 2 == 1))).astype(np.uint8)
    code |= np.signbit(b).astype(np.uint8) << 3
    code[bad] = 0
    code = code.reshape(rows, cols)
    return code[:, ::2] | code[:, 1::2] << 4, scale


def values(codes, scales):
    """The values that codes and scales (uint8 arrays or tensors) stand for, float64 [rows, cols]."""
    c, s = (np.asarray(t.cpu() if torch.is_tensor(t) else t) for t in (codes, scales))
    code = np.stack([c & 15, c >> 4], -1).reshape(c.shape[0], -1)
    v = np.where(code & 8, -1.0, 1.0) * GRID[code & 7]
    sc = np.where(s == 255, np.nan, np.exp2(s.astype(np.float64) - 127))
    return v * np.repeat(sc, 32, axis=1)
