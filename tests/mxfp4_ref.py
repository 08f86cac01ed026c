"""MXFP4 and MXFP8 in plain numpy, 64 bits: what the kernels are compared with."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def _floor_log2(a):
    return np.frexp(a)[1] - 1


def quantize_mxfp4(x):
    """Values [..., K] -> GGUF blocks [..., K / 32 * 17]."""
    x = np.asarray(x, dtype=np.float64)
    b = x.reshape(-1, 32)
    amax = np.abs(b).max(1)
    bad = ~np.isfinite(amax)
    e = np.where(amax > 0, _floor_log2(np.where(bad | (amax == 0), 1.0, amax)), -1000)
    e = np.maximum(e, -126)                                    # fp32 numbers below the normal ones share the lowest exponents
    s = np.where(np.abs(b).max(1) >= 2.0 ** -126, np.maximum(e - 2, -127), -127)
    v = np.where(bad[:, None], 0, b) * 2.0 ** -s[:, None].astype(np.float64)
    a = np.minimum(np.abs(v), 6)
    unit = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
    a = np.rint(a / unit) * unit                               # np.rint: ties to even multiples, which are the even codes
    code = np.searchsorted(E2M1, a).astype(np.uint8) | np.where(np.signbit(v), 8, 0).astype(np.uint8)
    out = np.empty((len(b), 17), dtype=np.uint8)
    out[:, 0] = np.where(bad, 255, s + 127)
    out[:, 1:] = np.where(bad[:, None], 0, code[:, :16] | (code[:, 16:] << 4))
    return out.reshape(x.shape[:-1] + (-1,))


def dequantize_mxfp4(w):
    """GGUF blocks, flat bytes -> values [blocks, 32]."""
    b = np.asarray(w, dtype=np.uint8).reshape(-1, 17)
    c = np.concatenate([b[:, 1:] & 15, b[:, 1:] >> 4], 1)
    v = np.where(c & 8, -E2M1[c & 7], E2M1[c & 7])
    scale = np.where(b[:, 0] == 255, np.nan, 2.0 ** (b[:, 0].astype(np.float64) - 127))
    return v * scale[:, None]


def mxfp8(x):
    """fp32 rows [M, K] -> the values that MXFP8 holds for them; blocks with an infinity or a NaN are NaN."""
    x = np.asarray(x, dtype=np.float64)
    b = x.reshape(-1, 32)
    amax = np.abs(b).max(1)
    bad = ~np.isfinite(amax)
    safe = np.where(bad | (amax < 2.0 ** -126), 2.0 ** -126, amax)
    e = _floor_log2(safe)
    s = np.maximum(e - 8 + (safe > 1.75 * 2.0 ** e), -127).astype(np.float64)
    v = np.where(bad[:, None], 0, b) * 2.0 ** -s[:, None]
    step = 2.0 ** (np.maximum(_floor_log2(np.maximum(np.abs(v), 2.0 ** -40)), -6) - 3)
    q = np.rint(v / step) * step * 2.0 ** s[:, None]
    return np.where(bad[:, None], np.nan, q).reshape(x.shape)


def product(x, w):
    """(y, mass): y = xq . w^T and the sums of the terms' magnitudes, in 64 bits; x fp32 [M, K], w values [N, K]."""
    import torch
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    xq, wt = torch.from_numpy(mxfp8(x)).to(dev), torch.from_numpy(np.ascontiguousarray(w)).to(dev).t()
    return (xq @ wt).cpu().numpy(), (xq.abs() @ wt.abs()).cpu().numpy()


def tolerance(K, mass):
    """A sum of K products goes into an fp32 accumulator 32 at a time, and at most 32 such sums are added up at the end. Every one of
    these steps truncates to 24 bits at worst: 2^-23 of a partial sum, none of which is over the mass."""
    return (K / 32 + 32) * 2.0 ** -23 * mass
