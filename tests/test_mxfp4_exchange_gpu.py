"""MXFP4 products whose k is shared by several CTAs: sums sent through a cluster's shared memory, in kernels of a handful of rows and of middle sizes. Sizes at which
buffers, slots and accumulators are used again, and tiles are more than a call's plan reckons with; each says which kernel it has to reach."""
import numpy as np
import pytest

from laplace_b200.ggml import GGMLType, any_row_bytes
from tests import mxfp4_ref as ref
from tests.test_mxfp4_gpu import _act, _close, _dev

pytestmark = pytest.mark.gpu
SMALL, SINGLE, PAIR = 1, 2, 3                                  # laplace_cuda_mxfp4_last_kernel, + 16 x the CTAs that share k


def _weights(seed, rows, K):
    """Random blocks on the GPU, flat bytes."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randint(0, 256, (rows * (K // 32), 17), dtype=torch.uint8, device="cuda", generator=g)
    w[:, 0] = w[:, 0] % 6 + 118
    return w.view(-1)


def _product(xq, w, N, K):
    """(y, mass) in 64 bits, of the values that dequantize gives (they are the definition's to the bit, see test_mxfp4_gpu.py)."""
    import torch
    from laplace_b200 import device
    rb, ys, ms = any_row_bytes(39, K), [], []
    for r in range(0, N, 16384):
        n = min(16384, N - r)
        v = device.dequantize(w[r * rb:(r + n) * rb], GGMLType.MXFP4, n * K).view(n, K).double().t()
        ys.append(xq @ v)
        ms.append(xq.abs() @ v.abs())
    return torch.cat(ys, 1).cpu().numpy(), torch.cat(ms, 1).cpu().numpy()


def _experts(x, w, expert, row, E, N, K, y0):
    """The same pair by pair; pairs of a negative expert keep y0."""
    import torch
    per = N * any_row_bytes(39, K)
    y, mass, xq = y0.astype(np.float64), np.zeros(y0.shape), torch.from_numpy(ref.mxfp8(x)).cuda()
    for e in range(E):
        at = np.flatnonzero(expert == e)
        if len(at):
            y[at], mass[at] = _product(xq[torch.from_numpy(at if row is None else row[at].astype(np.int64)).cuda()], w[e * per:(e + 1) * per], N, K)
    return y, mass


def _kernel():
    from laplace_b200 import device
    return device.lib().laplace_cuda_mxfp4_last_kernel()


# ---- clusters ------------------------------------------------------------------------------------------------------------

# The last four have several tiles for a cluster of 148 or 296: a receiving slot of two CTAs is used again from the fifth on, an accumulator from the ninth.
@pytest.mark.parametrize("M,K,N,C", [(1, 4096, 1024, 8), (8, 4096, 4096, 4), (3, 14336, 4096, 4), (2, 4096, 76700, 2), (8, 4096, 76700, 2), (1, 8192, 115150, 2), (7, 256, 400000, 1)])
def test_handful_of_rows(M, K, N, C):
    import torch
    from laplace_b200 import device
    w = _weights(1600 + C, N, K)
    x = _act(1601 + N, M, K)
    packed, xd = device.mxfp4_pack(w, N, K), _dev(x)
    y = device.mxfp4_gemm(xd, packed, M, K, N)
    device.sync()
    assert _kernel() == SMALL + 16 * C
    _close(y, *_product(torch.from_numpy(ref.mxfp8(x)).cuda(), w, N, K), K, f"M={M} K={K} N={N}")
    for _ in range(5):
        assert torch.equal(device.mxfp4_gemm(xd, packed, M, K, N), y)
    device.sync()


@pytest.mark.parametrize("P,E,K,N,C", [(32, 32, 256, 16384, 1), (32, 32, 4096, 2400, 2), (30, 3, 4096, 512, 4), (12, 4, 2048, 512, 4)])
@pytest.mark.parametrize("form", ["own", "elsewhere"])
def test_handful_of_pairs(P, E, K, N, C, form):
    import torch
    from laplace_b200 import device
    w = _weights(1610 + E, E * N, K)
    expert = (np.arange(P) * 7 % E).astype(np.int32)
    row = None
    if form == "elsewhere":
        expert[1::5] = -3
        row = (np.arange(P, dtype=np.int32) * 5 % 9).astype(np.int32)
    x = _act(1611 + P, 9 if row is not None else P, K)
    packed, args = device.mxfp4_pack(w, N, K, E), (_dev(expert), None if row is None else _dev(row), E, K, N)
    y0 = torch.full((P, N), 7.0, device="cuda")
    y = device.mxfp4_moe_grouped(_dev(x), packed, *args, y=y0.clone())
    device.sync()
    assert _kernel() == SMALL + 16 * C
    _close(y, *_experts(x, w, expert, row, E, N, K, y0.cpu().numpy()), K, f"P={P} E={E} K={K} N={N} {form}")
    for _ in range(5):
        assert torch.equal(device.mxfp4_moe_grouped(_dev(x), packed, *args, y=y0.clone()), y)
    device.sync()


# widths of 32, 64 and 128 tokens; 24 and 9 x 14336 x 10240: 80 tiles for some 33 clusters of four
@pytest.mark.parametrize("M,K,N,C", [(24, 14336, 10240, 4), (9, 14336, 10240, 4), (24, 8192, 6000, 2), (48, 4096, 1000, 8), (64, 14336, 8192, 2), (100, 14336, 8000, 2), (77, 8192, 1100, 8), (300, 14336, 256, 8),
                                     (260, 8192, 1200, 4)])
def test_rows_of_middle_sizes(M, K, N, C):
    import torch
    from laplace_b200 import device
    w = _weights(1620 + C, N, K)
    x = _act(1621 + M, M, K)
    packed, xd = device.mxfp4_pack(w, N, K), _dev(x)
    y = device.mxfp4_gemm(xd, packed, M, K, N)
    device.sync()
    assert _kernel() == SINGLE + 16 * C
    _close(y, *_product(torch.from_numpy(ref.mxfp8(x)).cuda(), w, N, K), K, f"M={M} K={K} N={N}")
    for _ in range(5):
        assert torch.equal(device.mxfp4_gemm(xd, packed, M, K, N), y)
    device.sync()


# pairs of the experts one after the other. Tiles of 32, 64 and 128 tokens, evenly and with more token tiles than experts: the plan reckons with one an expert, and the
# last three have more tiles than clusters
GROUPED = [((30, 30, 30, 30), 2048, 1000, 4), ((50, 50, 50, 50), 4096, 600, 4), ((110, 110, 110, 110), 4096, 600, 4), ((9, 0, 31, 1, 40), 2816, 900, 2), ((61, 3), 4096, 300, 8),
           ((65, 1, 31, 31), 2048, 1000, 4), ((129, 65, 1, 61), 4096, 1000, 4), ((193, 63), 4096, 2000, 4)]


@pytest.mark.parametrize("counts,K,N,C", GROUPED)
@pytest.mark.parametrize("form", ["own", "shared", "elsewhere", "bad rows"])
def test_pairs_of_middle_sizes(counts, K, N, C, form):
    import torch
    from laplace_b200 import device
    from laplace_b200.matmul import LaplaceCudaError
    E, P = len(counts), sum(counts)
    rng = np.random.default_rng(1630)
    expert = rng.permutation(np.repeat(np.arange(E), counts)).astype(np.int32)
    row, X = None, P
    if form != "own":
        X = 21
        row = rng.integers(0, X, P).astype(np.int32)
    if form == "elsewhere":
        expert[::9] = -1
    ok = expert.copy()
    if form == "bad rows":
        row[3::11], ok[3::11] = X, -1
    w = _weights(1631 + P, E * N, K)
    x = _act(1632 + P, X, K)
    packed, args = device.mxfp4_pack(w, N, K, E), (_dev(expert), None if row is None else _dev(row), E, K, N)
    y0 = torch.full((P, N), 7.0, device="cuda")
    y = device.mxfp4_moe_grouped(_dev(x), packed, *args, y=y0.clone())
    if form == "bad rows":
        with pytest.raises(LaplaceCudaError):
            device.sync()
    device.sync()
    assert _kernel() == SINGLE + 16 * C
    _close(y, *_experts(x, w, ok, row, E, N, K, y0.cpu().numpy()), K, f"{counts} K={K} N={N} {form}")
    if form != "bad rows":
        for _ in range(5):
            assert torch.equal(device.mxfp4_moe_grouped(_dev(x), packed, *args, y=y0.clone()), y)
        device.sync()
