"""MXFP4 on the CPU: the plain forms that the GPU tests compare with, the type's geometry, sizes, and calls without a GPU."""
import numpy as np
import pytest

from laplace_b200 import _lib
from laplace_b200.ggml import ALL_GEOM, GGMLType, any_row_bytes
from tests import mxfp4_ref as ref


def test_type_and_geometry():
    assert int(GGMLType.MXFP4) == 39 and ALL_GEOM[GGMLType.MXFP4] == (32, 17)
    assert any_row_bytes(39, 4096) == 4096 // 32 * 17


def test_sizes():
    L = _lib.load()
    for e, n, k in ((1, 1, 32), (1, 128, 128), (1, 129, 160), (3, 4096, 14336)):
        assert L.laplace_cuda_mxfp4_packed_size(e, n, k) == e * -(-n // 128) * -(-k // 128) * (128 * 64 + 512)
    for bad in ((0, 1, 32), (1, 0, 32), (1, 1, 0), (1, 1, 33), (-1, 1, 32)):
        assert L.laplace_cuda_mxfp4_packed_size(*bad) == 0


def test_no_gpu_means_error():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    L = _lib.load()
    b = np.zeros(4096, dtype=np.uint8)
    p = b.ctypes.data
    assert L.laplace_cuda_mxfp4_workspace_size(40, 0, 256, 64) == 0
    assert L.laplace_cuda_mxfp4_quantize_dev(p, 0, p, 32, None) == -3
    assert L.laplace_cuda_mxfp4_pack_dev(p, p, 1, 1, 32, None) == -3
    assert L.laplace_cuda_mxfp4_gemm_dev(p, p, p, 1, 32, 1, None, 0, None) == -3
    assert L.laplace_cuda_mxfp4_moe_grouped_dev(p, 1, p, p, None, 1, 1, p, 32, 1, None, 0, None) == -3


def test_plain_quantizer_is_nearest_with_ties_to_even():
    """Against the definition by search: of the codes the nearest, of two equally near ones the even one, over 6 the largest."""
    rng = np.random.default_rng(5)
    x = np.concatenate([rng.standard_normal((50, 32)), np.round(rng.standard_normal((50, 32)) * 4) / 4])
    x[0] = 0
    w = ref.quantize_mxfp4(x).reshape(-1, 17)
    codes = np.concatenate([w[:, 1:] & 15, w[:, 1:] >> 4], 1)
    for b in range(len(x)):
        top = np.abs(x[b]).max()
        s = np.floor(np.log2(top)) - 2 if top else -127
        assert w[b, 0] == s + 127
        for v, c in zip(x[b] / 2.0 ** s, codes[b]):
            d = np.abs(ref.E2M1 - min(abs(v), 6))
            near = np.flatnonzero(d == d.min())
            assert (c & 7) == (near[0] if len(near) == 1 else near[near % 2 == 0][0]) and (c >> 3) == np.signbit(v)
    assert np.array_equal(ref.quantize_mxfp4(ref.dequantize_mxfp4(w).reshape(x.shape)).reshape(-1, 17)[1:, 1:] & 7, w[1:, 1:] & 7)


def test_plain_mxfp8_is_torchs_e4m3():
    import torch
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((40, 64)) * np.exp(2 * rng.standard_normal((40, 1)))).astype(np.float32)
    x[3, :32] = 0
    x[4, 5] = np.inf
    q = ref.mxfp8(x)
    assert np.isnan(q[4, :32]).all() and np.isfinite(q[4, 32:]).all() and not q[3, :32].any()
    for row in (0, 1, 2, 5, 6):
        for b in range(2):
            v = x[row, 32 * b:32 * b + 32].astype(np.float64)
            p = 1.0
            while np.abs(v).max() > 448 * p:
                p *= 2
            while np.abs(v).max() <= 224 * p:
                p /= 2
            want = torch.from_numpy(v / p).float().to(torch.float8_e4m3fn).double().numpy() * p
            assert np.array_equal(q[row, 32 * b:32 * b + 32], want)


def test_gguf_file_with_mxfp4_tensors(tmp_path):
    """The loader sizes type 39 and hands out its rows and experts like those of every other type."""
    from laplace_b200.gguf import GgufFile
    from tests.gguf_file import write_gguf
    K, N, E, NE = 64, 300, 4, 48
    w = ref.quantize_mxfp4(np.random.default_rng(7).standard_normal((N + E * NE, K)))
    path = tmp_path / "m.gguf"
    write_gguf(path, [("general.architecture", "str", "llama")], [("blk.0.w", [K, N], 39, w[:N].tobytes()), ("blk.0.exps", [K, NE, E], 39, w[N:].tobytes())], alignment=32)
    for rank in range(2):
        g = GgufFile(path, rank, 2)
        try:
            t, e = g.tensor("blk.0.w"), g.tensor("blk.0.exps")
            assert t.type == 39 and t.kind == 1 and t.nbytes == (t.rows[1] - t.rows[0]) * 34
            assert e.kind == 2 and e.experts == (2 * rank, 2 * rank + 2) and e.nbytes == 2 * NE * 34
        finally:
            g.close()


def test_sizes_at_the_end_of_the_range():
    """Tiles are counted in more than 32 bits: 2^24 - 1 of them are the most that a call takes (2^31 rows of packed bytes), above that the size is 0."""
    L = _lib.load()
    most = (1 << 24) - 1
    assert L.laplace_cuda_mxfp4_packed_size(1, most * 128, 32) == most * (128 * 64 + 512)
    assert L.laplace_cuda_mxfp4_packed_size(1, 1, most * 128) == most * (128 * 64 + 512)
    assert L.laplace_cuda_mxfp4_packed_size(most, 1, 32) == most * (128 * 64 + 512)
    for over in ((1, most * 128 + 1, 32), (1, 2 ** 31 - 1, 32), (1, 1, most * 128 + 32), (1, 1, 2 ** 31 - 32), (most + 1, 1, 32), (2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 32)):
        assert L.laplace_cuda_mxfp4_packed_size(*over) == 0, over
