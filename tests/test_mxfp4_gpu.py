"""The MXFP4 operators against plain 64-bit forms: quantizer, packing, product with MXFP8 activations, expert-grouped product."""
import numpy as np
import pytest

from laplace_b200.ggml import GGMLType
from tests import mxfp4_ref as ref
from tests import synth

pytestmark = pytest.mark.gpu
MX = GGMLType.MXFP4


def _dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _blocks(seed, n, k, std=0.02):
    """GGUF blocks of an N(0, std^2) matrix, and its values."""
    w = ref.quantize_mxfp4((synth.normal_f32(seed, (n, k)) * std).astype(np.float32))
    return w.reshape(-1), ref.dequantize_mxfp4(w).reshape(n, k)


def _act(seed, m, k):
    return (synth.normal_f32(seed, (m, k)) * np.exp(0.5 * synth.normal_f32(seed + 1, (k,)))).astype(np.float32)


def _close(y, want, mass, K, what=""):
    y = y.cpu().numpy().astype(np.float64)
    assert y.shape == want.shape
    bad = ~(np.abs(y - want) <= ref.tolerance(K, mass))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} off, first at {np.argwhere(bad)[0]}: {y[bad][0]} for {want[bad][0]}"
    norm = np.linalg.norm(want)
    assert np.linalg.norm(y - want) <= 1e-6 * norm, f"{what}: relative error {np.linalg.norm(y - want) / norm:.2e}"


# ---- quantizer, blocks -----------------------------------------------------------------------------------------------

def _edge_values():
    rows = [np.zeros(32), np.full(32, -0.0), np.full(32, 2.0 ** -149), np.full(32, 2.0 ** -126), np.full(32, 3.4e38), np.full(32, 7.0), np.full(32, -7.99)]
    ties = np.zeros(32)                                        # 6 sets the scale to 1: every midpoint between two codes, both signs
    ties[:16] = [6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5, -6]
    rows += [ties, ties * 2.0 ** -100, ties * 2.0 ** 100, np.nextafter(ties, 10).astype(np.float32), np.nextafter(ties, -10).astype(np.float32)]
    one = np.ones(32)
    for v in (np.inf, -np.inf, np.nan):
        r = one.copy(); r[17] = v
        rows.append(r)
    with np.errstate(over="ignore"):
        return np.array(rows).astype(np.float32)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (1, 4096), (65, 2848), (1000, 64), (2001, 2848), (1501, 14336)])
def test_quantize(dtype, shape):
    import torch
    from laplace_b200 import device
    x = _dev(synth.normal_f32(900, shape)).to(getattr(torch, dtype))
    w = device.mxfp4_quantize(x)
    assert w.numel() == x.numel() // 32 * 17
    want = ref.quantize_mxfp4(x.float().cpu().numpy())
    assert np.array_equal(w.cpu().numpy(), want.reshape(-1))
    v = device.dequantize(w, MX, x.numel()).cpu().numpy()
    assert np.array_equal(v, ref.dequantize_mxfp4(want).reshape(-1).astype(np.float32))


def test_quantize_edges():
    from laplace_b200 import device
    x = _edge_values()
    got = device.mxfp4_quantize(_dev(x)).cpu().numpy().reshape(-1, 17)
    assert np.array_equal(got, ref.quantize_mxfp4(x).reshape(-1, 17))


def test_quantize_into_the_middle_of_a_buffer():
    """Blocks may start at any byte; what lies around them stays."""
    import torch
    from laplace_b200 import device
    x = _dev(synth.normal_f32(901, (7, 160)))
    n = x.numel() // 32 * 17
    for off in (0, 1, 5, 16, 17):
        buf = torch.full((n + 64,), 0xAB, dtype=torch.uint8, device="cuda")
        device.mxfp4_quantize(x, buf[off:off + n])
        assert torch.equal(buf[off:off + n], device.mxfp4_quantize(x))
        assert (buf[:off] == 0xAB).all() and (buf[off + n:] == 0xAB).all()


def test_dequantize_every_scale_and_code():
    from laplace_b200 import device
    w = np.empty((256, 17), dtype=np.uint8)
    w[:, 0] = np.arange(256)
    w[:, 1:] = np.arange(16) + 16 * ((np.arange(16) + np.arange(256)[:, None]) % 16)
    for off in (0, 1, 3):
        import torch
        buf = torch.zeros(w.size + 8, dtype=torch.uint8, device="cuda")
        buf[off:off + w.size] = _dev(w.reshape(-1))
        v = device.dequantize(buf[off:], MX, 256 * 32).cpu().numpy()
        with np.errstate(over="ignore"):
            assert np.array_equal(v, ref.dequantize_mxfp4(w).reshape(-1).astype(np.float32), equal_nan=True)


def test_embed_rows():
    import torch
    from laplace_b200 import device
    w, v = _blocks(902, 50, 2848)
    tok = [3, 0, 49, 3]
    y = device.embed_rows(_dev(w), MX, torch.tensor(tok, dtype=torch.int32, device="cuda"), 2848, 50, scale=2.0)
    assert np.array_equal(y.cpu().numpy(), (2 * v[tok]).astype(np.float32))


@pytest.mark.parametrize("experts,n,k", [(1, 1, 32), (1, 128, 128), (3, 130, 160), (2, 300, 96), (1, 257, 1024)])
@pytest.mark.parametrize("off", [0, 3])
def test_pack_layout(experts, n, k, off):
    import torch
    from laplace_b200 import device
    w, _ = _blocks(903, experts * n, k)
    buf = torch.zeros(w.size + 8, dtype=torch.uint8, device="cuda")
    buf[off:off + w.size] = _dev(w)
    p = device.mxfp4_pack(buf[off:off + w.size], n, k, experts).cpu().numpy()
    rts, kts = -(-n // 128), -(-k // 128)
    b = np.zeros((experts, rts * 128, kts * 4, 17), dtype=np.uint8)
    b[..., 0] = 127
    b[:, :n, :k // 32] = w.reshape(experts, n, k // 32, 17)
    c = np.concatenate([b[..., 1:] & 15, b[..., 1:] >> 4], -1).reshape(experts, rts, 128, kts, 128)
    q = (c[..., 0::2] | (c[..., 1::2] << 4)).transpose(0, 1, 3, 2, 4)
    sf = b[..., 0].reshape(experts, rts, 4, 32, kts, 4).transpose(0, 1, 4, 3, 2, 5)
    assert np.array_equal(p, np.concatenate([q.reshape(-1), sf.reshape(-1)]))


# ---- product -----------------------------------------------------------------------------------------------------------

SHAPES = [(1, 32, 1), (1, 64, 129), (1, 4096, 1024), (2, 160, 200), (7, 288, 64), (8, 2848, 384), (9, 512, 4096), (16, 128, 128), (17, 96, 1000), (24, 14336, 256), (31, 1024, 640),
          (32, 2816, 130), (33, 4096, 512), (64, 160, 300), (65, 2048, 257), (77, 2816, 1056), (96, 544, 4000), (128, 1024, 128), (129, 4096, 384), (200, 256, 2000), (255, 352, 513),
          (256, 4096, 1024), (257, 1056, 700), (300, 14336, 256), (512, 2048, 2816), (777, 768, 1411), (1030, 96, 2100), (2048, 512, 1024), (5000, 64, 300), (1200, 14336, 256), (260, 4096, 200), (9, 14336, 1000), (100, 14336, 64)]


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_product(M, K, N):
    from laplace_b200 import device
    w, v = _blocks(910 + M, N, K)
    x = _act(911 + N, M, K)
    y = device.mxfp4_gemm(_dev(x), device.mxfp4_pack(_dev(w), N, K), M, K, N)
    device.sync()
    _close(y, *ref.product(x, v), K, f"M={M} K={K} N={N}")


@pytest.mark.parametrize("M,K,N", [(640, 4096, 4100), (600, 8192, 2100), (1030, 4096, 2600), (512, 14336, 3900)])
def test_product_on_pairs_of_sms(M, K, N):
    """Shapes whose tiles go to pairs of SMs (the workspace then holds parts of cut tiles): odd numbers of row tiles, ragged last tiles of both kinds, k cut."""
    from laplace_b200 import device
    assert device.lib().laplace_cuda_mxfp4_workspace_size(M, 0, K, N) > 148 * 2 * 256 * 512
    rng = np.random.default_rng(912)
    w = rng.integers(0, 256, (N * K // 32, 17), dtype=np.uint8)
    w[:, 0] = 118 + w[:, 0] % 6
    x = _act(913, M, K)
    y = device.mxfp4_gemm(_dev(x), device.mxfp4_pack(_dev(w.reshape(-1)), N, K), M, K, N)
    device.sync()
    _close(y, *ref.product(x, ref.dequantize_mxfp4(w).reshape(N, K)), K, f"M={M} K={K} N={N}")


@pytest.mark.parametrize("M", [1, 20, 150, 260, 1000])
def test_every_value_counts_once(M):
    """Weights that are a single 1 per row: y picks single activations, whose value and place must be right for every k and scale."""
    from laplace_b200 import device
    K = N = 416
    v = np.eye(N, K, dtype=np.float32) * 2.0 ** (np.arange(N) % 9 - 4)[:, None].astype(np.float32)
    w = ref.quantize_mxfp4(v)
    x = (_act(920, M, K) * 2.0 ** (np.arange(M) % 60 - 30)[:, None]).astype(np.float32)
    y = device.mxfp4_gemm(_dev(x), device.mxfp4_pack(_dev(w.reshape(-1)), N, K), M, K, N)
    device.sync()
    assert np.array_equal(y.cpu().numpy(), (ref.mxfp8(x) * np.diag(v).astype(np.float64)).astype(np.float32))


@pytest.mark.parametrize("M", [1, 40, 200])
def test_bad_values_stay_in_their_row_and_column(M):
    """Infinities and NaN in a block of x make that row NaN, a NaN block of the weights that column, and nothing else."""
    from laplace_b200 import device
    K, N = 384, 300
    w, v = _blocks(930, N, K)
    w = w.reshape(N, K // 32, 17).copy()
    w[257, 5, 0] = 255
    x = _act(931, M, K)
    bad = {0: np.inf} if M == 1 else {0: np.inf, M // 2: np.nan, M - 1: -np.inf}
    for m, value in bad.items():
        x[m, 100 + m] = value
    y = device.mxfp4_gemm(_dev(x), device.mxfp4_pack(_dev(w.reshape(-1)), N, K), M, K, N)
    device.sync()
    got = y.cpu().numpy()
    nan = np.zeros((M, N), dtype=bool)
    nan[list(bad)] = True
    nan[:, 257] = True
    assert np.array_equal(np.isnan(got), nan)
    want, mass = ref.product(np.where(np.isfinite(x), x, 0), v)
    ok = ~nan
    assert (np.abs(got - want)[ok] <= ref.tolerance(K, mass)[ok]).all()


def test_zeros_and_extreme_scales():
    from laplace_b200 import device
    M, K, N = 5, 256, 70
    w, v = _blocks(940, N, K)
    packed = device.mxfp4_pack(_dev(w), N, K)
    x = _act(941, M, K)
    x[1] = 0
    x[2, :128] *= np.float32(2.0 ** 90)
    x[3] *= np.float32(2.0 ** -90)
    y = device.mxfp4_gemm(_dev(x), packed, M, K, N)
    device.sync()
    want, mass = ref.product(x, v)
    assert (np.abs(y.cpu().numpy() - want) <= ref.tolerance(K, mass)).all() and not y[1].any()


@pytest.mark.parametrize("M", [1, 20, 200])
def test_scales_from_end_to_end_of_their_range(M):
    """Scales far from 1 on one side and as far the other way on the other: results are ordinary numbers, or so small that fp32 holds them with
    fewer bits (there a step may be off by the smallest number that it holds)."""
    from laplace_b200 import device
    K, N = 64, 130
    rng = np.random.default_rng(942)
    for we, xe in ((0, 100), (1, 120), (20, 100), (60, 40), (127, -126), (200, -60), (250, -130), (20, -40)):
        w = np.zeros((N, K // 32, 17), dtype=np.uint8)
        w[..., 0] = we
        w[..., 1:] = rng.integers(0, 256, (N, K // 32, 16))
        x = (rng.standard_normal((M, K)) * 2.0 ** xe).astype(np.float32)
        y = device.mxfp4_gemm(_dev(x), device.mxfp4_pack(_dev(w.reshape(-1)), N, K), M, K, N)
        device.sync()
        want, mass = ref.product(x, ref.dequantize_mxfp4(w).reshape(N, K))
        assert (np.abs(y.cpu().numpy() - want) <= ref.tolerance(K, mass) + (K / 32 + 32) * 2.0 ** -149).all(), (we, xe)


def test_rows_behind_the_last_stay():
    import torch
    from laplace_b200 import device
    for M in (1, 33, 130):
        K, N = 256, 200
        w, _ = _blocks(950, N, K)
        packed, x = device.mxfp4_pack(_dev(w), N, K), _dev(_act(951, M, K))
        y = torch.full((M + 3, N), 7.0, device="cuda")
        assert device.mxfp4_gemm(x, packed, M, K, N, y=y) is y
        assert (y[M:] == 7).all() and torch.equal(y[:M], device.mxfp4_gemm(x, packed, M, K, N))
    assert device.mxfp4_gemm(x[:0], packed, 0, K, N).shape == (0, N)
    device.sync()


# ---- experts -----------------------------------------------------------------------------------------------------------

def _grouped_ref(x, v, expert, row, y0):
    """(y, mass) pair by pair; v [E, N, K]."""
    y, mass = y0.astype(np.float64).copy(), np.zeros(y0.shape)
    for e in set(int(i) for i in expert if i >= 0):
        at = np.flatnonzero(expert == e)
        y[at], mass[at] = ref.product(x[at if row is None else row[at]], v[e])
    return y, mass


def _routing(seed, T, E, k, skew):
    logits = synth.normal_f32(seed, (T, E)) + skew * synth.normal_f32(seed + 1, (E,))
    return np.argsort(-logits, axis=1)[:, :k].astype(np.int32).reshape(-1)


@pytest.mark.parametrize("T,E,k,K,N,skew", [(1, 32, 8, 2048, 384, 0.), (1, 4, 1, 32, 1, 0.), (4, 32, 8, 352, 300, 3.), (5, 4, 2, 160, 200, 1.), (24, 60, 4, 768, 130, 1.), (100, 8, 3, 256, 520, 2.),
                                            (256, 32, 8, 512, 256, 1.5), (600, 4, 2, 96, 257, 1.), (700, 128, 8, 128, 96, 2.), (40, 1, 1, 288, 300, 0.), (1400, 3, 2, 1056, 700, 1.),
                                            (3000, 8, 2, 96, 130, 2.), (32, 1, 1, 288, 300, 0.), (31, 2, 1, 96, 140, 3.), (33, 1, 1, 64, 64, 0.), (20000, 4, 1, 32, 40, 1.), (2000, 1500, 3, 64, 24, 2.), (700, 600, 3, 32, 33, 3.), (60000, 3, 1, 32, 8, 1.)])
@pytest.mark.parametrize("form", ["shared", "own", "elsewhere"])
def test_grouped(T, E, k, K, N, skew, form):
    from laplace_b200 import device
    w, v = _blocks(960, E * N, K)
    expert = _routing(961 + T, T, E, k, skew)
    row = np.repeat(np.arange(T, dtype=np.int32), k)
    if form == "elsewhere":                                    # half of the experts on another GPU, pairs in no order
        expert = np.where(expert % 2 == 1, np.int32(-1 - expert), expert).astype(np.int32)
        order = np.random.default_rng(962).permutation(len(expert))
        expert, row = expert[order], row[order]
    x = _act(963, len(expert) if form == "own" else T, K)
    y0 = np.full((len(expert), N), 7.0, dtype=np.float32)
    y = device.mxfp4_moe_grouped(_dev(x), device.mxfp4_pack(_dev(w), N, K, E), _dev(expert), None if form == "own" else _dev(row), E, K, N, y=_dev(y0))
    device.sync()
    want, mass = _grouped_ref(x, v.reshape(E, N, K), expert, None if form == "own" else row, y0)
    _close(y, want, mass, K, f"T={T} E={E} k={k} K={K} N={N} {form}")


def test_grouped_same_expert_and_row_twice_and_none():
    import torch
    from laplace_b200 import device
    E, K, N = 6, 256, 140
    w, v = _blocks(970, E * N, K)
    packed, x = device.mxfp4_pack(_dev(w), N, K, E), _act(971, 3, K)
    expert, row = np.array([5, 5, 5, 2, 5], dtype=np.int32), np.array([1, 1, 0, 2, 1], dtype=np.int32)
    y = device.mxfp4_moe_grouped(_dev(x), packed, _dev(expert), _dev(row), E, K, N)
    assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[4])
    want, mass = _grouped_ref(x, v.reshape(E, N, K), expert, row, np.zeros((5, N)))
    _close(y, want, mass, K)
    none = device.mxfp4_moe_grouped(_dev(x), packed, _dev(np.full(5, -1, dtype=np.int32)), _dev(row), E, K, N, y=torch.full((5, N), 3.0, device="cuda"))
    assert (none == 3).all()
    assert device.mxfp4_moe_grouped(_dev(x), packed, _dev(expert[:0]), None, E, K, N).shape == (0, N)
    device.sync()


def test_grouped_bad_indices_are_skipped_and_reported():
    import torch
    from laplace_b200 import device
    from laplace_b200.matmul import LaplaceCudaError
    E, K, N = 3, 128, 128
    w, v = _blocks(975, E * N, K)
    packed, x = device.mxfp4_pack(_dev(w), N, K, E), _act(976, 2, K)
    for expert, row, bad in (([0, 3, 2], [0, 1, 1], 1), ([0, 1, 2], [0, 2, 1], 1), ([0, 1, 2], [0, 1, -1], 2), ([2147483647, 1, 2], [0, 1, 1], 0)):
        y = device.mxfp4_moe_grouped(_dev(x), packed, _dev(np.array(expert, dtype=np.int32)), _dev(np.array(row, dtype=np.int32)), E, K, N, y=torch.full((3, N), 7.0, device="cuda"))
        with pytest.raises(LaplaceCudaError):
            device.sync()
        device.sync()                                          # reported once
        assert (y[bad] == 7).all()
        for p in range(3):
            if p != bad:
                want, mass = ref.product(x[row[p]:row[p] + 1], v.reshape(E, N, K)[expert[p]])
                _close(y[p:p + 1], want, mass, K)


# ---- large ones ---------------------------------------------------------------------------------------------------------------

def test_results_behind_the_32_bit_range():
    """More than 2^31 results: rows from everywhere are right."""
    import torch
    from laplace_b200 import device
    M, K, N = 140001, 64, 16400
    w, v = _blocks(1400, N, K)
    g = torch.Generator(device="cuda").manual_seed(1401)
    x = torch.randn(M, K, device="cuda", generator=g)
    y = device.mxfp4_gemm(x, device.mxfp4_pack(_dev(w), N, K), M, K, N)
    device.sync()
    for m in (0, 1, 65535, 130943, 130944, 131072, M - 1):
        _close(y[m:m + 1], *ref.product(x[m:m + 1].cpu().numpy(), v), K, f"row {m}")


def test_weights_behind_the_32_bit_range():
    """Experts of more than 2^32 packed bytes: the first and the last are right, for a few pairs, for many, and as one matrix's rows."""
    import torch
    from laplace_b200 import device
    E, K, N = 66, 8192, 16384
    g = torch.Generator(device="cuda").manual_seed(1410)
    w = torch.randint(0, 256, (E * N * (K // 32), 17), dtype=torch.uint8, device="cuda", generator=g)
    w[:, 0] = w[:, 0] % 8 + 116
    packed = device.mxfp4_pack(w.view(-1), N, K, E)
    assert packed.numel() > 1 << 32
    per = N * (K // 32)
    values = {e: ref.dequantize_mxfp4(w[e * per:e * per + 64 * (K // 32)].cpu().numpy()).reshape(64, K) for e in (0, E - 1)}      # of the expert's first 64 rows
    del w
    for T in (3, 200, 1000):
        x = _act(1411, T, K)
        expert = np.where(np.arange(T) % 3 == 0, 0, E - 1).astype(np.int32)
        y = device.mxfp4_moe_grouped(_dev(x), packed, _dev(expert), None, E, K, N)
        device.sync()
        for p in (0, 1, T - 1):
            _close(y[p:p + 1, :64], *ref.product(x[p:p + 1], values[int(expert[p])]), K, f"{T} pairs, pair {p}")


# ---- streams, graphs, timing ----------------------------------------------------------------------------------------------

def _calls(seed):
    """Calls of every operator on data of their own."""
    from laplace_b200 import device
    K, N, E = 1024, 640, 8
    w, _ = _blocks(seed, N, K)
    we, _ = _blocks(seed + 1, E * N, K)
    packed, experts = device.mxfp4_pack(_dev(w), N, K), device.mxfp4_pack(_dev(we), N, K, E)
    xs = [_dev(_act(seed + 2 + m, m, K)) for m in (1, 50, 300)]
    big, wide = _dev(_act(seed + 7, 640, 4096)), device.mxfp4_pack(device.mxfp4_quantize(_dev(synth.normal_f32(seed + 8, (4100, 4096)) * 0.02)), 4100, 4096)      # on pairs of SMs
    expert, row = _dev(_routing(seed + 9, 50, E, 3, 1.)), _dev(np.repeat(np.arange(50, dtype=np.int32), 3))
    many = _dev(_routing(seed + 10, 300, E, 1, 3.))
    return [lambda x=x: device.mxfp4_gemm(x, packed, x.shape[0], K, N) for x in xs] + [
        lambda: device.mxfp4_moe_grouped(xs[1], experts, expert, row, E, K, N), lambda: device.mxfp4_quantize(xs[2]),
        lambda: device.mxfp4_gemm(big, wide, 640, 4096, 4100), lambda: device.mxfp4_moe_grouped(xs[2], experts, many, None, E, K, N)]


def test_the_same_call_gives_the_same_bits():
    import torch
    from laplace_b200 import device
    for call in _calls(980):
        first = call()
        for _ in range(20):
            assert torch.equal(call(), first)
    device.sync()


def test_streams_side_by_side():
    import torch
    from laplace_b200 import device
    a, b = _calls(1000), _calls(1020)
    want = [[f() for f in c] for c in (a, b)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i in range(len(a)):
            for side, calls in enumerate((a, b)):
                with torch.cuda.stream(streams[side]):
                    got[side].append(calls[i]())
    torch.cuda.synchronize()
    for side in (0, 1):
        for n, y in enumerate(got[side]):
            assert torch.equal(y, want[side][n % len(a)])
    device.sync()


def test_two_graphs_replayed_side_by_side():
    import torch
    from laplace_b200 import device
    sets = [_calls(1040), _calls(1060)]
    want = [[f() for f in c] for c in sets]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for c in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([f() for f in c])
        graphs.append(g)
    for _ in range(5):
        for o in outs:
            for y in o:
                y.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(y, z) for y, z in zip(o, w))
    device.sync()


# ---- refusals -----------------------------------------------------------------------------------------------------------------

def test_refusals():
    import torch
    from laplace_b200 import device
    from laplace_b200.matmul import LaplaceCudaError
    L = device.lib()
    K, N, E = 256, 130, 2
    w, _ = _blocks(990, E * N, K)
    w = _dev(w)
    packed = device.mxfp4_pack(w, N, K, E)
    x = _dev(_act(991, 4, K))
    expert = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (lambda: device.mxfp4_quantize(x.double()), lambda: device.mxfp4_quantize(x.t()), lambda: device.mxfp4_quantize(x.cpu()), lambda: device.mxfp4_quantize(x[:, :16].contiguous()),
                lambda: device.mxfp4_quantize(x, torch.empty(4, dtype=torch.uint8, device="cuda")), lambda: device.mxfp4_pack(w[:-1], N, K, E), lambda: device.mxfp4_gemm(x, packed[:5000], 4, K, N),
                lambda: device.mxfp4_gemm(x, packed, 5, K, N), lambda: device.mxfp4_gemm(x, packed, -1, K, N), lambda: device.mxfp4_gemm(x.half(), packed, 4, K, N), lambda: device.mxfp4_gemm(x, packed, 4, K, N, y=torch.empty(3, N, device="cuda")),
                lambda: device.mxfp4_moe_grouped(x, packed, expert.long(), None, E, K, N), lambda: device.mxfp4_moe_grouped(x, packed, expert, expert[:3], E, K, N),
                lambda: device.mxfp4_moe_grouped(x, packed, expert, None, E + 1, K, N)):
        with pytest.raises(AssertionError):
            bad()
    off = torch.zeros(4 * K + 1, device="cuda")[1:].view(4, K)      # x not 16-byte aligned
    for bad in (lambda: device.mxfp4_quantize(off), lambda: device.mxfp4_gemm(off, packed, 4, K, N), lambda: device.mxfp4_gemm(x, packed, 4, 0, N),
                lambda: device.mxfp4_gemm(x, packed, 4, 48, N), lambda: device.mxfp4_gemm(x, packed, 4, K, 0), lambda: device.mxfp4_gemm(x, torch.zeros(packed.numel() + 1, dtype=torch.uint8, device="cuda")[1:], 4, K, N),
                lambda: device.mxfp4_moe_grouped(x[:3], packed, expert, None, E, K, N), lambda: device.mxfp4_moe_grouped(x, packed, expert, None, 0, K, N)):
        with pytest.raises(LaplaceCudaError):
            bad()
    M = 40
    assert L.laplace_cuda_mxfp4_workspace_size(8, 0, K, N) == 0 and L.laplace_cuda_mxfp4_workspace_size(32, E, K, N) == 0       # none is needed
    for bad in ((0, 0, K, N), (M, -1, K, N), (M, 0, 48, N), (M, 0, K, 0)):
        assert L.laplace_cuda_mxfp4_workspace_size(*bad) == 0
    assert L.laplace_cuda_mxfp4_packed_size(1, N, 48) == 0 and L.laplace_cuda_mxfp4_packed_size(0, N, K) == 0
    x = _dev(_act(992, M, K))
    ws = torch.empty(L.laplace_cuda_mxfp4_workspace_size(M, 0, K, N), dtype=torch.uint8, device="cuda")
    y = torch.empty(M, N, device="cuda")
    args = [x.data_ptr(), packed.data_ptr(), y.data_ptr(), M, K, N, ws.data_ptr()]
    assert L.laplace_cuda_mxfp4_gemm_dev(*args, ws.numel(), 1) == 0
    assert L.laplace_cuda_mxfp4_gemm_dev(*args, ws.numel() - 1, 1) == -1
    assert L.laplace_cuda_mxfp4_gemm_dev(*args[:6], None, ws.numel(), 1) == -1
    assert L.laplace_cuda_mxfp4_gemm_dev(*args[:6], ws.data_ptr() + 16, ws.numel(), 1) == -1
    assert L.laplace_cuda_mxfp4_gemm_dev(*args[:3], -1, K, N, ws.data_ptr(), ws.numel(), 1) == -1
    assert L.laplace_cuda_mxfp4_gemm_dev(*args[:3], 1 << 25, K, N, ws.data_ptr(), ws.numel(), 1) == -5
    for i in range(3):
        assert L.laplace_cuda_mxfp4_gemm_dev(*(args[:i] + [None] + args[i + 1:]), ws.numel(), 1) == -1
    assert L.laplace_cuda_mxfp4_quantize_dev(x.data_ptr(), 2, w.data_ptr(), 32, 1) == 1
    assert L.laplace_cuda_mxfp4_moe_grouped_dev(x.data_ptr(), 4, packed.data_ptr(), expert.data_ptr(), None, 4, 4001, y.data_ptr(), K, N, ws.data_ptr(), 1 << 40, 1) == -5
    assert L.laplace_cuda_gemm_dev(x.data_ptr(), w.data_ptr(), 39, y.data_ptr(), 4, K, N, 1) == 1
    device.sync()


# ---- together -------------------------------------------------------------------------------------------------------------------

def test_expert_layer_and_head():
    """From bf16 weights to logits: quantize, pack, route, gate / up, gated activation, down, weighted sum, head; against the same steps in
    64 bits. What a step makes is the next one's input on both sides, so that a rounding at a step's border is not carried on."""
    import torch
    from laplace_b200 import device
    T, E, k, H, I, V = 21, 8, 3, 512, 288, 1000

    def weights(seed, n, kk):
        x = _dev(synth.normal_f32(seed, (n, kk)) * 0.05).bfloat16()
        return device.mxfp4_quantize(x), ref.dequantize_mxfp4(ref.quantize_mxfp4(x.float().cpu().numpy()))

    (gu, gu_v), (dn, dn_v), (head, head_v) = weights(1100, E * 2 * I, H), weights(1101, E * H, I), weights(1102, V, H)
    gu_p, dn_p, head_p = device.mxfp4_pack(gu, 2 * I, H, E), device.mxfp4_pack(dn, H, I, E), device.mxfp4_pack(head, V, H)
    x = _act(1103, T, H)
    idx, wts = device.moe_route(_dev(synth.normal_f32(1104, (T, E))), k)
    expert, row = idx.reshape(-1), torch.arange(T, dtype=torch.int32, device="cuda").repeat_interleave(k)
    h = device.mxfp4_moe_grouped(_dev(x), gu_p, expert, row, E, H, 2 * I)
    act = (torch.nn.functional.silu(h[:, :I]) * h[:, I:]).contiguous()
    d = device.mxfp4_moe_grouped(act, dn_p, expert, None, E, I, H)
    out = (d.view(T, k, H) * wts[..., None]).sum(1)
    logits = device.mxfp4_gemm(out, head_p, T, H, V)
    device.sync()
    e = expert.cpu().numpy()
    _close(h, *_grouped_ref(x, gu_v.reshape(E, 2 * I, H), e, row.cpu().numpy(), np.zeros((T * k, 2 * I))), H, "gate / up")
    _close(d, *_grouped_ref(act.cpu().numpy(), dn_v.reshape(E, H, I), e, None, np.zeros((T * k, H))), I, "down")
    _close(logits, *ref.product(out.cpu().numpy(), head_v.reshape(V, H)), H, "head")


def test_native_and_general_paths_agree():
    import torch
    from laplace_b200 import device
    device.lib()
    assert device._native is not None
    w, _ = _blocks(1200, 64, 96)
    calls = _calls(1210) + [lambda: device.dequantize(_dev(w), MX, 64 * 96)]
    native = device._native
    fast = [f() for f in calls]
    try:
        device._native = None
        slow = [f() for f in calls]
    finally:
        device._native = native
    assert all(torch.equal(a, b) and a.dtype == b.dtype and a.shape == b.shape for a, b in zip(fast, slow))
    x = _dev(_act(1220, 2, 96))
    p = device.mxfp4_pack(_dev(w), 64, 96)
    for bad in (lambda v: device.mxfp4_gemm(v, p, 1, 96, 64), lambda v: device.mxfp4_quantize(v.reshape(1, -1)),
                lambda v: device.mxfp4_moe_grouped(v, p, torch.zeros(1, dtype=torch.int32, device="cuda"), None, 1, 96, 64)):
        def f(v):                                               # inside a transform tensors have no storage
            with pytest.raises(RuntimeError):
                bad(v)
            return v.sum()
        torch.vmap(f)(x)
    device.sync()


def test_from_a_gguf_file(tmp_path):
    """A file's MXFP4 matrix and this GPU's half of its experts: loaded, packed, multiplied."""
    import torch
    from laplace_b200 import device
    from laplace_b200.gguf import GgufFile
    from tests.gguf_file import write_gguf
    K, N, E, NE = 96, 300, 4, 48
    (w, v), (we, ve) = _blocks(1300, N, K), _blocks(1301, E * NE, K)
    path = tmp_path / "m.gguf"
    write_gguf(path, [("general.architecture", "str", "llama")], [("norm", [K], 0, np.ones(K, dtype=np.float32).tobytes()), ("w", [K, N], 39, w.tobytes()), ("exps", [K, NE, E], 39, we.tobytes())],
               alignment=32)
    device.lib()
    g = GgufFile(path, 1, 2)
    try:
        g.upload()
        t, e = g.tensor("w"), g.tensor("exps")
        rows = t.rows[1] - t.rows[0]
        packed, experts = device.mxfp4_pack(t.as_torch(), rows, K), device.mxfp4_pack(e.as_torch(), NE, K, 2)
        x = _act(1302, 11, K)
        y = device.mxfp4_gemm(_dev(x), packed, 11, K, rows)
        pick = np.arange(11, dtype=np.int32) % 3 - 1
        z = device.mxfp4_moe_grouped(_dev(x), experts, _dev(pick), None, 2, K, NE, y=torch.zeros(11, NE, device="cuda"))
        device.sync()
        _close(y, *ref.product(x, v[t.rows[0]:t.rows[1]]), K)
        _close(z, *_grouped_ref(x, ve.reshape(E, NE, K)[2:], pick, None, np.zeros((11, NE))), K)
    finally:
        g.close()


def test_more_pairs_than_one_block_counts_and_bad_rows_among_them():
    """Rows of x out of range among thousands of pairs, in each size class of the products: skipped, reported, the others right."""
    import torch
    from laplace_b200 import device
    from laplace_b200.matmul import LaplaceCudaError
    for T, E, k, K, N in ((60, 8, 2, 64, 140), (300, 4, 2, 64, 140), (2500, 4, 2, 64, 140)):
        w, v = _blocks(1310, E * N, K)
        expert, row = _routing(1311, T, E, k, 0.5), np.repeat(np.arange(T, dtype=np.int32), k)
        bad = np.arange(5, T * k, 37)
        row[bad] = np.where(bad % 2, T, -1)
        x = _act(1312, T, K)
        y0 = np.full((T * k, N), 7.0, dtype=np.float32)
        y = device.mxfp4_moe_grouped(_dev(x), device.mxfp4_pack(_dev(w), N, K, E), _dev(expert), _dev(row), E, K, N, y=_dev(y0))
        with pytest.raises(LaplaceCudaError):
            device.sync()
        device.sync()
        ok = expert.copy()
        ok[bad] = -1
        _close(y, *_grouped_ref(x, v.reshape(E, N, K), ok, np.clip(row, 0, T - 1), y0), K, f"{T}")
        assert torch.equal(y[torch.from_numpy(bad).cuda()], torch.full((len(bad), N), 7.0, device="cuda"))


def test_sizes_beyond_the_limits_are_refused():
    """Each limit of the header: the call says so, and the size of a workspace is 0. No pointer is looked at before."""
    from laplace_b200 import device
    L = device.lib()
    p, K, N = 4096, 2 ** 31 - 32, 1                            # (an address that nothing reads)
    for rows, experts, k, n in ((1, 0, K, 1), (40, 0, K, 1), (1, 0, 32, 2 ** 31 - 1), (300, 0, 32, 2 ** 31 - 1), ((1 << 24) + 1, 0, 32, 1), (2 ** 31 - 1, 0, 32, 1), (1 << 24, 0, 32, 1 << 20),
                                (40, 1 << 20, 4096, 128), (40, 4001, 32, 1), ((1 << 24) + 1, 4, 32, 1), (2 ** 31 - 1, 4, 32, 1), (40, 2, K, 1)):
        assert L.laplace_cuda_mxfp4_workspace_size(rows, experts, k, n) == 0, (rows, experts, k, n)
        if experts:
            rc = L.laplace_cuda_mxfp4_moe_grouped_dev(p, 2 ** 31 - 1, p, p, None, rows, experts, p, k, n, p, 1 << 60, 1)
        else:
            rc = L.laplace_cuda_mxfp4_gemm_dev(p, p, p, rows, k, n, p, 1 << 60, 1)
        assert rc == -5, (rows, experts, k, n)
    assert L.laplace_cuda_mxfp4_pack_dev(p, p, 1, 1, K, 1) == -5 and L.laplace_cuda_mxfp4_pack_dev(p, p, 1, 2 ** 31 - 1, 32, 1) == -5
    device.sync()


def test_sizes_above_32_bits_are_refused():
    """2^32 more than a right size is not that size."""
    import torch
    from laplace_b200 import device
    K, N, E = 64, 40, 2
    w, _ = _blocks(1500, E * N, K)
    w, x = _dev(w), _dev(_act(1501, 4, K))
    packed, one, expert = device.mxfp4_pack(w, N, K, E), device.mxfp4_pack(w, N, K), torch.zeros(4, dtype=torch.int32, device="cuda")
    big = 2 ** 32
    wide = torch.empty((big + K) // 32 * 17, dtype=torch.uint8, device="cuda")      # a row of 2^32 + 64 values
    for bad in (lambda: device.mxfp4_pack(wide, 1, big + K), lambda: device.mxfp4_gemm(x, one, 1, K, big + N), lambda: device.mxfp4_gemm(x, one, 0, big + K, N),
                lambda: device.mxfp4_moe_grouped(x, packed, expert, None, big + E, K, N), lambda: device.mxfp4_moe_grouped(x, packed, expert[:1], None, E, K, big + N),
                lambda: device.mxfp4_moe_grouped(x, packed, expert[:0], None, E, big + K, N)):
        with pytest.raises(AssertionError):
            bad()
    device.sync()


def test_products_right_behind_a_long_kernel():
    """A kernel of some milliseconds that lets the next one start early, and a product of its results behind it: the same bits as with a pause in between."""
    import torch
    from laplace_b200 import device
    M, K, N = 4096, 4096, 4096
    q = device.upload_weights(synth.weights(GGMLType.Q4_K, K, N, seed=1510, how="affine"))
    w, _ = _blocks(1511, 600, N)
    packed = device.mxfp4_pack(_dev(w), 600, N)
    x = _dev(_act(1512, M, K))
    for rows in (1, 8, 40, 300):
        got = []
        for pause in (True, False, False):
            h = device.gemm(x, q, GGMLType.Q4_K, M, K, N)
            if pause:
                torch.cuda.synchronize()
            got.append(device.mxfp4_gemm(h[M - rows:], packed, rows, N, 600))
        device.sync()
        assert torch.isfinite(got[0]).all() and torch.equal(got[0], got[1]) and torch.equal(got[0], got[2]), rows


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_quantize_edges_of_16_bits(dtype):
    """Zeros, numbers below the normal ones, the largest ones, ties, infinities and NaN in the types that have a way of their own to the largest magnitude; then every
    number of the type as its block's largest."""
    import torch
    from laplace_b200 import device
    t = getattr(torch, dtype)
    info = torch.finfo(t)
    edges = torch.from_numpy(_edge_values()).clamp(-info.max, info.max).to(t)
    tiny = torch.tensor([info.smallest_normal, info.smallest_normal / 2, info.smallest_normal * info.eps, 3 * info.smallest_normal * info.eps, info.max, -info.max, info.max / 2], dtype=torch.float64).to(t)
    bad = torch.ones(4, 32, dtype=t)
    bad[0, 0], bad[1, 31], bad[2, 16], bad[3, 15] = float("inf"), -float("inf"), float("nan"), -float("nan")
    every = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(t)
    g = torch.Generator().manual_seed(1520)
    blocks = (every.float()[:, None] * torch.rand(1 << 16, 32, generator=g)).to(t)
    blocks[torch.arange(1 << 16), torch.arange(1 << 16) % 32] = every
    for x in (edges, tiny[:, None].expand(-1, 32).contiguous(), torch.cat([tiny, -tiny, torch.zeros(18, dtype=t)])[None].contiguous(), bad, blocks):
        got = device.mxfp4_quantize(x.cuda()).cpu().numpy().reshape(-1, 17)
        assert np.array_equal(got, ref.quantize_mxfp4(x.float().numpy()).reshape(-1, 17))
