"""MXFP4 products whose k is shared by several CTAs: sums sent through a cluster's shared memory, in kernels of a handful of rows and of middle sizes, and parts of
cut tiles left in the workspace, on pairs of SMs. Sizes at which buffers, slots and accumulators are used again, runs lie across a tile's border, and tiles are more
than a call's plan reckons with; each says which kernel it has to reach."""
import numpy as np
import pytest

from laplace_b200.ggml import GGMLType, any_row_bytes
from tests import mxfp4_ref as ref
from tests.test_mxfp4_gpu import _act, _close, _dev

pytestmark = pytest.mark.gpu
SMALL, SINGLE, PAIR = 1, 2, 3                                  # laplace_cuda_mxfp4_last_kernel, + 16 x the CTAs that share k
MARK = 0xA5


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


# ---- cut tiles -----------------------------------------------------------------------------------------------------------------

def _round256(n):
    return (n + 255) & ~255


def _parts_left(ws, behind=0):
    """Parts of cut tiles that the even CTAs left in a workspace whose last `behind` bytes come after their area: of every cut tile all but the one whose pair was the last.
    Two slots a pair of SMs, 128 KB for each of its CTAs."""
    from laplace_b200 import device
    area = 2 * device.lib().laplace_cuda_sm_count() * 256 * 128 * 4
    end = ws.numel() - behind
    return int((ws[end - area:end].view(-1, 2, 256 * 128 * 4)[:, 0] != MARK).any(1).sum())


# 300: 18 tiles in four; 600, 2000: 36 and 33 tiles in halves; 2048 x 2600: 14 tiles over 74 pairs of SMs, whose runs lie across the tiles' borders, then 74 whole ones;
# 1030: 6 tiles in twelve parts and more, then 74 whole ones; 640: none
@pytest.mark.parametrize("M,K,N,parts", [(300, 14336, 2100, 54), (600, 14336, 2100, 36), (2000, 8192, 700, 33), (2048, 14336, 2600, 72), (1030, 14336, 4096, 72), (640, 4096, 4100, 0)])
def test_cut_tiles(M, K, N, parts):
    import torch
    from laplace_b200 import device
    L = device.lib()
    w = _weights(1640 + M, N, K)
    x = _act(1641 + M, M, K)
    packed, xd = device.mxfp4_pack(w, N, K), _dev(x)
    n = L.laplace_cuda_mxfp4_workspace_size(M, 0, K, N)
    ws, y = torch.full((n,), MARK, dtype=torch.uint8, device="cuda"), torch.empty(M, N, device="cuda")
    assert L.laplace_cuda_mxfp4_gemm_dev(xd.data_ptr(), packed.data_ptr(), y.data_ptr(), M, K, N, ws.data_ptr(), n, 1) == 0
    device.sync()
    assert _kernel() == PAIR + 16 and _parts_left(ws) == parts
    _close(y, *_product(torch.from_numpy(ref.mxfp8(x)).cuda(), w, N, K), K, f"M={M} K={K} N={N}")
    for _ in range(5):
        assert torch.equal(device.mxfp4_gemm(xd, packed, M, K, N), y)
    device.sync()


# The plan is made on the GPU: 12 tiles in three; 24 in three, three experts; 10 in four, of ragged experts and an odd number of row tiles; 14 over 74 pairs of SMs, across the
# tiles' borders, then 74 whole ones
@pytest.mark.parametrize("counts,K,N,parts", [((150,), 8192, 3000, 24), ((300, 290, 400), 8192, 1000, 48), ((512, 0, 300, 150), 14336, 300, 30), ((450, 450), 5376, 5600, 72)])
@pytest.mark.parametrize("form", ["own", "elsewhere", "bad rows"])
def test_cut_tiles_of_experts(counts, K, N, parts, form):
    import torch
    from laplace_b200 import device
    from laplace_b200.matmul import LaplaceCudaError
    L = device.lib()
    E, P = len(counts), sum(counts)
    rng = np.random.default_rng(1650)
    expert = rng.permutation(np.repeat(np.arange(E), counts)).astype(np.int32)
    row, X = None, P
    if form != "own":
        X = 33
        row = rng.integers(0, X, P).astype(np.int32)
    if form == "elsewhere":
        expert[::50] = -2
    ok = expert.copy()
    if form == "bad rows":
        row[3::11], ok[3::11] = -1, -1
    w = _weights(1651 + P, E * N, K)
    x = _act(1652 + P, X, K)
    packed, xd, ed = device.mxfp4_pack(w, N, K, E), _dev(x), _dev(expert)
    rd = None if row is None else _dev(row)
    n = L.laplace_cuda_mxfp4_workspace_size(P, E, K, N)
    y0 = torch.full((P, N), 7.0, device="cuda")
    ws, y = torch.full((n,), MARK, dtype=torch.uint8, device="cuda"), y0.clone()
    assert L.laplace_cuda_mxfp4_moe_grouped_dev(xd.data_ptr(), X, packed.data_ptr(), ed.data_ptr(), None if rd is None else rd.data_ptr(), P, E, y.data_ptr(), K, N, ws.data_ptr(), n, 1) == 0
    if form == "bad rows":
        with pytest.raises(LaplaceCudaError):
            device.sync()
    device.sync()
    # behind the parts: places, rows of results, token tiles, the plan, counts
    rows, tiles = (P + 7 * min(E, P) + 7) & ~7, P // 256 + min(E, P)
    behind = _round256(8 * P) + _round256(4 * rows) + _round256(16 * tiles) + 256 + _round256(4 * E)
    assert _kernel() == PAIR + 16 and _parts_left(ws, behind) == parts
    _close(y, *_experts(x, w, ok, row, E, N, K, y0.cpu().numpy()), K, f"{counts} K={K} N={N} {form}")
    if form != "bad rows":
        for _ in range(5):
            assert torch.equal(device.mxfp4_moe_grouped(xd, packed, ed, rd, E, K, N, y=y0.clone()), y)
        device.sync()


# ---- side by side ------------------------------------------------------------------------------------------------------------------

def _calls(seed):
    """Calls that share k in every way, on data of their own: clusters of two kernels, one matrix and experts, more tiles than clusters, cut tiles before whole ones."""
    from laplace_b200 import device

    def dense(M, K, N):
        x, p = _dev(_act(seed + M, M, K)), device.mxfp4_pack(_weights(seed + N, N, K), N, K)
        return lambda: device.mxfp4_gemm(x, p, M, K, N)

    def experts(counts, K, N):
        expert = np.random.default_rng(seed).permutation(np.repeat(np.arange(len(counts)), counts)).astype(np.int32)
        x, p, e = _dev(_act(seed + K, len(expert), K)), device.mxfp4_pack(_weights(seed + N, len(counts) * N, K), N, K, len(counts)), _dev(expert)
        return lambda: device.mxfp4_moe_grouped(x, p, e, None, len(counts), K, N)

    return [dense(2, 4096, 76700), dense(4, 14336, 4096), experts((3, 3, 3, 3), 2048, 512), dense(24, 14336, 10240), experts((129, 65, 1, 61), 4096, 1000), dense(1030, 14336, 2048),
            dense(300, 14336, 2100), experts((450, 450), 5376, 5600)]


def test_streams_side_by_side():
    import torch
    from laplace_b200 import device
    sets = [_calls(1660), _calls(1670)]
    want = [[f() for f in c] for c in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for turn in range(10):
        for i in range(len(sets[0])):
            for side in (0, 1):
                with torch.cuda.stream(streams[side]):
                    got[side].append(sets[side][(i + side * turn) % len(sets[0])]())      # other calls meet each turn
    torch.cuda.synchronize()
    for side in (0, 1):
        for turn in range(10):
            for i in range(len(sets[0])):
                assert torch.equal(got[side][turn * len(sets[0]) + i], want[side][(i + side * turn) % len(sets[0])])
    device.sync()


def test_two_graphs_replayed_side_by_side():
    import torch
    from laplace_b200 import device
    sets = [_calls(1680), _calls(1690)]
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


# ---- first calls of a process --------------------------------------------------------------------------------------------------------

_FIRST = """
import sys, threading
import torch
from laplace_b200 import device
from tests.test_mxfp4_exchange_gpu import _calls
from tests.test_mxfp4_gpu import _calls as _more

sets = [_calls(1700 + 10 * i) + _more(1750 + 10 * i) for i in range({threads})]
torch.cuda.synchronize()
"""
_CAPTURE = _FIRST + """
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    outs = [f() for f in sets[0]]
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(y, f()) for y, f in zip(outs, sets[0]))
device.sync()
print("same")
"""
_THREADS = _FIRST + """
got, start = [[] for _ in sets], threading.Barrier(len(sets))
def work(i):
    start.wait()
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(5):
            for f in sets[i]:
                got[i].append(f())
        torch.cuda.current_stream().synchronize()
threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
[t.start() for t in threads]
[t.join() for t in threads]
for ys, calls in zip(got, sets):
    assert len(ys) == 5 * len(calls) and all(torch.equal(y, calls[i % len(calls)]()) for i, y in enumerate(ys))
device.sync()
print("same")
"""


@pytest.mark.parametrize("code,threads", [(_CAPTURE, 1), (_THREADS, 4)], ids=["captured", "threads"])
def test_first_calls(code, threads):
    """A process whose first products are captured into a graph, and one whose first products come from several threads at once: results as later."""
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", code.replace("{threads}", str(threads))], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stdout + r.stderr


# ---- experts whose rows end inside a k tile --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("tokens", [1, 8, 9, 20, 64, 257, 1100])
@pytest.mark.parametrize("gate_up", [True, False])
def test_top_4_of_32_experts_of_2880(tokens, gate_up):
    """Rows of 22.5 k tiles, four experts a token, from one token to a prompt: gate / up with a row per token, down with a row per pair."""
    import torch
    from laplace_b200 import device
    E, K, N = 32, 2880, 720 if gate_up else 360
    rng = np.random.default_rng(1720 + tokens)
    expert = np.argsort(-(rng.standard_normal((tokens, E)) + 1.5 * rng.standard_normal(E)), axis=1)[:, :4].astype(np.int32).reshape(-1)
    row = np.repeat(np.arange(tokens, dtype=np.int32), 4) if gate_up else None
    w, x = _weights(1721, E * N, K), _act(1722, tokens if gate_up else 4 * tokens, K)
    y = device.mxfp4_moe_grouped(_dev(x), device.mxfp4_pack(w, N, K, E), _dev(expert), None if row is None else _dev(row), E, K, N)
    device.sync()
    _close(y, *_experts(x, w, expert, row, E, N, K, np.zeros((4 * tokens, N))), K, f"{tokens} tokens")


# ---- a captured call, replayed with other inputs ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("P,E,K,N", [(20, 6, 2048, 600), (120, 4, 2048, 1000), (700, 4, 8192, 600), (5000, 40, 256, 300)])
def test_replayed_with_another_routing(P, E, K, N):
    """The plan of a call on experts is made on the GPU at every replay: routings from even to all pairs on one expert and to none here, each replay as the call itself."""
    import torch
    from laplace_b200 import device
    rng = np.random.default_rng(1730 + P)
    packed = device.mxfp4_pack(_weights(1731, E * N, K), N, K, E)
    x, y = torch.zeros(P, K, device="cuda"), torch.empty(P, N, device="cuda")
    expert, row = torch.zeros(P, dtype=torch.int32, device="cuda"), torch.zeros(P, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        device.mxfp4_moe_grouped(x, packed, expert, row, E, K, N, y=y)
    even = np.arange(P) % E
    for e in (even, np.full(P, E - 1), np.full(P, -1), np.where(np.arange(P) % 3 == 0, -1, even), rng.choice(E, P, p=rng.dirichlet(np.full(E, 0.3))), np.minimum(even, 1)):
        x.copy_(_dev(_act(1732 + int(e[0]), P, K)))
        expert.copy_(_dev(e.astype(np.int32)))
        row.copy_(_dev(rng.integers(0, P, P).astype(np.int32)))
        y.fill_(7.0)
        want = device.mxfp4_moe_grouped(x, packed, expert, row, E, K, N, y=y.clone())
        g.replay()
        device.sync()
        assert torch.equal(y, want) and (y[expert < 0] == 7).all() and not (y[expert >= 0] == 7).all(1).any()


@pytest.mark.parametrize("M,K,N", [(3, 4096, 600), (24, 4096, 600), (300, 14336, 2100)])
def test_replayed_with_other_rows(M, K, N):
    import torch
    from laplace_b200 import device
    packed = device.mxfp4_pack(_weights(1740, N, K), N, K)
    x, y = torch.zeros(M, K, device="cuda"), torch.empty(M, N, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        device.mxfp4_gemm(x, packed, M, K, N, y=y)
    for i in range(4):
        x.copy_(_dev(_act(1741 + i, M, K)))
        y.fill_(7.0)
        g.replay()
        assert torch.equal(y, device.mxfp4_gemm(x, packed, M, K, N))
    device.sync()
