"""The work that the microscaled 4-bit operators are measured on: MXFP4 weights (GGUF type 39), from the values of a
trained matrix to the products that a program which serves a model makes with them.

Formats. A block is 32 values of a row that share a power of two, 2^s. MXFP4 holds a value as e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6
and their negatives), MXFP8 as e4m3 (largest 448). A GGUF block is 17 bytes: s + 127, then 16 bytes whose low halves are the
values 0..15 and whose high halves the values 16..31.

Kinds of cases
  quantize   values [rows, k] in fp32, fp16 or bf16 -> GGUF blocks with s = floor(log2(largest magnitude)) - 2, to nearest,
             ties to even, magnitudes over 6 held as 6; returned as the values that the blocks stand for.
  product    y[m, j] = sum over the row of xq[m, :] * w[j, :], fp32 x quantized to MXFP8 with the smallest s that keeps the
             block's largest magnitude within 448 * 2^s.
  grouped    the same for (token, expert) pairs: y[p] = xq[row of p] . w[expert of p], experts with whatever number of pairs the
             router gave them, none included; a pair of expert -1 (another GPU's) leaves its row of y as it was.

Weights are N(0, 0.02^2), activations N(0, 1) times a spread over channels, as the inputs of a trained model's matrices have
it; router logits are N(0, 1) with a preference for some experts.
"""
import functools
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one row of a table that is updated in place: launch and latency are all there is
        {"name": "quantize_row", "kind": "quantize", "rows": 1, "k": 4096, "dtype": "f32"},
        # an fp16 matrix of odd extents
        {"name": "quantize_odd_f16", "kind": "quantize", "rows": 1001, "k": 2848, "dtype": "f16"},
        # the largest matrix of an 8B model's layer, from a bf16 file
        {"name": "quantize_matrix_bf16", "kind": "quantize", "rows": 14336, "k": 4096, "dtype": "bf16"},
        # a key or value projection in a decode step of one sequence
        {"name": "product_1_small", "kind": "product", "tokens": 1, "k": 4096, "n": 1024},
        # the gate matrix in the same step
        {"name": "product_1", "kind": "product", "tokens": 1, "k": 4096, "n": 14336},
        # two dozen sequences decoded together, the down matrix
        {"name": "product_24", "kind": "product", "tokens": 24, "k": 14336, "n": 4096},
        # a short prompt of ragged length, extents that are no powers of two
        {"name": "product_77", "kind": "product", "tokens": 77, "k": 2816, "n": 8448},
        # a prompt of 512 tokens, the gate matrix
        {"name": "product_512", "kind": "product", "tokens": 512, "k": 4096, "n": 14336},
        # the largest prompt chunk a server would take in one pass, the down matrix
        {"name": "product_2048", "kind": "product", "tokens": 2048, "k": 14336, "n": 4096},
        # one token through gate / up of its eight experts
        {"name": "grouped_1", "kind": "grouped", "tokens": 1, "top_k": 8, "experts": 128, "k": 2048, "n": 1536, "own_rows": False, "here": 1.0},
        # a batch of 256 tokens through the same, a shared input row per token
        {"name": "grouped_256", "kind": "grouped", "tokens": 256, "top_k": 8, "experts": 128, "k": 2048, "n": 1536, "own_rows": False, "here": 1.0},
        # a prompt chunk through the down matrices, an input row per pair, a quarter of the experts on another GPU
        {"name": "grouped_2048_down", "kind": "grouped", "tokens": 2048, "top_k": 8, "experts": 128, "k": 768, "n": 2048, "own_rows": True, "here": 0.75},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "product", "product", "grouped", "grouped"])
    if kind == "quantize":
        k = 32 * _log_int(rng, 2, 448)
        return {"kind": kind, "rows": _log_int(rng, 1, 14336 * 4096 // k), "k": k, "dtype": rng.choice(sorted(DTYPES))}
    if kind == "product":
        k, n = 32 * _log_int(rng, 2, 448), _log_int(rng, 40, 16384)
        most = min(2048, 2048 * 14336 * 4096 // (k * n))
        return {"kind": kind, "tokens": rng.choice([1, _log_int(rng, 1, 32), _log_int(rng, 1, most)]), "k": k, "n": n}
    experts = rng.choice([4, 8, 32, 60, 64, 128])
    k = 32 * _log_int(rng, 8, 64)
    n = _log_int(rng, 200, min(2048, 128 * 1536 * 2048 // (experts * k)))
    return {"kind": kind, "tokens": _log_int(rng, 1, 2048), "top_k": rng.randint(1, min(8, experts)), "experts": experts, "k": k, "n": n, "own_rows": rng.random() < 0.5,
            "here": rng.choice([1.0, 1.0, 0.5])}


# ---------------------------------------------------------------- plain forms

def _pow2(s):
    return torch.exp2(s.double()).float()


def _exponent(amax):
    """floor(log2) of positive fp32 numbers; -127 for 0 and numbers below the normal ones."""
    return (amax.view(torch.int32) >> 23) - 127


def _mxfp4_codes(x):
    """Values [..., 32] -> (s + 127, e2m1 codes with the sign in bit 3)."""
    x = x.float()
    s = (_exponent(x.abs().amax(-1)) - 2).clamp_min(-127)
    v = (x * _pow2(-s)[..., None])
    a = v.abs()
    mids = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)
    code = sum(((a > m) if i % 2 == 0 else (a >= m)).to(torch.int32) for i, m in enumerate(mids))
    return s + 127, code + 8 * (v < 0).to(torch.int32)


@functools.cache
def _e2m1(device):
    return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=device)


def _mxfp4_values(e, code):
    return _e2m1(code.device)[code] * _pow2(e - 127)[..., None]


def _blocks(x):
    """Rows [n, k] -> GGUF blocks, flat bytes."""
    e, c = _mxfp4_codes(x.reshape(-1, 32))
    return torch.cat([e[:, None], c[:, :16] | (c[:, 16:] << 4)], 1).to(torch.uint8).reshape(-1)


def _unblock(w):
    """GGUF blocks -> values [blocks, 32]."""
    b = w.view(-1, 17).to(torch.int32)
    return _mxfp4_values(b[:, 0], torch.cat([b[:, 1:] & 15, b[:, 1:] >> 4], 1))


def _mxfp8(x):
    """fp32 [m, k] -> the values that MXFP8 holds for them."""
    b = x.reshape(x.shape[0], -1, 32)
    amax = b.abs().amax(-1)
    e = _exponent(amax)
    s = (e - 8 + (amax > 1.75 * _pow2(e)).to(torch.int32)).clamp_min(-127)
    v = b * _pow2(-s)[..., None]
    step = _pow2(_exponent(v.abs()).clamp_min(-6) - 3)
    return (torch.round(v / step) * step * _pow2(s)[..., None]).reshape(x.shape)


# ---------------------------------------------------------------- one pass

def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _activations(g, m, k):
    return _normal(g, m, k) * torch.exp(0.5 * _normal(g, k))


def _weights(g, n, k):
    out = torch.empty(n * (k // 32) * 17, dtype=torch.uint8, device="cuda")
    rb = k // 32 * 17
    for r in range(0, n, 16384):                  # in pieces: the fp32 values of a large matrix need not exist at once
        m = min(16384, n - r)
        out[r * rb:(r + m) * rb] = _blocks(_normal(g, m, k) * 0.02)
    return out


def _pairs(case, g):
    """The router's choice: (expert of each pair, -1 for another GPU's; token of each pair)."""
    t, k, e = case["tokens"], case["top_k"], case["experts"]
    logits = _normal(g, t, e) + 1.5 * _normal(g, e)
    idx = logits.topk(k, dim=1).indices
    kept = torch.arange(e, device="cuda") < max(1, int(case["here"] * e))
    return torch.where(kept[idx], idx, torch.full_like(idx, -1)).reshape(-1).int(), torch.arange(t, device="cuda").repeat_interleave(k).int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "quantize":
        return {"case": case, "x": (_normal(g, case["rows"], case["k"]) * 0.02).to(DTYPES[case["dtype"]])}
    k, n, e = case["k"], case["n"], case.get("experts", 1)
    s = {"case": case, "w": _weights(g, e * n, k)}
    if case["kind"] == "product":
        s["x"] = _activations(g, case["tokens"], k)
    else:
        expert, token = _pairs(case, g)
        pairs = expert.numel()
        s.update(expert=expert, row=None if case["own_rows"] else token, x=_activations(g, pairs if case["own_rows"] else case["tokens"], k), y=torch.zeros(pairs, n, device="cuda"),
                 most=int(torch.bincount(expert.clamp_min(0), minlength=e).max()))
    if own:                                       # weights laid out once, as at model load
        from laplace_b200 import device
        s["packed"] = device.mxfp4_pack(s["w"], n, k, e)
    return s


def run(s):
    c = s["case"]
    if own:
        from laplace_b200 import device
        from laplace_b200.ggml import GGMLType
        if c["kind"] == "quantize":
            return device.dequantize(device.mxfp4_quantize(s["x"]), GGMLType.MXFP4, c["rows"] * c["k"]).view(c["rows"], c["k"])
        if c["kind"] == "product":
            return device.mxfp4_gemm(s["x"], s["packed"], c["tokens"], c["k"], c["n"])
        return device.mxfp4_moe_grouped(s["x"], s["packed"], s["expert"], s["row"], c["experts"], c["k"], c["n"], y=s["y"])
    if c["kind"] == "quantize":
        return _unblock(_blocks(s["x"])).view(c["rows"], c["k"])
    w, xq = _unblock(s["w"]), _mxfp8(s["x"])
    if c["kind"] == "product":
        return xq @ w.view(c["n"], c["k"]).t()
    # pairs sorted into one slab of rows per expert (slab E takes those that are not computed here), one batched product
    e, expert = c["experts"], s["expert"].long()
    here = expert >= 0
    slab = torch.where(here, expert, torch.full_like(expert, e))
    rank = (slab[:, None] == torch.arange(e, device="cuda")).int().cumsum(0).gather(1, expert.clamp_min(0)[:, None])[:, 0].long() - 1
    rank = torch.where(here, rank, torch.zeros_like(rank))
    x = torch.zeros(e + 1, s["most"], c["k"], device="cuda")
    x[slab, rank] = xq if s["row"] is None else xq[s["row"].long()]
    y = torch.bmm(x[:e], w.view(e, c["n"], c["k"]).transpose(1, 2))
    return torch.where(here[:, None], y[expert.clamp_min(0), rank], s["y"])


# ------------------------------------------------- what a pass cannot do without

def work(case):
    k = case["k"]
    if case["kind"] == "quantize":
        v = case["rows"] * k
        return {"bytes": v * (4 if case["dtype"] == "f32" else 2) + v // 32 * 17 + 4 * v, "flops": 4 * v}
    n = case["n"]
    if case["kind"] == "product":
        m = case["tokens"]
        return {"bytes": 4 * m * k + n * k // 32 * 17 + 4 * m * n, "flops": 2 * m * n * k}
    pairs = case["tokens"] * case["top_k"]
    here = max(1, int(case["here"] * case["experts"]))
    computed = pairs * here // case["experts"]
    rows = computed if case["own_rows"] else case["tokens"]
    # experts that at least one pair goes to, were the router even-handed
    met = here * (1 - (1 - 1 / case["experts"]) ** pairs)
    return {"bytes": int(4 * rows * k + met * n * (k // 32) * 17 + 8 * pairs + 4 * computed * n), "flops": 2 * computed * n * k}


# ------------------------------------------------- the definition, in 64 bits

def _exact_mxfp4(x):
    b = x.double().reshape(-1, 32)
    top = b.abs().amax(1, keepdim=True)
    p = 2.0 ** torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))).sub(2)
    v = (b / p).clamp(-6, 6)
    unit = 2.0 ** torch.floor(torch.log2(v.abs().clamp_min(1.0))).sub(1)
    return torch.round(v / unit) * unit * p


def _exact_mxfp8(x):
    b = x.double().reshape(-1, 32)
    top = b.abs().amax(1, keepdim=True)
    p = 2.0 ** torch.ceil(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / 448.0))
    p = torch.where(top > 448.0 * p, 2 * p, torch.where(top <= 224.0 * p, p / 2, p))      # where the logarithm was rounded over a whole number
    return ((b / p).float().to(torch.float8_e4m3fn).double() * p).reshape(x.shape)


def _exact_weights(w):
    b = w.view(-1, 17)
    n = torch.stack([b[:, 1:] % 16, b[:, 1:] // 16], 1).reshape(-1, 32).long()
    size = n % 8
    mag = torch.where(size < 2, 0.5 * size.double(), (1 + 0.5 * (size % 2).double()) * 2.0 ** (size // 2 - 1).double())
    return torch.where(n >= 8, -mag, mag) * 2.0 ** (b[:, :1].double() - 127)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        return _exact_mxfp4(s["x"]).view(case["rows"], case["k"])
    n, k = case["n"], case["k"]
    w, x = _exact_weights(s["w"]).view(-1, n, k), _exact_mxfp8(s["x"])
    if case["kind"] == "product":
        return x @ w[0].t()
    y = s["y"].double()
    for e in range(case["experts"]):
        at = torch.nonzero(s["expert"] == e)[:, 0]
        if at.numel():
            y[at] = x[at if s["row"] is None else s["row"][at].long()] @ w[e].t()
    return y
