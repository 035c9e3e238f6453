"""Microscaled 4-bit floating point as a user of this library has it run: quantisation and read-back of matrices, the
product of two such matrices, and a mixture-of-experts layer for a few tokens with 4-bit weights.

Two formats.  A matrix is cut into blocks along its rows; a block holds E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives) and one scale:

  mxfp4   blocks of 32, scale 2^max(-127, floor(log2 amax) - 2) (E8M0)
  nvfp4   blocks of 16, scale E4M3 nearest to amax / 6 of the values times 2^-exponent, within [2^-9, 448]

Codes are the nearest E2M1 value of value / scale (ties to even), saturated at 6.  Packed rows hold element 2 i in the low
half of byte i.  Scales lie in tiles of 128 rows x 4 blocks, 512 bytes: row r, block b of a tile at (r % 32) * 16 +
(r / 32) * 4 + b; tiles follow each other along a row of tiles, what lies outside the matrix is 0.

``own`` false computes the plain form, true calls the library.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

# nothing drawn costs more than the largest listed case of its kind
MATRIX_MAX = 8192 * 4096
PRODUCT_MAX = 4096 * 14336 * 4096
EXPERT_WEIGHTS_MAX = 64 * 768 * 2048


# ---- cases ------------------------------------------------------------------------------------------------
def matrix(kind, rows, cols, dtype, fmt, exponent=0):
    return dict(kind=kind, rows=rows, cols=cols, dtype=dtype, fmt=fmt, exponent=exponent)


def product(M, N, K, dtype, fmt, bias):
    return dict(kind="product", M=M, N=N, K=K, dtype=dtype, fmt=fmt, bias=bias)


def moe(tokens, hidden, inner, experts, top_k, dtype, fmt, renormalise):
    return dict(kind="moe", tokens=tokens, hidden=hidden, inner=inner, experts=experts, top_k=top_k, dtype=dtype, fmt=fmt,
                renormalise=renormalise)


def listed():
    return [
        # activations of one token on their way into a linear layer: latency only
        dict(matrix("quantise", 1, 4096, "bf16", "nvfp4"), name="quantise_token"),
        # activations of a whole prompt, the rows and width of the LLM-style linear layer of the benchmark
        dict(matrix("quantise", 8192, 4096, "bf16", "mxfp4"), name="quantise_prompt"),
        # weights straight from training: 32-bit, small values (tensor exponent)
        dict(matrix("quantise", 4096, 4096, "f32", "nvfp4", -6), name="quantise_weights"),
        # an odd width: rows that start at any byte, a last block that is not full
        dict(matrix("quantise", 1023, 2049, "f16", "mxfp4"), name="quantise_ragged"),
        # stored weights read back for a layer that computes in 16 bits
        dict(matrix("read_back", 8192, 4096, "bf16", "nvfp4", -6), name="read_back_weights"),
        # a stored table of odd width read back in 32 bits
        dict(matrix("read_back", 333, 1001, "f32", "mxfp4"), name="read_back_ragged"),
        # one token through a square projection: weights read once, latency
        dict(product(1, 4096, 4096, "bf16", "nvfp4", True), name="product_token"),
        # a decoding batch through the wide projection: bound by the weights' bytes
        dict(product(24, 14336, 4096, "f16", "mxfp4", False), name="product_batch"),
        # a prompt through the wide projection: bound by the tensor cores
        dict(product(4096, 14336, 4096, "bf16", "nvfp4", False), name="product_prompt"),
        # ragged in every dimension, 32-bit logits
        dict(product(333, 1001, 2050, "f32", "mxfp4", True), name="product_ragged"),
        # one token through an expert layer: eight experts' weights are all there is to read
        dict(moe(1, 2048, 768, 64, 8, "bf16", "nvfp4", True), name="moe_token"),
        # a decoding batch: most experts are hit by a few tokens each
        dict(moe(48, 2048, 768, 64, 4, "f16", "mxfp4", True), name="moe_batch"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantise", "read_back", "product", "product", "moe"])
    fmt = rng.choice(["mxfp4", "nvfp4"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind in ("quantise", "read_back"):
        cols = _log(rng, 16, 16384)
        rows = _log(rng, 1, max(1, min(16384, MATRIX_MAX // cols)))
        if rng.random() < 0.5:
            cols = max(32, cols // 32 * 32)
        return matrix(kind, rows, cols, dtype, fmt, rng.choice([0, -6, 3]) if fmt == "nvfp4" else 0)
    if kind == "product":
        M = _log(rng, 1, 8192)
        K = _log(rng, 64, 14336)
        N = _log(rng, 64, max(64, min(16384, PRODUCT_MAX // (M * K))))
        if rng.random() < 0.6:
            N, K = max(64, N // 64 * 64), max(64, K // 64 * 64)
        return product(M, N, K, dtype, fmt, rng.random() < 0.5)
    tokens = _log(rng, 1, 128)
    experts = rng.choice([8, 16, 32, 60, 64, 128])
    hidden = 16 * _log(rng, 16, 256)
    inner = 16 * _log(rng, 8, max(8, min(256, EXPERT_WEIGHTS_MAX // (experts * hidden * 16))))
    return moe(tokens, hidden, inner, experts, rng.choice([1, 2, 4, 6, 8]), rng.choice(["f16", "bf16"]), fmt, rng.random() < 0.7)


# ---- inputs -----------------------------------------------------------------------------------------------
def _pitch(cols):
    """Bytes between packed rows: the next multiple of 16."""
    return (cols + 31) // 32 * 16


def _blocks(cols, fmt):
    return -(-cols // BLOCK[fmt])


def _pow2(n):
    """2^n of whole n, float32, from the bits of a double (a power function may be off by a step)."""
    return ((n.to(torch.int64) + 1023) << 52).view(torch.float64).to(torch.float32)


def _quantise(x, fmt, exponent):
    """(E2M1 values, block scales without the exponent) of a float32 matrix, values [rows, blocks, block]."""
    rows, cols = x.shape
    block = BLOCK[fmt]
    t = torch.nn.functional.pad(x * 2.0 ** -exponent, (0, -cols % block)).reshape(rows, -1, block)
    amax = t.abs().amax(dim=2, keepdim=True)
    if fmt == "mxfp4":
        scale = _pow2((torch.frexp(amax).exponent - 3).clamp(min=-127))
    else:
        scale = (amax / torch.full_like(amax, 6.0)).clamp(2.0 ** -9, 448.0)  # a true division: a scalar divisor becomes a product
        scale = scale.to(torch.float8_e4m3fn).to(torch.float32)
    scale = torch.where(amax > 0, scale, 0.0)
    a = t.abs() / torch.where(amax > 0, scale, 1.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp(max=6.0)
    return torch.copysign(q, t), scale[:, :, 0]


def _pack(q, scale, fmt, cols):
    """Packed codes (rows at the pitch) and tiled scale bytes of what _quantise returns."""
    rows, nb = scale.shape
    index = torch.zeros(13, dtype=torch.uint8, device=q.device)
    index[torch.tensor([int(2 * v) for v in GRID], device=q.device)] = torch.arange(8, dtype=torch.uint8, device=q.device)
    codes = index[(2 * q.abs()).to(torch.int32)] | (torch.signbit(q).to(torch.uint8) << 3)
    codes = codes.reshape(rows, -1)[:, :cols]
    codes = torch.nn.functional.pad(codes, (0, 2 * _pitch(cols) - cols))
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    if fmt == "mxfp4":
        byte = torch.where(scale > 0, torch.frexp(scale).exponent - 1 + 127, 0).to(torch.uint8)
    else:
        byte = scale.to(torch.float8_e4m3fn).view(torch.uint8)
    byte = torch.nn.functional.pad(byte, (0, -nb % 4, 0, -rows % 128))
    tiles = byte.reshape(byte.shape[0] // 128, 4, 32, byte.shape[1] // 4, 4).permute(0, 3, 2, 1, 4)
    return packed.contiguous(), tiles.contiguous()


def _normal(gen, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def _weights(gen, rows, cols, fmt, std):
    """A packed weight matrix and what its values are to be multiplied by."""
    exponent = math.floor(math.log2(std)) if fmt == "nvfp4" else 0
    packed, tiles = _pack(*_quantise(_normal(gen, (rows, cols), std=std), fmt, exponent), fmt, cols)
    return packed, tiles, 2.0 ** exponent


def _experts(gen, experts, rows, cols, fmt, std):
    """One packed matrix per expert: codes [experts * rows, pitch], scale tiles of every expert on their own."""
    parts = [_weights(gen, rows, cols, fmt, std) for _ in range(experts)]
    return torch.cat([p[0] for p in parts]), torch.stack([p[1] for p in parts]), parts[0][2]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, fmt = case["kind"], case["fmt"]
    state = dict(case)
    if kind in ("quantise", "read_back"):
        rows, cols = case["rows"], case["cols"]
        std = 2.0 ** case["exponent"]
        x = _normal(gen, (rows, cols), std=std) * torch.exp(0.5 * _normal(gen, (1, cols)))  # columns of unequal size
        if kind == "quantise":
            state["x"] = x.to(DTYPE[case["dtype"]])
            state["packed"] = torch.zeros((rows, _pitch(cols)), dtype=torch.uint8, device="cuda")
            state["scales"] = torch.zeros((-(-rows // 128), -(-_blocks(cols, fmt) // 4), 512), dtype=torch.uint8, device="cuda")
        else:
            state["packed"], state["scales"] = _pack(*_quantise(x, fmt, case["exponent"]), fmt, cols)
        state["out"] = torch.empty((rows, cols), dtype=DTYPE[case["dtype"]], device="cuda")
    elif kind == "product":
        M, N, K = case["M"], case["N"], case["K"]
        state["a"], state["a_scales"], _ = _weights(gen, M, K, fmt, 1.0)
        state["b"], state["b_scales"], state["alpha"] = _weights(gen, N, K, fmt, 1.0 / math.sqrt(K))
        state["bias"] = _normal(gen, (N,)) if case["bias"] else None
        state["out"] = torch.empty((M, N), dtype=DTYPE[case["dtype"]], device="cuda")
    else:
        T, H, F, E = case["tokens"], case["hidden"], case["inner"], case["experts"]
        state["x"] = _normal(gen, (T, H), DTYPE[case["dtype"]])
        state["logits"] = _normal(gen, (T, E))
        state["gate"] = _experts(gen, E, F, H, fmt, 1.0 / math.sqrt(H))
        state["up"] = _experts(gen, E, F, H, fmt, 1.0 / math.sqrt(H))
        state["down"] = _experts(gen, E, H, F, fmt, 1.0 / math.sqrt(F))
        state["out"] = torch.empty((T, H), dtype=DTYPE[case["dtype"]], device="cuda")
    return state


# ---- the plain form ---------------------------------------------------------------------------------------
def _decode(packed, tiles, fmt, cols):
    """Values of packed rows with one set of scale tiles, float32 [..., rows, cols] (leading dimensions alike)."""
    table = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float32, device=packed.device)
    rows, nb = packed.shape[-2], _blocks(cols, fmt)
    codes = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2)[..., :cols]
    lead = packed.shape[:-2]
    byte = tiles.reshape(lead + (-(-rows // 128), -(-nb // 4), 32, 4, 4)).movedim(-2, -4).movedim(-2, -3)
    byte = byte.reshape(lead + (-(-rows // 128) * 128, -(-nb // 4) * 4))[..., :rows, :nb]
    if fmt == "mxfp4":
        scale = _pow2(byte.to(torch.int64) - 127)
    else:
        scale = byte.contiguous().view(torch.float8_e4m3fn).to(torch.float32)
    return table[codes.to(torch.int32)] * scale.repeat_interleave(BLOCK[fmt], dim=-1)[..., :cols]


def _round_trip(x, fmt):
    q, scale = _quantise(x, fmt, 0)
    return (q * scale[:, :, None]).flatten(1)[:, :x.shape[1]]


def _gate(logits, top_k, renormalise):
    """Chosen experts [T, k] (the largest logits, equal ones by index) and their weights."""
    order = torch.argsort(logits, dim=1, descending=True, stable=True)[:, :top_k]
    chosen = torch.gather(logits, 1, order)
    if renormalise:
        return order, torch.softmax(chosen, dim=1)
    return order, torch.exp(chosen - torch.logsumexp(logits, dim=1, keepdim=True))


def _moe_plain(s):
    T, H, F, E, k, fmt = s["tokens"], s["hidden"], s["inner"], s["experts"], min(s["top_k"], s["experts"]), s["fmt"]
    ids, p = _gate(s["logits"], k, s["renormalise"])
    x = _round_trip(s["x"].float(), fmt)
    few = T * k <= E // 2  # only the chosen experts are decoded, else every one once

    def values(w, rows, cols):
        codes, tiles = w[0].view(E, rows, -1), w[1]
        if few:
            codes, tiles = codes[ids.flatten()], tiles[ids.flatten()]
        return _decode(codes, tiles, fmt, cols) * w[2]

    if few:  # [T * k, ...]: every pair of a token and an expert on its own
        xs = x.repeat_interleave(k, dim=0)[:, :, None]
        g, u = torch.matmul(values(s["gate"], F, H), xs)[:, :, 0], torch.matmul(values(s["up"], F, H), xs)[:, :, 0]
        h = _round_trip(p.flatten()[:, None] * torch.nn.functional.silu(g) * u, fmt)
        y = torch.matmul(values(s["down"], H, F), h[:, :, None])[:, :, 0]
        return y.view(T, k, H).sum(dim=1)
    weight = torch.zeros((T, E), dtype=torch.float32, device=x.device).scatter(1, ids, p)  # 0: not chosen
    g, u = torch.matmul(x, values(s["gate"], F, H).mT), torch.matmul(x, values(s["up"], F, H).mT)  # [E, T, F]
    h = weight.T[:, :, None] * torch.nn.functional.silu(g) * u
    h = _round_trip(h.reshape(E * T, F), fmt).view(E, T, F)
    return torch.matmul(h, values(s["down"], H, F).mT).sum(dim=0)


def _plain(s):
    kind, dtype = s["kind"], DTYPE[s["dtype"]]
    if kind == "quantise":
        q, scale = _quantise(s["x"].float(), s["fmt"], s["exponent"])
        return (q * (scale[:, :, None] * 2.0 ** s["exponent"])).flatten(1)[:, :s["cols"]].to(dtype)
    if kind == "read_back":
        return (_decode(s["packed"], s["scales"], s["fmt"], s["cols"]) * 2.0 ** s["exponent"]).to(dtype)
    if kind == "product":
        a, b = _decode(s["a"], s["a_scales"], s["fmt"], s["K"]), _decode(s["b"], s["b_scales"], s["fmt"], s["K"])
        y = torch.matmul(a, b.T) * s["alpha"]
        return (y + s["bias"] if s["bias"] is not None else y).to(dtype)
    return _moe_plain(s).to(dtype)


# ---- the library's calls ----------------------------------------------------------------------------------
_kept = {}


def _context():
    """The context a program keeps for its stream (the default stream's handle is the same on every device)."""
    import computelibrary_b200 as cl

    at = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream
    if at not in _kept:
        _kept[at] = cl.Context(*at)
    return _kept[at]


def _describe(s):
    """The descriptor (and workspace) a program fills in once for tensors of these shapes."""
    from computelibrary_b200 import capi

    fmt = {"mxfp4": capi.MXFP4, "nvfp4": capi.NVFP4}[s["fmt"]]
    dtype = {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}[s["dtype"]]
    if s["kind"] in ("quantise", "read_back"):
        s["desc"] = capi.make_mx_desc(s["rows"], s["cols"], fmt, dtype, tensor_exponent=s["exponent"])
    elif s["kind"] == "product":
        s["desc"] = capi.make_mx_gemm_desc(s["M"], s["N"], s["K"], fmt, dtype, alpha=s["alpha"], has_bias=s["bias"] is not None)
    else:
        s["desc"] = capi.make_mx_moe_desc(s["tokens"], s["hidden"], s["inner"], s["experts"], min(s["top_k"], s["experts"]), fmt, dtype,
                                          renormalize=s["renormalise"], gate_alpha=s["gate"][2], up_alpha=s["up"][2],
                                          down_alpha=s["down"][2])
        s["workspace"] = torch.empty(capi.mx_moe_workspace_bytes(s["desc"]), dtype=torch.uint8, device="cuda")
    return s["desc"]


def _library(s):
    ctx = _context()
    desc = s.get("desc") or _describe(s)
    kind = s["kind"]
    if kind == "quantise":  # written and read back: codes are returned as the values they stand for
        ctx.mx_quantize(desc, s["x"], s["packed"], s["scales"])
        ctx.mx_dequantize(desc, s["packed"], s["scales"], s["out"])
    elif kind == "read_back":
        ctx.mx_dequantize(desc, s["packed"], s["scales"], s["out"])
    elif kind == "product":
        ctx.mx_gemm(desc, s["a"], s["a_scales"], s["b"], s["b_scales"], s["bias"], s["out"])
    else:
        ctx.mx_moe(desc, s["x"], s["logits"], s["gate"][:2], s["up"][:2], s["down"][:2], s["out"], s["workspace"])
    return s["out"]


def run(state):
    return _library(state) if own else _plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------
def work(case):
    kind, fmt = case["kind"], case["fmt"]
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]

    def stored(rows, cols):  # codes and scales
        return rows * (cols / 2 + _blocks(cols, fmt))

    if kind == "quantise":  # read, store, read back
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * size + 2 * stored(case["rows"], case["cols"]), "flops": 4 * n}
    if kind == "read_back":
        n = case["rows"] * case["cols"]
        return {"bytes": n * size + stored(case["rows"], case["cols"]), "flops": 2 * n}
    if kind == "product":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": stored(M, K) + stored(N, K) + M * N * size + (4 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    T, H, F, E = case["tokens"], case["hidden"], case["inner"], case["experts"]
    k = min(case["top_k"], E)
    hit = E * (1 - (1 - k / E) ** T)  # experts that at least one token is expected to choose
    return {"bytes": hit * (2 * stored(F, H) + stored(H, F)) + 2 * T * H * size + 4 * T * E, "flops": 6 * T * k * H * F}


# ---- the definition in 64 bits ----------------------------------------------------------------------------
def _exponent(v):
    """floor(log2 v) (a logarithm may land on the wrong side of a power of two)."""
    return torch.frexp(v).exponent.long() - 1


def _two_to(n):
    return torch.tensor([2.0 ** i for i in range(-160, 161)], dtype=torch.float64, device=n.device)[n + 160]


def _exact_scale(amax, fmt):
    if fmt == "mxfp4":
        return torch.where(amax > 0, _two_to((_exponent(amax) - 2).clamp(min=-127)), 0.0)
    v = (amax / torch.full_like(amax, 6.0)).clamp(2.0 ** -9, 448.0)
    ulp = _two_to(_exponent(v).clamp(min=-6) - 3)  # three bits behind the leading one, subnormals below 2^-6
    return torch.where(amax > 0, torch.round(v / ulp) * ulp, 0.0)


def _exact_values(x, fmt, exponent):
    """What x holds once stored, float64."""
    rows, cols = x.shape
    block = BLOCK[fmt]
    t = torch.zeros((rows, _blocks(cols, fmt) * block), dtype=torch.float64, device=x.device)
    t[:, :cols] = x.double() * 2.0 ** -exponent
    t = t.view(rows, -1, block)
    scale = _exact_scale(t.abs().amax(2, keepdim=True), fmt)
    r = t.abs() / torch.where(scale > 0, scale, 1.0)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    below, above = torch.bucketize(r, mid, right=False), torch.bucketize(r, mid, right=True)  # differ at a tie only
    v = grid[torch.where(below % 2 == 0, below, above)]
    return (torch.sign(t) * v * scale * 2.0 ** exponent).view(rows, -1)[:, :cols]


def _exact_decode(packed, tiles, fmt, cols):
    """The values at every (row, column), by index arithmetic on the layout."""
    packed = packed.long()
    rows = packed.shape[0]
    r = torch.arange(rows, device=packed.device)[:, None]
    c = torch.arange(cols, device=packed.device)[None, :]
    code = (packed[r, c // 2] >> (4 * (c % 2))) & 15
    b = c // BLOCK[fmt]
    across = -(-_blocks(cols, fmt) // 4)
    byte = tiles.reshape(-1).long()[((r // 128) * across + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4]
    if fmt == "mxfp4":
        scale = _two_to(byte - 127)
    else:
        e, m = byte // 8, (byte % 8).double()
        scale = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * _two_to(e - 7))
    m, e = (code & 1).double(), (code >> 1) & 3
    v = torch.where(e == 0, m / 2, (1 + m / 2) * _two_to(e - 1))
    return torch.where(code >= 8, -v, v) * scale


def exact(case, seed):
    s = prepare(case, seed)
    kind, fmt = case["kind"], case["fmt"]
    if kind == "quantise":
        return _exact_values(s["x"], fmt, case["exponent"])
    if kind == "read_back":
        return _exact_decode(s["packed"], s["scales"], fmt, case["cols"]) * 2.0 ** case["exponent"]
    if kind == "product":
        K = case["K"]
        y = _exact_decode(s["a"], s["a_scales"], fmt, K) @ _exact_decode(s["b"], s["b_scales"], fmt, K).T * s["alpha"]
        return y + s["bias"].double() if s["bias"] is not None else y
    T, H, F, E = case["tokens"], case["hidden"], case["inner"], case["experts"]
    k = min(case["top_k"], E)
    x = _exact_values(s["x"], fmt, 0)
    logits = s["logits"].double().cpu().numpy()
    y = torch.zeros((T, H), dtype=torch.float64, device="cuda")
    ids = np.stack([np.lexsort((np.arange(E), -row))[:k] for row in logits])
    for e in range(E):
        tokens = np.nonzero((ids == e).any(axis=1))[0]
        if not len(tokens):
            continue
        among = np.stack([logits[t] if not case["renormalise"] else logits[t][ids[t]] for t in tokens])
        p = torch.from_numpy(1 / np.exp(among - logits[tokens, e][:, None]).sum(axis=1)).cuda()
        at = torch.from_numpy(tokens).cuda()
        w = [_exact_decode(s[n][0].view(E, rows, -1)[e], s[n][1][e], fmt, cols) * s[n][2]
             for n, rows, cols in (("gate", F, H), ("up", F, H), ("down", H, F))]
        g, u = x[at] @ w[0].T, x[at] @ w[1].T
        h = _exact_values(p[:, None] * g / (1 + torch.exp(-g)) * u, fmt, 0)
        y[at] += h @ w[2].T
    return y
