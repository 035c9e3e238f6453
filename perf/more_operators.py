"""Expert layers of prompts with microscaled 4-bit weights, step by step, and low-rank adapters of many requests, as a user of this
library has them run.

  route      the top_k largest logits of every token, their weights, and a place for every choice: the rows of an expert lie together
             (a group), in the order of the tokens; groups start at multiples of 128 rows
  group      activations quantised to 4 bits, written to the rows of their choices (and read back: codes are returned as the
             values they stand for)
  experts    products of every group with its expert's weights, plain or as SwiGLU of two products
  combine    the rows of a token's choices, times their weights, added up
  lora       dst = base + scale * (x . A^T) . B^T with the adapter of the token's request

The formats are those of perf/operators.py: blocks of 32 with power-of-two scales (mxfp4) or of 16 with E4M3 scales (nvfp4), E2M1
codes, scales in tiles of 128 rows x 4 blocks.

``own`` false computes the plain form, true calls the library.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
ALIGN = 128  # rows at whose multiples groups start

# about what the largest listed cases cost; a drawn case that still costs more than those of its kind is drawn again
ROUTE_MAX = 8192 * 128 * 2       # bytes of logits
GROUP_MAX = 4096 * 4 * 4096 * 2  # bytes of values read back
ROWS_MAX = 4096 * 8              # rows of all groups
WEIGHT_MAX = 64 * 1536 * 2048    # values
RESULT_MAX = 4096 * 8 * 2048 * 2 # bytes
LORA_MAX = 4096 * 4096           # values of one matrix


# ---- cases ------------------------------------------------------------------------------------------------
def route(tokens, experts, top_k, dtype, renormalise):
    return dict(kind="route", tokens=tokens, experts=experts, top_k=top_k, dtype=dtype, renormalise=renormalise)


def group(tokens, cols, experts, top_k, dtype, fmt):
    return dict(kind="group", tokens=tokens, cols=cols, experts=experts, top_k=top_k, dtype=dtype, fmt=fmt)


def experts_(tokens, experts, top_k, N, K, dtype, fmt, swiglu, bias=False):
    return dict(kind="experts", tokens=tokens, experts=experts, top_k=top_k, N=N, K=K, dtype=dtype, fmt=fmt, swiglu=swiglu, bias=bias)


def combine(tokens, cols, experts, top_k, src_dtype, dtype):
    return dict(kind="combine", tokens=tokens, cols=cols, experts=experts, top_k=top_k, src_dtype=src_dtype, dtype=dtype)


def lora(tokens, requests, adapters, rank, K, N, dtype, dst):
    return dict(kind="lora", tokens=tokens, requests=requests, adapters=adapters, rank=rank, K=K, N=N, dtype=dtype, dst=dst)


def listed():
    return [
        # the gate of one token: latency only
        dict(route(1, 64, 8, "f32", True), name="route_token"),
        # the gate of a long prompt, logits as a 16-bit layer leaves them (many of them alike)
        dict(route(8192, 128, 8, "bf16", False), name="route_prompt"),
        # a decoding batch on its way into the experts
        dict(group(48, 2048, 64, 4, "f16", "mxfp4"), name="group_batch"),
        # a prompt on its way into the experts
        dict(group(4096, 4096, 64, 4, "bf16", "nvfp4"), name="group_prompt"),
        # a decoding batch through gate and up: most experts hold a few rows each, their weights' bytes bound it
        dict(experts_(48, 64, 4, 768, 2048, "f16", "mxfp4", True), name="experts_batch"),
        # a prompt through gate and up: bound by the tensor cores
        dict(experts_(4096, 64, 8, 768, 2048, "bf16", "nvfp4", True), name="experts_prompt_up"),
        # and through down: short sums, wide rows
        dict(experts_(4096, 64, 8, 2048, 768, "bf16", "nvfp4", False), name="experts_prompt_down"),
        # ragged in every dimension, few experts with biases, 32-bit results
        dict(experts_(777, 6, 2, 1001, 530, "f32", "mxfp4", False, True), name="experts_ragged"),
        # a decoding batch back from the experts
        dict(combine(48, 2048, 64, 4, "f16", "f16"), name="combine_batch"),
        # a prompt back from the experts
        dict(combine(4096, 2048, 64, 8, "bf16", "bf16"), name="combine_prompt"),
        # a decoding batch, every request with one token and an adapter of its own choice, beside the wide projection
        dict(lora(24, 24, 16, 16, 4096, 14336, "bf16", "bf16"), name="lora_batch"),
        # prompts of a few requests beside the square projection, added before its result is rounded
        dict(lora(4096, 7, 5, 64, 4096, 4096, "f16", "f32"), name="lora_prompts"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    while True:
        case = _draw(rng)
        most = [work(c) for c in listed() if c["kind"] == case["kind"]]
        if all(work(case)[n] <= max(w[n] for w in most) for n in ("bytes", "flops")):
            return case


def _draw(rng):
    kind = rng.choice(["route", "group", "experts", "experts", "combine", "lora", "lora"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    fmt = rng.choice(["mxfp4", "nvfp4"])
    experts = rng.choice([5, 8, 16, 32, 60, 64, 128])
    top_k = rng.choice([k for k in (1, 2, 4, 6, 8) if k <= experts])
    if kind == "route":
        experts = rng.choice([1, 3, 8, 60, 64, 128, 256, 500])
        return route(_log(rng, 1, min(16384, ROUTE_MAX // (experts * SIZE[dtype]))), experts, min(top_k, experts), dtype, rng.random() < 0.6)
    if kind == "group":
        tokens = _log(rng, 1, ROWS_MAX // 2 // top_k)
        cols = _log(rng, 16, min(8192, GROUP_MAX // (tokens * top_k * SIZE[dtype])))
        if rng.random() < 0.6:
            cols = max(32, cols // 32 * 32)
        return group(tokens, cols, experts, top_k, dtype, fmt)
    if kind == "experts":
        swiglu = rng.random() < 0.5
        tokens = _log(rng, 1, ROWS_MAX // top_k)
        K = _log(rng, 64, 4096)
        rows, pair = tokens * top_k, 2 if swiglu else 1
        N = _log(rng, 64, min(4096, WEIGHT_MAX // (experts * K * pair), ROWS_MAX * 1536 * 2048 // (rows * K * pair), RESULT_MAX // (rows * SIZE[dtype])))
        if rng.random() < 0.6:
            N, K = max(64, N // 64 * 64), max(64, K // 64 * 64)
        return experts_(tokens, experts, top_k, N, K, dtype, fmt, swiglu, not swiglu and rng.random() < 0.3)
    if kind == "combine":
        tokens = _log(rng, 1, ROWS_MAX // top_k)
        src_dtype = rng.choice(["f16", "bf16", "f32"])
        cols = _log(rng, 16, min(8192, RESULT_MAX // (tokens * top_k * SIZE[src_dtype])))
        if rng.random() < 0.6:
            cols = max(8, cols // 8 * 8)
        return combine(tokens, cols, experts, top_k, src_dtype, dtype)
    tokens = _log(rng, 1, 4096)
    requests = tokens if rng.random() < 0.4 and tokens <= 256 else _log(rng, 1, min(64, tokens))
    K, N = _log(rng, 64, min(8192, LORA_MAX // tokens)), _log(rng, 64, min(14336, LORA_MAX // tokens))
    if rng.random() < 0.6:
        N, K = max(64, N // 64 * 64), max(64, K // 64 * 64)
    sixteen = rng.choice(["f16", "bf16"])
    return lora(tokens, requests, rng.choice([1, 3, 16, 40]), rng.choice([4, 8, 16, 32, 64]), K, N, sixteen, rng.choice([sixteen, "f32"]))


# ---- inputs -----------------------------------------------------------------------------------------------
def _rows(case):
    """Rows that hold any groups of these choices: every expert that is chosen leaves at most 127 rows empty."""
    total = case["tokens"] * case["top_k"]
    return (total + (ALIGN - 1) * min(case["experts"], total)) // ALIGN * ALIGN


def _pitch(cols):
    return (cols + 31) // 32 * 16


def _blocks(cols, fmt):
    return -(-cols // BLOCK[fmt])


def _pow2(n):
    """2^n of whole n, float32, from the bits of a double."""
    return ((n.to(torch.int64) + 1023) << 52).view(torch.float64).to(torch.float32)


def _quantise(x, fmt):
    """(E2M1 values [rows, blocks, block], block scales [rows, blocks]) of a float32 matrix."""
    cols, block = x.shape[1], BLOCK[fmt]
    t = torch.nn.functional.pad(x, (0, -cols % block)).reshape(x.shape[0], -1, block)
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
    codes = torch.nn.functional.pad(codes.reshape(rows, -1)[:, :cols], (0, 2 * _pitch(cols) - cols))
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


def _logits(gen, case, dtype=torch.float32):
    """Logits of a gate that likes some experts more than others."""
    return (_normal(gen, (case["tokens"], case["experts"])) + 0.7 * _normal(gen, (1, case["experts"]))).to(dtype)


def _weights(gen, E, rows, cols, fmt):
    """Packed rows of E experts, the scale tiles of each and a factor for each (nvfp4: kept apart from the scales)."""
    factor = torch.exp2(torch.randint(-2, 3, (E,), generator=gen, device="cuda").float()) * 1.25 if fmt == "nvfp4" else torch.ones(E, device="cuda")
    parts = [_pack(*_quantise(_normal(gen, (rows, cols)), fmt), fmt, cols) for _ in range(E)]
    return torch.cat([p[0] for p in parts]), torch.stack([p[1] for p in parts]), factor / math.sqrt(cols)


def _lengths(case, seed):
    """Tokens of every request: as many requests as tokens have one each; else a few long ones, some with none."""
    if case["requests"] == case["tokens"]:
        return [1] * case["tokens"]
    share = np.random.default_rng(seed).lognormal(0.0, 1.0, case["requests"])
    edges = np.round(np.cumsum(share) / share.sum() * case["tokens"]).astype(int)
    return np.diff(np.concatenate([[0], edges])).tolist()


def _adapter_ranks(case):
    return [max(1, case["rank"] >> (i % 3)) for i in range(case["adapters"])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, s = case["kind"], dict(case)
    if kind == "lora":
        M, R, A, r, K, N = (case[n] for n in ("tokens", "requests", "adapters", "rank", "K", "N"))
        dt = DTYPE[case["dtype"]]
        s["lengths"] = _lengths(case, seed)
        s["picks"] = np.random.default_rng(seed + 1).integers(-1 if R > 3 else 0, A, R).tolist()  # -1: a request without adapter
        s["rank_list"] = _adapter_ranks(case)
        pitch = (r + 7) // 8 * 8  # rows of B at multiples of 16 bytes
        s["x"] = _normal(gen, (M, K), dt)
        s["a"] = _normal(gen, (A, r, K), dt, 1.0 / math.sqrt(K))
        s["b"] = _normal(gen, (A, N, pitch), dt, 0.5 / math.sqrt(r))
        s["base"] = _normal(gen, (M, N), DTYPE[case["dst"]])
        s["starts"] = torch.tensor([0] + np.cumsum(s["lengths"]).tolist(), dtype=torch.int32, device="cuda")
        s["request_adapters"] = torch.tensor(s["picks"], dtype=torch.int32, device="cuda")
        s["ranks"] = torch.tensor(s["rank_list"], dtype=torch.int32, device="cuda")
        s["scales"] = 0.5 + torch.rand((A,), generator=gen, device="cuda")
        s["out"] = torch.zeros((M, N), dtype=DTYPE[case["dst"]], device="cuda")
        return s
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    if kind == "route":
        s["logits"] = _logits(gen, case, DTYPE[case["dtype"]])
        s["ids"], s["slots"] = (torch.zeros((T, k), dtype=torch.int32, device="cuda") for _ in range(2))
        s["p"] = torch.zeros((T, k), dtype=torch.float32, device="cuda")
        s["groups"] = torch.zeros((E, 2), dtype=torch.int32, device="cuda")
        return s
    rows = s["rows"] = _rows(case)
    _, s["p"], s["slots"], s["groups"] = _route(_logits(gen, case), k, True)
    s["group_list"] = s["groups"].tolist()
    if kind == "group":
        x = _normal(gen, (T, case["cols"])) * torch.exp(0.5 * _normal(gen, (1, case["cols"])))  # columns of unequal size
        s["x"] = x.to(DTYPE[case["dtype"]])
        s["packed"] = torch.zeros((rows, _pitch(case["cols"])), dtype=torch.uint8, device="cuda")
        s["tiles"] = torch.zeros((rows // 128, -(-_blocks(case["cols"], case["fmt"]) // 4), 512), dtype=torch.uint8, device="cuda")
        s["out"] = torch.zeros((rows, case["cols"]), dtype=DTYPE[case["dtype"]], device="cuda")
    elif kind == "experts":
        N, K, fmt = case["N"], case["K"], case["fmt"]
        x = _pack(*_quantise(_normal(gen, (T, K))[_source(s["slots"], rows)], fmt), fmt, K)
        s["a"], s["a_tiles"] = x
        s["b"] = _weights(gen, E, N, K, fmt)
        s["up"] = _weights(gen, E, N, K, fmt) if case["swiglu"] else None
        s["bias"] = _normal(gen, (E, N)) if case["bias"] else None
        s["out"] = torch.zeros((rows, N), dtype=DTYPE[case["dtype"]], device="cuda")
    else:
        s["src"] = _normal(gen, (rows, case["cols"]), DTYPE[case["src_dtype"]])
        s["out"] = torch.zeros((T, case["cols"]), dtype=DTYPE[case["dtype"]], device="cuda")
    return s


# ---- the plain form ---------------------------------------------------------------------------------------
def _route(logits, top_k, renormalise):
    """(ids, weights, slots [T, k], groups [E, 2]) of finite logits."""
    T, E = logits.shape
    logits = logits.float()
    ids = torch.argsort(logits, dim=1, descending=True, stable=True)[:, :top_k]
    chosen = torch.gather(logits, 1, ids)
    top = chosen[:, :1]
    total = torch.exp((chosen if renormalise else logits) - top).sum(dim=1, keepdim=True)
    weights = torch.exp(chosen - top) / total
    hit = torch.zeros((T, E), dtype=torch.int64, device=logits.device).scatter(1, ids, 1)
    counts = hit.sum(dim=0)
    room = (counts + ALIGN - 1) // ALIGN * ALIGN
    starts = torch.cumsum(room, 0) - room
    place = torch.cumsum(hit, 0) - hit + starts[None, :]
    slots = torch.gather(place, 1, ids)
    return ids.to(torch.int32), weights, slots.to(torch.int32), torch.stack([starts, counts], dim=1).to(torch.int32)


def _source(slots, rows):
    """The token of every row of the groups, 0 for rows between them."""
    source = torch.zeros(rows, dtype=torch.int64, device=slots.device)
    tokens = torch.arange(slots.shape[0], device=slots.device)[:, None].expand_as(slots)
    source[slots.flatten().long()] = tokens.flatten()
    return source


def _decode(packed, tiles, fmt, cols):
    """Values of packed rows with their scale tiles, float32 [..., rows, cols] (leading dimensions alike)."""
    table = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float32, device=packed.device)
    lead, rows, nb = packed.shape[:-2], packed.shape[-2], _blocks(cols, fmt)
    codes = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2)[..., :cols]
    byte = tiles.reshape(lead + (-(-rows // 128), -(-nb // 4), 32, 4, 4)).movedim(-2, -4).movedim(-2, -3)
    byte = byte.reshape(lead + (-(-rows // 128) * 128, -(-nb // 4) * 4))[..., :rows, :nb]
    scale = _pow2(byte.to(torch.int64) - 127) if fmt == "mxfp4" else byte.contiguous().view(torch.float8_e4m3fn).to(torch.float32)
    return table[codes.to(torch.int32)] * scale.repeat_interleave(BLOCK[fmt], dim=-1)[..., :cols]


def _plain(s):
    kind = s["kind"]
    if kind == "route":
        return _route(s["logits"], s["top_k"], s["renormalise"])
    dtype = DTYPE[s["dst" if kind == "lora" else "dtype"]]
    if kind == "group":
        q, scale = _quantise(s["x"].float(), s["fmt"])
        values = (q * scale[:, :, None]).flatten(1)[:, :s["cols"]].to(dtype)
        out = torch.zeros_like(s["out"])
        for j in range(s["top_k"]):
            out[s["slots"][:, j].long()] = values
        return out
    if kind == "experts":
        N, K, fmt = s["N"], s["K"], s["fmt"]
        a = _decode(s["a"], s["a_tiles"], fmt, K)
        out = torch.zeros_like(s["out"])
        hit = [e for e, (_, count) in enumerate(s["group_list"]) if count > 0]  # only the chosen experts are decoded

        def values(w):
            return _decode(w[0].view(s["experts"], N, -1)[hit], w[1][hit], fmt, K) * w[2][hit, None, None]

        b, up = values(s["b"]), values(s["up"]) if s["swiglu"] else None
        for i, e in enumerate(hit):
            start, count = s["group_list"][e]
            rows = a[start:start + count]
            y = torch.matmul(rows, b[i].T)
            if s["swiglu"]:
                y = y * torch.sigmoid(y) * torch.matmul(rows, up[i].T)
            if s["bias"] is not None:
                y = y + s["bias"][e]
            out[start:start + count] = y.to(dtype)
        return out
    if kind == "combine":
        y = torch.zeros(s["out"].shape, dtype=torch.float32, device=s["src"].device)
        for j in range(s["top_k"]):
            y = y + s["p"][:, j:j + 1] * s["src"][s["slots"][:, j].long()].float()
        return y.to(dtype)
    adapters = np.repeat(s["picks"], s["lengths"])  # of every token
    out = s["base"].clone()
    for i in sorted(set(adapters.tolist()) - {-1}):
        r, rows = s["rank_list"][i], torch.from_numpy(np.nonzero(adapters == i)[0]).cuda()
        v = torch.matmul(s["x"][rows].float(), s["a"][i, :r].float().T)
        delta = torch.matmul(v, s["b"][i, :, :r].float().T) * s["scales"][i]
        out[rows] = (s["base"][rows].float() + delta).to(dtype)
    return out


# ---- the library's calls ----------------------------------------------------------------------------------
_kept = {}


def _context():
    """The context a program keeps for its device and stream."""
    import computelibrary_b200 as cl

    at = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream
    if at not in _kept:
        _kept[at] = cl.Context(*at)
    return _kept[at]


def _describe(s):
    """The descriptors (and workspace) a program fills in once for tensors of these shapes."""
    from computelibrary_b200 import capi

    fmt = {"mxfp4": capi.MXFP4, "nvfp4": capi.NVFP4}.get(s.get("fmt"))
    types = {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}
    dtype, kind = types[s["dtype"]], s["kind"]
    need = 0
    if kind == "route":
        s["desc"] = capi.make_moe_route_desc(s["tokens"], s["experts"], s["top_k"], dtype, renormalize=s["renormalise"])
        need = capi.moe_route_workspace_bytes(s["desc"])
    elif kind == "group":
        s["desc"] = capi.make_mx_group_desc(s["tokens"], s["top_k"], s["cols"], s["rows"], fmt, dtype)
        s["back"] = capi.make_mx_desc(s["rows"], s["cols"], fmt, dtype)
    elif kind == "experts":
        s["desc"] = capi.make_mx_grouped_gemm_desc(s["experts"], s["rows"], s["N"], s["K"], fmt, dtype,
                                                   expected_rows=s["tokens"] * s["top_k"], swiglu=s["swiglu"],
                                                   has_bias=s["bias"] is not None)
    elif kind == "combine":
        s["desc"] = capi.make_moe_combine_desc(s["tokens"], s["top_k"], s["cols"], s["rows"], types[s["src_dtype"]], dtype)
    else:
        s["desc"] = capi.make_lora_desc(s["tokens"], s["requests"], s["adapters"], s["rank"], s["K"], s["N"], dtype, types[s["dst"]],
                                        ld_b=2 * s["b"].shape[2])
        need = capi.lora_workspace_bytes(s["desc"])
    s["workspace"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    return s["desc"]


def _library(s):
    ctx = _context()
    desc = s.get("desc") or _describe(s)
    kind = s["kind"]
    if kind == "route":
        ctx.moe_route(desc, s["logits"], s["ids"], s["p"], s["slots"], s["groups"], s["workspace"])
        return s["ids"], s["p"], s["slots"], s["groups"]
    if kind == "group":  # written and read back: codes are returned as the values they stand for
        ctx.mx_quantize_grouped(desc, s["x"], s["slots"], s["packed"], s["tiles"])
        ctx.mx_dequantize(s["back"], s["packed"], s["tiles"], s["out"])
    elif kind == "experts":
        ctx.mx_grouped_gemm(desc, s["a"], s["a_tiles"], s["groups"], s["b"], s["out"], up=s["up"], bias=s["bias"])
    elif kind == "combine":
        ctx.moe_combine(desc, s["src"], s["slots"], s["p"], s["out"])
    else:
        ctx.lora(desc, s["x"], s["starts"], s["request_adapters"], s["ranks"], s["scales"], s["a"], s["b"], s["base"], s["out"],
                 s["workspace"])
    return s["out"]


def run(state):
    return _library(state) if own else _plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "lora":
        M, R, A, K, N = (case[n] for n in ("tokens", "requests", "adapters", "K", "N"))
        ranks = _adapter_ranks(case)
        rank, none = sum(ranks) / A, 1 / (A + 1) if R > 3 else 0.0
        used = A * (1 - (1 - (1 - none) / A) ** R)  # adapters that at least one request is expected to have
        return {"bytes": M * K * 2 + 2 * M * N * SIZE[case["dst"]] + used * rank * (K + N) * 2, "flops": 2 * M * (1 - none) * rank * (K + N)}
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    if kind == "route":
        return {"bytes": T * E * SIZE[case["dtype"]] + 12 * T * k + 8 * E, "flops": 2 * T * E}
    if kind == "group":
        n, stored = T * case["cols"], T * k * (case["cols"] / 2 + _blocks(case["cols"], case["fmt"]))
        size = SIZE[case["dtype"]]
        return {"bytes": n * size + 4 * T * k + 2 * stored + k * n * size, "flops": 2 * (k + 1) * n}
    if kind == "experts":
        N, K, fmt, pairs = case["N"], case["K"], case["fmt"], 2 if case["swiglu"] else 1
        hit = E * (1 - (1 - k / E) ** T)  # experts that at least one token is expected to choose
        row = K / 2 + _blocks(K, fmt)
        return {"bytes": T * k * row + pairs * hit * N * row + T * k * N * SIZE[case["dtype"]] + (4 * hit * N if case["bias"] else 0),
                "flops": 2 * pairs * T * k * N * K}
    n = T * case["cols"]
    return {"bytes": k * n * SIZE[case["src_dtype"]] + 8 * T * k + n * SIZE[case["dtype"]], "flops": 2 * k * n}


# ---- the definition in 64 bits ----------------------------------------------------------------------------
def _two_to(n):
    return torch.tensor([2.0 ** i for i in range(-160, 161)], dtype=torch.float64, device=n.device)[n + 160]


def _exact_values(x, fmt):
    """What x holds once stored, float64."""
    rows, cols = x.shape
    t = torch.zeros((rows, _blocks(cols, fmt) * BLOCK[fmt]), dtype=torch.float64, device=x.device)
    t[:, :cols] = x.double()
    t = t.view(rows, -1, BLOCK[fmt])
    amax = t.abs().amax(2, keepdim=True)

    def log2(v):
        return torch.frexp(v).exponent.long() - 1

    if fmt == "mxfp4":
        scale = torch.where(amax > 0, _two_to((log2(amax) - 2).clamp(min=-127)), 0.0)
    else:
        v = (amax / torch.full_like(amax, 6.0)).clamp(2.0 ** -9, 448.0)
        ulp = _two_to(log2(v).clamp(min=-6) - 3)  # three bits behind the leading one, subnormals below 2^-6
        scale = torch.where(amax > 0, torch.round(v / ulp) * ulp, 0.0)
    r = t.abs() / torch.where(scale > 0, scale, 1.0)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    below, above = torch.bucketize(r, mid, right=False), torch.bucketize(r, mid, right=True)  # differ at a tie only
    v = grid[torch.where(below % 2 == 0, below, above)]
    return (torch.sign(t) * v * scale).view(rows, -1)[:, :cols]


def _exact_decode(packed, tiles, fmt, cols):
    """The values at every (row, column), by index arithmetic on the layout, float64."""
    packed = packed.long()
    r = torch.arange(packed.shape[0], device=packed.device)[:, None]
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


def _exact_route(s):
    """Choices by sorting on the host, weights in 64 bits, places one token after the other."""
    logits = s["logits"].double().cpu().numpy()
    T, E = logits.shape
    k = s["top_k"]
    ids = np.empty((T, k), np.int64)
    for t in range(T):
        ids[t] = np.lexsort((np.arange(E), -logits[t]))[:k]
    chosen = np.take_along_axis(logits, ids, 1)
    among = chosen if s["renormalise"] else logits
    weights = 1 / np.exp(among[:, None, :] - chosen[:, :, None]).sum(axis=2)
    counts = np.bincount(ids.ravel(), minlength=E)
    starts, at = np.zeros(E, np.int64), 0
    for e in range(E):
        starts[e] = at
        at += -(-counts[e] // ALIGN) * ALIGN
    following, slots = starts.copy(), np.empty((T, k), np.int64)
    for t in range(T):
        slots[t] = following[ids[t]]
        following[ids[t]] += 1

    def whole(v):
        return torch.from_numpy(v.astype(np.int32)).cuda()

    return whole(ids), torch.from_numpy(weights).cuda(), whole(slots), whole(np.stack([starts, counts], axis=1))


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        return _exact_route(s)
    y = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    if kind == "group":
        y[s["slots"].flatten().long()] = _exact_values(s["x"], case["fmt"]).repeat_interleave(case["top_k"], dim=0)
    elif kind == "experts":
        N, K, fmt = case["N"], case["K"], case["fmt"]
        for e in range(case["experts"]):
            first, count = s["group_list"][e]
            if count:
                rows = slice(first, first + count)
                a = _exact_decode(s["a"][rows], s["a_tiles"][first // 128:-(-(first + count) // 128)], fmt, K)
                w = [_exact_decode(m[0].view(case["experts"], N, -1)[e], m[1][e], fmt, K) * m[2][e].double() for m in (s["b"], s["up"]) if m]
                z = a @ w[0].T
                y[rows] = z / (1 + torch.exp(-z)) * (a @ w[1].T) if case["swiglu"] else z
                if case["bias"]:
                    y[rows] += s["bias"][e].double()
    elif kind == "combine":
        y = (s["src"].double()[s["slots"].long()] * s["p"].double()[:, :, None]).sum(dim=1)
    else:
        ends = s["starts"].tolist()
        for request, adapter in enumerate(s["picks"]):
            rows = slice(ends[request], ends[request + 1])
            y[rows] = s["base"][rows].double()
            if adapter >= 0:
                r = s["rank_list"][adapter]
                weight = (s["b"][adapter].double()[:, :r] @ s["a"][adapter].double()[:r]) * s["scales"][adapter].double()
                y[rows] += s["x"][rows].double() @ weight.T
    return y
