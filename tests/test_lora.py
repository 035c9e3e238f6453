"""Low-rank adapters of many requests against sums in 64 bits.

Tolerance.  v = x . A^T: a matrix instruction adds 16 products, which are exact in 32 bits, and is off by at most one step of 24 bits of
the magnitudes added so far; the warps' and the CTAs' shares add up to 16 steps more: ceil(K / 16) + 16 steps of 2^-23.  v in parts: two of
bf16 leave 2^-17 of it, three 2^-25; two of f16 2^-21 and 2^-24 of the token's largest.  The second product: a step for 16 ranks and part,
and the last sum; then half a step of the destination type."""
import ctypes as C

import numpy as np
import pytest

from computelibrary_b200 import capi
from test_mx_gemm import HALF_STEP, torch_dtype

TYPES = [(capi.F16, capi.F16), (capi.BF16, capi.BF16), (capi.F16, capi.F32), (capi.BF16, capi.F32)]


# ---- without a GPU ----------------------------------------------------------------------------------------
def test_descriptor_layout():
    assert C.sizeof(capi.LoraDesc) == 8 * 4 + 5 * 8 and capi.LoraDesc.ld_x.offset == 32


@pytest.mark.parametrize("change,word", [
    (dict(tokens=-1), "tokens"), (dict(requests=-1), "requests"), (dict(adapters=0), "adapters"), (dict(max_rank=0), "max_rank"), (dict(max_rank=129), "max_rank"),
    (dict(N=0), "N"), (dict(K=0), "K"), (dict(K=2 ** 31 - 1), "too large"), (dict(dtype=capi.F32), "dtype"), (dict(dst_dtype=capi.BF16), "dst_dtype"),
    (dict(ld_x=126), "ld_x"), (dict(ld_x=201), "ld_x"), (dict(ld_a=126), "ld_a"), (dict(ld_b=8), "ld_b"), (dict(ld_b=24), "ld_b"), (dict(ld_base=126), "ld_base"),
    (dict(ld_dst=201), "ld_dst"), (dict(tokens=2 ** 30, requests=2 ** 20), "65535")])
def test_validate_refuses(change, word):
    d = capi.make_lora_desc(10, 3, 2, 8, 64, 64, capi.F16, capi.F16)
    assert capi.lora_validate(d)[0] == 0
    for k, v in change.items():
        setattr(d, k, v)
    st, why = capi.lora_validate(d)
    assert st == capi.INVALID_ARGUMENT and word in why
    assert capi.lora_workspace_bytes(d) == 0


def test_null_context_is_refused():
    d = capi.make_lora_desc(10, 3, 2, 8, 64, 64, capi.F16, capi.F16)
    assert capi.load_library().cugl_lora(None, C.byref(d), *[None] * 10, 0) == capi.INVALID_ARGUMENT
    assert capi.lora_workspace_bytes(d) >= 10 * (16 * 4 + 4)


# ---- on the GPU -------------------------------------------------------------------------------------------
def matrix(values, dtype, pad=0, offset=0, fill=float("nan")):
    """Values [.., rows, cols] on the device, rows `pad` elements apart, the first `offset` elements into an allocation."""
    import torch
    lead, cols = values.shape[:-1], values.shape[-1]
    flat = torch.full((int(np.prod(lead)) * (cols + pad) + offset + 8,), fill, dtype=dtype, device="cuda")
    m = flat[offset:offset + int(np.prod(lead)) * (cols + pad)].view(*lead, cols + pad)
    m[..., :cols] = torch.from_numpy(values).to(dtype).cuda()
    return m


def check(ctx, lengths, picks, max_rank, K, N, dtype, dst, ranks=None, in_place=False, pad=0, offset=0, behind=2, adapters=None, seed=0, size=1.0, before=0):
    import torch
    rng = np.random.default_rng(seed + 3 * K + 5 * N + max_rank)
    R, M = len(lengths), before + sum(lengths) + behind
    E = adapters if adapters is not None else max([p for p in picks if p < 1000] + [0]) + 1
    el, od = torch_dtype(dtype), torch_dtype(dst)
    x = matrix(rng.standard_normal((M, K)) * size, el, pad, offset)
    a = rng.standard_normal((E, max_rank, K)) / np.sqrt(K)
    b = rng.standard_normal((E, N, max_rank)) / np.sqrt(max_rank)
    if ranks is not None:  # what lies behind an adapter's ranks counts nothing
        for i, r in enumerate(ranks):
            a[i, r:], b[i, :, r:] = np.nan, np.inf
    a = matrix(a, el, pad, offset)
    b = matrix(b, el, -max_rank % 8)
    scales = rng.uniform(-2, 2, E).astype(np.float32)
    base = matrix(rng.standard_normal((M, N)), od, pad, offset, fill=3.0)
    out = base if in_place else torch.full((M, N + pad), 7.0, dtype=od, device="cuda")
    starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32) + before
    want_base = base[:, :N].double().cpu().numpy()
    old = out.clone()
    es = base.element_size()
    d = capi.make_lora_desc(M, R, E, max_rank, K, N, dtype, dst, ld_x=2 * (K + pad), ld_a=2 * (K + pad), ld_base=(N + pad) * es, ld_dst=(N + pad) * es)
    assert d.ld_b == 2 * b.shape[2]
    ws = torch.full((capi.lora_workspace_bytes(d) + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    up = lambda v, t: torch.tensor(v, dtype=t, device="cuda")
    args = (d, x, up(starts, torch.int32), up(picks, torch.int32), up(ranks, torch.int32) if ranks is not None else None, up(scales, torch.float32), a, b, base, out,
            ws[:capi.lora_workspace_bytes(d)])
    ctx.lora(*args)
    ctx.sync()
    assert (ws[-64:] == 0xFF).all()
    got = out[:, :N].double().cpu().numpy()
    vx, va, vb = (t.double().cpu().numpy() for t in (x, a, b))
    parts = 3 if (dtype, dst) == (capi.BF16, capi.F32) else 2
    for i in range(R):
        rows = slice(starts[i], starts[i + 1])
        e = picks[i]
        r = (ranks[e] if ranks is not None else max_rank) if 0 <= e < E else 0
        if r <= 0:
            assert (got[rows] == want_base[rows]).all()
            continue
        xs, A, B = vx[rows, :K], va[e, :r, :K], vb[e, :, :r]
        v, size1 = xs @ A.T, np.abs(xs) @ np.abs(A).T
        ev = 2.0 ** -23 * (-(-K // 16) + 16) * size1
        if dtype == capi.F16:
            lost = 2.0 ** -21 * (np.abs(v) + ev) + 2.0 ** -24 * (np.abs(v) + ev).max(axis=1, keepdims=True, initial=0)
        else:
            lost = (2.0 ** -17 if parts == 2 else 2.0 ** -25) * (np.abs(v) + ev)
        delta = scales[e].astype(np.float64) * (v @ B.T)
        tol = abs(float(scales[e])) * ((ev + lost) @ np.abs(B).T + 2.0 ** -23 * (parts * -(-r // 16) + 1) * ((np.abs(v) + ev) @ np.abs(B).T))
        want = want_base[rows] + delta
        tol = tol + 2.0 ** -24 * (np.abs(want) + tol)
        tol = tol + HALF_STEP[dst] * (np.abs(want) + tol) + (2.0 ** -25 if dst == capi.F16 else 0)
        bad = ~(np.abs(got[rows] - want) <= tol)
        assert not bad.any(), f"request {i}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[:3].tolist()}: {got[rows][bad][:3]} for {want[bad][:3]}"
    mine = np.zeros(M, bool)
    mine[starts[0]:starts[-1]] = True
    keep = torch.from_numpy(~mine).cuda()
    assert torch.equal(out[keep], old[keep])  # tokens of no request
    assert torch.equal(out[:, N:], old[:, N:])
    return out, args


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dst", TYPES)
@pytest.mark.parametrize("max_rank", [1, 3, 8, 16, 17, 32, 48, 64, 65, 128])
def test_ranks(ctx, max_rank, dtype, dst):
    check(ctx, [1, 40, 0, 130, 16], [0, 1, 1, 2, 0], max_rank, 256, 520, dtype, dst)
    check(ctx, [33, 65], [1, 0], max_rank, 100, 264, dtype, dst, ranks=[max(1, max_rank // 3), max_rank])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dst", TYPES)
@pytest.mark.parametrize("K", [1, 7, 8, 31, 32, 33, 255, 512, 1000, 4096, 9001])
def test_k(ctx, K, dtype, dst):
    check(ctx, [1, 70, 17], [0, 1, 2], 16, K, 96, dtype, dst)
    check(ctx, [129], [0], 64, K, 96, dtype, dst)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dst", TYPES)
@pytest.mark.parametrize("N", [1, 2, 7, 8, 31, 33, 255, 256, 257, 1000, 4104])
def test_channels(ctx, N, dtype, dst):
    check(ctx, [1, 70, 17], [0, -1, 2], 8, 128, N, dtype, dst)
    check(ctx, [50], [0], 32, 128, N, dtype, dst, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dst", TYPES)
def test_strides_and_alignment(ctx, dtype, dst):
    check(ctx, [20, 70], [1, 0], 16, 200, 200, dtype, dst, pad=8)
    check(ctx, [20, 70], [1, 0], 16, 200, 200, dtype, dst, pad=3)
    check(ctx, [20, 70], [1, 0], 16, 200, 200, dtype, dst, offset=1)
    check(ctx, [20, 70], [1, 0], 16, 200, 200, dtype, dst, pad=8, offset=8, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("max_rank", [16, 128])
@pytest.mark.parametrize("lengths", [[1], [15], [16], [17], [31], [32], [33], [63], [64], [65], [127], [128], [129], [300], [0, 0, 5], [5, 0, 0], [0]], ids=str)
def test_lengths(ctx, lengths, max_rank):
    check(ctx, lengths, [1] * len(lengths), max_rank, 320, 300, capi.BF16, capi.F32, adapters=3)
    check(ctx, lengths, [0] * len(lengths), max_rank, 320, 304, capi.F16, capi.F16, before=3)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [1, 24, 255, 256, 257, 700])
def test_many_requests(ctx, R):
    """One token each, more requests than threads of a block."""
    rng = np.random.default_rng(R)
    check(ctx, [1] * R, rng.integers(-1, 9, R).tolist(), 16, 256, 264, capi.BF16, capi.BF16, adapters=9)
    lengths = rng.integers(0, 4, R).tolist()
    check(ctx, lengths, rng.integers(-1, 9, R).tolist(), 8, 64, 40, capi.F16, capi.F32, adapters=9, ranks=rng.integers(0, 9, 9).tolist())


@pytest.mark.gpu
def test_no_adapter(ctx):
    check(ctx, [5, 70, 3, 9], [-1, 4, 10 ** 9, -2 ** 31], 16, 128, 136, capi.F16, capi.F32, adapters=4)
    check(ctx, [5, 70, 3], [0, 1, 2], 16, 128, 136, capi.BF16, capi.BF16, ranks=[0, -3, 16])
    check(ctx, [5, 70, 3], [0, 1, 2], 16, 128, 136, capi.BF16, capi.BF16, ranks=[0, 0, 0], in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-6, 300.0])
def test_f16_sums_beyond_the_type(ctx, size):
    """v of f16 operands far above and below what f16 holds."""
    check(ctx, [3, 90], [0, 1], 16, 4096, 64, capi.F16, capi.F32, size=size)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dst", TYPES)
def test_nan_and_infinity_stay_with_their_token(ctx, dtype, dst):
    import torch
    out, args = check(ctx, [10, 60], [0, 1], 16, 128, 72, dtype, dst)
    want, x = out.clone(), args[1]
    x[3, 5] = float("nan")
    x[40, 100] = float("inf")
    ctx.lora(*args)
    ctx.sync()
    bad = torch.zeros(out.shape[0], dtype=torch.bool, device="cuda")
    bad[3] = bad[40] = True
    assert torch.equal(out[~bad], want[~bad])
    assert torch.isnan(out[3]).all() and not torch.isfinite(out[40]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[1] * 24, [700, 3, 1000]], ids=len)
def test_equal_calls_give_equal_bits(ctx, lengths):
    import torch
    out, args = check(ctx, lengths, [i % 3 for i in range(len(lengths))], 64, 2048, 1032, capi.F16, capi.F32)
    want = out.clone()
    for _ in range(3):
        out.fill_(7)
        ctx.lora(*args)
        ctx.sync()
        rows = sum(lengths)
        assert torch.equal(out[:rows], want[:rows])


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,rank,k_block", [([1] * 24, 16, 0), ([1] * 24, 16, 3), ([200, 70], 64, 5), ([200, 70], 128, 2)])
def test_wait_limit(ctx, lengths, rank, k_block):
    """Operand copies that never come: the call ends by its wait limit and says so; the next one is as always."""
    import torch
    out, args = check(ctx, lengths, [i % 3 for i in range(len(lengths))], rank, 4096, 264, capi.BF16, capi.F32)
    want = out.clone()
    ctx.set_wait_limit_us(20000)
    try:
        ctx.withhold_copy_once(k_block)
        ctx.lora(*args)
        with pytest.raises(capi.CuglError) as e:
            ctx.sync()
        assert e.value.status == capi.RUNTIME_ERROR and "wait ran out" in e.value.message
    finally:
        ctx.set_wait_limit_us(0)
    out[:sum(lengths)] = 7
    ctx.lora(*args)
    ctx.sync()
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,rank", [(10, 16), (64, 32), (64, 64), (32, 128)])
def test_gives_up_in_flight(ctx, tokens, rank):
    """A limit far below the time of a tile: the kernel gives up with copies and products under way."""
    import torch
    from test_mx_give_up import check as give_up
    K, N = 2 ** 23, 64
    g = torch.Generator(device="cuda").manual_seed(rank)
    x = torch.randint(-8, 8, (tokens, K), generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    a = torch.randint(-8, 8, (1, rank, K), generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    b = torch.randn((1, N, rank), generator=g, device="cuda").to(torch.bfloat16)
    base, out = torch.randn((tokens, N), generator=g, device="cuda"), torch.zeros((tokens, N), device="cuda")
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    d = capi.make_lora_desc(tokens, 1, 1, rank, K, N, capi.BF16, capi.F32)
    ws = torch.zeros(capi.lora_workspace_bytes(d), dtype=torch.uint8, device="cuda")
    starts, picks, scales = i(0, tokens), i(0), torch.full((1,), 2.0 ** -20, device="cuda")
    give_up(ctx, lambda: ctx.lora(d, x, starts, picks, None, scales, a, b, base, out, ws), out)


@pytest.mark.gpu
def test_starts_out_of_order(ctx):
    """Requests that overlap, lie outside or end before they begin are cut to the tokens there are; nothing else is written."""
    import torch
    M, R, N = 300, 600, 72
    d = capi.make_lora_desc(M, R, 2, 16, 128, N, capi.F16, capi.F16)
    x = torch.ones((M, 128), dtype=torch.float16, device="cuda")
    a, b = torch.ones((2, 16, 128), dtype=torch.float16, device="cuda"), torch.ones((2, N, 16), dtype=torch.float16, device="cuda")
    base = torch.zeros((M, N), dtype=torch.float16, device="cuda")
    out = torch.full((M + 4, N), 7.0, dtype=torch.float16, device="cuda")
    ws = torch.full((capi.lora_workspace_bytes(d) + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(0)
    for starts in (rng.integers(-2 ** 31, 2 ** 31 - 1, R + 1), np.where(np.arange(R + 1) % 2, 10 ** 9, -5), rng.integers(-400, 700, R + 1), np.arange(R, -1, -1)):
        picks = rng.integers(-3, 5, R)
        ctx.lora(d, x, torch.tensor(starts, dtype=torch.int32, device="cuda"), torch.tensor(picks, dtype=torch.int32, device="cuda"), None,
                 torch.ones(2, device="cuda"), a, b, base, out, ws[:capi.lora_workspace_bytes(d)])
        ctx.sync()
        assert (out[M:] == 7).all() and (ws[-64:] == 0xFF).all()
        got = out[:M].double().cpu().numpy()  # a token is left alone, copied, or given its adapter's 16 * 128
        assert np.isin(got, [7.0, 0.0, 2048.0]).all()


@pytest.mark.gpu
def test_nothing_to_do(ctx):
    for M, R in ((0, 3), (3, 0)):
        ctx.lora(capi.make_lora_desc(M, R, 2, 8, 64, 64, capi.F16, capi.F16), *[None] * 10)
    ctx.sync()


@pytest.mark.gpu
@pytest.mark.parametrize("change,word", [("null", "NULL"), ("b", "16-byte"), ("x", "aligned"), ("workspace", "too small"), ("ld", "in place")])
def test_call_refuses(ctx, change, word):
    import torch
    f = torch.zeros(64 * 64, dtype=torch.float16, device="cuda")
    i = torch.zeros(64, dtype=torch.int32, device="cuda")
    s = torch.zeros(64, device="cuda")
    d = capi.make_lora_desc(10, 3, 2, 8, 64, 64, capi.F16, capi.F16, ld_dst=160 if change == "ld" else None)
    with pytest.raises(capi.CuglError) as e:
        ctx.lora(d, f.view(torch.uint8)[1:] if change == "x" else f, i, i, None, None if change == "null" else s, f, f[4:] if change == "b" else f, f, f, f,
                 workspace_bytes=100 if change == "workspace" else None)
    assert e.value.status == capi.INVALID_ARGUMENT and word in e.value.message


# ---- short requests: both products in one launch; long ones in two -----------------------------------------------
SHORT = [1, 2, 0, 17, 1, 33, 1, 1, 16, 1, 0, 1, 1, 3, 1, 15]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dst", TYPES)
@pytest.mark.parametrize("max_rank", [1, 4, 8, 16, 20, 30, 32, 48, 64])
def test_short_requests(ctx, max_rank, dtype, dst):
    picks = [i % 4 - (i % 7 == 3) for i in range(len(SHORT))]
    check(ctx, SHORT, picks, max_rank, 200, 520, dtype, dst, adapters=4)
    check(ctx, SHORT, picks, max_rank, 72, 7000, dtype, dst, adapters=4, ranks=[max_rank, 0, max(1, max_rank // 3), max_rank - 1])
    check(ctx, SHORT, picks, max_rank, 1032, 1001, dtype, dst, adapters=4, before=2)  # rows of base and dst start anywhere
    check(ctx, SHORT, picks, max_rank, 64, 296, dtype, dst, adapters=4, in_place=True, pad=8)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [8, 60, 150, 300, 700])
@pytest.mark.parametrize("max_rank", [16, 64])
def test_many_short_requests(ctx, R, max_rank):
    """Clusters of eight CTAs down to single ones, more blocks of channels than a CTA has asked for ahead."""
    rng = np.random.default_rng(R)
    check(ctx, rng.integers(0, 4, R).tolist(), rng.integers(-1, 3, R).tolist(), max_rank, 136, 2056, capi.BF16, capi.BF16, adapters=3)
    check(ctx, [1] * R, rng.integers(-1, 3, R).tolist(), max_rank, 64, 1288, capi.F16, capi.F32, adapters=3, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1, 8, 63, 64, 65, 130, 4096])
def test_short_requests_k(ctx, K):
    """Fewer blocks of K than CTAs of a cluster, and more than stages."""
    check(ctx, [1] * 9, [i % 3 for i in range(9)], 16, K, 264, capi.BF16, capi.F32, pad=-K % 8)
    check(ctx, [2], [0], 32, K, 256, capi.F16, capi.F16, pad=-K % 8)


@pytest.mark.gpu
@pytest.mark.parametrize("max_rank", [16, 128])
def test_many_long_requests(ctx, max_rank):
    rng = np.random.default_rng(max_rank)
    lengths = rng.integers(9, 21, 300).tolist()
    check(ctx, lengths, rng.integers(-1, 3, 300).tolist(), max_rank, 64, 264, capi.BF16, capi.BF16, adapters=3)
    check(ctx, lengths, rng.integers(-1, 3, 300).tolist(), max_rank, 36, 259, capi.F16, capi.F32, adapters=3)


@pytest.mark.gpu
@pytest.mark.parametrize("rank,k_block", [(16, 1), (64, 0), (64, 7)])
def test_wait_limit_of_short_requests(ctx, rank, k_block):
    test_wait_limit(ctx, [1] * 24, rank, k_block)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,rank", [(1, 16), (8, 32), (5, 64)])
def test_short_requests_give_up_in_flight(ctx, tokens, rank):
    test_gives_up_in_flight(ctx, tokens, rank)


@pytest.mark.gpu
def test_starts_of_long_requests_out_of_order(ctx):
    import torch
    M, R, N = 3000, 200, 72
    d = capi.make_lora_desc(M, R, 2, 16, 128, N, capi.F16, capi.F16)
    x = torch.ones((M, 128), dtype=torch.float16, device="cuda")
    a, b = torch.ones((2, 16, 128), dtype=torch.float16, device="cuda"), torch.ones((2, N, 16), dtype=torch.float16, device="cuda")
    base = torch.zeros((M, N), dtype=torch.float16, device="cuda")
    out = torch.full((M + 4, N), 7.0, dtype=torch.float16, device="cuda")
    ws = torch.full((capi.lora_workspace_bytes(d) + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(0)
    for starts in (rng.integers(-2 ** 31, 2 ** 31 - 1, R + 1), np.where(np.arange(R + 1) % 2, 10 ** 9, -5), np.arange(R, -1, -1)):
        ctx.lora(d, x, torch.tensor(starts, dtype=torch.int32, device="cuda"), torch.tensor(rng.integers(-3, 5, R), dtype=torch.int32, device="cuda"), None,
                 torch.ones(2, device="cuda"), a, b, base, out, ws[:capi.lora_workspace_bytes(d)])
        ctx.sync()
        assert (out[M:] == 7).all() and (ws[-64:] == 0xFF).all()
        assert np.isin(out[:M].double().cpu().numpy(), [7.0, 0.0, 2048.0]).all()


@pytest.mark.gpu
def test_captured_short_requests(ctx):
    """A captured call, replayed with other requests in the same buffers, gives what the call gives."""
    import torch
    out, args = check(ctx, [1] * 24, [i % 3 for i in range(24)], 16, 256, 1288, capi.BF16, capi.BF16)
    stream = torch.cuda.Stream()
    own = capi.Context(0, stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            own.lora(*args)
        for turn in range(3):
            args[3].copy_(torch.tensor([(i + turn) % 4 - 1 for i in range(24)], dtype=torch.int32))
            torch.cuda.synchronize()
            ctx.lora(*args)
            ctx.sync()
            want = out.clone()
            out.fill_(7)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[:24], want[:24])
        del graph
    finally:
        own.close()
