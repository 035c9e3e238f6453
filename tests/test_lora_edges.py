"""Low-rank adapters at the edges: long sums, calls beside each other."""
import numpy as np
import pytest

from computelibrary_b200 import capi
from test_lora import check
from test_mx_gemm import torch_dtype


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [capi.F16, capi.BF16])
@pytest.mark.parametrize("requests,each,rank", [(300, 1, 16), (300, 1, 64), (150, 64, 32), (300, 32, 128)])
def test_long_sums_are_four_shorter_ones(ctx, requests, each, rank, dtype):
    """Blocks of 64 columns of K go to four sums in turn, which are added up as floats (requests enough that no CTAs share K).  So v is that of
    the four quarters by themselves, where the other sums are zero, added up: bit for bit with BF16, whose three parts hold all of a float;
    with F16 within what the parts of five values leave, 2^-21 of each and 2^-24 of the token's largest, and four roundings.  One sum, which is
    cut to 24 bits at each of its 256 steps, is off by 9e-6 and 2.4e-5 with these inputs.  B picks one rank, base is zero."""
    import torch
    M, K, N = requests * each, 4096, rank
    el = torch_dtype(dtype)
    g = torch.Generator(device="cuda").manual_seed(rank)
    x = (torch.rand((M, K), generator=g, device="cuda") + 0.5).to(el)
    a = (torch.rand((1, rank, K), generator=g, device="cuda") + 0.5).to(el)
    b = torch.eye(N, device="cuda").to(el).view(1, N, rank).contiguous()
    base = torch.zeros((M, N), device="cuda")
    starts = torch.arange(0, M + 1, each, dtype=torch.int32, device="cuda")
    picks, scale = torch.zeros(requests, dtype=torch.int32, device="cuda"), torch.ones(1, device="cuda")
    d = capi.make_lora_desc(M, requests, 1, rank, K, N, dtype, capi.F32)
    ws = torch.zeros(capi.lora_workspace_bytes(d), dtype=torch.uint8, device="cuda")

    def v(a):
        out = torch.zeros((M, N), device="cuda")
        ctx.lora(d, x, starts, picks, None, scale, a, b, base, out, ws)
        ctx.sync()
        return out

    block = torch.arange(K, device="cuda") // 64 % 4
    want = torch.zeros((M, N), device="cuda")
    for q in range(4):
        want += v(torch.where(block == q, a, torch.zeros_like(a)))
    got = v(a)
    if dtype == capi.BF16:
        assert torch.equal(got, want)
        return
    tol = 2 * 2.0 ** -21 * want + 5 * 2.0 ** -24 * want.amax(1, keepdim=True) + 4 * 2.0 ** -24 * want  # (the quarters add up to one value)
    off = (got - want).abs()
    assert (off <= tol).all(), f"off by {(off / want).max().item():.2e}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [capi.F16, capi.BF16])
@pytest.mark.parametrize("rank", [16, 32, 64, 128])
def test_calls_on_three_streams(ctx, rank, dtype):
    """Short requests, long ones and products at once, again and again: every call gives what it gives alone.  (Their clusters share SMs and
    their tensor memory.)"""
    import torch
    from test_mx_inputs_ahead import stored
    streams = [torch.cuda.Stream() for _ in range(3)]
    own = [capi.Context(0, s.cuda_stream) for s in streams]
    g = torch.Generator(device="cuda").manual_seed(1)
    a, b = stored(g, 48, 4096, capi.NVFP4), stored(g, 2048, 4096, capi.NVFP4)
    product = torch.zeros((48, 2048), device="cuda")
    d = capi.make_mx_gemm_desc(48, 2048, 4096, capi.NVFP4, capi.F32)
    try:
        short, short_args = check(ctx, [1] * 28, [i % 3 for i in range(28)], min(rank, 64), 4096, 1032, dtype, capi.F32)
        long, long_args = check(ctx, [200, 1, 77, 300], [0, 1, 2, 0], rank, 4096, 1032, dtype, capi.F32)
        ctx.mx_gemm(d, *a, *b, None, product)
        ctx.sync()
        outs = (short, long, product)
        want = [o.clone() for o in outs]
        for o in outs:
            o.fill_(7)
        torch.cuda.synchronize()
        for _ in range(200):
            own[0].lora(*short_args)
            own[1].lora(*long_args)
            own[2].mx_gemm(d, *a, *b, None, product)
        for c in own:
            c.sync()
        for o, w in zip(outs, want):
            rows = w != 7
            assert torch.equal(o[rows], w[rows])
    finally:
        for c in own:
            c.close()


@pytest.mark.gpu
def test_wide_results_of_high_ranks_fill_the_gpu_once(ctx):
    """Rank 64 in three parts leaves room for one CTA of the second launch to an SM: more items than CTAs, whole and ragged rows."""
    check(ctx, [700, 3, 1000, 64], [0, 1, 2, 0], 64, 512, 4096, capi.BF16, capi.F32)
    check(ctx, [700, 3, 1000, 64], [0, 1, -1, 0], 50, 512, 2051, capi.BF16, capi.F32, ranks=[50, 7, 33], adapters=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dst", [capi.BF16, capi.F32])
def test_two_calls_of_short_requests_at_once(ctx, dst):
    """Each on its stream with its own workspace, again and again."""
    import torch
    streams = [torch.cuda.Stream() for _ in range(2)]
    own = [capi.Context(0, s.cuda_stream) for s in streams]
    try:
        calls = [check(ctx, [1] * 24, [(i + turn) % 4 - 1 for i in range(24)], rank, 1024, 2056, capi.BF16, dst, adapters=3, seed=turn)
                 for turn, rank in enumerate((16, 64))]
        want = [out.clone() for out, _ in calls]
        for out, _ in calls:
            out[:24] = 7
        torch.cuda.synchronize()
        for _ in range(100):
            for c, (_, args) in zip(own, calls):
                c.lora(*args)
        for c in own:
            c.sync()
        for (out, _), w in zip(calls, want):
            assert torch.equal(out, w)
    finally:
        for c in own:
            c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("R", [7, 8, 33, 34, 71, 72, 119, 148, 149])
def test_numbers_of_short_requests_where_clusters_change(ctx, R):
    rng = np.random.default_rng(R)
    check(ctx, [1] * R, rng.integers(-1, 3, R).tolist(), 16, 1024, 2312, capi.BF16, capi.BF16, adapters=3)
    check(ctx, rng.integers(1, 4, R).tolist(), rng.integers(-1, 3, R).tolist(), 40, 1000, 521, capi.F16, capi.F32, adapters=3, ranks=[40, 3, 17])
