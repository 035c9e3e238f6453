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
