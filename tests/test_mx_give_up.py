"""Waits that run out while everything is still under way: a limit far below the time a tile takes, so that a kernel gives up with
its copies and MMAs in flight.  The call says so, and what runs after it (on the same tensor memory and SMs) is as always.  The limit
is looked at every 256 polls of a barrier, up to a millisecond: hence tiles of two milliseconds and more."""
import pytest

from computelibrary_b200 import capi

pytestmark = pytest.mark.gpu


def packed(g, rows, cols, fmt):
    """Random codes and scales made on the device (the matrices are large)."""
    import torch
    q = torch.randint(0, 256, (rows, capi.mx_pitch(cols)), generator=g, device="cuda", dtype=torch.uint8)
    low, high = (125, 130) if fmt == capi.MXFP4 else (40, 72)
    return q, torch.randint(low, high, (capi.mx_scale_bytes(rows, cols, fmt),), generator=g, device="cuda", dtype=torch.uint8)


def gives_up(ctx, call, limit):
    """Whether the call ran out of its limit (it may have been faster)."""
    ctx.set_wait_limit_us(limit)
    try:
        call()
        ctx.sync()
        return False
    except capi.CuglError as e:
        assert e.status == capi.RUNTIME_ERROR and "wait ran out" in e.message
        return True
    finally:
        ctx.set_wait_limit_us(0)


def check(ctx, call, out, sure=True):
    import torch
    call()
    ctx.sync()
    want = out.clone()
    assert torch.isfinite(want).all()
    given_up = [gives_up(ctx, call, limit) for limit in (1, 20, 100, 1, 50)]
    assert any(given_up) or not sure
    for _ in range(2):
        out.zero_()
        call()
        ctx.sync()
        assert torch.equal(out, want)


@pytest.mark.parametrize("fmt", [capi.MXFP4, capi.NVFP4])
@pytest.mark.parametrize("M,N,K", [(16, 128, 2 ** 24), (30, 256, 2 ** 24), (64, 128, 2 ** 24), (100, 128, 2 ** 24),  # K shared by a cluster
                                   (40, 19200, 2 ** 20), (100, 4864, 2 ** 21),                                      # a CTA per tile
                                   (512, 4096, 2 ** 21), (2048, 8192, 2 ** 20)])                                    # SM pairs, halves of tiles, both
def test_products(ctx, fmt, M, N, K):
    import torch
    g = torch.Generator(device="cuda").manual_seed(M)
    a, b = packed(g, M, K, fmt), packed(g, N, K, fmt)
    out = torch.zeros((M, N), dtype=torch.float32, device="cuda")
    d = capi.make_mx_gemm_desc(M, N, K, fmt, capi.F32, alpha=2.0 ** -20)
    check(ctx, lambda: ctx.mx_gemm(d, *a, *b, None, out), out)


@pytest.mark.parametrize("fmt", [capi.MXFP4, capi.NVFP4])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k,sure", [
    (1, 2 ** 20, 128, 1, 1, False), (100, 2 ** 20, 128, 1, 1, True),     # long rows of gate and up (the first is over in half a millisecond)
    (1, 128, 2 ** 20, 16, 16, True), (100, 128, 2 ** 20, 16, 16, True)])  # of down
def test_expert_layer(ctx, fmt, tokens, hidden, inner, experts, top_k, sure):
    import torch
    g = torch.Generator(device="cuda").manual_seed(tokens)
    # the tiles of an expert's scales are its own: where rows are a multiple of 128 those of all experts are one matrix'
    gate, up, down = packed(g, experts * inner, hidden, fmt), packed(g, experts * inner, hidden, fmt), packed(g, experts * hidden, inner, fmt)
    x = torch.randn((tokens, hidden), generator=g, device="cuda").to(torch.bfloat16)
    logits = torch.randn((tokens, experts), generator=g, device="cuda")
    d = capi.make_mx_moe_desc(tokens, hidden, inner, experts, top_k, fmt, capi.BF16, gate_alpha=2.0 ** -14, up_alpha=2.0 ** -14, down_alpha=2.0 ** -14)
    ws = torch.zeros(capi.mx_moe_workspace_bytes(d), dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(x)
    check(ctx, lambda: ctx.mx_moe(d, x, logits, gate, up, down, out, ws), out, sure)
