"""Small inputs (factors, biases, logits, scales, tokens) that the launch right ahead on the stream writes: every call reads what was
written for it.  cugl_moe_combine writes them here, itself launched so that its successor starts early."""
import numpy as np
import pytest

from computelibrary_b200 import capi

pytestmark = pytest.mark.gpu


class Writer:
    """Writes one of `turns` random vectors to `n` floats (or another type)."""

    def __init__(self, ctx, n, dtype=capi.F32, seed=0, turns=4):
        import torch
        self.ctx, self.n = ctx, n
        self.values = torch.from_numpy(np.random.default_rng(seed).uniform(0.5, 2.0, (turns, n)).astype(np.float32)).cuda()
        self.out = torch.zeros(n, dtype={capi.F32: torch.float32, capi.BF16: torch.bfloat16}[dtype], device="cuda")
        self.slots = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
        self.one = torch.ones((1, 1), device="cuda")
        self.desc = capi.make_moe_combine_desc(1, 1, n, 1, capi.F32, dtype)

    def write(self, turn):
        self.ctx.moe_combine(self.desc, self.values[turn], self.slots, self.one, self.out)


def compare(ctx, writers, call, out):
    """What the call gives when everything has been written long before is what it gives right behind the writes."""
    import torch
    turns = writers[0].values.shape[0]
    want = []
    for t in range(turns):
        for w in writers:
            w.write(t)
        ctx.sync()
        call()
        ctx.sync()
        want.append(out.clone())
    assert not torch.equal(want[0], want[1])
    for _ in range(20):
        got = []
        for t in range(turns):
            for w in writers:
                w.write(t)
            call()
            got.append(out.clone())
        ctx.sync()
        for g, w in zip(got, want):
            assert torch.equal(g, w)


def stored(g, rows, cols, fmt):
    import torch
    q = torch.randint(0, 256, (rows, capi.mx_pitch(cols)), generator=g, device="cuda", dtype=torch.uint8)
    low, high = (125, 130) if fmt == capi.MXFP4 else (40, 72)
    return q, torch.randint(low, high, (capi.mx_scale_bytes(rows, cols, fmt),), generator=g, device="cuda", dtype=torch.uint8)


@pytest.mark.parametrize("expected", [1, 10 ** 6])
@pytest.mark.parametrize("swiglu", [False, True])
def test_factors_and_bias_of_groups(ctx, swiglu, expected):
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)
    E, N, K, fmt = 4, 256, 64, capi.NVFP4
    a, b, up = stored(g, 512, K, fmt), stored(g, E * N, K, fmt), stored(g, E * N, K, fmt)
    groups = torch.tensor([[0, 100], [128, 3], [256, 128], [384, 0]], dtype=torch.int32, device="cuda")
    out = torch.zeros((512, N), device="cuda")
    d = capi.make_mx_grouped_gemm_desc(E, 512, N, K, fmt, capi.F32, expected_rows=expected, swiglu=swiglu, has_bias=not swiglu, alpha=0.01)
    f, other = Writer(ctx, E, seed=1), Writer(ctx, E if swiglu else E * N, seed=2)
    call = lambda: ctx.mx_grouped_gemm(d, *a, groups, (*b, f.out), out, up=(*up, other.out) if swiglu else None, bias=None if swiglu else other.out)
    compare(ctx, [f, other], call, out)


@pytest.mark.parametrize("M", [1, 300])
def test_bias_of_a_product(ctx, M):
    import torch
    g = torch.Generator(device="cuda").manual_seed(2)
    N, K, fmt = 512, 64, capi.MXFP4
    a, b = stored(g, M, K, fmt), stored(g, N, K, fmt)
    out = torch.zeros((M, N), device="cuda")
    d = capi.make_mx_gemm_desc(M, N, K, fmt, capi.F32, has_bias=True)
    bias = Writer(ctx, N)
    compare(ctx, [bias], lambda: ctx.mx_gemm(d, *a, *b, bias.out, out), out)


def test_logits_and_tokens_of_the_expert_layer(ctx):
    import torch
    g = torch.Generator(device="cuda").manual_seed(3)
    E, H, F, fmt = 16, 256, 128, capi.NVFP4
    gate, up, down = stored(g, E * F, H, fmt), stored(g, E * F, H, fmt), stored(g, E * H, F, fmt)
    logits, x = Writer(ctx, E, seed=1), Writer(ctx, H, capi.BF16, seed=2)
    out = torch.zeros((1, H), dtype=torch.bfloat16, device="cuda")
    d = capi.make_mx_moe_desc(1, H, F, E, 4, fmt, capi.BF16, renormalize=False, gate_alpha=0.01, up_alpha=0.01, down_alpha=0.01)
    ws = torch.zeros(capi.mx_moe_workspace_bytes(d), dtype=torch.uint8, device="cuda")
    compare(ctx, [logits, x], lambda: ctx.mx_moe(d, x.out.view(1, H), logits.out.view(1, E), gate, up, down, out, ws), out)


@pytest.mark.parametrize("lengths", [[1] * 24, [70, 3]], ids=len)
def test_scales_of_adapters(ctx, lengths):
    import torch
    g = torch.Generator(device="cuda").manual_seed(4)
    R, M, A, K, N, r = len(lengths), sum(lengths), 3, 128, 520, 16
    x, a, b = (torch.randn(s, generator=g, device="cuda").to(torch.bfloat16) for s in ((M, K), (A, r, K), (A, N, r)))
    base, out = torch.randn((M, N), generator=g, device="cuda"), torch.zeros((M, N), device="cuda")
    starts = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda")
    picks = torch.arange(R, device="cuda", dtype=torch.int32) % A
    d = capi.make_lora_desc(M, R, A, r, K, N, capi.BF16, capi.F32)
    ws = torch.zeros(capi.lora_workspace_bytes(d), dtype=torch.uint8, device="cuda")
    scales = Writer(ctx, A)
    compare(ctx, [scales], lambda: ctx.lora(d, x, starts, picks, None, scales.out, a, b, base, out, ws), out)
