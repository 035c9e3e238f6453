"""The microscaled 4-bit calls as a program uses them: one after the other, two at a time, over large matrices, with and without
overlapped launches.  Tolerances are those of test_mx_gemm.py and test_mx_moe.py."""
import numpy as np
import pytest

import mx_helpers as mx
import test_mx_gemm
import test_mx_moe
from computelibrary_b200 import capi

FORMATS = [capi.MXFP4, capi.NVFP4]


# ---- without a GPU ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("change", [dict(gate_alpha=1e30, x_exponent=64), dict(up_alpha=-1e30, x_exponent=64), dict(down_alpha=1e30, h_exponent=64)])
def test_alphas_that_overflow_with_their_exponent(change):
    d = capi.make_mx_moe_desc(4, 64, 32, 8, 2, capi.NVFP4, capi.BF16)
    for k, v in change.items():
        setattr(d, k, v)
    st, why = capi.mx_moe_validate(d)
    assert st == capi.INVALID_ARGUMENT and "alpha" in why
    d.x_exponent = d.h_exponent = 0
    assert capi.mx_moe_validate(d)[0] == 0


@pytest.mark.parametrize("dtype", [capi.F16, capi.BF16])
@pytest.mark.parametrize("which", ["a_dtype", "b_dtype", "dst_dtype"])
def test_integer_products_take_no_16_bit_floats(dtype, which):
    for stage, dst in ((capi.STAGE_NONE, capi.S32), (capi.STAGE_FIXEDPOINT, capi.U8)):
        d, keep = capi.make_gemm_desc(16, 16, 16, capi.U8, capi.U8, dst, stage=stage)
        setattr(d, which, dtype)
        assert capi.gemm_validate(d)[0] != 0


# ---- on the GPU -------------------------------------------------------------------------------------------
def quantized(ctx, x, fmt, dtype, exponent=0):
    import torch
    rows, cols = x.shape
    q = torch.zeros((rows, capi.mx_pitch(cols)), dtype=torch.uint8, device="cuda")
    s = torch.zeros(capi.mx_scale_bytes(rows, cols, fmt), dtype=torch.uint8, device="cuda")
    ctx.mx_quantize(capi.make_mx_desc(rows, cols, fmt, dtype, tensor_exponent=exponent), x, q, s)
    return q, s


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens", [1, 20, 128])
def test_a_block_of_a_model(ctx, fmt, tokens):
    """Projection, gate logits and expert layer, the last in place, nothing awaited between the calls."""
    import torch
    hidden, experts, top_k = 320, 12, 3
    g = torch.Generator().manual_seed(tokens)
    layer = test_mx_moe.Layer(21, hidden, 144, experts, fmt)
    x = torch.randn((tokens, hidden), generator=g).to(torch.bfloat16).cuda()
    w = (torch.randn((hidden, hidden), generator=g) * hidden ** -0.5).to(torch.bfloat16).cuda()
    r = (torch.randn((experts, hidden), generator=g) * hidden ** -0.5).to(torch.bfloat16).cuda()
    y, before = (torch.zeros((tokens, hidden), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    logits = torch.zeros((tokens, experts), device="cuda")
    d = layer.desc(tokens, top_k, capi.BF16)
    ws = test_mx_moe.workspace(d)
    wq, rq, xq = quantized(ctx, w, fmt, capi.BF16), quantized(ctx, r, fmt, capi.BF16), quantized(ctx, x, fmt, capi.BF16)
    gemm = capi.make_mx_gemm_desc(tokens, hidden, hidden, fmt, capi.BF16)
    ctx.mx_gemm(gemm, *xq, *wq, None, y)
    ctx.mx_gemm(gemm, *xq, *wq, None, before)
    yq = quantized(ctx, y, fmt, capi.BF16)
    ctx.mx_gemm(capi.make_mx_gemm_desc(tokens, experts, hidden, fmt, capi.F32), *yq, *rq, None, logits)
    ctx.mx_moe(d, y, logits, layer.gate, layer.up, layer.down, y, ws)
    ctx.sync()

    def values(t):
        return mx.values(*mx.quantize(t.double().cpu().numpy(), fmt), fmt)

    for got, a, b, half in ((before, x, w, 2.0 ** -8), (logits, before, r, 2.0 ** -24)):
        va, vb = values(a), values(b)
        want = va @ vb.T
        tol = (-(-hidden // 64) + 10) * 2.0 ** -23 * (np.abs(va) @ np.abs(vb).T) + half * np.abs(want)
        assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()
    want, tol = test_mx_moe.expected(layer, before, logits, top_k, capi.BF16)
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.gpu
def test_two_streams_at_a_time(ctx):
    """Contexts on two streams, products that share K in clusters, SM-pair products and expert layers beside each other: the bits
    are those of the calls alone."""
    import torch
    import computelibrary_b200 as cl
    rng = np.random.default_rng(4)
    sizes = [(1, 4096, 4096), (24, 1500, 2304), (100, 2048, 2048), (300, 2048, 1024), (2048, 2048, 512), (64, 20000, 256)]
    products = []
    for M, N, K in sizes:
        a, sa, _ = test_mx_gemm.operand(rng, M, K, capi.NVFP4)
        b, sb, _ = test_mx_gemm.operand(rng, N, K, capi.NVFP4)
        products.append((capi.make_mx_gemm_desc(M, N, K, capi.NVFP4, capi.F32), a, sa, b, sb, None))
    layer = test_mx_moe.Layer(31, 512, 320, 24, capi.MXFP4)
    g = torch.Generator().manual_seed(5)
    layers = []
    for tokens in (1, 40, 128):
        x, logits = torch.randn((tokens, 512), generator=g).to(torch.bfloat16).cuda(), torch.randn((tokens, 24), generator=g).cuda()
        layers.append((layer.desc(tokens, 4, capi.BF16), x, logits, layer.gate, layer.up, layer.down))

    def outputs():
        return ([torch.zeros((M, N), device="cuda") for M, N, _ in sizes],
                [torch.zeros_like(x) for _, x, *_ in layers], [test_mx_moe.workspace(d) for d, *_ in layers])

    def run(context, out, turn):
        order = list(range(len(products) + len(layers)))
        for i in order[turn:] + order[:turn]:
            if i < len(products):
                context.mx_gemm(*products[i], out[0][i])
            else:
                i -= len(products)
                context.mx_moe(*layers[i], out[1][i], out[2][i])

    want = outputs()
    run(ctx, want, 0)
    ctx.sync()
    contexts = [cl.Context(0, torch.cuda.Stream().cuda_stream) for _ in range(2)]
    sets = [outputs(), outputs()]
    torch.cuda.synchronize()
    for turn in range(9):
        for context, out, shift in zip(contexts, sets, (0, 4)):
            run(context, out, (turn + shift) % 9)
    for context in contexts:
        context.sync()
    for out in sets:
        for got, alone in zip(out[0] + out[1], want[0] + want[1]):
            assert torch.equal(got, alone)
    for context in contexts:
        context.close()


@pytest.mark.gpu
def test_threads_at_a_time(ctx):
    """Threads with contexts of their own make their calls at once (a kernel's first ones among them): the bits are those of one thread."""
    import threading
    import torch
    import computelibrary_b200 as cl
    rng = np.random.default_rng(6)
    jobs = []
    for fmt in FORMATS:
        for M, N, K in ((1, 500, 300), (20, 300, 600), (50, 300, 600), (100, 260, 900), (300, 2048, 2048)):
            a, sa, _ = test_mx_gemm.operand(rng, M, K, fmt)
            b, sb, _ = test_mx_gemm.operand(rng, N, K, fmt)
            jobs.append((capi.make_mx_gemm_desc(M, N, K, fmt, capi.F32), a, sa, b, sb))
    layers = []
    for fmt in FORMATS:
        layer = test_mx_moe.Layer(81, 256, 160, 12, fmt)
        for tokens in (2, 30, 60, 100):
            x, logits = torch.from_numpy(rng.standard_normal((tokens, 256))).to(torch.bfloat16).cuda(), torch.from_numpy(rng.standard_normal((tokens, 12))).float().cuda()
            layers.append((layer.desc(tokens, 3, capi.BF16), x, logits, layer.gate, layer.up, layer.down))

    def buffers():
        return ([torch.zeros((j[0].M, j[0].N), device="cuda") for j in jobs], [torch.zeros_like(x) for _, x, *_ in layers],
                [test_mx_moe.workspace(d) for d, *_ in layers])

    def run(context, out):
        for j, y in zip(jobs, out[0]):
            context.mx_gemm(*j, None, y)
        for j, y, ws in zip(layers, out[1], out[2]):
            context.mx_moe(*j, y, ws)

    sets = [buffers() for _ in range(5)]
    contexts = [cl.Context(0, torch.cuda.Stream().cuda_stream) for _ in range(4)]
    torch.cuda.synchronize()
    start, failed = threading.Barrier(4), []

    def thread(context, out):
        try:
            start.wait()
            for _ in range(3):
                run(context, out)
            context.sync()
        except BaseException as e:
            failed.append(e)

    threads = [threading.Thread(target=thread, args=a) for a in zip(contexts, sets)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    run(ctx, sets[4])
    ctx.sync()
    for out in sets[:4]:
        for got, alone in zip(out[0] + out[1], sets[4][0] + sets[4][1]):
            assert torch.equal(got, alone)
    for context in contexts:
        context.close()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_without_overlapped_launches(ctx, fmt):
    import torch
    g = torch.Generator().manual_seed(6)
    layer = test_mx_moe.Layer(41, 256, 160, 8, fmt)
    x, logits = torch.randn((30, 256), generator=g).to(torch.bfloat16).cuda(), torch.randn((30, 8), generator=g).cuda()
    w = torch.randn((700, 256), generator=g).cuda()
    d, gemm = layer.desc(30, 2, capi.BF16), capi.make_mx_gemm_desc(30, 700, 256, fmt, capi.F16)
    ws = test_mx_moe.workspace(d)
    results = []
    try:
        for on in (True, False):
            ctx.set_dependent_launch(on)
            y, z = torch.zeros_like(x), torch.zeros((30, 700), dtype=torch.float16, device="cuda")
            for _ in range(3):
                ctx.mx_moe(d, x, logits, layer.gate, layer.up, layer.down, y, ws)
                ctx.mx_gemm(gemm, *quantized(ctx, y, fmt, capi.BF16), *quantized(ctx, w, fmt, capi.F32), None, z)
            ctx.sync()
            results.append((y, z))
    finally:
        ctx.set_dependent_launch(True)
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [capi.F32, capi.BF16])
def test_results_past_32_bits(ctx, dtype):
    """More than 2^32 bytes of results, of a product and of a read-back."""
    import torch
    fmt, K = capi.NVFP4, 80
    M, N = (40000, 30000) if dtype == capi.F32 else (75000, 30000)
    g = torch.Generator(device="cuda").manual_seed(7)
    td = test_mx_gemm.torch_dtype(dtype)
    a, b = torch.randn((M, K), generator=g, device="cuda"), torch.randn((N, K), generator=g, device="cuda")
    aq, bq = quantized(ctx, a, fmt, capi.F32), quantized(ctx, b, fmt, capi.F32)
    out = torch.zeros((M, N), dtype=td, device="cuda")
    assert out.numel() * out.element_size() > 2 ** 32
    ctx.mx_gemm(capi.make_mx_gemm_desc(M, N, K, fmt, dtype), *aq, *bq, None, out)
    ctx.sync()
    rows = [0, 1, 17895, 17896, 35791, 35792, M - 2, M - 1]
    va, vb = mx.values(*mx.quantize(a[rows].double().cpu().numpy(), fmt), fmt), mx.values(*mx.quantize(b.double().cpu().numpy(), fmt), fmt)
    want = va @ vb.T
    tol = (-(-K // 64) + 10) * 2.0 ** -23 * (np.abs(va) @ np.abs(vb).T) + test_mx_gemm.HALF_STEP[dtype] * np.abs(want)
    assert (np.abs(out[rows].double().cpu().numpy() - want) <= tol).all()

    q, s = quantized(ctx, out, fmt, dtype)
    again = torch.zeros_like(out)
    ctx.mx_dequantize(capi.make_mx_desc(M, N, fmt, dtype), q, s, again)
    ctx.sync()
    code, byte = mx.quantize(out[rows].double().cpu().numpy(), fmt)
    want = mx.values(code, byte, fmt)
    assert np.array_equal(again[rows].double().cpu().numpy(), want)  # codes of four bits times scales of four: exact in either type


@pytest.mark.gpu
def test_weights_past_32_bits(ctx):
    """Experts at both ends of weights of more than 2^32 bytes; those that nobody chose hold NaN scales."""
    import torch
    fmt, hidden, inner, experts, pitch = capi.NVFP4, 2048, 1024, 512, 9216
    rng = np.random.default_rng(8)
    chosen = (0, 1, 455, 456, 511)

    def matrices(rows, cols):
        codes = torch.empty((experts, rows, pitch), dtype=torch.uint8, device="cuda")
        scales = torch.full((experts, capi.mx_scale_bytes(rows, cols, fmt)), 127, dtype=torch.uint8, device="cuda")
        vals = {}
        for e in chosen:
            code, byte, vals[e] = mx.matrix(rng, rows, cols, fmt, cols ** -0.5)
            codes[e] = torch.from_numpy(mx.pack(code, pitch)).cuda()
            scales[e] = torch.from_numpy(mx.tile(byte)).cuda()
        return (codes, scales), vals

    gate, vgate = matrices(inner, hidden)
    up, vup = matrices(inner, hidden)
    down, vdown = matrices(hidden, inner)
    assert gate[0].numel() > 2 ** 32
    tokens, top_k = 3, 4
    x = torch.from_numpy(rng.standard_normal((tokens, hidden))).to(torch.bfloat16).cuda()
    logits = torch.full((tokens, experts), -float("inf"), device="cuda")
    logits[:, list(chosen)] = torch.from_numpy(rng.standard_normal((tokens, len(chosen)))).float().cuda()
    d = capi.make_mx_moe_desc(tokens, hidden, inner, experts, top_k, fmt, capi.BF16, ld_gate_up=pitch, ld_down=pitch)
    ws = test_mx_moe.workspace(d)
    out = torch.zeros_like(x)
    ctx.mx_moe(d, x, logits, gate, up, down, out, ws)
    ctx.sync()
    small = type("Small", (), {})()
    small.fmt = fmt
    small.vgate, small.vup, small.vdown = (np.stack([v[e] for e in chosen]) for v in (vgate, vup, vdown))
    want, tol = test_mx_moe.expected(small, x, logits[:, list(chosen)], top_k, capi.BF16)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
