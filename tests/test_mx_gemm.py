"""Products of microscaled 4-bit matrices against sums in 64 bits.

Tolerance: one MMA adds 64 products to a float accumulator.  The products are exact (two significant bits each, times scales of
at most four), so each MMA is off by at most one step of 24 bits of the magnitudes added so far: ceil(K / 64) steps of 2^-23
times sum |a| |b|, as much again for the partial sums of a split K (at most 8), one fused multiply-add, and half a step of the
destination type."""
import ctypes as C

import numpy as np
import pytest

import mx_helpers as mx
from computelibrary_b200 import capi

FORMATS = [capi.MXFP4, capi.NVFP4]
DTYPES = [capi.F32, capi.F16, capi.BF16]
HALF_STEP = {capi.F32: 2.0 ** -24, capi.F16: 2.0 ** -11, capi.BF16: 2.0 ** -8}


def torch_dtype(dtype):
    import torch
    return {capi.F32: torch.float32, capi.F16: torch.float16, capi.BF16: torch.bfloat16}[dtype]


# ---- without a GPU ----------------------------------------------------------------------------------------
def test_descriptor_layout():
    assert C.sizeof(capi.MxGemmDesc) == 24 + 24 + 8 and capi.MxGemmDesc.alpha.offset == 48


@pytest.mark.parametrize("change,word", [
    (dict(M=-1), "M"), (dict(N=0), "N"), (dict(K=0), "K"), (dict(K=2 ** 31 - 1), "too large"), (dict(format=-1), "format"),
    (dict(dst_dtype=capi.S32), "dst_dtype"), (dict(lda=32), "lda"), (dict(lda=56), "lda"), (dict(ldb=72), "lda"), (dict(ldb=2 ** 40), "2^40"),
    (dict(ldd=198), "ldd"), (dict(ldd=201), "ldd"), (dict(alpha=float("inf")), "alpha"), (dict(alpha=float("nan")), "alpha")])
def test_validate_refuses(change, word):
    d = capi.make_mx_gemm_desc(4, 100, 100, capi.NVFP4, capi.BF16)
    assert capi.mx_gemm_validate(d)[0] == 0
    for k, v in change.items():
        setattr(d, k, v)
    st, why = capi.mx_gemm_validate(d)
    assert st == capi.INVALID_ARGUMENT and word in why


def test_null_context_is_refused():
    d = capi.make_mx_gemm_desc(4, 100, 100, capi.NVFP4, capi.BF16)
    assert capi.load_library().cugl_mx_gemm(None, C.byref(d), None, None, None, None, None, None) == capi.INVALID_ARGUMENT


# ---- on the GPU -------------------------------------------------------------------------------------------
def operand(rng, rows, cols, fmt, pitch=None):
    """Every code, scales that differ from block to block; rows behind the last have NaN scales, which must not matter."""
    import torch
    pitch = capi.mx_pitch(cols) if pitch is None else pitch
    code = rng.integers(0, 16, (rows, cols)).astype(np.uint8)
    nb = mx.blocks_of(cols, fmt)
    byte = (rng.integers(121, 133, (rows, nb)) if fmt == mx.MXFP4 else rng.integers(1, 127, (rows, nb))).astype(np.uint8)
    packed = mx.pack(code, pitch)
    packed[:, (cols + 1) // 2:] = 0xFF  # bytes between rows belong to nobody
    return (torch.from_numpy(packed).cuda(), torch.from_numpy(mx.tile(byte, fill=255 if fmt == mx.MXFP4 else 127)).cuda(),
            mx.values(code, byte, fmt))


def check(ctx, M, N, K, fmt, dtype, bias=False, alpha=1.0, seed=0, pad=0, lda=None, ldb=None):
    import torch
    rng = np.random.default_rng(seed + 7 * M + 13 * N + K)
    a, sa, va = operand(rng, M, K, fmt, lda)
    b, sb, vb = operand(rng, N, K, fmt, ldb)
    vbias = rng.standard_normal(N).astype(np.float32) * 100 if bias else None
    want = alpha * (va @ vb.T) + (vbias.astype(np.float64) if bias else 0)
    size = abs(alpha) * (np.abs(va) @ np.abs(vb).T) + (np.abs(vbias) if bias else 0)
    if dtype == capi.F16:  # keep within its range
        alpha = alpha * 2.0 ** -float(np.ceil(np.log2(max(1.0, np.abs(want).max() / 30000))))
        want = alpha * (va @ vb.T) + (vbias.astype(np.float64) if bias else 0)
        size = abs(alpha) * (np.abs(va) @ np.abs(vb).T) + (np.abs(vbias) if bias else 0)
    out = torch.full((M + 2, N + pad), 7.0, dtype=torch_dtype(dtype), device="cuda")
    d = capi.make_mx_gemm_desc(M, N, K, fmt, dtype, lda=lda, ldb=ldb, ldd=out.stride(0) * out.element_size(), alpha=alpha, has_bias=bias)
    dbias = torch.from_numpy(vbias).cuda() if bias else None
    ctx.mx_gemm(d, a, sa, b, sb, dbias, out)
    ctx.sync()
    got = out[:M, :N].double().cpu().numpy()
    assert np.isfinite(got).all()
    tol = (-(-K // 64) + 8 + 2) * 2.0 ** -23 * size + HALF_STEP[dtype] * np.abs(want) + (2.0 ** -25 if dtype == capi.F16 else 0)
    bad = np.abs(got - want) > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[:3].tolist()}: {got[bad][:3]} for {want[bad][:3]}"
    assert (out[M:] == 7).all() and (out[:, N:] == 7).all()
    return out, (d, a, sa, b, sb, dbias)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("K", [64, 128, 256, 512, 1, 2, 15, 16, 31, 33, 63, 65, 127, 129, 192, 255, 257, 321, 1000, 2050, 4096])
def test_k(ctx, fmt, K):
    check(ctx, 16, 128, K, fmt, capi.F32)
    check(ctx, 5, 300, K, fmt, capi.BF16, bias=True)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 511, 513, 700])
def test_tokens(ctx, fmt, M):
    check(ctx, M, 200, 512, fmt, capi.F32)
    check(ctx, M, 129, 320, fmt, capi.F16, bias=True, alpha=-0.375)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("N", [1, 2, 31, 32, 127, 128, 129, 255, 257, 384, 1001, 2049])
def test_channels(ctx, fmt, N):
    check(ctx, 7, N, 1024, fmt, capi.BF16, pad=3)
    check(ctx, 130, N, 256, fmt, capi.F32, bias=True, pad=1)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (40, 2500, 1536), (2048, 2048, 512), (4096, 640, 256), (300, 19000, 128), (1200, 2304, 4096), (2600, 1500, 1000)])
def test_larger(ctx, fmt, dtype, M, N, K):
    check(ctx, M, N, K, fmt, dtype, bias=dtype == capi.BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(512, 4096, 700), (257, 8200, 2048), (385, 4104, 2304), (140, 9472, 2050), (2100, 2800, 300)])
def test_halves_of_tiles(ctx, fmt, M, N, K):
    """Few tiles, or a few beyond whole waves: worked on as two halves of 128 tokens, the second of which may be empty."""
    check(ctx, M, N, K, fmt, capi.BF16)
    check(ctx, M, N, K, fmt, capi.F32, bias=True)
    check(ctx, M, N - 1, K, fmt, capi.F16)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,k_block", [(1, 4096, 4096, 1), (8, 512, 1024, 0), (64, 20000, 1024, 3), (100, 4096, 2048, 0), (512, 4096, 2048, 3),
                                           (2048, 4096, 2048, 9), (300, 1001, 2048, 1)])
def test_wait_limit(ctx, M, N, K, k_block):
    """Operand copies that never come: the call ends by its wait limit and says so; the next one is as always."""
    import torch
    rng = np.random.default_rng(0)
    a, sa, _ = operand(rng, M, K, capi.NVFP4)
    b, sb, _ = operand(rng, N, K, capi.NVFP4)
    want, out = (torch.zeros((M, N), dtype=torch.float32, device="cuda") for _ in range(2))
    d = capi.make_mx_gemm_desc(M, N, K, capi.NVFP4, capi.F32)
    ctx.mx_gemm(d, a, sa, b, sb, None, want)
    ctx.sync()
    ctx.set_wait_limit_us(20000)
    try:
        ctx.withhold_copy_once(k_block)
        ctx.mx_gemm(d, a, sa, b, sb, None, out)
        with pytest.raises(capi.CuglError) as e:
            ctx.sync()
        assert e.value.status == capi.RUNTIME_ERROR
    finally:
        ctx.set_wait_limit_us(0)
    ctx.mx_gemm(d, a, sa, b, sb, None, out)
    ctx.sync()
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,pad", [(4097, 0), (4098, 0), (4098, 1), (4100, 2)])
def test_large_ragged_rows(ctx, dtype, N, pad):
    """Many tiles, long K and rows that bulk stores cannot write: odd, two-byte and four-byte aligned ones."""
    check(ctx, 1210, N, 3900, capi.NVFP4 if N % 2 else capi.MXFP4, dtype, bias=True, pad=pad)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_long_k(ctx, fmt):
    check(ctx, 3, 130, 70001, fmt, capi.F32)
    check(ctx, 200, 300, 16384, fmt, capi.F32)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_strides(ctx, fmt):
    check(ctx, 20, 150, 300, fmt, capi.F32, lda=160, ldb=256, pad=5)
    check(ctx, 300, 300, 300, fmt, capi.BF16, lda=176, ldb=192, pad=2)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 1000, 4096), (16, 256, 8192), (300, 700, 512), (1500, 1500, 1024)])
def test_equal_calls_give_equal_bits(ctx, M, N, K):
    import torch
    out, (d, *args) = check(ctx, M, N, K, capi.NVFP4, capi.F32)
    again = torch.full_like(out, 7.0)
    for _ in range(3):
        ctx.mx_gemm(d, *args, again)
        ctx.sync()
        assert torch.equal(out, again)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_nan_scales_stay_in_their_row(ctx, fmt):
    import torch
    rng = np.random.default_rng(3)
    x, w = rng.standard_normal((40, 512)), rng.standard_normal((300, 512))
    x[5, 100], w[77, 300] = np.nan, np.inf
    d = []
    for m in (x, w):
        t = torch.from_numpy(m).float().cuda()
        q = torch.zeros((m.shape[0], 256), dtype=torch.uint8, device="cuda")
        s = torch.zeros(capi.mx_scale_bytes(*m.shape, fmt), dtype=torch.uint8, device="cuda")
        ctx.mx_quantize(capi.make_mx_desc(*m.shape, fmt, capi.F32), t, q, s)
        d += [q, s]
    out = torch.zeros((40, 300), dtype=torch.float32, device="cuda")
    ctx.mx_gemm(capi.make_mx_gemm_desc(40, 300, 512, fmt, capi.F32), *d, None, out)
    ctx.sync()
    bad = torch.isnan(out).cpu().numpy()
    want = np.zeros((40, 300), bool)
    want[5], want[:, 77] = True, True
    assert np.array_equal(bad, want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens", [1, 33, 300])
def test_linear_layer(ctx, fmt, tokens):
    """As a program runs it: weights quantised once, activations quantised, multiplied, and both captured into a graph that is
    replayed on new activations."""
    import torch
    import computelibrary_b200 as cl
    stream = torch.cuda.Stream()
    own = cl.Context(0, stream.cuda_stream)
    N, K, exponent = 640, 1056, -5 if fmt == capi.NVFP4 else 0
    g = torch.Generator().manual_seed(tokens)
    w = torch.randn((N, K), generator=g) * 0.03
    wq, ws = torch.zeros((N, capi.mx_pitch(K)), dtype=torch.uint8, device="cuda"), torch.zeros(capi.mx_scale_bytes(N, K, fmt), dtype=torch.uint8, device="cuda")
    x = torch.zeros((tokens, K), dtype=torch.bfloat16, device="cuda")
    xq, xs = torch.zeros((tokens, capi.mx_pitch(K)), dtype=torch.uint8, device="cuda"), torch.zeros(capi.mx_scale_bytes(tokens, K, fmt), dtype=torch.uint8, device="cuda")
    y = torch.zeros((tokens, N), dtype=torch.bfloat16, device="cuda")
    wd = w.cuda()
    torch.cuda.synchronize()
    own.mx_quantize(capi.make_mx_desc(N, K, fmt, capi.F32, tensor_exponent=exponent), wd, wq, ws)
    own.sync()
    xd, gd = capi.make_mx_desc(tokens, K, fmt, capi.BF16), capi.make_mx_gemm_desc(tokens, N, K, fmt, capi.BF16, alpha=2.0 ** exponent)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        own.mx_quantize(xd, x, xq, xs)
        own.mx_gemm(gd, xq, xs, wq, ws, None, y)
    vw = mx.values(*mx.quantize(w.double().numpy(), fmt, exponent), fmt, exponent)
    for _ in range(2):
        x.copy_(torch.randn((tokens, K), generator=g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        vx = mx.values(*mx.quantize(x.double().cpu().numpy(), fmt), fmt)
        want = vx @ vw.T
        tol = (-(-K // 64) + 10) * 2.0 ** -23 * (np.abs(vx) @ np.abs(vw).T) + 2.0 ** -8 * np.abs(want)
        assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()
    del graph
    own.sync()
    own.close()


@pytest.mark.gpu
def test_nothing_to_do_and_refusals(ctx):
    import torch
    p = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda").data_ptr()
    ctx.mx_gemm(capi.make_mx_gemm_desc(0, 64, 64, capi.MXFP4, capi.F32), None, None, None, None, None, None)
    d, db = capi.make_mx_gemm_desc(2, 64, 64, capi.MXFP4, capi.F32), capi.make_mx_gemm_desc(2, 64, 64, capi.MXFP4, capi.F32, has_bias=True)
    for args in ((d, None, p, p, p, None, p), (d, p, None, p, p, None, p), (d, p, p, None, p, None, p), (d, p, p, p, None, None, p),
                 (d, p, p, p, p, None, None), (d, p, p, p, p, p, p), (db, p, p, p, p, None, p), (d, p + 8, p, p, p, None, p),
                 (d, p, p + 4, p, p, None, p), (d, p, p, p + 1, p, None, p), (d, p, p, p, p + 2, None, p), (d, p, p, p, p, None, p + 2),
                 (db, p, p, p, p, p + 1, p)):
        with pytest.raises(capi.CuglError) as e:
            ctx.mx_gemm(*args)
        assert e.value.status == capi.INVALID_ARGUMENT
    ctx.sync()
