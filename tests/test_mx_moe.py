"""The expert layer with 4-bit weights against the formulas in 64 bits.

Tolerance: what float sums can change, carried through the layer (mx_helpers.moe): a code of h may fall the other way where its
midpoint lies within the error of h, and then counts as a whole step times its weight; plus half a step of the result's type."""
import ctypes as C

import numpy as np
import pytest

import mx_helpers as mx
from computelibrary_b200 import capi

FORMATS = [capi.MXFP4, capi.NVFP4]
HALF_STEP = {capi.F16: 2.0 ** -11, capi.BF16: 2.0 ** -8}


def torch_dtype(dtype):
    import torch
    return {capi.F16: torch.float16, capi.BF16: torch.bfloat16}[dtype]


# ---- without a GPU ----------------------------------------------------------------------------------------
def test_descriptor_layout():
    assert C.sizeof(capi.MxMoeDesc) == 13 * 4 + 4 + 5 * 8 and capi.MxMoeDesc.ld_x.offset == 56


@pytest.mark.parametrize("change,word", [
    (dict(tokens=-1), "tokens"), (dict(tokens=129), "tokens"), (dict(hidden=8), "hidden"), (dict(hidden=100), "hidden"),
    (dict(intermediate=24), "hidden"), (dict(intermediate=2 ** 20 + 16), "hidden"), (dict(experts=0), "experts"), (dict(experts=513), "experts"),
    (dict(top_k=0), "top_k"), (dict(top_k=9), "top_k"), (dict(top_k=17, experts=64, ld_logits=256), "top_k"), (dict(format=3), "format"),
    (dict(dtype=capi.F32), "dtype"), (dict(ld_x=126), "ld_x"), (dict(ld_x=129), "ld_x"), (dict(ld_dst=100), "ld_x"), (dict(ld_logits=28), "ld_logits"),
    (dict(ld_logits=34), "ld_logits"), (dict(ld_gate_up=40), "ld_gate_up"), (dict(ld_gate_up=16), "ld_gate_up"), (dict(ld_down=8), "ld_gate_up"),
    (dict(x_exponent=1), "exponent"), (dict(h_exponent=-1), "exponent"), (dict(format=capi.NVFP4, h_exponent=65), "exponent"),
    (dict(gate_alpha=float("nan")), "alpha"), (dict(down_alpha=float("inf")), "alpha"),
    (dict(experts=512, hidden=2 ** 20, ld_x=2 ** 21, ld_dst=2 ** 21, ld_gate_up=2 ** 19, intermediate=2 ** 20, ld_down=2 ** 19, ld_logits=2048), None)])
def test_validate_refuses(change, word):
    d = capi.make_mx_moe_desc(4, 64, 32, 8, 2, capi.MXFP4, capi.BF16)
    assert capi.mx_moe_validate(d)[0] == 0 and capi.mx_moe_workspace_bytes(d) > 0
    for k, v in change.items():
        setattr(d, k, v)
    st, why = capi.mx_moe_validate(d)
    if word is None:  # the largest rows count that still fits
        assert st == 0
        return
    assert st == capi.INVALID_ARGUMENT and word in why and capi.mx_moe_workspace_bytes(d) == 0


def test_null_context_is_refused():
    d = capi.make_mx_moe_desc(4, 64, 32, 8, 2, capi.MXFP4, capi.BF16)
    assert capi.load_library().cugl_mx_moe(None, C.byref(d), *[None] * 10, 0) == capi.INVALID_ARGUMENT


def test_choice_of_the_reference():
    nan, inf = float("nan"), float("inf")
    picks = mx.choose([[1, 3, 3, 0], [nan, -inf, -inf, 2], [nan, nan, -inf, -inf], [0, 0, 0, 0]], 2, True)
    assert [[e for e, _ in p] for p in picks] == [[1, 2], [3], [], [0, 1]]
    assert picks[0][0][1] == 0.5 and picks[1][0][1] == 1.0


@pytest.mark.parametrize("size", [1.0, 0.1])
def test_h_exponent_follows_the_gate_weight(size):
    """What the header says of it: with small weights E4M3 scales of h run out at exponent 0, and with one that follows their size the
    error is that of h quantised without them."""
    rng = np.random.default_rng(3)
    h, p = rng.standard_normal((256, 256)) * size, 1 / 128
    w = rng.standard_normal((256, 64))

    def error(stored):
        return np.linalg.norm((stored - p * h) @ w) / np.linalg.norm(p * h @ w)

    apart = error(p * mx.values(*mx.quantize(h, mx.NVFP4), mx.NVFP4))
    folded = {e: error(mx.values(*mx.quantize(p * h, mx.NVFP4, e), mx.NVFP4, e)) for e in (0, -6, -9)}
    assert folded[0] > 1.3 * apart and folded[-9] < 1.05 * apart
    if size == 1.0:
        assert folded[-6] < 1.05 * apart


# ---- on the GPU -------------------------------------------------------------------------------------------
class Layer:
    def __init__(self, seed, hidden, inner, experts, fmt, pitch_extra=0):
        import torch
        rng = np.random.default_rng(seed)
        self.hidden, self.inner, self.experts, self.fmt = hidden, inner, experts, fmt
        self.pitches = (capi.mx_pitch(hidden) + pitch_extra, capi.mx_pitch(inner) + pitch_extra)

        def matrices(rows, cols, pitch, std):
            codes, tiles, vals = [], [], []
            for _ in range(experts):
                code, byte, v = mx.matrix(rng, rows, cols, fmt, std)
                packed = mx.pack(code, pitch)
                packed[:, cols // 2:] = 0xFF
                codes.append(packed)
                tiles.append(mx.tile(byte, fill=255 if fmt == mx.MXFP4 else 127))  # NaN behind the last row
                vals.append(v)
            return (torch.from_numpy(np.concatenate(codes)).cuda(), torch.from_numpy(np.concatenate(tiles)).cuda()), np.stack(vals)

        std = 1.0 / np.sqrt(hidden)
        self.gate, self.vgate = matrices(inner, hidden, self.pitches[0], std)
        self.up, self.vup = matrices(inner, hidden, self.pitches[0], std)
        self.down, self.vdown = matrices(hidden, inner, self.pitches[1], 1.0 / np.sqrt(inner))

    def desc(self, tokens, top_k, dtype, **more):
        return capi.make_mx_moe_desc(tokens, self.hidden, self.inner, self.experts, top_k, self.fmt, dtype, ld_gate_up=self.pitches[0],
                                     ld_down=self.pitches[1], **more)


def workspace(d):
    import torch
    n = capi.mx_moe_workspace_bytes(d)
    return torch.full((n + 256,), 0xFF, dtype=torch.uint8, device="cuda")[:n]  # NaN scales wherever nothing is written


def expected(layer, x, logits, top_k, dtype, renormalize=True, x_exponent=0, h_exponent=0, alphas=(1, 1, 1)):
    vx = mx.values(*mx.quantize(x.double().cpu().numpy(), layer.fmt, x_exponent), layer.fmt, x_exponent)
    y, tol = mx.moe(vx, logits.double().cpu().numpy(), layer.vgate, layer.vup, layer.vdown, top_k, renormalize, layer.fmt, h_exponent, alphas)
    return y, tol + HALF_STEP[dtype] * (np.abs(y) + tol) + (2.0 ** -25 if dtype == capi.F16 else 0)


def check(ctx, layer, tokens, top_k, dtype=capi.BF16, seed=0, logits=None, pad=0, renormalize=True, **more):
    import torch
    g = torch.Generator().manual_seed(seed + tokens)
    x = torch.randn((tokens, layer.hidden + pad), generator=g).to(torch_dtype(dtype)).cuda()
    logits = torch.randn((tokens, layer.experts + pad), generator=g) * 1.5 if logits is None else logits
    logits = logits.cuda()
    out = torch.full((tokens + 1, layer.hidden + pad), 7.0, dtype=torch_dtype(dtype), device="cuda")
    d = layer.desc(tokens, top_k, dtype, renormalize=renormalize, ld_x=2 * x.stride(0), ld_logits=4 * logits.stride(0), ld_dst=2 * out.stride(0),
                   **{k: v for k, v in more.items() if k != "alphas"}, **dict(zip(("gate_alpha", "up_alpha", "down_alpha"), more.get("alphas", (1, 1, 1)))))
    ws = workspace(d)
    ctx.mx_moe(d, x, logits, layer.gate, layer.up, layer.down, out, ws)
    ctx.sync()
    y, tol = expected(layer, x[:, :layer.hidden], logits[:, :layer.experts], top_k, dtype, renormalize, more.get("x_exponent", 0),
                      more.get("h_exponent", 0), more.get("alphas", (1, 1, 1)))
    got = out[:tokens, :layer.hidden].double().cpu().numpy()
    bad = ~(np.abs(got - y) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[:3].tolist()}: {got[bad][:3]} for {y[bad][:3]} +- {tol[bad][:3]}"
    assert (out[tokens:] == 7).all() and (out[:, layer.hidden:] == 7).all()
    return out, (d, x, logits, layer.gate, layer.up, layer.down)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hidden,inner,experts,top_k", [(64, 64, 1, 1), (128, 128, 4, 2), (16, 16, 3, 1), (272, 144, 9, 3), (512, 320, 40, 8), (2048, 768, 6, 6)])
def test_layer(ctx, fmt, hidden, inner, experts, top_k):
    layer = Layer(hidden + inner, hidden, inner, experts, fmt)
    for tokens in (1, 7):
        check(ctx, layer, tokens, top_k)
    check(ctx, layer, 20, top_k, capi.F16, renormalize=False)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128])
def test_tokens(ctx, fmt, tokens):
    layer = Layer(5, 320, 208, 24, fmt)
    check(ctx, layer, tokens, 4, capi.F16)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(1, 768, 640, 10, 8), (3, 1104, 512, 12, 4), (8, 2032, 208, 24, 3), (1, 3600, 1056, 4, 2),
                                                               (100, 3600, 1056, 4, 2), (2, 7184, 272, 8, 4), (70, 7184, 272, 4, 2)])
def test_parts_of_k(ctx, fmt, tokens, hidden, inner, experts, top_k):
    """Sizes whose K is shared by two or four CTAs in either product, in uneven parts."""
    check(ctx, Layer(hidden + inner, hidden, inner, experts, fmt), tokens, top_k)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(1, 2320, 640, 10, 8), (8, 2864, 640, 10, 8), (1, 3056, 768, 8, 8), (7, 3344, 640, 10, 8)])
def test_parts_of_longer_rows(ctx, fmt, tokens, hidden, inner, experts, top_k):
    """Rows of ten to fourteen chunks over two or four CTAs, few tokens and enough units for one CTA per SM."""
    check(ctx, Layer(hidden + inner, hidden, inner, experts, fmt), tokens, top_k)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens,hidden,inner", [(2, 18944, 48), (2, 18960, 48), (30, 19088, 32), (60, 19200, 16), (100, 19216, 32), (3, 38032, 16)])
def test_long_rows(ctx, fmt, tokens, hidden, inner):
    """From 148 output blocks on the down product runs without clusters, from 296 on in several waves."""
    check(ctx, Layer(hidden, hidden, inner, 3, fmt), tokens, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_many_experts(ctx, fmt):
    """More units of work than SMs: a CTA works through several."""
    layer = Layer(6, 256, 144, 512, fmt)
    check(ctx, layer, 128, 16)
    check(ctx, layer, 60, 8)
    check(ctx, layer, 30, 16)
    check(ctx, layer, 10, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_what_cannot_be_chosen(ctx, fmt):
    """Masked experts, NaN, equal logits, tokens with fewer choices than top_k, with none, a call in which nobody has any."""
    import torch
    layer = Layer(7, 96, 80, 12, fmt)
    inf, nan = float("inf"), float("nan")
    logits = torch.randn((20, 12), generator=torch.Generator().manual_seed(9))
    logits[0] = -inf
    logits[1] = nan
    logits[2, 3:] = -inf
    logits[3, ::2], logits[3, 1::2] = nan, -inf
    logits[3, 5] = -3.0
    logits[4] = 2.5
    logits[5, 4:8] = logits[5].max() + 1
    logits[6] = torch.finfo(torch.float32).min
    logits[7, :6] = torch.finfo(torch.float32).min
    logits[8] = torch.linspace(-300, 300, 12)
    logits[9] = -0.0
    logits[9, 6] = 0.0
    for renormalize in (True, False):
        out, _ = check(ctx, layer, 20, 4, logits=logits, renormalize=renormalize)
        assert (out[[0, 1], :] == 0).all()
    out, _ = check_empty(ctx, layer)
    assert (out == 0).all()


def check_empty(ctx, layer):
    import torch
    logits = torch.full((5, layer.experts), -float("inf"), device="cuda")
    x = torch.randn((5, layer.hidden), device="cuda").to(torch.bfloat16)
    out = torch.full_like(x, 7.0)
    d = layer.desc(5, 3, capi.BF16)
    ctx.mx_moe(d, x, logits, layer.gate, layer.up, layer.down, out, workspace(d))
    ctx.sync()
    return out, d


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [1, 3, 8])
def test_strides(ctx, pad):
    check(ctx, Layer(8, 160, 112, 5, capi.NVFP4, pitch_extra=32), 19, 2, pad=pad)


@pytest.mark.gpu
def test_exponents_and_alphas(ctx):
    layer = Layer(9, 128, 160, 6, capi.NVFP4)
    check(ctx, layer, 9, 2, x_exponent=-2, h_exponent=-5, alphas=(0.5, -0.25, 3.0))
    check(ctx, Layer(9, 128, 160, 6, capi.MXFP4), 9, 2, alphas=(2.0, 0.75, -1.5))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_nan_stays_with_its_token(ctx, fmt):
    import torch
    layer = Layer(10, 192, 96, 8, fmt)
    g = torch.Generator().manual_seed(4)
    x, logits = torch.randn((18, 192), generator=g).to(torch.bfloat16), torch.randn((18, 8), generator=g)
    x[3, 17], x[16, 100], logits[7, 2] = float("nan"), float("inf"), float("inf")
    x, logits = x.cuda(), logits.cuda()
    out = torch.zeros_like(x)
    d = layer.desc(18, 2, capi.BF16)
    ctx.mx_moe(d, x, logits, layer.gate, layer.up, layer.down, out, workspace(d))
    ctx.sync()
    bad = torch.isnan(out).any(dim=1).cpu().tolist()
    assert bad == [t in (3, 7, 16) for t in range(18)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 30, 128])
def test_equal_calls_give_equal_bits(ctx, tokens):
    import torch
    layer = Layer(11, 512, 256, 32, capi.MXFP4)
    out, (d, *args) = check(ctx, layer, tokens, 4)
    ws = workspace(d)
    for _ in range(4):
        again = torch.full_like(out, 7.0)
        ctx.mx_moe(d, *args, again, ws)
        ctx.sync()
        assert torch.equal(out, again)


@pytest.mark.gpu
def test_calls_in_a_row_share_a_workspace_and_a_graph(ctx):
    """Two layers one after the other on one workspace, captured and replayed on new tokens."""
    import torch
    import computelibrary_b200 as cl
    stream = torch.cuda.Stream()
    own = cl.Context(0, stream.cuda_stream)
    first, second = Layer(12, 160, 96, 10, capi.NVFP4), Layer(13, 160, 128, 10, capi.NVFP4)
    tokens = 6
    x = torch.zeros((tokens, 160), dtype=torch.bfloat16, device="cuda")
    mid, y, again = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    logits = torch.zeros((tokens, 10), device="cuda")
    d1, d2 = first.desc(tokens, 3, capi.BF16), second.desc(tokens, 2, capi.BF16)
    ws = workspace(max((d1, d2), key=capi.mx_moe_workspace_bytes))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        own.mx_moe(d1, x, logits, first.gate, first.up, first.down, mid, ws)
        own.mx_moe(d2, mid, logits, second.gate, second.up, second.down, y, ws)
        own.mx_moe(d1, x, logits, first.gate, first.up, first.down, again, ws)
    for seed in (1, 2, 3):
        g = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn((tokens, 160), generator=g))
        logits.copy_(torch.randn((tokens, 10), generator=g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(mid, again)
        for layer, src, dst, k in ((first, x, mid, 3), (second, mid, y, 2)):
            want, tol = expected(layer, src, logits, k, capi.BF16)
            assert (np.abs(dst.double().cpu().numpy() - want) <= tol).all()
    del graph
    own.sync()
    own.close()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 20])
@pytest.mark.parametrize("fmt", FORMATS)
def test_many_calls_in_a_row_on_one_workspace(ctx, fmt, tokens):
    """Other experts in every call, nothing awaited in between: a launch that runs ahead reads the choices of its own call."""
    import torch
    layer = Layer(61, 512, 256, 48, fmt)
    g = torch.Generator().manual_seed(tokens)
    calls = 300
    x = torch.randn((calls, tokens, 512), generator=g).to(torch.bfloat16).cuda()
    logits = torch.randn((calls, tokens, 48), generator=g).cuda()
    d = layer.desc(tokens, 4, capi.BF16)
    ws = workspace(d)
    alone, row = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    for i in range(calls):
        ctx.mx_moe(d, x[i], logits[i], layer.gate, layer.up, layer.down, alone[i], ws)
        ctx.sync()
    for i in range(calls):
        ctx.mx_moe(d, x[i], logits[i], layer.gate, layer.up, layer.down, row[i], ws)
    ctx.sync()
    assert torch.equal(row, alone)
    want, tol = expected(layer, x[calls - 1], logits[calls - 1], 4, capi.BF16)
    assert (np.abs(row[-1].double().cpu().numpy() - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,k_block", [(1, 6, 0), (40, 40, 3), (128, 40, 2), (1, 6, 65536), (40, 40, 65539), (128, 40, 65537)])
def test_wait_limit(ctx, tokens, experts, k_block):
    """Operand copies that never come, in the gate and up products or in the down product: the call ends by its wait limit and says
    so; the next one is as always.  (1 token: four chunks of K over four CTAs, one copy each to withhold.)"""
    import torch
    layer = Layer(51, 1024, 1152, experts, capi.NVFP4)
    g = torch.Generator().manual_seed(tokens)
    x, logits = torch.randn((tokens, 1024), generator=g).to(torch.bfloat16).cuda(), torch.randn((tokens, experts), generator=g).cuda()
    d = layer.desc(tokens, 4, capi.BF16)
    ws, want, out = workspace(d), torch.zeros_like(x), torch.zeros_like(x)
    args = (d, x, logits, layer.gate, layer.up, layer.down)
    ctx.mx_moe(*args, want, ws)
    ctx.sync()
    ctx.set_wait_limit_us(20000)
    try:
        ctx.withhold_copy_once(k_block)
        ctx.mx_moe(*args, out, ws)
        with pytest.raises(capi.CuglError) as e:
            ctx.sync()
        assert e.value.status == capi.RUNTIME_ERROR
    finally:
        ctx.set_wait_limit_us(0)
    ctx.mx_moe(*args, out, ws)
    ctx.sync()
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hidden,inner,experts", [(1024, 256, 6), (1024, 128, 20)])
def test_time_of_the_second_launch_counts_in_no_wait_of_the_third(ctx, fmt, hidden, inner, experts):
    """A copy withheld in the gate and up products keeps the second launch busy for the whole limit.  The third, all of which is on the
    device by then, has waited for nothing of its own: it carries on and writes its results, whatever they are, although the call
    says that a wait ran out.  (Both would run out of the limit within microseconds of each other: which comes first is chance, so
    this can pass without the wait it is about.)"""
    import torch
    layer = Layer(71, hidden, inner, experts, fmt)
    g = torch.Generator().manual_seed(1)
    x, logits = torch.randn((1, hidden), generator=g).to(torch.bfloat16).cuda(), torch.randn((1, experts), generator=g).cuda()
    d = layer.desc(1, 4, capi.BF16)
    ws = workspace(d)
    for limit in (3000, 20000):
        out = torch.full_like(x, 7.0)
        ctx.set_wait_limit_us(limit)
        try:
            ctx.withhold_copy_once(0)
            ctx.mx_moe(d, x, logits, layer.gate, layer.up, layer.down, out, ws)
            with pytest.raises(capi.CuglError) as e:
                ctx.sync()
            assert e.value.status == capi.RUNTIME_ERROR
        finally:
            ctx.set_wait_limit_us(0)
        assert not (out == 7).any()


@pytest.mark.gpu
def test_nothing_to_do_and_refusals(ctx):
    import torch
    p = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda").data_ptr()
    d = capi.make_mx_moe_desc(2, 64, 32, 4, 2, capi.MXFP4, capi.BF16)
    n = capi.mx_moe_workspace_bytes(d)
    none = capi.make_mx_moe_desc(0, 64, 32, 4, 2, capi.MXFP4, capi.BF16)
    ctx.mx_moe(none, None, None, (None, None), (None, None), (None, None), None, None, 0)
    good = [p, p, (p, p), (p, p), (p, p), p, p, n]
    for at, bad in ((0, None), (1, None), (2, (None, p)), (2, (p, None)), (3, (None, p)), (3, (p, None)), (4, (None, p)), (4, (p, None)),
                    (5, None), (6, None), (0, p + 1), (1, p + 2), (2, (p + 8, p)), (3, (p, p + 4)), (4, (p + 1, p)), (5, p + 1), (6, p + 128),
                    (7, n - 1)):
        args = list(good)
        args[at] = bad
        with pytest.raises(capi.CuglError) as e:
            ctx.mx_moe(d, *args)
        assert e.value.status == capi.INVALID_ARGUMENT
    ctx.sync()
