"""Expert layers of prompts, step after step, and adapters beside a projection, as a program runs them: nothing awaited between the
calls, captured and replayed on new inputs, on two streams at once, over rows further apart than 32 bits count.  Every step is held
against 64 bits on what the step before it left; the tolerances are those of the steps' own tests."""
import numpy as np
import pytest

import mx_helpers as mx
import test_lora
import test_moe_steps
from computelibrary_b200 import capi
from test_mx_gemm import FORMATS
from test_mx_together import quantized

pytestmark = pytest.mark.gpu


class Layer:
    """An expert layer with every buffer its steps need, for up to `tokens` tokens."""

    def __init__(self, fmt, tokens, hidden, inner, experts, top_k, seed=0, device_rng=None):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.fmt, self.T, self.H, self.F, self.E, self.k = fmt, tokens, hidden, inner, experts, top_k
        self.rows = capi.mx_group_rows(experts, tokens * top_k)

        def packed(rows, cols, std):
            w = torch.randn((experts, rows, cols), generator=g, device="cuda") * std
            return w

        self.plain = [packed(inner, hidden, hidden ** -0.5), packed(inner, hidden, hidden ** -0.5), packed(hidden, inner, inner ** -0.5)]
        self.factors = [torch.rand(experts, generator=g, device="cuda") + 0.5 for _ in range(3)]
        self.weights = None
        b = lambda *s, dt=torch.uint8: torch.zeros(s, dtype=dt, device="cuda")
        self.x = b(tokens, hidden, dt=torch.bfloat16)
        self.logits = b(tokens, experts, dt=torch.float32)
        self.ids, self.slots = b(tokens, top_k, dt=torch.int32), b(tokens, top_k, dt=torch.int32)
        self.p, self.groups = b(tokens, top_k, dt=torch.float32), b(experts, 2, dt=torch.int32)
        self.xq, self.xs = b(self.rows, capi.mx_pitch(hidden)), b(capi.mx_scale_bytes(self.rows, hidden, fmt))
        self.h = b(self.rows, inner, dt=torch.bfloat16)
        self.hq, self.hs = b(self.rows, capi.mx_pitch(inner)), b(capi.mx_scale_bytes(self.rows, inner, fmt))
        self.d = b(self.rows, hidden, dt=torch.bfloat16)
        self.y = b(tokens, hidden, dt=torch.bfloat16)
        self.route = capi.make_moe_route_desc(tokens, experts, top_k)
        self.ws = b(capi.moe_route_workspace_bytes(self.route))

    def quantize_weights(self, ctx):
        import torch
        out = []
        for w in self.plain:
            parts = [quantized(ctx, w[e].contiguous(), self.fmt, capi.F32) for e in range(self.E)]
            out.append((torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])))
        self.weights = [w + (f,) for w, f in zip(out, self.factors)]

    def fill(self, seed):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.x.copy_(torch.randn(self.x.shape, generator=g, device="cuda"))
        self.logits.copy_(torch.randn(self.logits.shape, generator=g, device="cuda") + torch.randn(self.E, generator=g, device="cuda"))

    def run(self, ctx):
        T, k, fmt, n = self.T, self.k, self.fmt, self.T * self.k
        ctx.moe_route(self.route, self.logits, self.ids, self.p, self.slots, self.groups, self.ws)
        ctx.mx_quantize_grouped(capi.make_mx_group_desc(T, k, self.H, self.rows, fmt, capi.BF16), self.x, self.slots, self.xq, self.xs)
        ctx.mx_grouped_gemm(capi.make_mx_grouped_gemm_desc(self.E, self.rows, self.F, self.H, fmt, capi.BF16, expected_rows=n, swiglu=True),
                            self.xq, self.xs, self.groups, self.weights[0], self.h, up=self.weights[1])
        ctx.mx_quantize_grouped(capi.make_mx_group_desc(T, k, self.F, self.rows, fmt, capi.BF16, src_grouped=True), self.h, self.slots, self.hq, self.hs)
        ctx.mx_grouped_gemm(capi.make_mx_grouped_gemm_desc(self.E, self.rows, self.H, self.F, fmt, capi.BF16, expected_rows=n),
                            self.hq, self.hs, self.groups, self.weights[2], self.d)
        ctx.moe_combine(capi.make_moe_combine_desc(T, k, self.H, self.rows, capi.BF16, capi.BF16), self.d, self.slots, self.p, self.y)

    def check(self):
        """Every step against 64 bits on what the step before it left."""
        ids, weights, rel, slots, groups = test_moe_steps.route_reference(self.logits.double().cpu().numpy(), self.k, True)
        np.testing.assert_array_equal(self.slots.cpu().numpy(), slots)
        np.testing.assert_array_equal(self.groups.cpu().numpy(), groups)
        p = self.p.double().cpu().numpy()
        assert (np.abs(p - weights) <= rel * weights).all()
        wv = [[mx.values(*mx.quantize(w[e].double().cpu().numpy(), self.fmt), self.fmt) * float(f[e]) for e in range(self.E)]
              for w, f in zip(self.plain, self.factors)]
        x, h, d, y = (t.double().cpu().numpy() for t in (self.x, self.h, self.d, self.y))

        def stored(v):
            return mx.values(*mx.quantize(v, self.fmt), self.fmt)

        xv = stored(x)
        for e, (start, count) in enumerate(groups):
            if count == 0:
                continue
            rows = slice(start, start + count)
            tokens = [t for t in range(self.T) if e in ids[t]]
            a = xv[tokens]
            steps = 2.0 ** -23 * (-(-self.H // 64) + 10)
            g, u = a @ wv[0][e].T, a @ wv[1][e].T
            eg, eu = steps * (np.abs(a) @ np.abs(wv[0][e]).T), steps * (np.abs(a) @ np.abs(wv[1][e]).T)
            silu = g / (1 + np.exp(-g))
            tol = (1.1 * eg + (2.0 ** -20 + 2.0 ** -23 * np.abs(g)) * np.abs(silu)) * (np.abs(u) + eu) + np.abs(silu) * eu
            assert (np.abs(h[rows] - silu * u) <= tol + 2.0 ** -8 * (np.abs(silu * u) + tol)).all()
            hv = stored(h[rows])
            want = hv @ wv[2][e].T
            tol = 2.0 ** -23 * (-(-self.F // 64) + 10) * (np.abs(hv) @ np.abs(wv[2][e]).T)
            assert (np.abs(d[rows] - want) <= tol + 2.0 ** -8 * (np.abs(want) + tol)).all()
        want, size = np.zeros_like(y), np.zeros_like(y)
        for j in range(self.k):
            want += p[:, j:j + 1] * d[slots[:, j]]
            size += np.abs(p[:, j:j + 1] * d[slots[:, j]])
        tol = self.k * 2.0 ** -24 * size
        assert (np.abs(y - want) <= tol + 2.0 ** -8 * (np.abs(want) + tol)).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 12, 3), (130, 12, 3), (700, 5, 2), (900, 4, 4)])
def test_an_expert_layer(ctx, fmt, tokens, experts, top_k):
    layer = Layer(fmt, tokens, 320, 144, experts, top_k, seed=tokens)
    layer.quantize_weights(ctx)
    for seed in (1, 2):  # buffers hold what the last call left
        layer.fill(seed)
        layer.run(ctx)
        ctx.sync()
        layer.check()


@pytest.mark.parametrize("tokens", [40, 600])
def test_an_expert_layer_captured(ctx, tokens):
    """One graph, replayed on other inputs, beside another one of its own buffers."""
    import torch
    import computelibrary_b200 as cl
    layers = [Layer(capi.NVFP4, tokens, 320, 144, 12, 3, seed=i) for i in range(2)]
    for layer in layers:
        layer.quantize_weights(ctx)
        layer.fill(0)
        layer.run(ctx)  # loads the kernels
    ctx.sync()
    streams = [torch.cuda.Stream() for _ in layers]
    contexts = [cl.Context(0, s.cuda_stream) for s in streams]
    graphs = []
    for layer, s, c in zip(layers, streams, contexts):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            layer.run(c)
        graphs.append(g)
    for seed in (5, 6, 7):
        for layer in layers:
            layer.fill(seed)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        got = [layer.y.clone() for layer in layers]
        for layer, y in zip(layers, got):
            layer.y.zero_()
            layer.run(ctx)
            ctx.sync()
            assert torch.equal(layer.y, y) and bool(y.any())
    layers[0].check()
    del graphs
    for c in contexts:
        c.sync()
        c.close()


def test_two_streams_at_once(ctx):
    import torch
    import computelibrary_b200 as cl
    layers = [Layer(capi.MXFP4, 500, 512, 256, 16, 4, seed=i) for i in range(2)]
    wants = []
    for i, layer in enumerate(layers):
        layer.quantize_weights(ctx)
        layer.fill(i)
        layer.run(ctx)
        ctx.sync()
        wants.append(layer.y.clone())
    streams = [torch.cuda.Stream() for _ in layers]
    contexts = [cl.Context(0, s.cuda_stream) for s in streams]
    for _ in range(20):
        for layer, c in zip(layers, contexts):
            layer.run(c)
    for c in contexts:
        c.sync()
        c.close()
    for layer, want in zip(layers, wants):
        assert torch.equal(layer.y, want)


def test_without_overlapped_launches(ctx):
    import torch
    layer = Layer(capi.NVFP4, 300, 320, 144, 12, 3)
    layer.quantize_weights(ctx)
    layer.fill(3)
    layer.run(ctx)
    ctx.sync()
    want = layer.y.clone()
    ctx.set_dependent_launch(False)
    try:
        layer.y.zero_()
        layer.run(ctx)
        ctx.sync()
    finally:
        ctx.set_dependent_launch(True)
    assert torch.equal(layer.y, want)


# ---- adapters beside a projection -------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,requests", [(1, 1), (24, 24), (300, 5)])
def test_projection_with_adapters(ctx, tokens, requests):
    """The shared 4-bit projection, then the adapters on top of its result in place; captured with both and replayed after the requests
    have changed."""
    import torch
    import computelibrary_b200 as cl
    K, N, E, r = 512, 776, 4, 16
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randn((tokens, K), generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn((N, K), generator=g, device="cuda") * K ** -0.5).to(torch.bfloat16)
    a = (torch.randn((E, r, K), generator=g, device="cuda") * K ** -0.5).to(torch.bfloat16)
    b = (torch.randn((E, N, r), generator=g, device="cuda") * r ** -0.5).to(torch.bfloat16)
    scales = torch.rand(E, generator=g, device="cuda") + 0.5
    ranks = torch.tensor([16, 8, 3, 16], dtype=torch.int32, device="cuda")
    wq, xq = quantized(ctx, w, capi.NVFP4, capi.BF16), quantized(ctx, x, capi.NVFP4, capi.BF16)
    y, base = (torch.zeros((tokens, N), device="cuda") for _ in range(2))
    starts, picks = torch.zeros(requests + 1, dtype=torch.int32, device="cuda"), torch.zeros(requests, dtype=torch.int32, device="cuda")
    gemm = capi.make_mx_gemm_desc(tokens, N, K, capi.NVFP4, capi.F32)
    lora = capi.make_lora_desc(tokens, requests, E, r, K, N, capi.BF16, capi.F32)
    ws = torch.zeros(capi.lora_workspace_bytes(lora), dtype=torch.uint8, device="cuda")

    def call(c):
        c.mx_gemm(gemm, *xq, *wq, None, y)
        c.lora(lora, x, starts, picks, ranks, scales, a, b, y, y, ws)

    ctx.mx_gemm(gemm, *xq, *wq, None, base)
    starts.copy_(torch.tensor([tokens * i // requests for i in range(requests + 1)], dtype=torch.int32))
    call(ctx)
    ctx.sync()
    s = torch.cuda.Stream()
    c = cl.Context(0, s.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        call(c)
    rng = np.random.default_rng(tokens)
    vx, va, vb, vy = (t.double().cpu().numpy() for t in (x, a, b, base))
    for turn in range(3):
        edges = [0] + sorted(rng.integers(0, tokens + 1, requests - 1).tolist()) + [tokens]
        chosen = rng.integers(-1, E, requests).tolist()
        starts.copy_(torch.tensor(edges, dtype=torch.int32))
        picks.copy_(torch.tensor(chosen, dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        got = y.double().cpu().numpy()
        y.zero_()
        call(ctx)
        ctx.sync()
        assert (y.double().cpu().numpy() == got).all()
        for i, e in enumerate(chosen):
            rows = slice(edges[i], edges[i + 1])
            if e < 0:
                assert (got[rows] == vy[rows]).all()
                continue
            n = int(ranks[e])
            v, size = vx[rows] @ va[e, :n].T, np.abs(vx[rows]) @ np.abs(va[e, :n]).T
            ev = 2.0 ** -23 * (K // 16 + 16) * size
            sc = float(scales[e])
            want = vy[rows] + sc * (v @ vb[e, :, :n].T)
            tol = sc * ((ev + 2.0 ** -25 * (np.abs(v) + ev)) @ np.abs(vb[e, :, :n]).T + 2.0 ** -23 * 4 * ((np.abs(v) + ev) @ np.abs(vb[e, :, :n]).T))
            assert (np.abs(got[rows] - want) <= tol + 2.0 ** -23 * (np.abs(want) + tol)).all()
    del graph
    c.sync()
    c.close()


def test_two_adapter_calls_at_once(ctx):
    import torch
    import computelibrary_b200 as cl
    outs = [test_lora.check(ctx, [200, 1, 77], [0, 1, 2], 32, 1024, 1032, capi.BF16, capi.BF16, seed=i) for i in range(2)]
    wants = [o.clone() for o, _ in outs]
    streams = [torch.cuda.Stream() for _ in outs]
    contexts = [cl.Context(0, s.cuda_stream) for s in streams]
    torch.cuda.synchronize()
    for _ in range(20):
        for (_, args), c in zip(outs, contexts):
            c.lora(*args)
    for c in contexts:
        c.sync()
        c.close()
    for (o, _), want in zip(outs, wants):
        assert torch.equal(o, want)


# ---- rows further apart than 32 bits count ------------------------------------------------------------------------
FAR = 1 << 20  # bytes between rows


def far(rows, cols, dtype, fill=None):
    """rows x cols elements, rows FAR bytes apart."""
    import torch
    flat = torch.empty(rows * FAR, dtype=torch.uint8, device="cuda")
    m = flat.view(dtype).view(rows, -1)[:, :cols]
    if fill is not None:
        m.copy_(fill)
    return m


def test_far_rows(ctx):
    import torch
    T, k, cols, rows = 2500, 2, 96, 5120
    assert rows * FAR > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(0)
    near = torch.randn((rows, cols), generator=g, device="cuda").to(torch.bfloat16)
    slots = torch.randperm(rows, generator=g, device="cuda")[:T * k].to(torch.int32).view(T, k).contiguous()
    p = torch.rand((T, k), generator=g, device="cuda")
    src = far(rows, cols, torch.bfloat16, near)
    y, want = (torch.zeros((T, cols), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ctx.moe_combine(capi.make_moe_combine_desc(T, k, cols, rows, capi.BF16, capi.BF16), near, slots, p, want)
    ctx.moe_combine(capi.make_moe_combine_desc(T, k, cols, rows, capi.BF16, capi.BF16, ld_src=FAR), src, slots, p, y)
    ctx.sync()
    assert torch.equal(y, want)
    # quantised from and to far rows, then multiplied into far rows
    q0, q1 = torch.zeros((rows, 48), dtype=torch.uint8, device="cuda"), far(rows, 48, torch.uint8)
    q1.zero_()
    s0, s1 = (torch.zeros(capi.mx_scale_bytes(rows, cols, capi.NVFP4), dtype=torch.uint8, device="cuda") for _ in range(2))
    ctx.mx_quantize_grouped(capi.make_mx_group_desc(T, k, cols, rows, capi.NVFP4, capi.BF16, src_grouped=True), near, slots, q0, s0)
    ctx.mx_quantize_grouped(capi.make_mx_group_desc(T, k, cols, rows, capi.NVFP4, capi.BF16, src_grouped=True, ld=FAR, ld_packed=FAR), src, slots, q1, s1)
    ctx.sync()
    assert torch.equal(q0, q1) and torch.equal(s0, s1)
    w, sw = quantized(ctx, torch.randn((3 * 128, cols), generator=g, device="cuda"), capi.NVFP4, capi.F32)
    groups = torch.tensor([[0, 1000], [1024, 2000], [4992, 128]], dtype=torch.int32, device="cuda")
    for expected in (1, 10 ** 6):
        o0, o1 = torch.zeros((rows, 128), dtype=torch.bfloat16, device="cuda"), far(rows, 128, torch.bfloat16)
        o1.zero_()
        d = lambda **kw: capi.make_mx_grouped_gemm_desc(3, rows, 128, cols, capi.NVFP4, capi.BF16, expected_rows=expected, **kw)
        ctx.mx_grouped_gemm(d(), q0, s0, groups, (w, sw), o0)
        ctx.mx_grouped_gemm(d(lda=FAR, ldd=FAR), q1, s1, groups, (w, sw), o1)
        ctx.sync()
        assert torch.equal(o0, o1) and bool(o0[4992:].any())
        del o1
    del q1, src


def test_far_rows_of_adapters(ctx):
    import torch
    M, K, N, r = 4200, 64, 72, 8
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn((M, K), generator=g, device="cuda").to(torch.float16)
    base = torch.randn((M, N), generator=g, device="cuda").to(torch.float16)
    a = torch.randn((2, r, K), generator=g, device="cuda").to(torch.float16)
    b = torch.randn((2, N, r), generator=g, device="cuda").to(torch.float16)
    starts = torch.tensor([0, 4100, M], dtype=torch.int32, device="cuda")
    picks = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    scales = torch.ones(2, device="cuda")
    want = torch.zeros((M, N), dtype=torch.float16, device="cuda")
    d = lambda **kw: capi.make_lora_desc(M, 2, 2, r, K, N, capi.F16, capi.F16, **kw)
    ws = torch.zeros(capi.lora_workspace_bytes(d()), dtype=torch.uint8, device="cuda")
    ctx.lora(d(), x, starts, picks, None, scales, a, b, base, want, ws)
    fx, fb, fo = far(M, K, torch.float16, x), far(M, N, torch.float16, base), far(M, N, torch.float16)
    ctx.lora(d(ld_x=FAR, ld_base=FAR, ld_dst=FAR), fx, starts, picks, None, scales, a, b, fb, fo, ws)
    ctx.sync()
    assert torch.equal(fo, want) and bool((want != base).any(dim=1).all())


# ---- threads ----------------------------------------------------------------------------------------------------
def test_from_a_thread_without_a_context():
    """A thread that has made no CUDA call before, with a context of its own."""
    import threading
    import torch
    import computelibrary_b200 as cl
    failed = []
    layer = Layer(capi.NVFP4, 200, 320, 144, 12, 3)

    def run():
        try:
            c = cl.Context(0, torch.cuda.default_stream().cuda_stream)
            layer.quantize_weights(c)
            layer.fill(1)
            layer.run(c)
            c.sync()
            c.close()
        except BaseException as e:
            failed.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    assert not failed, failed
    layer.check()
