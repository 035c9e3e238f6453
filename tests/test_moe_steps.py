"""The steps of an expert layer around its products: the gate with the rows of its choices, quantisation into groups, combination."""
import ctypes as C

import numpy as np
import pytest

import mx_helpers as mx
from computelibrary_b200 import capi
from test_mx_gemm import DTYPES, FORMATS, HALF_STEP, torch_dtype


# ---- without a GPU ----------------------------------------------------------------------------------------
def test_descriptor_layouts():
    assert C.sizeof(capi.MoeRouteDesc) == 32 and capi.MoeRouteDesc.ld_logits.offset == 24
    assert C.sizeof(capi.MxGroupDesc) == 48 and capi.MxGroupDesc.ld.offset == 32
    assert C.sizeof(capi.MoeCombineDesc) == 40 and capi.MoeCombineDesc.ld_src.offset == 24


def refuses(desc, validate, change, word):
    assert validate(desc)[0] == 0
    for k, v in change.items():
        setattr(desc, k, v)
    st, why = validate(desc)
    assert st == capi.INVALID_ARGUMENT and word in why


@pytest.mark.parametrize("change,word", [
    (dict(tokens=-1), "tokens"), (dict(experts=0), "experts"), (dict(experts=513), "experts"), (dict(top_k=0), "top_k"), (dict(top_k=17), "top_k"),
    (dict(top_k=9), "top_k"), (dict(dtype=capi.U8), "dtype"), (dict(ld_logits=28), "ld_logits"), (dict(ld_logits=34), "ld_logits"),
    (dict(tokens=2 ** 30, top_k=2), "32 bits")])
def test_route_refuses(change, word):
    refuses(capi.make_moe_route_desc(5, 8, 3), capi.moe_route_validate, change, word)


@pytest.mark.parametrize("change,word", [
    (dict(tokens=-1), "tokens"), (dict(rows=-1), "rows"), (dict(top_k=0), "top_k"), (dict(top_k=17), "top_k"), (dict(tokens=2 ** 30, top_k=2), "too large"),
    (dict(cols=0), "cols"), (dict(format=3), "format"), (dict(dtype=capi.S32), "dtype"), (dict(ld=198), "ld"), (dict(ld=201), "ld"),
    (dict(ld_packed=49), "ld_packed"), (dict(tensor_exponent=65), "tensor_exponent")])
def test_group_refuses(change, word):
    refuses(capi.make_mx_group_desc(5, 3, 100, 512, capi.NVFP4, capi.BF16), capi.mx_group_validate, change, word)


@pytest.mark.parametrize("change,word", [
    (dict(tokens=-1), "tokens"), (dict(rows=-1), "rows"), (dict(cols=0), "cols"), (dict(cols=2 ** 31 - 5), "too large"), (dict(top_k=0), "top_k"),
    (dict(top_k=17), "top_k"), (dict(src_dtype=capi.S8), "dtypes"), (dict(dst_dtype=capi.S8), "dtypes"), (dict(ld_src=399), "ld_src"), (dict(ld_dst=201), "ld_dst")])
def test_combine_refuses(change, word):
    refuses(capi.make_moe_combine_desc(5, 3, 100, 512, capi.F32, capi.BF16), capi.moe_combine_validate, change, word)


def test_null_contexts_are_refused():
    lib = capi.load_library()
    assert lib.cugl_moe_route(None, C.byref(capi.make_moe_route_desc(5, 8, 3)), *[None] * 6, 0) == capi.INVALID_ARGUMENT
    assert lib.cugl_mx_quantize_grouped(None, C.byref(capi.make_mx_group_desc(5, 3, 100, 512, capi.NVFP4, capi.BF16)), *[None] * 4) == capi.INVALID_ARGUMENT
    assert lib.cugl_moe_combine(None, C.byref(capi.make_moe_combine_desc(5, 3, 100, 512, capi.F32, capi.BF16)), *[None] * 4) == capi.INVALID_ARGUMENT


def test_workspace_of_the_gate():
    assert capi.moe_route_workspace_bytes(capi.make_moe_route_desc(129, 8, 3)) >= 3 * 8 * 4
    assert capi.moe_route_workspace_bytes(capi.make_moe_route_desc(5, 8, 9)) == 0


# ---- on the GPU -------------------------------------------------------------------------------------------
def route_reference(logits, top_k, renormalize):
    """(ids, weights, bound of their relative error, slots, groups) in 64 bits.  A logit less the largest one is off by half a step of 24
    bits, which its exponential takes over times that difference; the exponential is off by two steps, a sum of up to 512 terms (sixteen per
    lane, five exchanges) by 21, the quotient by one."""
    T, E = logits.shape
    ids, slots = np.full((T, top_k), -1, np.int64), np.full((T, top_k), -1, np.int64)
    weights, rel = np.zeros((T, top_k)), np.zeros((T, top_k))
    hits = [[] for _ in range(E)]
    for t, row in enumerate(logits):
        order = [e for e in np.lexsort((np.arange(E), -np.where(np.isnan(row), -np.inf, row))) if row[e] > -np.inf]
        chosen = order[:top_k]
        among = row[chosen] if renormalize else row[order]
        for j, e in enumerate(chosen):
            ids[t, j] = e
            d = among - row[chosen[0]]
            total = np.exp(d).sum()
            weights[t, j] = np.exp(row[e] - row[chosen[0]]) / total
            rel[t, j] = 2.0 ** -23 * (abs(row[e] - row[chosen[0]]) + (np.abs(d) * np.exp(d)).sum() / total + 2 + 2 + 21 + 1)
            hits[e].append((t, j))
    groups, at = np.zeros((E, 2), np.int64), 0
    for e in range(E):
        groups[e] = at, len(hits[e])
        for i, (t, j) in enumerate(hits[e]):
            slots[t, j] = at + i
        at += -(-len(hits[e]) // 128) * 128
    return ids, weights, rel, slots, groups


def check_route(ctx, logits, top_k, dtype=capi.F32, renormalize=True, pad=0):
    import torch
    T, E = logits.shape
    x = torch.full((T, E + pad), 1e4, dtype=torch_dtype(dtype), device="cuda")  # what lies between rows is not looked at
    x[:, :E] = torch.from_numpy(logits).to(torch_dtype(dtype)).cuda()
    d = capi.make_moe_route_desc(T, E, top_k, dtype, renormalize, ld_logits=x.stride(0) * x.element_size() if T else None)
    ids, slots = (torch.full((T + 1, top_k), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    w = torch.full((T + 1, top_k), 77.0, device="cuda")
    groups = torch.full((E + 1, 2), 77, dtype=torch.int32, device="cuda")
    ws = torch.full((capi.moe_route_workspace_bytes(d),), 255, dtype=torch.uint8, device="cuda")
    ctx.moe_route(d, x, ids, w, slots, groups, ws)
    ctx.sync()
    want = route_reference(x[:, :E].double().cpu().numpy(), top_k, renormalize)
    assert (ids[T] == 77).all() and (slots[T] == 77).all() and (w[T] == 77).all() and (groups[E] == 77).all()
    np.testing.assert_array_equal(ids[:T].cpu().numpy(), want[0])
    np.testing.assert_array_equal(groups[:E].cpu().numpy(), want[4])
    np.testing.assert_array_equal(slots[:T].cpu().numpy(), want[3])
    got = w[:T].double().cpu().numpy()
    assert (np.abs(got - want[1]) <= want[2] * want[1] + 2.0 ** -149).all()
    assert (slots[:T].max().item() if T else -1) < capi.mx_group_rows(E, T * top_k)
    return ids, w, slots, groups


@pytest.mark.gpu
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 8), (2, 3, 3), (33, 8, 2), (128, 64, 8), (129, 64, 8), (200, 500, 16), (1000, 128, 6), (64, 512, 16),
                                   (4097, 60, 4), (3, 33, 1), (700, 5, 5), (20000, 7, 2), (16384, 3, 1),
                                   (16385, 4, 2), (40000, 40, 3)])
def test_route(ctx, T, E, k, renormalize):
    rng = np.random.default_rng(T + E)
    logits = (rng.standard_normal((T, E)) * 3 + rng.standard_normal(E)).astype(np.float32)
    check_route(ctx, logits, k, renormalize=renormalize, pad=T % 3)
    check_route(ctx, logits, k, capi.BF16, renormalize)
    check_route(ctx, logits, k, capi.F16, renormalize, pad=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [5, 300])
def test_route_ties_and_nothing_to_choose(ctx, T, dtype):
    rng = np.random.default_rng(T)
    logits = rng.integers(-1, 2, (T, 40)).astype(np.float32)  # many alike; -0 and 0 are
    logits[logits == 0] *= rng.choice([-1.0, 1.0], (logits == 0).sum())
    logits[0] = -np.inf                                   # nothing
    logits[1, 2:] = np.nan                                # two
    logits[2] = np.where(np.arange(40) == 7, 1.0, -np.inf)  # one
    logits[3] = np.nan
    logits[4] = -60000.0                                  # all alike, far below zero
    check_route(ctx, logits, 6, dtype)
    check_route(ctx, logits, 6, dtype, renormalize=False)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 150])
def test_route_extremes(ctx, T):
    logits = np.tile(np.array([3.4e38, -3.4e38, 0.0, 1e-45, -1e-45, 3.4e38], np.float32), (T, 1))
    check_route(ctx, logits, 4)
    check_route(ctx, np.full((T, 9), -3.0e38, np.float32), 9, renormalize=False)


@pytest.mark.gpu
def test_route_one_expert_for_all(ctx):
    logits = np.zeros((500, 16), np.float32)
    logits[:, 11] = 5
    ids, _, _, groups = check_route(ctx, logits, 1)
    assert groups[11].tolist() == [0, 500] and groups[12].tolist() == [512, 0]


@pytest.mark.gpu
def test_route_without_tokens(ctx):
    import torch
    d = capi.make_moe_route_desc(0, 10, 3)
    groups = torch.full((10, 2), 9, dtype=torch.int32, device="cuda")
    ctx.moe_route(d, None, None, None, None, groups, None)
    ctx.sync()
    assert (groups == 0).all()


def some_slots(rng, T, k, rows, missing=0.0):
    slots = rng.permutation(rows)[:T * k].reshape(T, k).astype(np.int32)
    slots[rng.random((T, k)) < missing] = -1
    return slots


def check_group(ctx, T, k, cols, fmt, dtype, src_grouped=False, pad=0, pitch=None, exponent=0, missing=0.2, offset=0, seed=0):
    import torch
    rng = np.random.default_rng(seed + T * k + cols)
    rows = -(-(T * k + 40) // 128) * 128 - 3  # the last slab need not be whole
    slots = some_slots(rng, T, k, rows, missing)
    if T > 1:
        slots[1, 0] = rows            # outside: skipped
        slots[0, -1] = -2 ** 31
    n = rows if src_grouped else T
    el = torch_dtype(dtype)
    flat = torch.full((n * (cols + pad) + offset + 8,), float("nan"), dtype=el, device="cuda")
    src = flat[offset:offset + n * (cols + pad)].view(n, cols + pad)
    src[:, :cols] = torch.from_numpy(rng.standard_normal((n, cols)) * np.exp(rng.standard_normal(cols)) * 2.0 ** exponent).to(el).cuda()
    d = capi.make_mx_group_desc(T, k, cols, rows, fmt, dtype, ld=(cols + pad) * src.element_size(), ld_packed=pitch, tensor_exponent=exponent,
                                src_grouped=src_grouped)
    packed = torch.full((rows, d.ld_packed), 0xA5, dtype=torch.uint8, device="cuda")
    tiles = torch.full((capi.mx_scale_bytes(rows, cols, fmt),), 0xA5, dtype=torch.uint8, device="cuda")
    dslots = torch.from_numpy(slots).cuda()
    ctx.mx_quantize_grouped(d, src, dslots, packed, tiles)
    ctx.sync()
    codes, byte = mx.quantize(src[:, :cols].double().cpu().numpy(), fmt, exponent)
    nb = mx.blocks_of(cols, fmt)
    want = np.full((rows, d.ld_packed), 0xA5, np.uint8)
    scales = np.full((rows, -(-nb // 4) * 4), 0xA5, np.uint8)
    for t in range(T):
        for r in slots[t]:
            if 0 <= r < rows:
                i = r if src_grouped else t
                want[r, :(cols + 1) // 2] = mx.pack(codes[i:i + 1], (cols + 1) // 2)[0]
                scales[r] = 0
                scales[r, :nb] = byte[i]
    np.testing.assert_array_equal(packed.cpu().numpy(), want)
    np.testing.assert_array_equal(mx.untile(tiles.cpu().numpy(), rows, scales.shape[1]), scales)
    return d, src, dslots, packed, tiles


@pytest.mark.gpu
@pytest.mark.parametrize("src_grouped", [False, True])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,cols", [(1, 1, 1), (1, 8, 2048), (48, 4, 2048), (3, 2, 15), (20, 3, 16), (65, 2, 33), (9, 16, 100), (40, 2, 257), (300, 1, 130),
                                      (130, 4, 1024), (700, 6, 1500)])
def test_group(ctx, T, k, cols, dtype, fmt, src_grouped):
    check_group(ctx, T, k, cols, fmt, dtype, src_grouped)


@pytest.mark.gpu
@pytest.mark.parametrize("src_grouped", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_group_strides(ctx, dtype, src_grouped):
    check_group(ctx, 50, 3, 500, capi.NVFP4, dtype, src_grouped, pad=3, exponent=-6, offset=1)
    check_group(ctx, 50, 3, 512, capi.MXFP4, dtype, src_grouped, pad=8, pitch=257)
    check_group(ctx, 50, 3, 512, capi.NVFP4, dtype, src_grouped, offset=3)


@pytest.mark.gpu
@pytest.mark.parametrize("src_grouped", [False, True])
@pytest.mark.parametrize("cols", [4096, 1100, 4100, 3001])
def test_group_wide(ctx, cols, src_grouped):
    """Enough rows for four segments at a time, with and without choices that are missing."""
    check_group(ctx, 4000 // (3 if src_grouped else 1), 3, cols, capi.NVFP4, capi.BF16, src_grouped, missing=0.0)
    check_group(ctx, 4000, 2, cols, capi.MXFP4, capi.F32, src_grouped, missing=0.5)


@pytest.mark.gpu
def test_group_same_row_twice(ctx):
    import torch
    d, src, slots, packed, tiles = check_group(ctx, 30, 4, 256, capi.NVFP4, capi.BF16, missing=0.0)
    want = packed.clone(), tiles.clone()
    slots[2:, 3] = slots[2:, 1]
    ctx.mx_quantize_grouped(d, src, slots, packed, tiles)
    ctx.sync()
    assert torch.equal(packed, want[0]) and torch.equal(tiles, want[1])


@pytest.mark.gpu
def test_group_nothing(ctx):
    for T, rows in ((0, 128), (4, 0)):
        ctx.mx_quantize_grouped(capi.make_mx_group_desc(T, 2, 64, rows, capi.NVFP4, capi.F32), None, None, None, None)
    ctx.sync()


def check_combine(ctx, T, k, cols, src_dtype, dst_dtype, pad=0, offset=0, missing=0.2, seed=0):
    import torch
    rng = np.random.default_rng(seed + T + cols)
    rows = T * k + 5
    slots = some_slots(rng, T, k, rows, missing)
    if T > 1:
        slots[0, 0], slots[1, -1] = rows, -7
    named = set(slots[(slots >= 0) & (slots < rows)].tolist())
    flat = torch.full((rows * (cols + pad) + offset + 8,), float("nan"), dtype=torch_dtype(src_dtype), device="cuda")
    src = flat[offset:offset + rows * (cols + pad)].view(rows, cols + pad)
    keep = torch.tensor(sorted(named), dtype=torch.int64, device="cuda")
    src[keep, :cols] = torch.from_numpy(rng.standard_normal((len(named), cols))).to(src.dtype).cuda()  # all other rows are NaN
    w = rng.random((T, k)).astype(np.float32)
    out = torch.full((T + 1, cols + pad), 7.0, dtype=torch_dtype(dst_dtype), device="cuda")
    d = capi.make_moe_combine_desc(T, k, cols, rows, src_dtype, dst_dtype, ld_src=(cols + pad) * src.element_size(), ld_dst=(cols + pad) * out.element_size())
    ctx.moe_combine(d, src, torch.from_numpy(slots).cuda(), torch.from_numpy(w).cuda(), out)
    ctx.sync()
    s = src[:, :cols].double().cpu().numpy()
    want, size = np.zeros((T, cols)), np.zeros((T, cols))
    for t in range(T):
        for j in range(k):
            if 0 <= slots[t, j] < rows:
                want[t] += w[t, j].astype(np.float64) * s[slots[t, j]]
                size[t] += np.abs(w[t, j].astype(np.float64) * s[slots[t, j]])
    got = out[:T, :cols].double().cpu().numpy()
    tol = k * 2.0 ** -24 * size  # a rounding per choice
    tol = tol + HALF_STEP[dst_dtype] * (np.abs(want) + tol) + (2.0 ** -25 if dst_dtype == capi.F16 else 0)
    assert (np.abs(got - want) <= tol).all()
    assert (out[T] == 7).all() and (out[:, cols:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("src_dtype", DTYPES)
@pytest.mark.parametrize("dst_dtype", DTYPES)
@pytest.mark.parametrize("T,k,cols", [(1, 1, 1), (1, 8, 2048), (3, 16, 9), (48, 4, 2048), (129, 5, 777), (600, 8, 1000), (2, 2, 7), (70, 9, 64)])
def test_combine(ctx, T, k, cols, src_dtype, dst_dtype):
    check_combine(ctx, T, k, cols, src_dtype, dst_dtype)
    check_combine(ctx, T, k, cols, src_dtype, dst_dtype, pad=3, offset=1)


@pytest.mark.gpu
def test_combine_nothing(ctx):
    import torch
    ctx.moe_combine(capi.make_moe_combine_desc(0, 2, 64, 10, capi.F32, capi.F32), None, None, None, None)
    out = torch.full((3, 64), 7.0, device="cuda")  # tokens without choices get zeros
    slots = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    ctx.moe_combine(capi.make_moe_combine_desc(3, 2, 64, 0, capi.F32, capi.F32), None, slots, torch.ones((3, 2), device="cuda"), out)
    ctx.sync()
    assert (out == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("call", ["route", "route workspace", "group", "combine"])
def test_calls_refuse(ctx, call):
    import torch
    x = torch.zeros(4096, device="cuda")
    i = torch.zeros(4096, dtype=torch.int32, device="cuda")
    with pytest.raises(capi.CuglError) as e:
        if call == "route":
            ctx.moe_route(capi.make_moe_route_desc(5, 8, 3), x, i, x, i, i[1:], x)
        elif call == "route workspace":
            ctx.moe_route(capi.make_moe_route_desc(500, 8, 3), x, i, x, i, i, x, workspace_bytes=100)
        elif call == "group":
            ctx.mx_quantize_grouped(capi.make_mx_group_desc(5, 3, 100, 128, capi.NVFP4, capi.F32), x, i, x, x[1:])
        else:
            ctx.moe_combine(capi.make_moe_combine_desc(5, 3, 100, 128, capi.F32, capi.F32), x, None, x, x)
    assert e.value.status == capi.INVALID_ARGUMENT
