"""Products of groups of microscaled rows against sums in 64 bits.

Tolerance of a sum as for the plain product: ceil(K / 64) + 10 steps of 2^-23 of its magnitudes (its MMAs, the factors, one fused
multiply-add).  SwiGLU: the slope of silu is below 1.1; the exponential, the division and the products are off by 2^-20 of the result
at most; 16-bit results take 2^(-g log2 e) of a product that is off by two half steps (the constant's and its own), 2^-23 |g| log2 e, which
makes 2^-23 |g| of the exponential.  Half a step of the destination type on top."""
import ctypes as C

import numpy as np
import pytest

import mx_helpers as mx
from computelibrary_b200 import capi
from test_mx_gemm import DTYPES, FORMATS, HALF_STEP, torch_dtype


# ---- without a GPU ----------------------------------------------------------------------------------------
def test_descriptor_layout():
    assert C.sizeof(capi.MxGroupedGemmDesc) == 9 * 4 + 8 + 4 + 24 and capi.MxGroupedGemmDesc.alpha.offset == 36
    assert capi.MxGroupedGemmDesc.lda.offset == 48


@pytest.mark.parametrize("groups,rows,want", [(1, 1, 128), (4, 0, 0), (4, 2, 256), (64, 192, 8320), (3, 128, 384), (2, 129, 256),
                                              (2, 130, 384), (1, 128, 128), (8, 10 ** 9, (10 ** 9 + 127 * 8) // 128 * 128), (0, 5, 0), (-1, 5, 0), (5, -1, 0)])
def test_group_rows(groups, rows, want):
    assert capi.mx_group_rows(groups, rows) == want


@pytest.mark.parametrize("groups,rows", [(1, 1), (2, 129), (2, 130), (3, 5), (5, 700), (7, 3)])
def test_group_rows_hold_every_split(groups, rows):
    rng = np.random.default_rng(groups)
    for _ in range(200):
        counts = np.bincount(rng.integers(0, groups, rows), minlength=groups)
        assert sum(-(-c // 128) * 128 for c in counts) <= capi.mx_group_rows(groups, rows)


@pytest.mark.parametrize("change,word", [
    (dict(groups=0), "groups"), (dict(groups=513), "groups"), (dict(rows=-1), "rows"), (dict(N=0), "N"), (dict(K=0), "K"),
    (dict(K=2 ** 31 - 1), "too large"), (dict(expected_rows=-1), "expected_rows"), (dict(format=2), "format"), (dict(dst_dtype=capi.S32), "dst_dtype"),
    (dict(swiglu=1, has_bias=1), "bias"), (dict(lda=32), "lda"), (dict(lda=56), "lda"), (dict(ldb=72), "lda"), (dict(ldb=2 ** 40), "2^40"),
    (dict(ldd=198), "ldd"), (dict(ldd=201), "ldd"), (dict(ldd=2 ** 40), "2^40"), (dict(alpha=float("inf")), "alpha"), (dict(up_alpha=float("nan")), "alpha"),
    (dict(groups=512, N=2 ** 22, ldd=2 ** 24), "scale tiles"), (dict(rows=2 ** 31 - 2 ** 11, N=2 ** 15, ldd=2 ** 17), "output tiles")])
def test_validate_refuses(change, word):
    d = capi.make_mx_grouped_gemm_desc(4, 512, 100, 100, capi.NVFP4, capi.BF16)
    assert capi.mx_grouped_gemm_validate(d)[0] == 0
    for k, v in change.items():
        setattr(d, k, v)
    st, why = capi.mx_grouped_gemm_validate(d)
    assert st == capi.INVALID_ARGUMENT and word in why


def test_null_context_is_refused():
    d = capi.make_mx_grouped_gemm_desc(4, 512, 100, 100, capi.NVFP4, capi.BF16)
    assert capi.load_library().cugl_mx_grouped_gemm(None, C.byref(d), *[None] * 11) == capi.INVALID_ARGUMENT


# ---- on the GPU -------------------------------------------------------------------------------------------
FEW, MANY = 1, 10 ** 6  # expected rows that choose one kernel or the other


def operand(rng, rows, cols, fmt, pitch=None, valid=None, matrices=1):
    """`matrices` matrices one behind the other: every code, scales that differ from block to block, NaN scales behind the last row
    and in rows that are not valid; (packed, tiles, values [matrices * rows, cols])."""
    import torch
    pitch = capi.mx_pitch(cols) if pitch is None else pitch
    nb, nan = mx.blocks_of(cols, fmt), 255 if fmt == mx.MXFP4 else 127
    code = rng.integers(0, 16, (matrices * rows, cols)).astype(np.uint8)
    byte = (rng.integers(121, 133, (matrices * rows, nb)) if fmt == mx.MXFP4 else rng.integers(1, 127, (matrices * rows, nb))).astype(np.uint8)
    values = mx.values(code, byte, fmt)
    if valid is not None:
        byte[~valid] = nan
    packed = mx.pack(code, pitch)
    packed[:, (cols + 1) // 2:] = 0xFF  # bytes between rows belong to nobody
    tiles = np.concatenate([mx.tile(byte[i * rows:(i + 1) * rows], fill=nan) for i in range(matrices)])
    return torch.from_numpy(packed).cuda(), torch.from_numpy(tiles).cuda(), values


def layout(counts, gap=0):
    """(groups [E, 2], rows): groups one behind the other, `gap` empty slabs between them."""
    groups, at = [], 0
    for c in counts:
        groups.append((at, c))
        at += -(-c // 128) * 128 + gap * 128
    return np.array(groups, np.int32), max(at, 128)


def check(ctx, counts, N, K, fmt, dtype, swiglu=False, bias=False, factors=False, expected=FEW, pad=0, lda=None, ldb=None, gap=0, seed=0, shuffle=False,
          alpha=1.0, cut=0):
    import torch
    E = len(counts)
    rng = np.random.default_rng(seed + 3 * sum(counts) + 13 * N + K)
    groups, rows = layout(counts, gap)
    rows -= cut  # the last slab need not be whole
    if shuffle:  # experts need not lie in order
        order = rng.permutation(E)
        groups = groups[order]
        counts = [counts[i] for i in order]
    valid = np.zeros(rows, bool)
    for start, count in groups:
        valid[start:start + count] = True
    a, sa, va = operand(rng, rows, K, fmt, lda, valid)
    weights = [operand(rng, N, K, fmt, ldb, matrices=E) for _ in range(2 if swiglu else 1)]
    vf = [rng.uniform(0.5, 2.0, E).astype(np.float32) if factors else None for _ in weights]
    vbias = (rng.standard_normal((E, N)) * 100).astype(np.float32) if bias else None
    alphas = [alpha, 1.0]
    spread = np.sqrt(K) * np.abs(va).mean() * np.abs(weights[0][2]).mean()
    if swiglu:  # the gate's values of size 1, the result's of size 1
        alphas = [alpha / spread, 1.0 / spread]
    elif dtype == capi.F16:  # keep within its range
        alphas[0] = alpha * 2.0 ** -float(np.ceil(np.log2(max(1.0, 8 * spread / 30000))))
    out = torch.full((rows, N + pad), 7.0, dtype=torch_dtype(dtype), device="cuda")
    d = capi.make_mx_grouped_gemm_desc(E, rows, N, K, fmt, dtype, expected_rows=expected, swiglu=swiglu, has_bias=bias, alpha=alphas[0], up_alpha=alphas[1],
                                       lda=lda, ldb=ldb, ldd=out.stride(0) * out.element_size())
    alphas = [d.alpha, d.up_alpha]  # as 32-bit numbers
    gw = [(w[0], w[1], torch.from_numpy(f).cuda() if factors else None) for w, f in zip(weights, vf)]
    dbias = torch.from_numpy(vbias).cuda() if bias else None
    args = (d, a, sa, torch.from_numpy(groups).cuda(), gw[0], out)
    kw = dict(up=gw[1] if swiglu else None, bias=dbias)
    ctx.mx_grouped_gemm(*args, **kw)
    ctx.sync()
    got = out[:, :N].double().cpu().numpy()
    steps = (-(-K // 64) + 10) * 2.0 ** -23
    for e, (start, count) in enumerate(groups):
        if count == 0:
            continue
        x = va[start:start + count]
        sums, sizes = [], []
        for w, f, al in zip(weights, vf, alphas):
            scale = al * (float(f[e]) if factors else 1.0)
            m = w[2][e * N:(e + 1) * N]
            sums.append(scale * (x @ m.T))
            sizes.append(abs(scale) * (np.abs(x) @ np.abs(m).T))
        if swiglu:
            g, u = sums
            eg, eu = steps * sizes[0], steps * sizes[1]
            with np.errstate(over="ignore"):
                silu = g / (1 + np.exp(-g))
            want = silu * u
            rel = 2.0 ** -20 + (2.0 ** -23 * np.abs(g) if dtype != capi.F32 else 0)
            tol = (1.1 * eg + rel * np.abs(silu)) * (np.abs(u) + eu) + np.abs(silu) * eu
        else:
            want = sums[0] + (vbias[e].astype(np.float64) if bias else 0)
            tol = steps * (sizes[0] + (np.abs(vbias[e]) if bias else 0))
        tol = tol + HALF_STEP[dtype] * (np.abs(want) + tol) + (2.0 ** -25 if dtype == capi.F16 else 0)
        mine = got[start:start + count]
        if dtype == capi.F16:  # values from 65520 (halfway between the largest, 65504, and the next one up, 65536) are infinite
            beyond = np.abs(want) - tol >= 65520
            assert (mine[beyond] == np.sign(want[beyond]) * np.inf).all()
            near = (np.abs(want) + tol >= 65520) & ~beyond & np.isinf(mine)  # either is right
            mine, want = np.where(beyond | near, 0, mine), np.where(beyond | near, 0, want)
        assert np.isfinite(mine).all()
        bad = np.abs(mine - want) > tol
        assert not bad.any(), f"group {e}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[:3].tolist()}: {mine[bad][:3]} for {want[bad][:3]}"
    full = out.double().cpu().numpy()
    assert (full[~valid] == 7).all() and (full[:, N:] == 7).all()  # rows of no group are left as they were
    return out, args, kw


COUNTS = [[1], [16, 0, 17], [0, 5, 128, 129, 0], [127, 31, 33, 64, 65, 96, 97], [300, 1, 256, 257, 0, 128, 511]]


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("counts", COUNTS, ids=len)
def test_counts(ctx, counts, fmt, swiglu, expected):
    check(ctx, counts, 256, 512, fmt, capi.BF16, swiglu, expected=expected)
    check(ctx, counts, 200, 320, fmt, capi.F32, swiglu, factors=True, expected=expected, gap=1, shuffle=True)


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("K", [1, 2, 15, 33, 64, 65, 127, 192, 255, 256, 257, 530, 1000, 2050])
def test_k(ctx, fmt, K, expected):
    check(ctx, [3, 40, 0, 200], 136, K, fmt, capi.F32, bias=True, expected=expected)
    check(ctx, [3, 40, 0, 200], 136, K, fmt, capi.F16, swiglu=True, expected=expected)


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 2, 7, 8, 31, 127, 128, 129, 255, 257, 384, 1001, 1288])
def test_channels(ctx, dtype, N, expected):
    check(ctx, [7, 0, 290], N, 256, capi.NVFP4, dtype, bias=True, factors=True, expected=expected)
    check(ctx, [7, 0, 290], N, 256, capi.MXFP4, dtype, swiglu=True, expected=expected, pad=3)


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
def test_strides(ctx, expected):
    check(ctx, [50, 140], 264, 300, capi.NVFP4, capi.BF16, expected=expected, pad=8, lda=160 + 32, ldb=160 + 64)
    check(ctx, [50, 140], 264, 300, capi.MXFP4, capi.F32, swiglu=True, expected=expected, pad=1, lda=160 + 32, ldb=160 + 64)
    check(ctx, [50, 140], 264, 300, capi.MXFP4, capi.BF16, expected=expected, cut=100)  # a last slab of 28 rows
    check(ctx, [500] * 3, 264, 300, capi.MXFP4, capi.F16, swiglu=True, factors=True, expected=expected, cut=10, alpha=-3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
@pytest.mark.parametrize("fmt", FORMATS)
def test_many_groups(ctx, fmt, expected):
    """More items than SMs, tiles of all sizes in turn, groups without rows."""
    rng = np.random.default_rng(5)
    counts = [int(c) for c in rng.choice([0, 1, 2, 9, 30, 64, 70, 128, 150, 400], 96)]
    check(ctx, counts, 384, 512, fmt, capi.BF16, swiglu=True, expected=expected)
    check(ctx, counts, 384, 512, fmt, capi.BF16, expected=expected)
    check(ctx, counts, 250, 130, fmt, capi.F32, swiglu=True, factors=True, expected=expected)
    check(ctx, [1, 0] * 256, 128, 64, fmt, capi.F32, bias=True, expected=expected)


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
def test_saturated_gate(ctx, expected):
    """Gates far from zero on both sides: silu is the identity or nothing."""
    check(ctx, [20, 130], 256, 256, capi.NVFP4, capi.F32, swiglu=True, expected=expected, alpha=300.0)


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
@pytest.mark.parametrize("swiglu", [False, True])
def test_nothing_to_do(ctx, expected, swiglu):
    check(ctx, [0, 0, 0], 256, 256, capi.NVFP4, capi.BF16, swiglu=swiglu, expected=expected)


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
@pytest.mark.parametrize("swiglu", [False, True])
def test_equal_calls_give_equal_bits(ctx, expected, swiglu):
    out, args, kw = check(ctx, [300, 64, 5, 900, 0, 128], 640, 768, capi.NVFP4, capi.F32, swiglu=swiglu, expected=expected)
    want = out.clone()
    for _ in range(3):
        out.fill_(7)
        ctx.mx_grouped_gemm(*args, **kw)
        ctx.sync()
        assert bool((out == want).all())


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
@pytest.mark.parametrize("group", [(64, 10), (-128, 10), (0, -5), (128, 1000), (2 ** 30, 4), (0, 2 ** 31 - 1), (1024, 1)])
def test_groups_outside_are_left_out(ctx, group, expected):
    """A group that the rows do not hold counts as empty and is reported; the others are computed."""
    import torch
    out, args, kw = check(ctx, [30, 0, 400], 264, 256, capi.NVFP4, capi.F32, expected=expected)
    want, groups = out.clone(), args[3]
    good = groups.clone()
    groups[1] = torch.tensor(group, dtype=torch.int32, device="cuda")
    out.fill_(7)
    ctx.mx_grouped_gemm(*args, **kw)
    with pytest.raises(capi.CuglError) as e:
        ctx.sync()
    assert e.value.status == capi.RUNTIME_ERROR and "group" in e.value.message
    assert torch.equal(out, want)
    groups.copy_(good)
    ctx.mx_grouped_gemm(*args, **kw)
    ctx.sync()
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
def test_groups_that_overlap(ctx, expected):
    """512 groups of the same 512 rows have more tiles than the rows.  Nothing is computed, the next sync reports it, and the call after
    that is as ever."""
    import torch
    rng = np.random.default_rng(5)
    E, N, K, rows = 512, 8, 64, 512
    a, sa, _ = operand(rng, rows, K, capi.NVFP4)
    b, sb, _ = operand(rng, N, K, capi.NVFP4, matrices=E)
    groups = torch.zeros((E, 2), dtype=torch.int32, device="cuda")
    groups[:, 1] = rows
    out = torch.full((rows, N), 7.0, device="cuda")
    d = capi.make_mx_grouped_gemm_desc(E, rows, N, K, capi.NVFP4, capi.F32, expected_rows=expected)
    ctx.mx_grouped_gemm(d, a, sa, groups, (b, sb, None), out)
    with pytest.raises(capi.CuglError) as e:
        ctx.sync()
    assert e.value.status == capi.RUNTIME_ERROR and "overlap" in e.value.message
    assert bool((out == 7).all())
    groups[1:] = 0
    groups[0, 1] = rows
    ctx.mx_grouped_gemm(d, a, sa, groups, (b, sb, None), out)
    ctx.sync()
    assert bool((out != 7).any())


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("k_block", [0, 3, 7])
def test_wait_limit(ctx, expected, swiglu, k_block):
    """Operand copies that never come: the call ends by its wait limit and says so; the next one is as always."""
    import torch
    out, args, kw = check(ctx, [300, 64, 5, 900, 0, 128], 640, 2048, capi.NVFP4, capi.F32, swiglu=swiglu, expected=expected)
    want = out.clone()
    ctx.set_wait_limit_us(20000)
    try:
        ctx.withhold_copy_once(k_block)
        ctx.mx_grouped_gemm(*args, **kw)
        with pytest.raises(capi.CuglError) as e:
            ctx.sync()
        assert e.value.status == capi.RUNTIME_ERROR and "wait ran out" in e.value.message
    finally:
        ctx.set_wait_limit_us(0)
    out.fill_(7)
    ctx.mx_grouped_gemm(*args, **kw)
    ctx.sync()
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("expected,count", [(FEW, 40), (FEW, 100), (MANY, 512)])
def test_gives_up_in_flight(ctx, fmt, swiglu, expected, count):
    """A limit far below the time of a tile: the kernel gives up with copies and MMAs under way."""
    import torch
    from test_mx_give_up import check as give_up, packed
    N, K = 512, 2 ** 21
    g = torch.Generator(device="cuda").manual_seed(count)
    a, b, up = packed(g, 512, K, fmt), packed(g, N, K, fmt), packed(g, N, K, fmt)
    groups = torch.tensor([[0, count]], dtype=torch.int32, device="cuda")
    out = torch.zeros((512, N), dtype=torch.float32, device="cuda")
    d = capi.make_mx_grouped_gemm_desc(1, 512, N, K, fmt, capi.F32, expected_rows=expected, swiglu=swiglu, alpha=2.0 ** -20, up_alpha=2.0 ** -20)
    give_up(ctx, lambda: ctx.mx_grouped_gemm(d, *a, groups, b, out, up=up if swiglu else None), out)


@pytest.mark.gpu
@pytest.mark.parametrize("change,word", [
    ("a", "16-byte"), ("groups", "8-byte"), ("dst", "aligned"), ("bias", "has_bias"), ("up", "swiglu"), ("null", "NULL")])
def test_call_refuses(ctx, change, word):
    import torch
    a = torch.zeros(512 * 64 + 16, dtype=torch.uint8, device="cuda")
    sf = torch.zeros(8192, dtype=torch.uint8, device="cuda")
    groups = torch.zeros(9, dtype=torch.int32, device="cuda")
    out = torch.zeros(512 * 100 + 2, dtype=torch.bfloat16, device="cuda")
    d = capi.make_mx_grouped_gemm_desc(4, 512, 100, 100, capi.NVFP4, capi.BF16)
    bias = torch.zeros(400, device="cuda") if change == "bias" else None
    up = (a, sf) if change == "up" else None
    with pytest.raises(capi.CuglError) as e:
        ctx.mx_grouped_gemm(d, a[1:] if change == "a" else a, sf, groups[1:] if change == "groups" else groups, (a, None if change == "null" else sf),
                            out.view(torch.uint8)[1:] if change == "dst" else out, up=up, bias=bias)
    assert e.value.status == capi.INVALID_ARGUMENT and word in e.value.message
