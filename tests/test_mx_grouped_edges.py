"""Grouped products at the edges of their formula: gates far below zero.

Gates here are exact: K = 64 products of a row of equal values and weights whose sum is known, halves of whole numbers, which a float sum
holds exactly.  What is left is silu.  h = exp(g / 2) is off by two of its steps (2^-22 of it, or 2^-148 where it is subnormal), and counts
twice; with three products that is below 2^-20 of the result, plus 2^-147 / h.  16-bit results above -80 take 2^(-g log2 e) of a rounded
product: 2^-20 + 2^-23 |g|.  Half a step of the destination type on top, of its subnormal numbers too."""
import numpy as np
import pytest

import mx_helpers as mx
from computelibrary_b200 import capi
from test_mx_gemm import DTYPES, FORMATS, HALF_STEP, torch_dtype

FEW, MANY = 1, 10 ** 6  # expected rows that choose one kernel or the other
ONE = {mx.MXFP4: 127, mx.NVFP4: 0x38}  # the scale byte of 1
HALF_SUBNORMAL = {capi.F32: 2.0 ** -150, capi.F16: 2.0 ** -25, capi.BF16: 2.0 ** -134}


def whole(sums, K=64):
    """Codes [len(sums), K] of E2M1 values whose sum is the given one (a half of a whole number, up to 6 K)."""
    code = np.zeros((len(sums), K), np.uint8)
    for row, s in zip(code, sums):
        sign, left, at = 8 * (s < 0), abs(s), 0
        while left > 0:
            i = np.searchsorted(mx.GRID, left, side="right") - 1
            row[at], left, at = i | sign, left - mx.GRID[i], at + 1
    return code


def stored(code, fmt):
    """(packed, tiles) of codes with scales of 1."""
    import torch
    byte = np.full((code.shape[0], mx.blocks_of(code.shape[1], fmt)), ONE[fmt], np.uint8)
    return torch.from_numpy(mx.pack(code, capi.mx_pitch(code.shape[1]))).cuda(), torch.from_numpy(mx.tile(byte)).cuda()


GATES = np.concatenate([np.arange(-92, -85, 0.5), np.arange(-200, -92, 7.5), np.arange(-82, -77, 0.5), [-60, -30.5, -17, -1, 0, 0.5, 3, 40, 88, 92, 200]])


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("pad", [0, 1])
def test_gates_far_below_zero(ctx, fmt, dtype, expected, pad):
    """silu(g) is g exp(g) there: a normal number down to -91 in 32 bits, and a result of any size beside a large second product."""
    import torch
    N = 2 * len(GATES) // 8 * 8 + 8  # rows of dst at multiples of 16 bytes where pad is 0
    gates = np.resize(GATES, N)
    ups = np.where(np.arange(N) % 3 == 1, -1.0, 1.0)
    rows = np.array([1.0, 0.5, 1.5, 2.0, 1.0])[np.arange(200) % 5]  # factors of a row: its 64 values
    a = stored(np.repeat(np.searchsorted(mx.GRID, rows).astype(np.uint8)[:, None], 64, axis=1), fmt)
    b, up = stored(whole(gates), fmt), stored(whole(ups), fmt)
    groups = torch.tensor([[0, 200]], dtype=torch.int32, device="cuda")
    g = rows[:, None] * gates
    for up_alpha in (1.0, 2.0 ** 60, 2.0 ** 120):
        out = torch.full((200, N + pad), 7.0, dtype=torch_dtype(dtype), device="cuda")
        d = capi.make_mx_grouped_gemm_desc(1, 200, N, 64, fmt, dtype, expected_rows=expected, swiglu=True, up_alpha=up_alpha,
                                           ldd=out.stride(0) * out.element_size())
        ctx.mx_grouped_gemm(d, *a, groups, b, out, up=up)
        ctx.sync()
        u = rows[:, None] * ups * up_alpha
        want = g / (1 + np.exp(-g)) * u
        rel = 2.0 ** -20 + np.where(g < -80, 2.0 ** -147 / np.exp(g / 2), 0 if dtype == capi.F32 else 2.0 ** -23 * np.abs(g))
        tol = rel * np.abs(want)
        tol = tol + HALF_STEP[dtype] * (np.abs(want) + tol) + HALF_SUBNORMAL[dtype] + 2.0 ** -149
        got = out[:, :N].double().cpu().numpy()
        if dtype == capi.F16:  # what lies beyond the type is infinite
            beyond = np.abs(want) >= 65520 + tol
            assert (got[beyond] == np.sign(want[beyond]) * np.inf).all()
            got, want, tol = (np.where(beyond, 0, v) for v in (got, want, tol))
        else:
            beyond = np.abs(want) >= 2.0 ** 128
            got, want, tol = (np.where(beyond, 0, v) for v in (got, want, tol))
        bad = ~(np.abs(got - want) <= tol)
        assert not bad.any(), f"{bad.sum()} of {bad.size} off at gates {np.unique(g[bad])[:8]}: {got[bad][:3]} for {want[bad][:3]}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("swiglu", [False, True])
def test_bits_depend_on_the_values_alone(ctx, fmt, swiglu, dtype):
    """expected_rows and the alignment of dst choose kernels and stores, never a result."""
    import torch
    from test_mx_grouped import check
    counts = [300, 64, 5, 900, 0, 128]
    want, args, _ = check(ctx, counts, 640, 768, fmt, dtype, swiglu, factors=True, expected=FEW)
    for expected in (FEW, 500, MANY):
        for pad in (0, 1, 2):
            out, _, _ = check(ctx, counts, 640, 768, fmt, dtype, swiglu, factors=True, expected=expected, pad=pad)
            for start, count in args[3].tolist():
                assert torch.equal(out[start:start + count, :640], want[start:start + count])


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
def test_a_bad_group_does_not_hide_a_wait_that_ran_out(ctx, expected):
    """Both in one launch: the sync says that results are invalid, and names the group too; the next call is as always."""
    import torch
    from test_mx_grouped import check
    out, args, kw = check(ctx, [300, 0, 5, 900], 640, 2048, capi.NVFP4, capi.F32, expected=expected)
    want, groups = out.clone(), args[3]
    groups[1] = torch.tensor([64, 10], dtype=torch.int32, device="cuda")
    ctx.set_wait_limit_us(20000)
    try:
        ctx.withhold_copy_once(1)
        ctx.mx_grouped_gemm(*args, **kw)
        with pytest.raises(capi.CuglError) as e:
            ctx.sync()
    finally:
        ctx.set_wait_limit_us(0)
    assert e.value.status == capi.RUNTIME_ERROR
    assert "wait ran out" in e.value.message and "invalid" in e.value.message and "group" in e.value.message
    ctx.mx_grouped_gemm(*args, **kw)  # each is forgotten by itself
    with pytest.raises(capi.CuglError) as e:
        ctx.sync()
    assert "group" in e.value.message and "wait ran out" not in e.value.message
    groups[1] = 0
    out.fill_(7)
    ctx.mx_grouped_gemm(*args, **kw)
    ctx.sync()
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("expected", [FEW, MANY])
def test_a_bad_group_does_not_hide_an_earlier_or_later_wait(ctx, expected):
    import torch
    from test_mx_grouped import check
    _, args, kw = check(ctx, [300, 0, 5, 900], 640, 2048, capi.NVFP4, capi.F32, expected=expected)
    bad = (*args[:3], args[3].clone(), *args[4:])
    bad[3][1] = torch.tensor([64, 10], dtype=torch.int32, device="cuda")
    for order in ((args, bad), (bad, args)):
        ctx.set_wait_limit_us(20000)
        try:
            for a in order:
                if a is args:
                    ctx.withhold_copy_once(1)
                ctx.mx_grouped_gemm(*a, **kw)
            with pytest.raises(capi.CuglError) as e:
                ctx.sync()
        finally:
            ctx.set_wait_limit_us(0)
        assert "wait ran out" in e.value.message and "group" in e.value.message
        ctx.sync()
