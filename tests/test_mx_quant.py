"""Quantisation to microscaled 4-bit floating point, the way back, and the order of scales: against the definition in 64 bits,
bit for bit (a code is a decision, a value read back has at most six significant bits)."""
import ctypes as C

import numpy as np
import pytest

import mx_helpers as mx
from computelibrary_b200 import capi

FORMATS = [capi.MXFP4, capi.NVFP4]
DTYPES = [capi.F32, capi.F16, capi.BF16]


def torch_dtype(dtype):
    import torch
    return {capi.F32: torch.float32, capi.F16: torch.float16, capi.BF16: torch.bfloat16}[dtype]


# ---- without a GPU ----------------------------------------------------------------------------------------
def test_descriptor_layout():
    assert C.sizeof(capi.MxDesc) == 16 + 16 + 8 and capi.MxDesc.tensor_exponent.offset == 32


def test_scale_bytes():
    assert capi.mx_scale_bytes(1, 1, capi.MXFP4) == 512
    assert capi.mx_scale_bytes(128, 128, capi.MXFP4) == 512
    assert capi.mx_scale_bytes(129, 129, capi.MXFP4) == 4 * 512
    assert capi.mx_scale_bytes(128, 65, capi.NVFP4) == 2 * 512
    assert capi.mx_scale_bytes(0, 64, capi.NVFP4) == 0
    assert capi.mx_scale_bytes(2 ** 31 - 1, 2 ** 30, capi.NVFP4) == 2 ** 24 * 2 ** 24 * 512  # beyond 32 bits
    assert capi.mx_scale_bytes(-1, 64, capi.NVFP4) == capi.mx_scale_bytes(1, 0, capi.NVFP4) == capi.mx_scale_bytes(1, 1, 2) == 0


@pytest.mark.parametrize("change,word", [
    (dict(rows=-1), "rows"), (dict(cols=0), "rows"), (dict(cols=2 ** 31 - 1), "too large"), (dict(format=2), "format"),
    (dict(dtype=capi.S8), "dtype"), (dict(dtype=capi.U8), "dtype"), (dict(ld=199), "ld"), (dict(ld=201), "ld"),
    (dict(ld_packed=49), "ld_packed"), (dict(tensor_exponent=1), "tensor_exponent"),
    (dict(format=capi.NVFP4, tensor_exponent=65), "-64"), (dict(format=capi.NVFP4, tensor_exponent=-65), "-64")])
def test_validate_refuses(change, word):
    d = capi.make_mx_desc(3, 100, capi.MXFP4, capi.BF16)
    assert capi.mx_validate(d)[0] == 0
    for k, v in change.items():
        setattr(d, k, v)
    st, why = capi.mx_validate(d)
    assert st == capi.INVALID_ARGUMENT and word in why


def test_null_context_is_refused():
    lib, d = capi.load_library(), capi.make_mx_desc(3, 100, capi.MXFP4, capi.BF16)
    assert lib.cugl_mx_quantize(None, C.byref(d), None, None, None) == capi.INVALID_ARGUMENT
    assert lib.cugl_mx_dequantize(None, C.byref(d), None, None, None) == capi.INVALID_ARGUMENT
    assert lib.cugl_mx_tile_scales(None, None, 4, 3, 100, capi.MXFP4, None) == capi.INVALID_ARGUMENT
    assert lib.cugl_mx_validate(None, None) == capi.INVALID_ARGUMENT


def test_reference_scales_are_e4m3():
    # every positive E4M3 value is its own scale and byte; the reference helper against the type's definition
    byte = np.arange(1, 127, dtype=np.uint8)
    v = mx.values(np.full((126, 1), 2, np.uint8), byte[:, None], mx.NVFP4)[:, 0]
    assert v[-1] == 448 and v[0] == 2.0 ** -9 and (np.diff(v) > 0).all()
    b, s = mx.scale_of(6 * v, mx.NVFP4)
    assert np.array_equal(b, byte) and np.array_equal(s, v)


# ---- on the GPU -------------------------------------------------------------------------------------------
class Stored:
    """Packed codes and tiles on the device, with guards around what belongs to the matrix."""

    def __init__(self, rows, cols, fmt, pitch=None):
        import torch
        self.rows, self.cols, self.fmt = rows, cols, fmt
        self.pitch = capi.mx_pitch(cols) if pitch is None else pitch
        self.raw = torch.full((rows * self.pitch + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        self.scales = torch.full((capi.mx_scale_bytes(rows, cols, fmt) + 64,), 0xA5, dtype=torch.uint8, device="cuda")

    def codes(self):
        return mx.unpack(self.raw[:self.rows * self.pitch].cpu().numpy().reshape(self.rows, self.pitch), self.cols)

    def bytes(self):
        return mx.untile(self.scales.cpu().numpy(), self.rows, mx.blocks_of(self.cols, self.fmt))

    def untouched(self):
        raw = self.raw.cpu().numpy()
        body = raw[:self.rows * self.pitch].reshape(self.rows, self.pitch)
        used = (self.cols + 1) // 2
        assert (raw[self.rows * self.pitch:] == 0xA5).all() and (body[:, used:] == 0xA5).all()
        if self.cols % 2:
            assert (body[:, used - 1] >> 4 == 0).all()  # the half byte behind an odd row
        nb = mx.blocks_of(self.cols, self.fmt)
        flat = self.scales.cpu().numpy()
        want = mx.tile(mx.untile(flat, self.rows, nb), fill=0xA5)  # zero behind each row, rows behind left alone
        assert np.array_equal(flat[:want.size], want) and (flat[want.size:] == 0xA5).all()


def same_values(got, want):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])


def round_trip(ctx, x, fmt, exponent=0, pitch=None):
    import torch
    rows, cols = x.shape
    dtype = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}[x.dtype]
    q = Stored(rows, cols, fmt, pitch)
    d = capi.make_mx_desc(rows, cols, fmt, dtype, ld=x.stride(0) * x.element_size() if rows > 1 else None,
                          ld_packed=q.pitch, tensor_exponent=exponent)
    ctx.mx_quantize(d, x, q.raw, q.scales)
    code, byte = mx.quantize(x.double().cpu().numpy(), fmt, exponent)
    fine = np.repeat(byte != (255 if fmt == capi.MXFP4 else 127), mx.block_of(fmt), axis=1)[:, :cols]
    assert np.array_equal(q.bytes(), byte)
    got = q.codes()
    zero = (got & 7 == 0) & (code & 7 == 0)  # a zero's sign says nothing
    assert np.array_equal(np.where(zero | ~fine, 0, got), np.where(zero | ~fine, 0, code))
    q.untouched()
    for out in DTYPES:
        y = torch.full((rows, cols + 3), 7.0, dtype=torch_dtype(out), device="cuda")
        ctx.mx_dequantize(capi.make_mx_desc(rows, cols, fmt, out, ld=y.stride(0) * y.element_size(), ld_packed=q.pitch,
                                            tensor_exponent=exponent), q.raw, q.scales, y)
        want = torch.from_numpy(mx.values(code, byte, fmt, exponent)).to(torch_dtype(out)).double().numpy()
        same_values(y[:, :cols].double().cpu().numpy(), want)
        assert (y[:, cols:] == 7).all()
    return q


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (1, 33), (3, 15), (2, 64), (5, 100), (129, 128), (130, 513), (7, 4096), (300, 1025)])
def test_round_trip(ctx, fmt, dtype, rows, cols):
    import torch
    g = torch.Generator().manual_seed(rows * 131 + cols)
    x = torch.randn((rows, cols), generator=g) * torch.exp(2 * torch.randn((rows, 1), generator=g))
    round_trip(ctx, x.to(torch_dtype(dtype)).cuda(), fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_scale_and_midpoint(ctx, fmt, dtype):
    """Rows whose first value sets the scale and whose others are the midpoints of E2M1 at that scale and their neighbours in
    the source's type."""
    import torch
    bits = {capi.F32: 23, capi.F16: 10, capi.BF16: 7}[dtype]
    tops = [6 * 2.0 ** e * (1 + m / 8) for e in range(-3, 4) for m in range(8)]
    rows = []
    for top in tops:
        top = float(torch.tensor(top).to(torch_dtype(dtype)))
        s = mx.scale_of([top], fmt)[1][0]
        near = [m * s * (1 + k * 2.0 ** -bits) for m in mx.MIDPOINTS for k in (-1, -.5, 0, .5, 1)]
        for i in range(0, len(near), 15):
            rows.append([top] + near[i:i + 15] + [0.0] * (15 - len(near[i:i + 15])) + ([0.0] * 16 if fmt == capi.MXFP4 else []))
    round_trip(ctx, torch.tensor(rows, dtype=torch.float64).to(torch_dtype(dtype)).cuda(), fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [capi.F16, capi.BF16])
@pytest.mark.parametrize("fmt", FORMATS)
def test_every_value_of_a_16_bit_type(ctx, fmt, dtype):
    """All 65536 bit patterns, NaNs and infinities among them, each in the company of a value of its own size and of others."""
    import torch
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch_dtype(dtype))
    round_trip(ctx, x.view(1024, 64).cuda(), fmt)
    round_trip(ctx, x[torch.randperm(65536, generator=torch.Generator().manual_seed(3))].view(512, 128).cuda(), fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_32_bit_corners(ctx, fmt):
    """Zeros of both signs, subnormals, the largest values, NaN and infinities of either sign in every place of a block."""
    import torch
    block = mx.block_of(fmt)
    tiny, big = 2.0 ** -149, torch.finfo(torch.float32).max
    rows = torch.zeros((24, 3 * block))
    rows[1] = -0.0
    rows[2], rows[3], rows[4] = tiny, -2.0 ** -127, 2.0 ** -126
    rows[5, ::3], rows[6, 1::2] = big, -big
    rows[7, 4], rows[8, block], rows[9, 3 * block - 1] = float("nan"), float("inf"), -float("inf")
    rows[10, :block], rows[11] = float("inf"), float("nan")
    rows[12, 5], rows[12, 6] = float("inf"), float("nan")
    g = torch.Generator().manual_seed(1)
    rows[13:] = torch.randn((11, 3 * block), generator=g) * torch.ldexp(torch.ones(11, 1), torch.arange(-140, 101, 24)[:11, None])
    round_trip(ctx, rows.cuda(), fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols,exponent", [(96, 0), (2048, 0), (77, 0), (96, -5), (1030, 7)])
def test_signs_of_zeros(ctx, fmt, dtype, cols, exponent):
    """A zero, or a value that rounds to it, keeps its sign in its code and on the way back, whatever type it comes from: codes bit for
    bit in every finite block."""
    import torch
    exponent = exponent if fmt == capi.NVFP4 else 0
    g = torch.Generator().manual_seed(cols)
    x = torch.randn((40, cols), generator=g)
    x[torch.rand((40, cols), generator=g) < 0.3] *= 1e-3
    x[torch.rand((40, cols), generator=g) < 0.3] *= 0.0
    x[1], x[2], x[3, ::2] = 0.0, -0.0, -0.0
    x = (x * 2.0 ** exponent).to(torch_dtype(dtype)).cuda()
    assert (torch.signbit(x) & (x == 0)).any()
    q = Stored(40, cols, fmt)
    d = capi.make_mx_desc(40, cols, fmt, dtype, tensor_exponent=exponent)
    ctx.mx_quantize(d, x, q.raw, q.scales)
    code, byte = mx.quantize(x.double().cpu().numpy(), fmt, exponent)
    assert np.array_equal(q.bytes(), byte) and np.array_equal(q.codes(), code)
    y = torch.full_like(x, 7.0)
    ctx.mx_dequantize(d, q.raw, q.scales, y)
    assert torch.equal(torch.signbit(y), torch.signbit(x))


@pytest.mark.gpu
@pytest.mark.parametrize("exponent", [-64, -6, 3, 64])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tensor_exponent(ctx, dtype, exponent):
    import torch
    g = torch.Generator().manual_seed(5)
    size = exponent if dtype != capi.F16 else max(-10, min(10, exponent))  # f16 does not reach 2^64: all saturates or vanishes
    x = torch.randn((9, 200), generator=g) * 2.0 ** size
    round_trip(ctx, x.to(torch_dtype(dtype)).cuda(), capi.NVFP4, exponent)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("offset,extra,pitch_extra", [(0, 8, 16), (1, 3, 1), (3, 5, 7), (4, 4, 8)])
def test_strides_and_alignment(ctx, fmt, offset, extra, pitch_extra):
    """Plain rows that start anywhere, packed rows at any pitch; bytes between rows stay as they are."""
    import torch
    for dtype in DTYPES:
        g = torch.Generator().manual_seed(offset)
        whole = torch.randn((6, 90 + extra + offset), generator=g).to(torch_dtype(dtype)).cuda()
        round_trip(ctx, whole[:, offset:offset + 90], fmt, pitch=capi.mx_pitch(90) + pitch_extra)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [4097, 4350, 5002])
def test_many_ragged_rows(ctx, fmt, dtype, cols):
    import torch
    g = torch.Generator().manual_seed(cols)
    round_trip(ctx, torch.randn((607, cols), generator=g).to(torch_dtype(dtype)).cuda(), fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(911, 4096), (1801, 2304), (911, 4097), (3600, 1031), (1203, 5002)])
def test_many_rows_of_several_segments(ctx, fmt, dtype, rows, cols):
    """As many items as the kernels that take four segments at a time want, aligned rows and others, last segments that are not full."""
    import torch
    g = torch.Generator().manual_seed(rows)
    round_trip(ctx, torch.randn((rows, cols), generator=g).to(torch_dtype(dtype)).cuda(), fmt)


@pytest.mark.gpu
def test_many_rows(ctx):
    """More rows than one launch has blocks of; the last ones are right."""
    import torch
    rows = 65535 * 64 + 77
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((rows, 16), generator=g, device="cuda").to(torch.bfloat16)
    q, s = torch.zeros((rows, 16), dtype=torch.uint8, device="cuda"), torch.zeros(capi.mx_scale_bytes(rows, 16, capi.NVFP4), dtype=torch.uint8, device="cuda")
    ctx.mx_quantize(capi.make_mx_desc(rows, 16, capi.NVFP4, capi.BF16, ld_packed=16), x, q, s)
    y = torch.empty_like(x)
    ctx.mx_dequantize(capi.make_mx_desc(rows, 16, capi.NVFP4, capi.BF16, ld_packed=16), q, s, y)
    for part in (slice(0, 200), slice(65535 * 64 - 50, rows)):
        code, byte = mx.quantize(x[part].double().cpu().numpy(), capi.NVFP4)
        same_values(y[part].double().cpu().numpy(), mx.values(code, byte, capi.NVFP4))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 100), (200, 130), (128, 4096)])
def test_tile_scales(ctx, fmt, rows, cols):
    import torch
    nb = mx.blocks_of(cols, fmt)
    byte = np.random.default_rng(rows).integers(1, 127, (rows, nb + 3)).astype(np.uint8)
    out = torch.full((capi.mx_scale_bytes(rows, cols, fmt) + 16,), 0xA5, dtype=torch.uint8, device="cuda")
    ctx.mx_tile_scales(torch.from_numpy(byte).cuda(), nb + 3, rows, cols, fmt, out)
    want = mx.tile(byte[:, :nb], fill=0xA5)
    got = out.cpu().numpy()
    assert np.array_equal(got[:-16], want) and (got[-16:] == 0xA5).all()


@pytest.mark.gpu
def test_nothing_to_do_and_refusals(ctx):
    import torch
    t = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    none = capi.make_mx_desc(0, 64, capi.MXFP4, capi.F32)
    ctx.mx_quantize(none, None, None, None)
    ctx.mx_dequantize(none, None, None, None)
    ctx.mx_tile_scales(None, 2, 0, 64, capi.MXFP4, None)
    d = capi.make_mx_desc(2, 64, capi.MXFP4, capi.F32)
    p = t.data_ptr()
    for call in (lambda: ctx.mx_quantize(d, None, p, p), lambda: ctx.mx_quantize(d, p, None, p), lambda: ctx.mx_quantize(d, p, p, None),
                 lambda: ctx.mx_quantize(d, p + 2, p, p), lambda: ctx.mx_quantize(d, p, p, p + 8),
                 lambda: ctx.mx_dequantize(d, p, p, p + 1), lambda: ctx.mx_dequantize(d, p, p + 4, p),
                 lambda: ctx.mx_tile_scales(p, 1, 2, 64, capi.MXFP4, p), lambda: ctx.mx_tile_scales(p, 2, 2, 64, capi.MXFP4, p + 4),
                 lambda: ctx.mx_tile_scales(p, 2, 2, 64, 7, p)):
        with pytest.raises(capi.CuglError) as e:
            call()
        assert e.value.status == capi.INVALID_ARGUMENT
    ctx.sync()


@pytest.mark.gpu
def test_other_stream_and_graph(ctx):
    """A context on another stream, and a captured pass that is replayed on new contents."""
    import torch
    import computelibrary_b200 as cl
    stream = torch.cuda.Stream()
    own = cl.Context(0, stream.cuda_stream)
    x = torch.zeros((40, 96), dtype=torch.bfloat16, device="cuda")
    q, s = torch.zeros((40, 48), dtype=torch.uint8, device="cuda"), torch.zeros(capi.mx_scale_bytes(40, 96, capi.MXFP4), dtype=torch.uint8, device="cuda")
    y = torch.zeros_like(x)
    d = capi.make_mx_desc(40, 96, capi.MXFP4, capi.BF16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        own.mx_quantize(d, x, q, s)
        own.mx_dequantize(d, q, s, y)
    for seed in (1, 2):
        x.copy_(torch.randn((40, 96), generator=torch.Generator().manual_seed(seed)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        code, byte = mx.quantize(x.double().cpu().numpy(), capi.MXFP4)
        same_values(y.double().cpu().numpy(), mx.values(code, byte, capi.MXFP4))
    del graph
    own.sync()
    own.close()
