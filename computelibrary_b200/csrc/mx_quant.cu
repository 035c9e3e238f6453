// Microscaled 4-bit matrices: quantisation, read-back and the re-ordering of scales.  One pass over the data each; the bytes
// moved bound all three.
#include "mx.cuh"

#include <cmath>
#include <cstring>
#include <utility>

namespace cugl
{
namespace
{
constexpr int kWarps = 8;

// Sixteen consecutive values of a row as floats, and the bits of the largest |value|.
template <typename T>
__device__ __forceinline__ uint32_t load16(const T *p, float (&v)[16])
{
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const float4 q = __ldg(reinterpret_cast<const float4 *>(p) + i);
            v[4 * i] = q.x, v[4 * i + 1] = q.y, v[4 * i + 2] = q.z, v[4 * i + 3] = q.w;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    else
    {
        uint32_t    w[8];
        const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p)), b = __ldg(reinterpret_cast<const uint4 *>(p) + 1);
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            m = __vmaxu2(m, w[i] & 0x7fff7fffu);
            T lo, hi;
            const uint16_t l = static_cast<uint16_t>(w[i]), h = static_cast<uint16_t>(w[i] >> 16);
            memcpy(&lo, &l, 2);
            memcpy(&hi, &h, 2);
            v[2 * i]     = to_float(lo);
            v[2 * i + 1] = to_float(hi);
        }
        const uint16_t top = static_cast<uint16_t>(max(m & 0xffffu, m >> 16));
        T              t;
        memcpy(&t, &top, 2);
        m = __float_as_uint(to_float(t)) & 0x7fffffffu;
    }
    return m;
}
template <typename T>
__device__ __forceinline__ uint32_t load16_part(const T *p, int n, float (&v)[16])
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
    {
        v[i] = i < n ? to_float(p[i]) : 0.f;
        m    = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    return m;
}

struct QuantParams
{
    const void *src;
    uint8_t    *dst, *scales;
    int64_t     ld, ld_packed, tiles; // bytes, bytes, scale tiles along a row
    int         rows, cols;
    int         chunks;     // pieces of sixteen columns a row is walked in: whole scale tiles
    int         lane_shift; // 2^lane_shift lanes of a warp share a row
    float       exponent_mul;
    int         vec_src, vec_dst; // 16-byte loads / 8-byte stores are aligned
};

// A lane owns sixteen columns: one NVFP4 block, or half an MXFP4 block whose other half is the neighbouring lane's.  The scale
// bytes of four blocks are gathered by shuffles and leave as one word of their tile.
template <typename T, int kFormat>
__global__ void __launch_bounds__(kWarps * 32) quantize_kernel(const QuantParams p)
{
    dependent_prologue();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per_row  = 1 << p.lane_shift;
    const int rows_per = 32 >> p.lane_shift;
    const int sub      = lane >> p.lane_shift;
    const int chunk    = blockIdx.x * per_row + (lane & (per_row - 1));
    const int c0       = chunk * 16;
    const int n        = min(16, p.cols - c0); // <= 0: behind the row, only the tile's zero scales
    for (int64_t row = (static_cast<int64_t>(blockIdx.y) * kWarps + warp) * rows_per + sub; __any_sync(0xffffffffu, row < p.rows);
         row += static_cast<int64_t>(gridDim.y) * kWarps * rows_per)
    {
        const bool in = row < p.rows && chunk < p.chunks;
        float      v[16];
        uint32_t   amax = 0;
        if (in && n > 0)
        {
            const T *src = reinterpret_cast<const T *>(static_cast<const uint8_t *>(p.src) + row * p.ld) + c0;
            amax         = (n == 16 && p.vec_src != 0) ? load16(src, v) : load16_part(src, n, v);
        }
        constexpr int kLanesPerBlock = kFormat == CUGL_NVFP4 ? 1 : 2;
        if (kLanesPerBlock == 2)
        {
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        }
        const MxScale s = mx_scale_of<kFormat>(amax, p.exponent_mul);
        uint32_t      word = s.byte << (8 * ((lane / kLanesPerBlock) & 3));
        word |= __shfl_xor_sync(0xffffffffu, word, kLanesPerBlock);
        word |= __shfl_xor_sync(0xffffffffu, word, 2 * kLanesPerBlock);
        if (!in)
        {
            continue;
        }
        if ((chunk & (4 * kLanesPerBlock - 1)) == 0)
        {
            *reinterpret_cast<uint32_t *>(p.scales + mx_scale_offset(row, chunk / kLanesPerBlock, p.tiles)) = word;
        }
        if (n > 0)
        {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = scale_to_code<kFormat, sizeof(T) == 4>(v[i], s, p.exponent_mul);
            const uint32_t lo = pack_e2m1x8(v), hi = pack_e2m1x8(v + 8);
            uint8_t       *d  = p.dst + row * p.ld_packed + c0 / 2;
            if (n == 16 && p.vec_dst != 0)
            {
                *reinterpret_cast<uint2 *>(d) = make_uint2(lo, hi);
            }
            else
            {
                const uint64_t w = (static_cast<uint64_t>(hi) << 32) | lo;
                for (int i = 0; i < (n + 1) / 2; ++i) d[i] = static_cast<uint8_t>(w >> (8 * i)); // values behind the row count as 0
            }
        }
    }
}

template <typename T, int kFormat>
__global__ void __launch_bounds__(kWarps * 32) dequantize_kernel(const QuantParams p, void *out)
{
    dependent_prologue();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per_row  = 1 << p.lane_shift;
    const int rows_per = 32 >> p.lane_shift;
    const int chunk    = blockIdx.x * per_row + (lane & (per_row - 1));
    const int c0       = chunk * 16;
    const int n        = min(16, p.cols - c0);
    if (n <= 0)
    {
        return;
    }
    for (int64_t row = (static_cast<int64_t>(blockIdx.y) * kWarps + warp) * rows_per + (lane >> p.lane_shift); row < p.rows;
         row += static_cast<int64_t>(gridDim.y) * kWarps * rows_per)
    {
        const uint8_t *src = static_cast<const uint8_t *>(p.src) + row * p.ld_packed + c0 / 2;
        uint32_t       w[2];
        if (n == 16 && p.vec_src != 0)
        {
            const uint2 q = __ldg(reinterpret_cast<const uint2 *>(src));
            w[0] = q.x, w[1] = q.y;
        }
        else
        {
            uint64_t q = 0;
            for (int i = 0; i < (n + 1) / 2; ++i) q |= static_cast<uint64_t>(__ldg(src + i)) << (8 * i);
            w[0] = static_cast<uint32_t>(q), w[1] = static_cast<uint32_t>(q >> 32);
        }
        const int   block = kFormat == CUGL_NVFP4 ? chunk : chunk >> 1;
        const float s     = mx_scale_value<kFormat>(__ldg(p.scales + mx_scale_offset(row, block, p.tiles))) * p.exponent_mul;
        T           v[16];
#pragma unroll
        for (int j = 0; j < 2; ++j)
        {
            __half2 h[4];
            unpack_e2m1x8(w[j], h);
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const float2 f         = __half22float2(h[i]);
                v[8 * j + 2 * i]     = from_float<T>(f.x * s);
                v[8 * j + 2 * i + 1] = from_float<T>(f.y * s);
            }
        }
        T *dst = reinterpret_cast<T *>(static_cast<uint8_t *>(out) + row * p.ld) + c0;
        if (n == 16 && p.vec_dst != 0)
        {
            uint4 q[sizeof(T)];
            memcpy(q, v, sizeof(v));
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) reinterpret_cast<uint4 *>(dst)[i] = q[i];
        }
        else
        {
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                if (i < n) dst[i] = v[i];
            }
        }
    }
}

// Row-major scale bytes into tiles: a thread per four blocks of a row.
__global__ void __launch_bounds__(256) tile_scales_kernel(const uint8_t *src, int64_t ld, int rows, int blocks, int64_t tiles, uint8_t *dst)
{
    dependent_prologue();
    const int64_t total = static_cast<int64_t>(rows) * tiles;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * blockDim.x)
    {
        const int64_t row = i / tiles, b0 = (i - row * tiles) * 4;
        uint32_t      w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            if (b0 + j < blocks) w |= static_cast<uint32_t>(__ldg(src + row * ld + b0 + j)) << (8 * j);
        }
        *reinterpret_cast<uint32_t *>(dst + mx_scale_offset(row, b0, tiles)) = w;
    }
}

bool aligned(const void *p, uintptr_t n)
{
    return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

QuantParams make_params(const cugl_mx_desc &d, const void *plain, const void *packed)
{
    QuantParams p{};
    p.ld        = d.ld;
    p.ld_packed = d.ld_packed;
    p.tiles     = mx_scale_tiles(d.cols, d.format);
    p.rows      = d.rows;
    p.cols      = d.cols;
    p.chunks    = static_cast<int>(p.tiles * 4 * mx_block(d.format) / 16);
    p.lane_shift = 5;
    // narrow rows: a power of two of lanes that holds one, at least those that share a word of scales
    while (p.lane_shift > (d.format == CUGL_NVFP4 ? 2 : 3) && (1 << (p.lane_shift - 1)) >= p.chunks) --p.lane_shift;
    const bool plain_vec = aligned(plain, 16) && d.ld % 16 == 0, packed_vec = aligned(packed, 8) && d.ld_packed % 8 == 0;
    p.vec_src = plain_vec;
    p.vec_dst = packed_vec;
    return p;
}

dim3 grid_of(const QuantParams &p)
{
    const int     per_row = 1 << p.lane_shift;
    const int64_t y       = (static_cast<int64_t>(p.rows) + kWarps * (32 / per_row) - 1) / (kWarps * (32 / per_row));
    return dim3(static_cast<unsigned>((p.chunks + per_row - 1) / per_row), static_cast<unsigned>(y < 65535 ? y : 65535));
}

template <typename T>
cudaError_t launch_quantize(cugl_context *ctx, int format, const QuantParams &p)
{
    const dim3      g     = grid_of(p);
    const long long units = static_cast<long long>(g.x) * g.y;
    return format == CUGL_NVFP4 ? launch_dependent(ctx, quantize_kernel<T, CUGL_NVFP4>, g, kWarps * 32, 0, units, p)
                                : launch_dependent(ctx, quantize_kernel<T, CUGL_MXFP4>, g, kWarps * 32, 0, units, p);
}
template <typename T>
cudaError_t launch_dequantize(cugl_context *ctx, int format, const QuantParams &p, void *out)
{
    const dim3      g     = grid_of(p);
    const long long units = static_cast<long long>(g.x) * g.y;
    return format == CUGL_NVFP4 ? launch_dependent(ctx, dequantize_kernel<T, CUGL_NVFP4>, g, kWarps * 32, 0, units, p, out)
                                : launch_dependent(ctx, dequantize_kernel<T, CUGL_MXFP4>, g, kWarps * 32, 0, units, p, out);
}

const char *validate_mx(const cugl_mx_desc *d, cugl_status *code)
{
    *code = CUGL_INVALID_ARGUMENT;
    if (d == nullptr) return "descriptor is NULL";
    if (d->rows < 0 || d->cols < 1) return "rows must not be negative and cols must be positive";
    if (d->cols > INT32_MAX - 1024) return "cols is too large";
    if (d->format != CUGL_MXFP4 && d->format != CUGL_NVFP4) return "format must be CUGL_MXFP4 or CUGL_NVFP4";
    if (!is_float_dtype(d->dtype)) return "dtype must be CUGL_F32, CUGL_F16 or CUGL_BF16";
    if (d->ld < static_cast<int64_t>(d->cols) * dtype_size(d->dtype) || d->ld % dtype_size(d->dtype) != 0)
        return "ld must hold a row and be a multiple of the element size";
    if (d->ld_packed < (static_cast<int64_t>(d->cols) + 1) / 2) return "ld_packed must hold a packed row";
    if (d->format == CUGL_MXFP4 && d->tensor_exponent != 0) return "tensor_exponent is for CUGL_NVFP4 (E8M0 scales have the whole range)";
    if (d->tensor_exponent < -64 || d->tensor_exponent > 64) return "tensor_exponent must lie within -64 .. 64";
    *code = CUGL_SUCCESS;
    return nullptr;
}

cugl_status check_mx(cugl_context *ctx, const char *name, const cugl_mx_desc *d, const void *plain, const void *packed, const void *scales)
{
    if (ctx == nullptr)
    {
        return fail(nullptr, CUGL_INVALID_ARGUMENT, "context is NULL");
    }
    cugl_status code;
    const char *why = validate_mx(d, &code);
    if (why == nullptr && d->rows > 0)
    {
        if (plain == nullptr || packed == nullptr || scales == nullptr) why = "NULL pointer";
        else if (!aligned(plain, static_cast<uintptr_t>(dtype_size(d->dtype)))) why = "the plain matrix is not aligned to its elements";
        else if (!aligned(scales, 16)) why = "scale tiles must be 16-byte aligned";
        if (why != nullptr) code = CUGL_INVALID_ARGUMENT;
    }
    return why == nullptr ? CUGL_SUCCESS : fail(ctx, code, std::string(name) + ": " + why);
}
} // namespace
} // namespace cugl

using namespace cugl;

extern "C"
{
    size_t cugl_mx_scale_bytes(int32_t rows, int32_t cols, int32_t format)
    {
        if (rows < 0 || cols < 1 || (format != CUGL_MXFP4 && format != CUGL_NVFP4))
        {
            return 0;
        }
        return static_cast<size_t>(mx_scale_size(rows, cols, format));
    }

    cugl_status cugl_mx_validate(const cugl_mx_desc *desc, const char **reason)
    {
        cugl_status code;
        const char *why = validate_mx(desc, &code);
        if (reason != nullptr)
        {
            *reason = why != nullptr ? why : "";
        }
        return code;
    }

    cugl_status cugl_mx_quantize(cugl_context *ctx, const cugl_mx_desc *desc, const void *d_src, void *d_dst, void *d_scales)
    {
        CUGL_TRY(check_mx(ctx, "cugl_mx_quantize", desc, d_src, d_dst, d_scales));
        if (desc->rows == 0) return CUGL_SUCCESS;
        const DeviceScope device(ctx);
        QuantParams       p = make_params(*desc, d_src, d_dst);
        p.src          = d_src;
        p.dst          = static_cast<uint8_t *>(d_dst);
        p.scales       = static_cast<uint8_t *>(d_scales);
        p.exponent_mul = std::ldexp(1.f, -desc->tensor_exponent);
        CUGL_CUDA_TRY(ctx, desc->dtype == CUGL_F32   ? launch_quantize<float>(ctx, desc->format, p)
                           : desc->dtype == CUGL_F16 ? launch_quantize<__half>(ctx, desc->format, p)
                                                     : launch_quantize<__nv_bfloat16>(ctx, desc->format, p));
        return CUGL_SUCCESS;
    }

    cugl_status cugl_mx_dequantize(cugl_context *ctx, const cugl_mx_desc *desc, const void *d_src, const void *d_scales, void *d_dst)
    {
        CUGL_TRY(check_mx(ctx, "cugl_mx_dequantize", desc, d_dst, d_src, d_scales));
        if (desc->rows == 0) return CUGL_SUCCESS;
        const DeviceScope device(ctx);
        QuantParams       p = make_params(*desc, d_dst, d_src);
        std::swap(p.vec_src, p.vec_dst);
        p.src          = d_src;
        p.scales       = const_cast<uint8_t *>(static_cast<const uint8_t *>(d_scales));
        p.exponent_mul = std::ldexp(1.f, desc->tensor_exponent);
        CUGL_CUDA_TRY(ctx, desc->dtype == CUGL_F32   ? launch_dequantize<float>(ctx, desc->format, p, d_dst)
                           : desc->dtype == CUGL_F16 ? launch_dequantize<__half>(ctx, desc->format, p, d_dst)
                                                     : launch_dequantize<__nv_bfloat16>(ctx, desc->format, p, d_dst));
        return CUGL_SUCCESS;
    }

    cugl_status cugl_mx_tile_scales(cugl_context *ctx, const void *d_src, int64_t ld, int32_t rows, int32_t cols, int32_t format, void *d_dst)
    {
        if (ctx == nullptr)
        {
            return fail(nullptr, CUGL_INVALID_ARGUMENT, "context is NULL");
        }
        if (rows < 0 || cols < 1 || (format != CUGL_MXFP4 && format != CUGL_NVFP4) || ld < mx_blocks(cols, format) ||
            (rows > 0 && (d_src == nullptr || d_dst == nullptr || !aligned(d_dst, 16))))
        {
            return fail(ctx, CUGL_INVALID_ARGUMENT, "cugl_mx_tile_scales: bad argument");
        }
        if (rows == 0) return CUGL_SUCCESS;
        const DeviceScope device(ctx);
        const int64_t     tiles = mx_scale_tiles(cols, format), blocks = (rows * tiles + 255) / 256;
        const int64_t     most  = static_cast<int64_t>(ctx->sm_count) * 16;
        const unsigned    grid  = static_cast<unsigned>(blocks < most ? blocks : most);
        CUGL_CUDA_TRY(ctx, launch_dependent(ctx, tile_scales_kernel, dim3(grid), 256, 0, grid, static_cast<const uint8_t *>(d_src), ld, rows,
                                            static_cast<int>(mx_blocks(cols, format)), tiles, static_cast<uint8_t *>(d_dst)));
        return CUGL_SUCCESS;
    }
}
