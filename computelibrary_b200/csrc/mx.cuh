// Microscaled 4-bit floating point (MXFP4 and NVFP4): what the quantiser, the product and the expert layer share.
//
// A matrix is cut into blocks along its rows.  A block is kBlock codes E2M1 (sign, two exponent bits, one mantissa bit:
// 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one scale byte:
//   MXFP4  blocks of 32, scale E8M0: 2^(byte - 127); 255 is NaN
//   NVFP4  blocks of 16, scale E4M3 (unsigned: bit 7 is 0); 0x7f is NaN
// Packed rows hold element 2 i in the low half of byte i.  Scale bytes lie in tiles of 128 rows x 4 blocks, 512 bytes,
// the order in which tcgen05.cp spreads them over tensor memory: row r, block b of a tile at (r % 32) * 16 + (r / 32) * 4 + b.
// The tiles of one group of 128 rows follow each other.
#pragma once

#include "kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>

namespace cugl
{
constexpr int kMxTileBytes = 512;

inline int mx_block(int format)
{
    return format == CUGL_NVFP4 ? 16 : 32;
}
inline int64_t mx_blocks(int64_t cols, int format)
{
    return (cols + mx_block(format) - 1) / mx_block(format);
}
inline int64_t mx_scale_tiles(int64_t cols, int format) // tiles along one group of 128 rows
{
    return (mx_blocks(cols, format) + 3) / 4;
}
inline int64_t mx_scale_size(int64_t rows, int64_t cols, int format)
{
    return (rows + 127) / 128 * mx_scale_tiles(cols, format) * kMxTileBytes;
}
inline int dtype_size(int dtype)
{
    return dtype == CUGL_F32 ? 4 : 2;
}
inline bool is_float_dtype(int dtype)
{
    return dtype == CUGL_F32 || dtype == CUGL_F16 || dtype == CUGL_BF16;
}

// The context's device for the duration of one call: the caller's current device may be another one.
class DeviceScope
{
public:
    explicit DeviceScope(const cugl_context *ctx)
    {
        if (cudaGetDevice(&before_) == cudaSuccess && before_ != ctx->device)
        {
            changed_ = true;
            (void)cudaSetDevice(ctx->device);
        }
    }
    ~DeviceScope()
    {
        if (changed_)
        {
            (void)cudaSetDevice(before_);
        }
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;

private:
    int  before_  = 0;
    bool changed_ = false;
};

__device__ __forceinline__ size_t mx_scale_offset(int64_t row, int64_t block, int64_t tiles)
{
    return static_cast<size_t>((row >> 7) * tiles + (block >> 2)) * kMxTileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// Eight values (already divided by their scale) to E2M1, v[0] in the lowest four bits: to nearest, ties to even, saturated.
__device__ __forceinline__ uint32_t pack_e2m1x8(const float *v)
{
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __nv_cvt_float2_to_fp4x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_E2M1, cudaRoundNearest);
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// Eight codes to f16 pairs (exact), the element of the lowest four bits first.
__device__ __forceinline__ void unpack_e2m1x8(uint32_t w, __half2 (&h)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        h[i] = __half2(__nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(w >> (8 * i)), __NV_E2M1));
    }
}

// A block's scale from the largest |value| in it (the bits of a non-negative float; NaN and infinity order above all
// finite values).  byte: what is stored.  mul: what a value is multiplied by on its way to a code.
//   MXFP4  2^max(-127, floor(log2 amax) - 2): the largest value lands in [4, 8), above 6 it saturates.  mul is a power of
//          two, so the codes are those of the exact quotient.
//   NVFP4  amax * 2^-exponent / 6 to the nearest E4M3 within [2^-9, 448].  Rounding the quotient to 24 bits first changes
//          nothing: a quotient that is not a midpoint of E4M3 (five bits) stays at least half a step of 24 bits away from it.
// A block of zeros gets the byte 0; one with a NaN or an infinity gets the NaN scale, all of it reads back as NaN.
struct MxScale
{
    uint32_t byte;
    float    mul;  // MXFP4: 1 / scale.  NVFP4: 2^-exponent / scale, rounded up, or to nearest where the source has 32 bits
    float    unit; // NVFP4, 32 bits: scale * 2^exponent, what a code of 1 stands for
};
// kExact false: values that were computed in float just now and carry its error; a product with 1 / 6 instead of the division.
template <int kFormat, bool kWide = false, bool kExact = true>
__device__ __forceinline__ MxScale mx_scale_of(uint32_t amax_bits, float exponent_mul)
{
    MxScale s;
    s.unit = 0.f;
    if (kFormat == CUGL_MXFP4)
    {
        const uint32_t e = amax_bits >> 23;
        s.byte           = e > 2 ? e - 2 : 0;
        s.mul            = __uint_as_float((254 - s.byte) << 23);
        if (amax_bits >= 0x7f800000u)
        {
            s.byte = 255;
            s.mul  = 0.f;
        }
        return s;
    }
    const float                amax = fminf(__uint_as_float(amax_bits) * exponent_mul, 4096.f); // all above 6 * 448 saturate alike
    float                      v    = amax * (1.f / 6.f);
    if (kExact) v                   = __fmaf_rn(__fmaf_rn(-6.f, v, amax), 1.f / 6.f, v); // correctly rounded, see scale_to_codes
    v                               = fminf(fmaxf(v, 0x1p-9f), 448.f);
    const __nv_fp8_storage_t   b    = __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
    const float                f    = __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
    s.byte                          = b;
    s.mul                           = (kWide ? __frcp_rn(f) : __frcp_ru(f)) * exponent_mul;
    if (kWide) s.unit               = f * __uint_as_float((254u << 23) - __float_as_uint(exponent_mul)); // exponent_mul: a power of two
    if (amax_bits == 0 || amax_bits >= 0x7f800000u)
    {
        s.byte = amax_bits == 0 ? 0 : 0x7f;
        s.mul  = 0.f;
    }
    return s;
}

// value / scale, near enough to the exact quotient that rounding it to E2M1 gives the quotient's code.
//   MXFP4            a product with a power of two
//   NVFP4, 16 bits   the reciprocal rounded up times the value, rounded towards zero: for every scale (four bits) and every
//                    value of up to eleven bits it compares with each midpoint of E2M1 as the exact quotient does (checked
//                    for all of them); one instruction
//   NVFP4, 32 bits   the correctly rounded quotient: as for the scale, a quotient that is no midpoint does not round onto one.
//                    Product with the reciprocal and one correction by the exact remainder (Markstein, Computation of
//                    elementary functions on the IBM RISC System/6000 processor, 1990).  A saturated block is bounded first:
//                    its products may overflow.
template <int kFormat, bool kWide, int kCount>
__device__ __forceinline__ void scale_to_codes(float (&v)[kCount], const MxScale &s)
{
    if (kFormat == CUGL_NVFP4 && kWide)
    {
        if (s.byte == 0x7e)
        {
#pragma unroll
            for (int i = 0; i < kCount; ++i) v[i] = fminf(fmaxf(v[i], -8.f * s.unit), 8.f * s.unit);
        }
#pragma unroll
        for (int i = 0; i < kCount; ++i)
        {
            const float q = __fmul_rn(v[i], s.mul);
            v[i]          = copysignf(__fmaf_rn(__fmaf_rn(-q, s.unit, v[i]), s.mul, q), v[i]); // -0: the remainder 0 would turn it into 0
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kCount; ++i) v[i] = kFormat == CUGL_MXFP4 ? v[i] * s.mul : __fmul_rz(v[i], s.mul);
}

// The value of a scale byte.
template <int kFormat>
__device__ __forceinline__ float mx_scale_value(uint32_t byte)
{
    if (kFormat == CUGL_MXFP4)
    {
        const uint32_t bits = byte == 0 ? 0x00400000u : byte << 23; // 2^-127 is subnormal
        return __uint_as_float(byte == 255 ? 0x7fc00000u : bits);
    }
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte & 0x7f), __NV_E4M3)));
}

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v)
{
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}
__device__ __forceinline__ float to_float(float v)
{
    return v;
}
__device__ __forceinline__ float to_float(__half v)
{
    return __half2float(v);
}
__device__ __forceinline__ float to_float(__nv_bfloat16 v)
{
    return __bfloat162float(v);
}
} // namespace cugl
