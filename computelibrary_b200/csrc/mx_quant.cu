// Microscaled 4-bit matrices: quantisation, read-back and the re-ordering of scales.  One pass over the data each; the bytes
// moved bound all three.
//
// us, and of the measured copy rate: 8192 x 4096 BF16 -> MXFP4 and back (170 MB, two launches) 31.0, 85 %; 4096 x 4096 F32 ->
// NVFP4 and back (153 MB) 28.0, 85 %; 8192 x 4096 NVFP4 -> BF16 (86 MB) 15.8, 84 %.  Rows that are not 16-byte aligned:
// 1023 x 2049 F16 there and back (10.6 MB) 7.5, two launches; 5780 x 3014 F32 -> MXFP4 22.2 and back 15.2 (79 MB, 12.2 at the copy
// rate), bound by the instructions of moving single elements and turning them over.
#include "mx.cuh"

#include <cmath>
#include <cstring>

namespace cugl
{
namespace
{
constexpr int kWarps = 8;
constexpr int kLaneCols = 8;               // consecutive columns of a lane
constexpr int kItemCols = 32 * kLaneCols;  // columns of a warp

struct QuantParams
{
    const uint8_t *src;
    uint8_t       *dst, *scales;
    int64_t        ld, ld_packed, tiles; // bytes, bytes, scale tiles along a row
    int            rows, cols, groups;   // groups of rows: what a block takes at a time
    int            lane_shift;           // 2^lane_shift lanes of a warp share a row
    float          exponent_mul;
    int            vec_plain, vec_packed; // the plain matrix is 16-byte aligned, the packed one 4-byte
    const int32_t *slots;                 // rows of groups (see Rows), within 0 .. group_rows - 1
    int            top_k, group_rows;
    int            wide_packed;           // packed rows are 16-byte aligned
};

// Which rows a row of the launch stands for.
//   kSame     row r of the plain matrix, row r of the packed one
//   kChoices  row r of the plain matrix, rows slots[r * top_k] and following of the packed one: a token's choices
//   kSlots    row slots[r] of both: rows of groups, choice by choice
// A slot outside the groups' rows stands for none.
enum Rows
{
    kSame,
    kChoices,
    kSlots
};
__device__ __forceinline__ int slot_of(const QuantParams &p, int64_t i)
{
    const int r = p.slots[i];
    return static_cast<unsigned>(r) < static_cast<unsigned>(p.group_rows) ? r : -1;
}
template <int kWhich>
__device__ __forceinline__ int source_row(const QuantParams &p, int row) // -1: none
{
    if (row >= p.rows) return -1;
    return kWhich == kSlots ? slot_of(p, row) : row;
}

// What a warp takes: kRows rows (or groups of narrow rows) of kSegs segments of 256 columns.  Segments lie 256 columns apart at
// addresses that differ by constants, so that a row's address is computed once.
struct Place
{
    int row, step; // first row, rows between items
    int c0;        // first column of the first segment
};
template <int kSegs, int kRows>
__device__ __forceinline__ Place place_of(const QuantParams &p, int group, int lane)
{
    Place q;
    q.step = 32 >> p.lane_shift;
    q.row  = (group * kWarps + static_cast<int>(threadIdx.x >> 5)) * kRows * q.step + (lane >> p.lane_shift);
    q.c0   = static_cast<int>(blockIdx.x) * kSegs * kItemCols + (lane & ((1 << p.lane_shift) - 1)) * kLaneCols;
    return q;
}

// Rows that start anywhere: a warp moves its 256 values as consecutive elements and turns them over in shared memory, where a
// lane's eight lie in a row.  row: of lane 0's columns; c0: the segment's first column.
template <typename T, int kWhich>
__device__ __forceinline__ void load_ragged(const QuantParams &p, int row, int c0, int lane, T (&v)[kLaneCols])
{
    if (p.lane_shift == 5) // the warp's values lie in one row
    {
        const int from = source_row<kWhich>(p, row);
        const T  *src  = reinterpret_cast<const T *>(p.src + from * p.ld) + c0 + lane;
        const int n    = from >= 0 ? p.cols - c0 - lane : 0;
#pragma unroll
        for (int i = 0; i < kLaneCols; ++i) v[i] = i * 32 < n ? src[i * 32] : from_float<T>(0.f);
        return;
    }
#pragma unroll
    for (int i = 0; i < kLaneCols; ++i)
    {
        const int at = i * 32 + lane, l = at / kLaneCols, r = row + (l >> p.lane_shift);
        const int c  = c0 + (l & ((1 << p.lane_shift) - 1)) * kLaneCols + at % kLaneCols;
        const int from = source_row<kWhich>(p, r);
        v[i]           = from_float<T>(0.f);
        if (from >= 0 && c < p.cols) v[i] = reinterpret_cast<const T *>(p.src + from * p.ld)[c];
    }
}
template <typename T>
__device__ __forceinline__ void turn_over(int lane, const T (&v)[kLaneCols], T *area)
{
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kLaneCols; ++i) area[i * 32 + lane] = v[i];
    __syncwarp();
}
template <typename T>
__device__ __forceinline__ void store_ragged(const QuantParams &p, int row, int c0, int lane, const T *area)
{
    __syncwarp();
    if (p.lane_shift == 5)
    {
        T        *dst = reinterpret_cast<T *>(p.dst + row * p.ld) + c0 + lane;
        const int n   = row < p.rows ? p.cols - c0 - lane : 0;
#pragma unroll
        for (int i = 0; i < kLaneCols; ++i)
        {
            if (i * 32 < n) dst[i * 32] = area[i * 32 + lane];
        }
        __syncwarp();
        return;
    }
#pragma unroll
    for (int i = 0; i < kLaneCols; ++i)
    {
        const int at = i * 32 + lane, l = at / kLaneCols, r = row + (l >> p.lane_shift);
        const int c  = c0 + (l & ((1 << p.lane_shift) - 1)) * kLaneCols + at % kLaneCols;
        if (r < p.rows && c < p.cols) reinterpret_cast<T *>(p.dst + r * p.ld)[c] = area[at];
    }
    __syncwarp();
}

// The bits of the largest |value| of eight (NaN above infinity above all others), and the values as floats.
template <typename T>
__device__ __forceinline__ uint32_t widen(const uint4 (&raw)[sizeof(T) / 2], float (&v)[kLaneCols])
{
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4)
    {
        memcpy(v, raw, sizeof(v));
#pragma unroll
        for (int i = 0; i < kLaneCols; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    else
    {
        const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            m = __vmaxu2(m, w[i] & 0x7fff7fffu);
            T two[2];
            memcpy(two, &w[i], 4);
            v[2 * i]     = to_float(two[0]);
            v[2 * i + 1] = to_float(two[1]);
        }
        const uint16_t top = static_cast<uint16_t>(max(m & 0xffffu, m >> 16));
        T              t;
        memcpy(&t, &top, 2);
        m = __float_as_uint(to_float(t)) & 0x7fffffffu;
    }
    return m;
}

// A lane owns eight columns of a segment: half an NVFP4 block or a quarter of an MXFP4 one; the largest value and the scale bytes
// of four blocks are gathered by shuffles, and the bytes leave as one word of their tile.  A warp has the loads of all its
// segments in flight.
//
// Floats: a lane's eight are two 16-byte units.  Lanes of a pair swap one each, so that an access of the warp covers whole
// 32-byte sectors (read-back of 4096 x 4096: 23.7 -> 16 us).
__device__ __forceinline__ void swap_units(uint4 &a, uint4 &b, int lane) // the even lane's b and the odd lane's a change places
{
    const bool odd  = (lane & 1) != 0;
    uint4      send = odd ? a : b;
    send.x = __shfl_xor_sync(0xffffffffu, send.x, 1);
    send.y = __shfl_xor_sync(0xffffffffu, send.y, 1);
    send.z = __shfl_xor_sync(0xffffffffu, send.z, 1);
    send.w = __shfl_xor_sync(0xffffffffu, send.w, 1);
    if (odd) a = send;
    else b = send;
}

// Four whole segments of a row to the rows of its choices.  w: a lane's eight codes of each segment; word: in every 4 kLanes-th lane, four
// blocks' scale bytes.  Four lanes turn their codes over, so that each has 16 bytes of one segment, and the scale words move to
// lanes that follow each other: two stores a choice instead of eight (4096 x 4096 BF16 to four choices, NVFP4, 22.5 -> 16.4 us).
template <int kFormat, int kLanes>
__device__ __forceinline__ void store_choices(const QuantParams &p, int row, int c0, int lane, uint32_t (&w)[4], const uint32_t (&word)[4])
{
    constexpr int kBlock = kFormat == CUGL_NVFP4 ? 16 : 32, kWords = 32 / (4 * kLanes); // scale words of a segment
    int           slot   = -1;
    if (lane < p.top_k) slot = slot_of(p, static_cast<int64_t>(row) * p.top_k + lane);
#pragma unroll
    for (int o = 1; o <= 2; o *= 2) // element i of lane l and element i ^ o of lane l ^ o change places
    {
        const bool     up = (lane & o) != 0;
        const uint32_t a = up ? w[0] : w[o], b = up ? w[3 - o] : w[3];
        const uint32_t ga = __shfl_xor_sync(0xffffffffu, a, o), gb = __shfl_xor_sync(0xffffffffu, b, o);
        if (up) w[0] = ga, w[3 - o] = gb;
        else w[o] = ga, w[3] = gb;
    }
    uint32_t scale = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g)
    {
        const uint32_t v = __shfl_sync(0xffffffffu, word[g], (lane % kWords) * 4 * kLanes);
        if (lane / kWords == g) scale = v;
    }
    const int     code_at = c0 / 2 + (lane & 3) * (kItemCols / 2) + (lane >> 2) * 16;
    const int64_t tile    = c0 / (4 * kBlock) + lane; // lanes up to 4 kWords
    for (int j = 0; j < p.top_k; ++j)
    {
        const int to = __shfl_sync(0xffffffffu, slot, j);
        if (to >= 0) // the same for the warp
        {
            *reinterpret_cast<uint4 *>(p.dst + to * p.ld_packed + code_at) = make_uint4(w[0], w[1], w[2], w[3]);
            if (lane < 4 * kWords) *reinterpret_cast<uint32_t *>(p.scales + mx_scale_offset(to, 0, p.tiles) + tile * kMxTileBytes) = scale;
        }
    }
}

// kWhole: every segment lies inside the matrix and all rows are aligned; nothing to test.
template <typename T, int kFormat, bool kVec, bool kWhole, int kSegs, int kRows, int kWhich>
__device__ __forceinline__ void quantize_group(const QuantParams &p, int group, T *area)
{
    constexpr int kBlock = kFormat == CUGL_NVFP4 ? 16 : 32;
    constexpr int kLanes = kBlock / kLaneCols; // of a block
    constexpr int kLoads = sizeof(T) / 2;
    constexpr int kTiles = kItemCols / (4 * kBlock); // scale tiles of a segment
    const int     lane   = threadIdx.x & 31;
    const Place   at     = place_of<kSegs, kRows>(p, group, lane);
    uint4         raw[kRows][kSegs][kLoads];
    T             loose[kRows][kVec ? 1 : kSegs][kLaneCols];
    if constexpr (!kVec)
    {
#pragma unroll
        for (int u = 0; u < kRows; ++u)
        {
#pragma unroll
            for (int g = 0; g < kSegs; ++g)
            {
                load_ragged<T, kWhich>(p, at.row + u * at.step - (lane >> p.lane_shift), (static_cast<int>(blockIdx.x) * kSegs + g) * kItemCols, lane, loose[u][g]);
            }
        }
    }
    else
    {
#pragma unroll
        for (int u = 0; u < kRows; ++u)
        {
            const int  row  = at.row + u * at.step, from = kWhich == kSlots ? source_row<kWhich>(p, row) : row;
            const bool in   = kWhich == kSlots ? from >= 0 : row < p.rows;
            const T   *src  = reinterpret_cast<const T *>(p.src + (kWhich == kSlots ? max(from, 0) : from) * p.ld) + at.c0; // none: row 0, not stored
#pragma unroll
            for (int g = 0; g < kSegs; ++g)
            {
                if constexpr (kWhole && kLoads == 2)
                {
                    const uint4 *unit = reinterpret_cast<const uint4 *>(src + g * kItemCols) - (lane & 1); // of the pair's first lane: + 2 per lane before it
                    raw[u][g][0]      = unit[0];
                    raw[u][g][1]      = unit[2];
                    continue;
                }
                const int n = kWhole || in ? p.cols - at.c0 - g * kItemCols : 0;
#pragma unroll
                for (int l = 0; l < kLoads; ++l)
                {
                    raw[u][g][l] = make_uint4(0, 0, 0, 0);
                    if (kWhole || n >= kLaneCols) raw[u][g][l] = reinterpret_cast<const uint4 *>(src + g * kItemCols)[l];
                }
                if (!kWhole && n > 0 && n < kLaneCols)
                {
                    T part[kLaneCols];
#pragma unroll
                    for (int i = 0; i < kLaneCols; ++i) part[i] = i < n ? src[g * kItemCols + i] : from_float<T>(0.f);
                    memcpy(raw[u][g], part, sizeof(part));
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u)
    {
        const int      row    = at.row + u * at.step;
        const int      block  = at.c0 / kBlock;
        uint8_t *const scales = p.scales + mx_scale_offset(row, block, p.tiles);
        uint8_t *const dst    = p.dst + row * p.ld_packed + at.c0 / 2;
        constexpr bool kFour  = kWhich == kChoices && kWhole && kSegs == 4;
        uint32_t       codes[kFour ? 4 : 1], words[kFour ? 4 : 1];
#pragma unroll
        for (int g = 0; g < kSegs; ++g)
        {
            if constexpr (!kVec)
            {
                turn_over(lane, loose[u][g], area);
#pragma unroll
                for (int l = 0; l < kLoads; ++l) raw[u][g][l] = reinterpret_cast<const uint4 *>(area + lane * kLaneCols)[l];
            }
            if constexpr (kWhole && kLoads == 2) swap_units(raw[u][g][0], raw[u][g][1], lane);
            float    v[kLaneCols];
            uint32_t amax = widen<T>(raw[u][g], v);
#pragma unroll
            for (int o = 1; o < kLanes; o *= 2) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            const MxScale s    = mx_scale_of<kFormat, sizeof(T) == 4>(amax, p.exponent_mul);
            uint32_t      word = s.byte << (8 * ((lane / kLanes) & 3));
            word |= __shfl_xor_sync(0xffffffffu, word, kLanes);
            word |= __shfl_xor_sync(0xffffffffu, word, 2 * kLanes);
            scale_to_codes<kFormat, sizeof(T) == 4>(v, s);
            const uint32_t w = pack_e2m1x8(v);
            if constexpr (kFour)
            {
                codes[g] = w;
                words[g] = word;
                continue;
            }
            auto store = [&](uint8_t *row_scales, uint8_t *row_dst) {
                if ((lane & (4 * kLanes - 1)) == 0 && (kWhole || block + g * 4 * kTiles < 4 * p.tiles))
                {
                    *reinterpret_cast<uint32_t *>(row_scales + g * kTiles * kMxTileBytes) = word; // blocks behind the row: 0
                }
                const int n = p.cols - at.c0 - g * kItemCols;
                uint8_t  *d = row_dst + g * kItemCols / 2;
                if (kWhole || (n >= kLaneCols && p.vec_packed != 0))
                {
                    *reinterpret_cast<uint32_t *>(d) = w;
                }
                else
                {
                    for (int i = 0; i < (min(n, kLaneCols) + 1) / 2; ++i) d[i] = static_cast<uint8_t>(w >> (8 * i)); // the half byte behind an odd row is 0
                }
            };
            if constexpr (kWhich == kSame)
            {
                if (kWhole || row < p.rows) store(scales, dst);
            }
            else if (kWhole || row < p.rows)
            {
                const int copies = kWhich == kChoices ? p.top_k : 1;
                for (int j = 0; j < copies; ++j)
                {
                    const int to = slot_of(p, static_cast<int64_t>(row) * copies + j);
                    if (to >= 0) store(p.scales + mx_scale_offset(to, block, p.tiles), p.dst + to * p.ld_packed + at.c0 / 2);
                }
            }
        }
        if constexpr (kFour) store_choices<kFormat, kLanes>(p, row, static_cast<int>(blockIdx.x) * kSegs * kItemCols, lane, codes, words);
    }
}

template <typename T, int kFormat, bool kVec, bool kWhole, int kSegs, int kRows>
__device__ __forceinline__ void dequantize_group(const QuantParams &p, int group, T *area)
{
    constexpr int kBlock = kFormat == CUGL_NVFP4 ? 16 : 32;
    constexpr int kTiles = kItemCols / (4 * kBlock); // scale tiles of a segment
    const int     lane   = threadIdx.x & 31;
    const Place   at     = place_of<kSegs, kRows>(p, group, lane);
    uint32_t      w[kRows][kSegs], byte[kRows][kSegs];
#pragma unroll
    for (int u = 0; u < kRows; ++u)
    {
        const int      row    = at.row + u * at.step;
        const uint8_t *src    = p.src + row * p.ld_packed + at.c0 / 2;
        const uint8_t *scales = p.scales + mx_scale_offset(row, at.c0 / kBlock, p.tiles);
#pragma unroll
        for (int g = 0; g < kSegs; ++g)
        {
            const int n = kWhole ? kLaneCols : row < p.rows ? p.cols - at.c0 - g * kItemCols : 0;
            w[u][g] = byte[u][g] = 0;
            if (n > 0) byte[u][g] = scales[g * kTiles * kMxTileBytes];
            if (kWhole || (n >= kLaneCols && p.vec_packed != 0))
            {
                w[u][g] = *reinterpret_cast<const uint32_t *>(src + g * kItemCols / 2);
            }
            else
            {
                for (int i = 0; i < (min(n, kLaneCols) + 1) / 2; ++i) w[u][g] |= static_cast<uint32_t>(src[g * kItemCols / 2 + i]) << (8 * i);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u)
    {
        const int row = at.row + u * at.step;
        T        *dst = reinterpret_cast<T *>(p.dst + row * p.ld) + at.c0;
#pragma unroll
        for (int g = 0; g < kSegs; ++g)
        {
            const float s = mx_scale_value<kFormat>(byte[u][g]) * p.exponent_mul;
            __half2     h[4];
            unpack_e2m1x8(w[u][g], h);
            T v[kLaneCols];
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const float2 f = __half22float2(h[i]);
                v[2 * i]       = from_float<T>(f.x * s);
                v[2 * i + 1]   = from_float<T>(f.y * s);
            }
            uint4 q[sizeof(T) / 2];
            memcpy(q, v, sizeof(v));
            if constexpr (!kVec)
            {
#pragma unroll
                for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) reinterpret_cast<uint4 *>(area + lane * kLaneCols)[i] = q[i];
                store_ragged(p, row - (lane >> p.lane_shift), (static_cast<int>(blockIdx.x) * kSegs + g) * kItemCols, lane, area);
            }
            else if constexpr (kWhole && sizeof(T) == 4)
            {
                swap_units(q[0], q[1], lane);
                uint4 *unit = reinterpret_cast<uint4 *>(dst + g * kItemCols) - (lane & 1);
                unit[0]     = q[0];
                unit[2]     = q[1];
            }
            else if (kWhole || row < p.rows)
            {
                const int n = p.cols - at.c0 - g * kItemCols;
                if (kWhole || n >= kLaneCols)
                {
#pragma unroll
                    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) reinterpret_cast<uint4 *>(dst + g * kItemCols)[i] = q[i];
                }
                else
                {
#pragma unroll
                    for (int i = 0; i < kLaneCols; ++i)
                    {
                        if (i < n) dst[g * kItemCols + i] = v[i];
                    }
                }
            }
        }
    }
}

template <typename T, int kFormat, bool kVec, int kSegs, int kRows, bool kBack, int kWhich = kSame>
__global__ void __launch_bounds__(kWarps * 32) mx_rows_kernel(const __grid_constant__ QuantParams p)
{
    __shared__ __align__(16) T areas[kVec ? 1 : kWarps][kVec ? 8 : kItemCols];
    dependent_prologue();
    T *area = areas[kVec ? 0 : threadIdx.x >> 5];
    for (int group = blockIdx.y; group < p.groups; group += gridDim.y)
    {
        const bool whole = kVec && p.lane_shift == 5 && (kWhich == kChoices ? p.wide_packed : p.vec_packed) != 0 && static_cast<int>(blockIdx.x + 1) * kSegs * kItemCols <= p.cols &&
                           (group + 1) * kWarps * kRows <= p.rows; // the same for the block
        if constexpr (kBack)
        {
            if (whole) dequantize_group<T, kFormat, kVec, kVec, kSegs, kRows>(p, group, area);
            else dequantize_group<T, kFormat, kVec, false, kSegs, kRows>(p, group, area);
        }
        else
        {
            if (whole) quantize_group<T, kFormat, kVec, kVec, kSegs, kRows, kWhich>(p, group, area);
            else quantize_group<T, kFormat, kVec, false, kSegs, kRows, kWhich>(p, group, area);
        }
    }
}

// Row-major scale bytes into tiles: a thread per four blocks of a row, read byte by byte, stored as a word.  Done once per weight, not
// made fast: 14336 x 4096 NVFP4 8.3 us (7.3 MB, 14 % of the copy rate), 65536 x 16384 113 (18 %).
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
            if (b0 + j < blocks) w |= static_cast<uint32_t>(src[row * ld + b0 + j]) << (8 * j);
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
    const int64_t lanes = p.tiles * 4 * mx_block(d.format) / kLaneCols; // of a row, whole scale tiles
    p.lane_shift = 5;
    // narrow rows: a power of two of lanes that holds one; those that share a word of scales stay together
    while (p.lane_shift > 3 && (1 << (p.lane_shift - 1)) >= lanes) --p.lane_shift;
    p.vec_plain  = aligned(plain, 16) && d.ld % 16 == 0;
    p.vec_packed = aligned(packed, 4) && d.ld_packed % 4 == 0;
    return p;
}

template <typename K>
cudaError_t launch_rows(cugl_context *ctx, K kernel, QuantParams p, int segs, int rows_per_warp)
{
    const int64_t per_block = static_cast<int64_t>(kWarps) * rows_per_warp * (32 >> p.lane_shift);
    const int64_t cols      = p.lane_shift < 5 ? p.cols : segs * kItemCols; // of a block: narrow rows lie in one
    p.groups                = static_cast<int>((p.rows + per_block - 1) / per_block);
    const dim3 grid(static_cast<unsigned>((p.cols + cols - 1) / cols), static_cast<unsigned>(p.groups < 65535 ? p.groups : 65535));
    return launch_dependent(ctx, kernel, grid, kWarps * 32, 0, static_cast<long long>(grid.x) * grid.y, p);
}
// Four segments of a row where there are enough rows and columns to keep the device busy that way, else one: from 24 items of four per
// SM on.  us with one segment / four, items rows * (cols / 1024): BF16 -> MXFP4 of 4096 columns, 2400 items 3.07 / 2.76, 3552 3.80 / 3.06,
// 11840 9.34 / 6.32, and back 2.59 / 2.98, 3.24 / 3.28, 7.47 / 5.78; F32 -> NVFP4 3.71 / 4.01, 4.84 / 4.10, 12.5 / 10.4, and back
// 3.09 / 3.82, 3.89 / 3.48, 8.84 / 8.70; read-back of F32 rows of 3014 4.9 / 5.8, 6.4 / 5.9, 18.0 / 14.2.  (Rows that end early in their
// last block of four are quantised slower by it at any size: 1281 columns, BF16 -> MXFP4, 11840 items 21.5 / 23.0.)
bool wide(const cugl_context *ctx, const QuantParams &p)
{
    return p.cols >= 4 * kItemCols && static_cast<int64_t>(p.rows) * (p.cols / (4 * kItemCols)) >= 24ll * ctx->sm_count;
}
template <typename T, int kFormat, bool kBack, int kWhich>
cudaError_t launch_matrix(cugl_context *ctx, const QuantParams &p)
{
    if (p.vec_plain == 0)
    {
        return wide(ctx, p) ? launch_rows(ctx, mx_rows_kernel<T, kFormat, false, 4, 1, kBack, kWhich>, p, 4, 1)
                            : launch_rows(ctx, mx_rows_kernel<T, kFormat, false, 1, 1, kBack, kWhich>, p, 1, 1);
    }
    return wide(ctx, p) ? launch_rows(ctx, mx_rows_kernel<T, kFormat, true, 4, 1, kBack, kWhich>, p, 4, 1)
                        : launch_rows(ctx, mx_rows_kernel<T, kFormat, true, 1, 1, kBack, kWhich>, p, 1, 1);
}
template <typename T, bool kBack, int kWhich>
cudaError_t launch_matrix(cugl_context *ctx, int format, const QuantParams &p)
{
    return format == CUGL_NVFP4 ? launch_matrix<T, CUGL_NVFP4, kBack, kWhich>(ctx, p) : launch_matrix<T, CUGL_MXFP4, kBack, kWhich>(ctx, p);
}
template <bool kBack, int kWhich = kSame>
cudaError_t launch_matrix(cugl_context *ctx, const cugl_mx_desc &d, const QuantParams &p)
{
    return d.dtype == CUGL_F32 ? launch_matrix<float, kBack, kWhich>(ctx, d.format, p)
           : d.dtype == CUGL_F16 ? launch_matrix<__half, kBack, kWhich>(ctx, d.format, p)
                                 : launch_matrix<__nv_bfloat16, kBack, kWhich>(ctx, d.format, p);
}

const char *validate_mx(const cugl_mx_desc *d, cugl_status *code)
{
    *code = CUGL_INVALID_ARGUMENT;
    if (d == nullptr) return "descriptor is NULL";
    if (d->rows < 0 || d->cols < 1) return "rows must not be negative and cols must be positive";
    if (d->cols > INT32_MAX - 1024) return "cols is too large";
    if (d->rows > INT32_MAX - (1 << 20)) return "rows is too large"; // row numbers behind the last one stay within 32 bits
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

// the descriptor of the matrix whose rows the launch goes through, or the reason why it cannot
const char *validate_group(const cugl_mx_group_desc *d, cugl_mx_desc *m)
{
    if (d == nullptr) return "descriptor is NULL";
    if (d->tokens < 0 || d->rows < 0) return "tokens and rows must not be negative";
    if (d->top_k < 1 || d->top_k > 16) return "top_k must lie within 1 .. 16";
    if (static_cast<int64_t>(d->tokens) * d->top_k > INT32_MAX - (1 << 20)) return "tokens is too large";
    *m                 = cugl_mx_desc{};
    m->rows            = d->src_grouped != 0 ? d->tokens * d->top_k : d->tokens;
    m->cols            = d->cols;
    m->format          = d->format;
    m->dtype           = d->dtype;
    m->ld              = d->ld;
    m->ld_packed       = d->ld_packed;
    m->tensor_exponent = d->tensor_exponent;
    cugl_status code;
    return validate_mx(m, &code);
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
        p.src          = static_cast<const uint8_t *>(d_src);
        p.dst          = static_cast<uint8_t *>(d_dst);
        p.scales       = static_cast<uint8_t *>(d_scales);
        p.exponent_mul = std::ldexp(1.f, -desc->tensor_exponent);
        CUGL_CUDA_TRY(ctx, launch_matrix<false>(ctx, *desc, p));
        return CUGL_SUCCESS;
    }

    cugl_status cugl_mx_dequantize(cugl_context *ctx, const cugl_mx_desc *desc, const void *d_src, const void *d_scales, void *d_dst)
    {
        CUGL_TRY(check_mx(ctx, "cugl_mx_dequantize", desc, d_dst, d_src, d_scales));
        if (desc->rows == 0) return CUGL_SUCCESS;
        const DeviceScope device(ctx);
        QuantParams       p = make_params(*desc, d_dst, d_src);
        p.src          = static_cast<const uint8_t *>(d_src);
        p.dst          = static_cast<uint8_t *>(d_dst);
        p.scales       = const_cast<uint8_t *>(static_cast<const uint8_t *>(d_scales));
        p.exponent_mul = std::ldexp(1.f, desc->tensor_exponent);
        CUGL_CUDA_TRY(ctx, launch_matrix<true>(ctx, *desc, p));
        return CUGL_SUCCESS;
    }

    cugl_status cugl_mx_group_validate(const cugl_mx_group_desc *desc, const char **reason)
    {
        cugl_mx_desc m;
        const char  *why = validate_group(desc, &m);
        if (reason != nullptr)
        {
            *reason = why != nullptr ? why : "";
        }
        return why == nullptr ? CUGL_SUCCESS : CUGL_INVALID_ARGUMENT;
    }

    cugl_status cugl_mx_quantize_grouped(cugl_context *ctx, const cugl_mx_group_desc *desc, const void *d_src, const int32_t *d_slots, void *d_dst,
                                         void *d_scales)
    {
        if (ctx == nullptr)
        {
            return fail(nullptr, CUGL_INVALID_ARGUMENT, "context is NULL");
        }
        cugl_mx_desc m;
        const char  *why = validate_group(desc, &m);
        if (why == nullptr && desc->tokens > 0 && desc->rows > 0 && (d_slots == nullptr || !aligned(d_slots, 4))) why = "d_slots must be given, aligned to its elements";
        if (why != nullptr)
        {
            return fail(ctx, CUGL_INVALID_ARGUMENT, std::string("cugl_mx_quantize_grouped: ") + why);
        }
        if (desc->tokens == 0 || desc->rows == 0) return CUGL_SUCCESS;
        CUGL_TRY(check_mx(ctx, "cugl_mx_quantize_grouped", &m, d_src, d_dst, d_scales));
        const DeviceScope device(ctx);
        QuantParams       p = make_params(m, d_src, d_dst);
        p.src          = static_cast<const uint8_t *>(d_src);
        p.dst          = static_cast<uint8_t *>(d_dst);
        p.scales       = static_cast<uint8_t *>(d_scales);
        p.exponent_mul = std::ldexp(1.f, -desc->tensor_exponent);
        p.slots        = d_slots;
        p.top_k        = desc->top_k;
        p.group_rows   = desc->rows;
        p.wide_packed  = aligned(d_dst, 16) && desc->ld_packed % 16 == 0;
        CUGL_CUDA_TRY(ctx, (desc->src_grouped != 0 ? launch_matrix<false, kSlots>(ctx, m, p) : launch_matrix<false, kChoices>(ctx, m, p)));
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
