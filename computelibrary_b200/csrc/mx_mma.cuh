// Block-scaled tensor-core products (tcgen05.mma with E2M1 operands): what the product and the expert layer share.
//
// Operand roles: the weights are the 128 rows of an MMA (accumulator lanes = output channels), the tokens its columns, as few
// as sixteen -- so a product with one token uses the same instructions as one with thousands, and a warp that drains the
// accumulator stores 32 consecutive channels of a token.
//
// K is walked in chunks of 256 elements: rows of 128 bytes in the 128-byte swizzle, as TMA writes them.  One MMA takes 64
// elements (32 bytes of each row) and the scales of its four (NVFP4) or two (MXFP4) blocks per row, which tcgen05.cp has
// brought from shared to tensor memory: a scale tile of 512 bytes becomes four columns, repeated in the four lane quarters.
#pragma once

#include "mx.cuh"
#include "sm100.cuh"

#include <atomic>

namespace cugl
{
namespace
{
constexpr int kMxChunk      = 256;            // elements of K per pipeline stage
constexpr int kMxChunkBytes = kMxChunk / 2;   // one swizzle row
constexpr int kMxStepK      = 64;             // elements of K per MMA
constexpr int kMxRows       = 128;            // weight rows per MMA
constexpr int kMxWBytes     = kMxRows * kMxChunkBytes;

template <int kFormat>
struct MxTraits
{
    static constexpr int kChunkTiles = kFormat == CUGL_NVFP4 ? 4 : 2; // scale tiles per chunk and 128 rows
    static constexpr int kChunkScale = kChunkTiles * kMxTileBytes;
    static constexpr int kChunkCols  = kChunkTiles * 4;               // their tensor-memory columns
};

// Instruction descriptor of kind::mxf4 / mxf4nvf4: E2M1 operands (1) in bits 7 and 10, columns / 8 in 17..22, scale type in 23
// (0 E4M3, 1 E8M0), rows / 16 in 24..28.  The byte of the scale word an MMA starts at goes to bits 4..5 (columns' operand)
// and 29..30 (rows' operand), see mx_scale_id.
inline uint32_t mx_idesc(int format, int rows, int cols)
{
    return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(cols >> 3) << 17) | ((format == CUGL_MXFP4 ? 1u : 0u) << 23) |
           (static_cast<uint32_t>(rows >> 4) << 24);
}
template <int kFormat>
__device__ __forceinline__ constexpr uint32_t mx_scale_id(int step) // two MXFP4 steps share a tile
{
    return kFormat == CUGL_MXFP4 ? (static_cast<uint32_t>((step & 1) * 2) << 4) | (static_cast<uint32_t>((step & 1) * 2) << 29) : 0u;
}
template <int kFormat>
__device__ __forceinline__ constexpr int mx_step_tile(int step)
{
    return kFormat == CUGL_MXFP4 ? step >> 1 : step;
}

// D[tmem] (+)= sum over 64 elements of (A code * A scale) * (B code * B scale), float accumulation
template <int kFormat>
__device__ __forceinline__ void umma_mx(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scale, uint32_t b_scale,
                                        uint32_t accumulate)
{
    if constexpr (kFormat == CUGL_MXFP4)
    {
        asm volatile("{\n\t"
                     ".reg .pred p;\n\t"
                     "setp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
                     "}"
                     :
                     : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scale), "r"(b_scale), "r"(accumulate)
                     : "memory");
    }
    else
    {
        asm volatile("{\n\t"
                     ".reg .pred p;\n\t"
                     "setp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
                     "}"
                     :
                     : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scale), "r"(b_scale), "r"(accumulate)
                     : "memory");
    }
}

// The same across an SM pair: 256 rows (128 per CTA, each with the scales of its own rows) x up to 256 columns (half of them
// staged by each CTA, the scales of all of them by both).
template <int kFormat>
__device__ __forceinline__ void umma_mx_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scale, uint32_t b_scale,
                                             uint32_t accumulate)
{
    if constexpr (kFormat == CUGL_MXFP4)
    {
        asm volatile("{\n\t"
                     ".reg .pred p;\n\t"
                     "setp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
                     "}"
                     :
                     : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scale), "r"(b_scale), "r"(accumulate)
                     : "memory");
    }
    else
    {
        asm volatile("{\n\t"
                     ".reg .pred p;\n\t"
                     "setp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
                     "}"
                     :
                     : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scale), "r"(b_scale), "r"(accumulate)
                     : "memory");
    }
}

// One scale tile (32 rows of 16 bytes in shared memory) to four tensor-memory columns, in all four lane quarters.
__device__ __forceinline__ void tmem_copy_scales(uint32_t d_tmem, uint64_t s_desc)
{
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(d_tmem), "l"(s_desc) : "memory");
}
// in both CTAs of a pair, each from its own shared memory
__device__ __forceinline__ void tmem_copy_scales_pair(uint32_t d_tmem, uint64_t s_desc)
{
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(d_tmem), "l"(s_desc) : "memory");
}
// Descriptor of a scale tile: no swizzle, groups of eight 16-byte rows 128 bytes apart.
__device__ __forceinline__ uint64_t make_scale_desc(uint32_t smem_addr)
{
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3ffff) >> 4);
    d |= static_cast<uint64_t>(1) << 16;
    d |= static_cast<uint64_t>(128 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    return d;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :
                 : "r"(dst), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
                 : "memory");
}

// Asks for a box of a tensor map to be brought into L2.  A hint: what another kernel writes there later is seen by whoever reads
// after it, so it may run ahead of griddepcontrol.wait.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap *map, int c0, int c1)
{
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1) : "memory");
}

// The lane that issues a warp's tcgen05 and TMA instructions.  The issuing loops are run by the whole warp and only the
// instructions themselves are guarded by this predicate: control flow stays uniform, so that descriptors and addresses are
// computed in uniform registers, which these instructions take their operands from.  Under a branch on the lane index each of
// them has to be moved there first: a copy of scales then takes 46 clocks instead of 16, an MMA of 16 columns 50 instead of 39.
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t"
                 ".reg .pred p;\n\t"
                 "elect.sync _|p, 0xffffffff;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t"
                 "}"
                 : "=r"(p));
    return p != 0;
}
// mbar_wait by a whole warp, which takes the decision to give up together
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int code, long long limit)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, code, limit));
}

// one column of a warp's 32 accumulator lanes
__device__ __forceinline__ void tmem_ld_x1(uint32_t taddr, uint32_t &v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr) : "memory");
}

// 16 accumulator lanes x 32 columns in the fragment layout of the matrix instructions: v[4 i + 0, 1] are columns 8 i + 2 (lane % 4)
// and the next of row lane / 4, v[4 i + 2, 3] the same columns of row lane / 4 + 8.
__device__ __forceinline__ void tmem_ld_frag32(uint32_t taddr, uint32_t (&v)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(taddr)
                 : "memory");
}
// Four 8 x 8 matrices of 16-bit values, transposed on the way to shared memory: lane l gives the address of row l % 8 of the
// transposed matrix l / 8.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Of a kernel that has given up: waits for the copies still in flight into the last STAGES of `issued` stages (their full barriers
// start at `bars`; withheld: a stage whose copies were left out) before the CTA leaves its shared memory.  Copies take
// microseconds; the bound is there for one that never comes, and long enough whatever limit the caller set.
template <int STAGES>
__device__ __forceinline__ void drain_stages(uint32_t bars, int issued, int withheld, long long limit)
{
    for (int i = max(0, issued - STAGES); i < issued; ++i)
    {
        const long long t0 = clock64(), bound = limit + 2000000;
        while (i != withheld && !mbar_try_wait(bars + 8u * (i % STAGES), static_cast<uint32_t>(i / STAGES) & 1u) && clock64() - t0 <= bound)
        {
        }
    }
    __syncwarp();
}

// Of a kernel that has given up, by the warp that issues its tcgen05 instructions: MMAs and copies of scales may still be reading
// shared and writing tensor memory, and their commits are still to arrive on this CTA's barriers.  Commits all of them once more to
// a barrier of its own and waits for it, before the tensor memory is freed and the CTA leaves.  (A commit covers what its thread
// has issued; elect.sync names the same lane every time.)  kPair: by the leader of an SM pair, whose barriers both get the arrival.
template <bool kPair>
__device__ __forceinline__ void drain_mmas(uint32_t bar, long long limit)
{
    if (elect_one())
    {
        if constexpr (kPair) umma_commit_pair(bar);
        else umma_commit(bar);
    }
    __syncwarp();
    const long long t0 = clock64(), bound = limit + 2000000;
    while (!mbar_try_wait(bar, 0) && clock64() - t0 <= bound)
    {
    }
    __syncwarp();
}

// drain_stages of an SM pair, by its leader, whose barriers count the copies of both CTAs: the producers may have stopped at different
// stages, so what the barrier of a stage that only one of them has filled still expects, or does not expect yet, is put right first.
// bytes: of one CTA's copies of a stage.  (The counts are at most STAGES apart: both wait for the same MMAs.)
template <int STAGES, typename Bytes>
__device__ __forceinline__ void drain_pair_stages(uint32_t bars, int issued, int peer, int withheld, long long limit, Bytes bytes)
{
    const int end = max(issued, peer);
    for (int i = max(0, end - STAGES); i < end; ++i)
    {
        const uint32_t bar = bars + 8u * (i % STAGES);
        const bool     own = i < issued && i != withheld, other = i < peer;
        if (own != other && elect_one())
        {
            if (own) mbar_complete_tx(bar, bytes(i)); // expected, but the peer never asked for it
            else mbar_expect_tx(bar, bytes(i));       // the other way round
        }
        __syncwarp();
        const long long t0 = clock64(), bound = limit + 2000000;
        while ((own || other) && !mbar_try_wait(bar, static_cast<uint32_t>(i / STAGES) & 1u) && clock64() - t0 <= bound)
        {
        }
    }
    __syncwarp();
}

// The MMAs of one chunk whose operands and scales have landed in shared memory.  steps: MMAs inside K (1 .. 4).  a_stage,
// b_stage: shared addresses of the operands; a_sf, b_sf: of their scale tiles; t_a, t_b: tensor-memory columns for those.
template <int kFormat>
__device__ __forceinline__ void mx_chunk(uint32_t d_tmem, uint32_t a_stage, uint32_t b_stage, uint32_t t_a, uint32_t t_b, uint32_t idesc, int steps,
                                         bool first)
{
    const uint64_t a_desc = make_kmajor_sw128_desc(a_stage), b_desc = make_kmajor_sw128_desc(b_stage);
#pragma unroll
    for (int k = 0; k < kMxChunk / kMxStepK; ++k)
    {
        if (k < steps)
        {
            const uint32_t col = static_cast<uint32_t>(mx_step_tile<kFormat>(k) * 4);
            umma_mx<kFormat>(d_tmem, a_desc + 2u * k, b_desc + 2u * k, idesc | mx_scale_id<kFormat>(k), t_a + col, t_b + col,
                             first && k == 0 ? 0u : 1u);
        }
    }
}
template <int kFormat>
__device__ __forceinline__ void mx_chunk_scales(uint32_t t_dst, uint32_t sf, int tiles)
{
    const uint64_t desc = make_scale_desc(sf);
#pragma unroll
    for (int t = 0; t < MxTraits<kFormat>::kChunkTiles; ++t)
    {
        if (t < tiles)
        {
            tmem_copy_scales(t_dst + 4 * t, desc + static_cast<uint64_t>(t * (kMxTileBytes >> 4)));
        }
    }
}

// First chunk of a rank's share of K.
__device__ __forceinline__ int chunk_share(int chunks, int rank, int ranks)
{
    return static_cast<int>(static_cast<int64_t>(chunks) * rank / ranks);
}

// Partial sums of a cluster whose 2^shift CTAs shared an accumulator's K.  Rank r owns channels r * (128 >> shift) and up.  The
// warp that drains 32 lanes of an accumulator writes them to the owners' shared memory, [rank][columns / 4][channel][4 columns],
// sixteen bytes per lane, and arrives on the owners' barrier; an owner that has all arrivals adds the parts up in the order of
// the ranks, the same every time.  stride: columns of a part.
// warps: of a CTA that drain the accumulator, one or two per lane quarter.  An owner's channels lie in one quarter or several.
__device__ __forceinline__ int partial_arrivals(int shift, int warps)
{
    return (1 << shift) * max(1, (kMxRows >> shift) / 32) * (warps / 4);
}
__device__ __forceinline__ uint32_t partial_address(uint32_t s_base, int ch, int rank, int shift, int stride)
{
    const int own = kMxRows >> shift;
    return map_to_cta(s_base, static_cast<uint32_t>(ch / own)) + 4u * static_cast<uint32_t>(rank * stride * own) + 16u * static_cast<uint32_t>(ch & (own - 1));
}
__device__ __forceinline__ void send_partial(uint32_t to, int shift, const uint32_t (&r)[16], int cols, bool has)
{
#pragma unroll
    for (int i = 0; i < 16; i += 4)
    {
        if (i < cols) // a rank without a share of K has no accumulator: zeros
        {
            st_cluster_v4(to + static_cast<uint32_t>(i) * (4u * kMxRows >> shift), has ? r[i] : 0u, has ? r[i + 1] : 0u, has ? r[i + 2] : 0u,
                          has ? r[i + 3] : 0u);
        }
    }
}
__device__ __forceinline__ void arrive_partial(uint32_t bar, int ch, int shift)
{
    __syncwarp();
    if ((ch & (min(kMxRows >> shift, 32) - 1)) == 0)
    {
        mbar_arrive_cluster(map_to_cta(bar, static_cast<uint32_t>(ch / (kMxRows >> shift))));
    }
}
// Four columns of one channel; at: (columns / 4) * (128 >> shift) + channel of the owner.
__device__ __forceinline__ float4 sum_partial(const float *part, int at, int shift, int stride)
{
    const float4 *p   = reinterpret_cast<const float4 *>(part) + at;
    const int     gap = stride * (kMxRows >> shift) / 4;
    float4        v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        if (i < (1 << shift)) v[i] = p[i * gap];
    }
    float4 sum = v[0];
#pragma unroll
    for (int i = 1; i < 8; ++i)
    {
        if (i < (1 << shift)) sum.x += v[i].x, sum.y += v[i].y, sum.z += v[i].z, sum.w += v[i].w;
    }
    return sum;
}

// silu(g) * u of gates far below zero, where 1 / (1 + exp(-g)) is exp(g) to 32 bits.  From -87 down that reciprocal is subnormal, and the
// fast divisions make it 0, while the result is a normal number for as long as u is large enough: hence exp(g) as the square of
// h = exp(g / 2), half of it on either factor.  h is normal down to g = -174, where the result is below 2^-115 whatever u is.
constexpr float kSiluTail = -80.f;
__device__ __forceinline__ float swiglu_tail(float g, float u)
{
    const float h = expf(0.5f * g);
    return (g * h) * (h * u);
}

// scale tiles as rows of 512 bytes; box = box_rows tiles
inline bool encode_scale_map(CUtensorMap *map, const void *base, int64_t tiles, int box_rows)
{
    EncodeTiledFn fn = get_encode_fn();
    if (fn == nullptr)
    {
        return false;
    }
    const cuuint64_t dims[2]    = {kMxTileBytes / 4, static_cast<cuuint64_t>(tiles)};
    const cuuint64_t strides[1] = {kMxTileBytes};
    const cuuint32_t box[2]     = {kMxTileBytes / 4, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estr[2]    = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// CTAs (a power of two up to `most`) that share the K of each of `tiles` tiles as a cluster.  With two CTAs to an SM the device
// holds 148 clusters of two, 71 of four or 33 of eight at once (cudaOccupancyMaxActiveClusters; clusters do not cross the
// boundaries between groups of SMs); one cluster more would run alone after all others.
inline int mx_split(long long tiles, int chunks, int most)
{
    if (most >= 8 && tiles <= 33 && chunks >= 8) return 8;
    if (most >= 4 && tiles <= 71 && chunks >= 4) return 4;
    if (most >= 2 && tiles <= 148 && chunks >= 2) return 2;
    return 1;
}

// Lets a kernel have its dynamic shared memory, once per device: set is the kernel's own.  Threads with contexts of their own may come
// here at once; each then sets the attribute, to the same value.
template <typename K>
cugl_status allow_smem(cugl_context *ctx, K kernel, int bytes, std::atomic<bool> (&set)[64])
{
    if (!set[ctx->device & 63].load(std::memory_order_acquire))
    {
        CUGL_CUDA_TRY(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        set[ctx->device & 63].store(true, std::memory_order_release);
    }
    return CUGL_SUCCESS;
}

// packed rows x (inner bytes), ld bytes apart; box = box_rows x 128 bytes in the 128-byte swizzle; what lies outside reads as 0
inline bool encode_packed_map(CUtensorMap *map, const void *base, int64_t rows, int64_t inner, int64_t ld, int box_rows)
{
    EncodeTiledFn fn = get_encode_fn();
    if (fn == nullptr)
    {
        return false;
    }
    const cuuint64_t dims[2]    = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
    const cuuint32_t box[2]     = {kMxChunkBytes, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estr[2]    = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
} // namespace
} // namespace cugl
