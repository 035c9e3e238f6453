// Product of two microscaled 4-bit matrices on the tensor cores: dst[m][n] = alpha * sum_k a[m][k] * b[n][k] + bias[n].
//
//   warp 0      TMA: 128 rows of weights (b) and NT rows of tokens (a), 128 bytes (256 elements) of each per stage, and the
//               scale tiles that belong to them as plain bulk copies
//   warp 1      copies the stage's scales to tensor memory and issues its MMAs (M = 128, N = NT, K = 64)
//   warps 2..   a tensor-memory lane quarter each (or half of its columns): accumulator * alpha + bias, rounded once, stored
//               as 32 consecutive channels per token
//
// Every stage has scale columns of its own in tensor memory: they are written again only after the stage's MMAs have been
// committed, like its shared memory.
//
// What bounds it: few tokens, the weights' bytes and the latency of one launch (1 x 4096 x 4096 NVFP4, 9.4 MB: 4.7 us in a
// captured run, 1.5 us at the copy rate; 24 x 14336 x 4096 MXFP4, 31 MB: 8.4 to 8.8 us, 3.6 TB/s).  Hence 64 to 74 KB of operands in
// flight per CTA, two CTAs per SM, K shared by a cluster where there are few tiles, and weights asked for before the launch
// ahead has ended.  Many tokens, the tensor cores: see the SM-pair kernel below.
#include "mx_mma.cuh"

#include <cstring>

namespace cugl
{
namespace
{
constexpr int kMmaWarp  = 1;
constexpr int kFirstEpi = 2;
constexpr int kPrefetch = 16; // chunks, 256 KB of weights per CTA

struct MxGemmParams
{
    const uint8_t *w_scales, *t_scales;
    uint8_t       *dst;
    const float   *bias;
    int64_t        ldd;
    int64_t        k_tiles; // scale tiles along K
    int            tokens, channels, K;
    int            dtype;
    int            pack_out; // two-byte results: rows of dst are words (4-byte aligned, an even number of channels)
    float          alpha;
    uint32_t       idesc, idesc_half; // SM pair: of a whole tile and of half a tile
    int            whole;             // SM pair: tiles that are not split
    int32_t       *status;
    long long      spin_limit;
    int            withhold; // see cugl_context_withhold_copy_once
};

template <int kFormat, int NT, int STAGES, bool kSplit>
struct MxPlan
{
    using F                          = MxTraits<kFormat>;
    // Epilogue warps: one per tensor-memory lane quarter, two where a tile has 64 columns or more (a warp has a scheduler
    // to itself and waits for its own instructions most of the time).
    static constexpr int EPI         = NT >= 64 ? 8 : 4;
    static constexpr int THREADS     = 32 * (kFirstEpi + EPI);
    static constexpr int T_BYTES     = NT * kMxChunkBytes;
    static constexpr int STAGE       = kMxWBytes + T_BYTES;
    static constexpr int SF_STAGE    = 2 * F::kChunkScale;
    static constexpr int OFF_SF      = STAGES * STAGE;
    // the partial sums of a cluster: an area of their own where there is room, else where the stages were
    static constexpr bool OWN_PART   = NT <= 32;
    [[maybe_unused]] static constexpr int OFF_PART    = OWN_PART ? OFF_SF + STAGES * SF_STAGE : 0;
    static constexpr int OFF_BAR     = OFF_SF + STAGES * SF_STAGE + (kSplit && OWN_PART ? NT * kMxRows * 4 : 0);
    static constexpr int OFF_MISC    = OFF_BAR + (2 * STAGES + 6) * 8;
    static constexpr int DYN_BYTES   = OFF_MISC + 16 + 1024;
    static constexpr int ACC         = kSplit || NT == 128 ? 1 : 2; // accumulators
    static constexpr int SF_COLS     = 2 * F::kChunkCols; // per stage
    static constexpr int COLS        = ACC * NT + STAGES * SF_COLS;
    static constexpr int TMEM_COLS   = COLS <= 32 ? 32 : COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    static_assert(TMEM_COLS <= 256 && DYN_BYTES <= 115200, "half the tensor and shared memory of an SM: two CTAs share it");
    static_assert(STAGES * STAGE >= NT * kMxRows * 4, "the partial sums of a cluster fit where the stages were");
};

// N accumulator columns (tokens m, m + 1, ..) of a lane's channel n to dst.  Two-byte results of neighbouring channels leave as
// one word: lanes exchange a column each, after which the even lane of a pair holds both channels of the first token and the
// odd lane those of the second.
template <typename T, int N>
__device__ __forceinline__ void store_block(const MxGemmParams &p, int m, int n, const uint32_t (&r)[N], int cols, float bias)
{
    uint8_t *dst = p.dst + static_cast<int64_t>(m) * p.ldd + static_cast<int64_t>(n) * static_cast<int>(sizeof(T));
    if (sizeof(T) == 2 && p.pack_out != 0)
    {
        const int odd = n & 1;
        dst += odd != 0 ? p.ldd - 2 : 0;
#pragma unroll
        for (int j = 0; j < N; j += 2)
        {
            const float a = __fmaf_rn(__uint_as_float(r[j]), p.alpha, bias), b = __fmaf_rn(__uint_as_float(r[j + 1]), p.alpha, bias);
            const float got = __shfl_xor_sync(0xffffffffu, odd != 0 ? a : b, 1);
            T           two[2] = {from_float<T>(odd != 0 ? got : a), from_float<T>(odd != 0 ? b : got)};
            if (j + odd < cols && n < p.channels)
            {
                *reinterpret_cast<uint32_t *>(dst + j * p.ldd) = *reinterpret_cast<const uint32_t *>(two);
            }
        }
        __syncwarp(); // aligned loads of tensor memory may be next
        return;
    }
    if (n < p.channels)
    {
#pragma unroll
        for (int j = 0; j < N; ++j)
        {
            if (j < cols) *reinterpret_cast<T *>(dst + j * p.ldd) = from_float<T>(__fmaf_rn(__uint_as_float(r[j]), p.alpha, bias));
        }
    }
    __syncwarp();
}
template <int N>
__device__ __forceinline__ void store_block(const MxGemmParams &p, int m, int n, const uint32_t (&r)[N], int cols, float bias)
{
    if (p.dtype == CUGL_F32) store_block<float>(p, m, n, r, cols, bias);
    else if (p.dtype == CUGL_F16) store_block<__half>(p, m, n, r, cols, bias);
    else store_block<__nv_bfloat16>(p, m, n, r, cols, bias);
}

// four tokens of one channel
template <typename T>
__device__ __forceinline__ void store_four(const MxGemmParams &p, int m, int n, const float4 &v, int cols, float bias)
{
    uint8_t    *dst  = p.dst + static_cast<int64_t>(m) * p.ldd + static_cast<int64_t>(n) * static_cast<int>(sizeof(T));
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
    {
        if (j < cols) *reinterpret_cast<T *>(dst + j * p.ldd) = from_float<T>(__fmaf_rn(f[j], p.alpha, bias));
    }
}
__device__ __forceinline__ void store_four(const MxGemmParams &p, int m, int n, const float4 &v, int cols, float bias)
{
    if (p.dtype == CUGL_F32) store_four<float>(p, m, n, v, cols, bias);
    else if (p.dtype == CUGL_F16) store_four<__half>(p, m, n, v, cols, bias);
    else store_four<__nv_bfloat16>(p, m, n, v, cols, bias);
}

template <int kFormat, int NT, int STAGES, bool kSplit>
__global__ void __launch_bounds__((MxPlan<kFormat, NT, STAGES, kSplit>::THREADS), 2)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_t, const __grid_constant__ MxGemmParams p)
{
    using P = MxPlan<kFormat, NT, STAGES, kSplit>;
    using F = MxTraits<kFormat>;
    constexpr int kEpi = P::EPI;
    extern __shared__ uint8_t smem_raw[];
    uint8_t       *smem      = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t s_stage   = smem_u32(smem);
    const uint32_t s_sf      = smem_u32(smem + P::OFF_SF);
    const uint32_t bar_base  = smem_u32(smem + P::OFF_BAR);
    auto           full_bar  = [&](int s) { return bar_base + 8u * s; };
    auto           empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto           tfull_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
    auto           tempty_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + 2 + a); };
    const uint32_t part_bar  = bar_base + 8u * (2 * STAGES + 4);
    const uint32_t gone_bar  = bar_base + 8u * (2 * STAGES + 5); // see drain_mmas
    uint32_t      *s_tmem    = reinterpret_cast<uint32_t *>(smem + P::OFF_MISC);
    volatile int  *s_abort   = reinterpret_cast<volatile int *>(smem + P::OFF_MISC + 4);
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int w_blocks = (p.channels + kMxRows - 1) / kMxRows;
    const int t_blocks = (p.tokens + NT - 1) / NT;
    const int tiles    = w_blocks * t_blocks;
    const int chunks   = (p.K + kMxChunk - 1) / kMxChunk;
    // the CTAs of a cluster share one tile's K; without split a CTA works through its tiles
    const int rank        = kSplit ? static_cast<int>(cluster_ctarank()) : 0;
    const int ranks       = kSplit ? static_cast<int>(gridDim.x) / static_cast<int>(num_clusters_x()) : 1;
    const int first_tile  = kSplit ? static_cast<int>(cluster_id_x()) : static_cast<int>(blockIdx.x);
    const int tile_stride = kSplit ? tiles : static_cast<int>(gridDim.x);
    const int c_begin     = chunk_share(chunks, rank, ranks);
    const int c_end       = chunk_share(chunks, rank + 1, ranks);

    if (threadIdx.x == 0)
    {
        for (int s = 0; s < STAGES; ++s)
        {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a)
        {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), kEpi);
        }
        mbar_init(part_bar, partial_arrivals(31 - __clz(ranks), kEpi));
        mbar_init(gone_bar, 1);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp)
    {
        tmem_alloc(smem_u32(s_tmem), P::TMEM_COLS);
    }
    tc_fence_before();
    __syncthreads();
    if (kSplit)
    {
        cluster_sync(); // every CTA runs and has its barriers before anything is sent to it
    }
    tc_fence_after();
    const uint32_t tmem_base = *s_tmem;
    griddep_launch_dependents();
    if (warp == 0 && first_tile < tiles)
    {
        // The weights of the first tile start on their way from memory while the kernels ahead finish: bringing them into L2
        // reads nothing that those kernels could still change.
        const bool el = elect_one();
        for (int c = c_begin; c < min(c_end, c_begin + kPrefetch); ++c)
        {
            if (el) tma_prefetch_2d(&tmap_w, c * kMxChunkBytes, first_tile % w_blocks * kMxRows);
            __syncwarp();
        }
    }
    griddep_wait(); // everything else touches global memory after the kernels ahead

    int issued = 0; // stages that the producer has filled
    if (warp == 0)
    {
        const bool el = elect_one();
        int g = 0;
        for (int tile = first_tile; tile < tiles; tile += tile_stride)
        {
            const int      wb = tile % w_blocks, tb = tile / w_blocks;
            const uint8_t *w_sf = p.w_scales + static_cast<int64_t>(wb) * p.k_tiles * kMxTileBytes;
            const uint8_t *t_sf = p.t_scales + static_cast<int64_t>(tb) * p.k_tiles * kMxTileBytes; // NT < 128: one block only
            for (int c = c_begin; c < c_end; ++c, ++g)
            {
                const int s = g % STAGES;
                if (!warp_wait(empty_bar(s), (static_cast<uint32_t>(g / STAGES) & 1u) ^ 1u, s_abort, DEV_TIMEOUT_PRODUCER, p.spin_limit))
                {
                    goto produced;
                }
                if (g == p.withhold && blockIdx.x == 0)
                {
                    continue;
                }
                const int      first = c * F::kChunkTiles;
                const int      n     = min(F::kChunkTiles, static_cast<int>(p.k_tiles) - first);
                const uint32_t bytes = static_cast<uint32_t>(n) * kMxTileBytes;
                const uint32_t dst   = s_stage + s * P::STAGE, sf = s_sf + s * P::SF_STAGE;
                if (el)
                {
                    mbar_expect_tx(full_bar(s), P::STAGE + 2 * bytes);
                    tma_load_2d(dst, &tmap_w, c * kMxChunkBytes, wb * kMxRows, full_bar(s));
                    tma_load_2d(dst + kMxWBytes, &tmap_t, c * kMxChunkBytes, tb * NT, full_bar(s));
                    bulk_load(sf, w_sf + static_cast<int64_t>(first) * kMxTileBytes, bytes, full_bar(s));
                    bulk_load(sf + F::kChunkScale, t_sf + static_cast<int64_t>(first) * kMxTileBytes, bytes, full_bar(s));
                }
                __syncwarp();
            }
        }
    produced:
        issued = g;
    }
    else if (warp == kMmaWarp)
    {
        const bool el = elect_one();
        int  g = 0, it = 0;
        bool ok = true;
        for (int tile = first_tile; tile < tiles && ok; tile += tile_stride, ++it)
        {
            const int as = it % P::ACC;
            ok = warp_wait(tempty_bar(as), (static_cast<uint32_t>(it / P::ACC) & 1u) ^ 1u, s_abort, DEV_TIMEOUT_MMA, p.spin_limit);
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + as * NT;
            for (int c = c_begin; c < c_end && ok; ++c, ++g)
            {
                const int s = g % STAGES;
                ok = warp_wait(full_bar(s), static_cast<uint32_t>(g / STAGES) & 1u, s_abort, DEV_TIMEOUT_MMA, p.spin_limit);
                if (!ok) break;
                tc_fence_after();
                const int      n     = min(F::kChunkTiles, static_cast<int>(p.k_tiles) - c * F::kChunkTiles);
                const int      steps = min(kMxChunk / kMxStepK, (p.K - c * kMxChunk + kMxStepK - 1) / kMxStepK);
                const uint32_t t_w   = tmem_base + P::ACC * NT + s * P::SF_COLS, t_t = t_w + F::kChunkCols;
                const uint32_t sf    = s_sf + s * P::SF_STAGE;
                if (el)
                {
                    mx_chunk_scales<kFormat>(t_w, sf, n);
                    mx_chunk_scales<kFormat>(t_t, sf + F::kChunkScale, n);
                    mx_chunk<kFormat>(d_tmem, s_stage + s * P::STAGE, s_stage + s * P::STAGE + kMxWBytes, t_w, t_t, p.idesc, steps, c == c_begin);
                    umma_commit(empty_bar(s));
                }
                __syncwarp();
            }
            if (ok && el)
            {
                umma_commit(tfull_bar(as));
            }
        }
        __syncwarp();
    }
    else if (!kSplit)
    {
        const int q = warp & 3, half = (warp - kFirstEpi) >> 2;
        int       it = 0;
        for (int tile = first_tile; tile < tiles; tile += tile_stride, ++it)
        {
            const int   wb = tile % w_blocks, tb = tile / w_blocks;
            const int   as = it % P::ACC;
            const int   n  = wb * kMxRows + q * 32 + lane;
            const float b  = p.bias != nullptr && n < p.channels ? __ldg(p.bias + n) : 0.f;
            if (!warp_wait(tfull_bar(as), static_cast<uint32_t>(it / P::ACC) & 1u, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit))
            {
                break;
            }
            tc_fence_after();
            const int cols = min(NT, p.tokens - tb * NT);
            for (int j = 16 * half; j < cols; j += 4 * kEpi)
            {
                uint32_t r[16];
                tmem_ld_x16(tmem_base + as * NT + j + (static_cast<uint32_t>(q * 32) << 16), r);
                tmem_ld_wait();
                store_block(p, tb * NT + j, n, r, cols - j, b);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty_bar(as));
        }
    }

    if constexpr (kSplit)
    {
        const int  tile = first_tile, wb = tile % w_blocks, tb = tile / w_blocks;
        const int  cols = min(NT, p.tokens - tb * NT), shift = 31 - __clz(ranks);
        const int  q = warp & 3, half = (warp - kFirstEpi) >> 2;
        bool       ok = true;
        if (warp >= kFirstEpi)
        {
            ok = warp_wait(tfull_bar(0), 0, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit);
            tc_fence_after();
        }
        if (!P::OWN_PART)
        {
            __syncthreads();
            cluster_sync(); // every CTA's MMAs have read their last stage
        }
        const uint32_t s_part = smem_u32(smem + P::OFF_PART);
        if (warp >= kFirstEpi && ok)
        {
            const int      ch = q * 32 + lane;
            const uint32_t to = partial_address(s_part, ch, rank, shift, NT);
            for (int j = 16 * half; j < cols; j += 4 * kEpi)
            {
                uint32_t r[16];
                tmem_ld_x16(tmem_base + j + (static_cast<uint32_t>(q * 32) << 16), r);
                tmem_ld_wait();
                send_partial(to + static_cast<uint32_t>(j) * (4u * kMxRows >> shift), shift, r, cols - j, c_begin < c_end);
            }
            arrive_partial(part_bar, ch, shift);
            ok = __all_sync(0xffffffffu, mbar_wait_cluster(part_bar, 0, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit));
        }
        if (warp >= kFirstEpi && ok)
        {
            const int    own = kMxRows >> shift, et = threadIdx.x - 32 * kFirstEpi;
            const int    n = wb * kMxRows + rank * own + (et & (own - 1));
            const float  b = p.bias != nullptr && n < p.channels ? __ldg(p.bias + n) : 0.f;
            const float *part = reinterpret_cast<const float *>(smem + P::OFF_PART);
            if (n < p.channels)
            {
                for (int at = et; at < (cols + 3) / 4 * own; at += 32 * kEpi)
                {
                    const int    j = (at >> (7 - shift)) * 4;
                    const float4 v = sum_partial(part, at, shift, NT);
                    store_four(p, tb * NT + j, n, v, cols - j, b);
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 0 && *s_abort != 0)
    {
        drain_stages<STAGES>(bar_base, issued, blockIdx.x == 0 ? p.withhold : -1, p.spin_limit);
    }
    if (warp == kMmaWarp)
    {
        if (*s_abort != 0) drain_mmas<false>(gone_bar, p.spin_limit);
        tc_fence_after();
        tmem_dealloc(tmem_base, P::TMEM_COLS);
    }
    if (kSplit && *s_abort != 0)
    {
        cluster_sync(); // this CTA may not have received all parts: it stays until the others have left or given up too
    }
    if (threadIdx.x == 0 && *s_abort != 0)
    {
        atomicCAS(p.status, 0, *s_abort);
    }
}

// ---- SM pair -------------------------------------------------------------------------------------------------
// 256 channels x 256 tokens per cluster of two CTAs: each stages its own 128 weight rows and half of the tokens, and the MMAs
// (M = 256, N = 256) of the leader read both halves -- 64 instead of 96 bytes from L2 per clock of tensor work and SM.  The
// scales of all 256 tokens go to both CTAs; they come as boxes of a tensor map because the bytes of both CTAs are credited to
// the leader's barrier.
// What bounds it: power.  4096 x 14336 x 4096 NVFP4 takes 96 us by itself (5.0 PFLOP/s) and 112 to 116 back to back, where the
// clock falls to 1.3 GHz; with operands of zeros K = 16384 runs at 7.1 PFLOP/s, with random ones at 5.65.
// Tensor memory: two accumulators of 256 columns that share 64 (0 .. 255 and 192 .. 447), so that the rest holds the scales of
// one chunk.  A chunk's scales overwrite those of the chunk before, by copies issued behind the MMAs that read them.  PTX lists copy
// before MMA among the pairs of tcgen05 instructions that keep the order of their issue, but not MMA before copy: this rests on one
// thread's copies and MMAs going through one queue, as public block-scaled main loops rely on too, and on every test of a tile with
// several chunks.  (Two sets of columns in turn, each copied to only after the commit of the MMAs that read it, cost a
// tenth: 4096 x 14336 x 4096 100 -> 110 us, 512 x 4096 x 4096 10.0 -> 11.3.)
// The epilogue drains the shared columns first; the next tile's MMAs start when it has, and the rest of the drain runs beside
// them.
// kBulk: blocks of 32 channels x 32 tokens leave through a warp's staging area as one bulk tensor store (rows of dst 16-byte
// aligned and whole 16-byte units long); two-byte results (kBulk = 2) are transposed by stmatrix on the way, floats (4) are
// stored as they lie.  A quarter of the instructions of stores from registers: 4096 x 14336 x 1024 to BF16 73 -> 44 us.
constexpr int kPairCols   = 256;
constexpr int kPairShared = 64;
constexpr int kPairEpi    = 8; // epilogue warps
constexpr int kPairThreads = 32 * (kFirstEpi + kPairEpi);

// Order of the tiles: strips of four blocks of channels, walked token block by token block, so that the tiles in flight share
// both operands in L2 and on the way to the SMs (channel blocks all the way: 4096 x 14336 x 16384 NVFP4 405 us, strips 346;
// K = 4096 101 and 102).
constexpr int kPairStrip = 4;

// Tiles of a last wave that fills at most half of the SM pairs are worked on as two halves of 128 tokens.  Items: whole tiles, then
// the halves.
struct PairItem
{
    int tile, half; // -1: whole
};
__device__ __forceinline__ PairItem pair_item(int item, int whole)
{
    return item < whole ? PairItem{item, -1} : PairItem{whole + ((item - whole) >> 1), (item - whole) & 1};
}
__device__ __forceinline__ void pair_tile(int tile, int w_blocks, int t_blocks, int &wb, int &tb)
{
    const int strip = tile / (kPairStrip * t_blocks), in = tile - strip * kPairStrip * t_blocks;
    const int width = min(kPairStrip, w_blocks - strip * kPairStrip);
    tb              = in / width;
    wb              = strip * kPairStrip + in - tb * width;
}

template <int kFormat>
struct MxPairPlan
{
    using F                       = MxTraits<kFormat>;
    static constexpr int STAGES   = 5;
    static constexpr int STAGE    = 2 * kMxWBytes;
    static constexpr int SF_STAGE = 3 * F::kChunkScale;
    static constexpr int OFF_OUT  = STAGES * STAGE; // staging: 4 KB per epilogue warp
    static constexpr int OFF_SF   = OFF_OUT + kPairEpi * 4096;
    static constexpr int OFF_BAR  = OFF_SF + STAGES * SF_STAGE;
    static constexpr int OFF_MISC = OFF_BAR + (2 * STAGES + 4) * 8;
    static constexpr int DYN_BYTES = OFF_MISC + 16 + 1024;
    static constexpr int SF_COL   = 2 * kPairCols - kPairShared;
    static_assert(SF_COL + 3 * F::kChunkCols <= 512 && DYN_BYTES <= 232448, "tensor and shared memory of an SM");
};

// 32 channels x 32 tokens of an accumulator (two halves of 16 lanes as fragments) to a staging area of 32 rows of 64 bytes in
// the 64-byte swizzle.  bias: of channels lane / 4 + 8 i.
template <typename T>
__device__ __forceinline__ void stage_block(uint32_t s_out, int lane, const uint32_t (&lo)[16], const uint32_t (&hi)[16], float alpha, const float (&bias)[4])
{
    auto pack = [&](uint32_t a, uint32_t b, float c) {
        const T  two[2] = {from_float<T>(__fmaf_rn(__uint_as_float(a), alpha, c)), from_float<T>(__fmaf_rn(__uint_as_float(b), alpha, c))};
        uint32_t w;
        memcpy(&w, two, 4);
        return w;
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) // eight tokens: matrix m holds channels 8 m .. 8 m + 7
    {
        const int      row  = 8 * i + (lane & 7), chunk = lane >> 3;
        const uint32_t addr = s_out + static_cast<uint32_t>(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
        stmatrix_x4_trans(addr, pack(lo[4 * i], lo[4 * i + 1], bias[0]), pack(lo[4 * i + 2], lo[4 * i + 3], bias[1]),
                          pack(hi[4 * i], hi[4 * i + 1], bias[2]), pack(hi[4 * i + 2], hi[4 * i + 3], bias[3]));
    }
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

template <int kFormat, int kBulk>
__global__ void __launch_bounds__(kPairThreads, 1)
    mx_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_t,
                        const __grid_constant__ CUtensorMap tmap_half,
                        const __grid_constant__ CUtensorMap tmap_wsf, const __grid_constant__ CUtensorMap tmap_tsf,
                        const __grid_constant__ CUtensorMap tmap_out, const __grid_constant__ MxGemmParams p)
{
    using P = MxPairPlan<kFormat>;
    using F = MxTraits<kFormat>;
    constexpr int STAGES = P::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t       *smem      = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t s_stage   = smem_u32(smem);
    const uint32_t s_sf      = smem_u32(smem + P::OFF_SF);
    const uint32_t bar_base  = smem_u32(smem + P::OFF_BAR);
    auto           full_bar  = [&](int s) { return bar_base + 8u * s; };            // used in the leader only
    auto           empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto           tfull_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
    const uint32_t tempty    = bar_base + 8u * (2 * STAGES + 2);                    // shared columns drained; leader only
    const uint32_t gone_bar  = bar_base + 8u * (2 * STAGES + 3);                    // see drain_mmas
    uint32_t      *s_tmem    = reinterpret_cast<uint32_t *>(smem + P::OFF_MISC);
    volatile int  *s_abort   = reinterpret_cast<volatile int *>(smem + P::OFF_MISC + 4);
    uint32_t      *s_peer    = reinterpret_cast<uint32_t *>(smem + P::OFF_MISC + 8); // stages the peer has filled; bit 31: it has given up
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int      rank = static_cast<int>(cluster_ctarank());

    const int w_blocks = (p.channels + 2 * kMxRows - 1) / (2 * kMxRows);
    const int t_blocks = (p.tokens + kPairCols - 1) / kPairCols;
    const int items    = p.whole + 2 * (w_blocks * t_blocks - p.whole);
    const int chunks   = (p.K + kMxChunk - 1) / kMxChunk;
    const int first    = static_cast<int>(cluster_id_x());
    const int stride   = static_cast<int>(num_clusters_x());

    if (threadIdx.x == 0)
    {
        for (int s = 0; s < STAGES; ++s)
        {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(tfull_bar(0), 1);
        mbar_init(tfull_bar(1), 1);
        mbar_init(tempty, 2 * kPairEpi);
        mbar_init(gone_bar, 1);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp)
    {
        tmem_alloc_pair(smem_u32(s_tmem), 512);
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync(); // the peer's barriers are initialised before anything is sent to them
    tc_fence_after();
    const uint32_t tmem_base = *s_tmem;
    griddep_launch_dependents();
    griddep_wait(); // the prologue above touched no global memory

    int issued = 0; // stages that the producer has filled
    if (warp == 0)
    {
        const bool el = elect_one();
        int g = 0;
        for (int v = first; v < items; v += stride)
        {
            const PairItem item = pair_item(v, p.whole);
            int            wb, tb;
            pair_tile(item.tile, w_blocks, t_blocks, wb, tb);
            for (int c = 0; c < chunks; ++c, ++g)
            {
                const int s = g % STAGES;
                if (!warp_wait(empty_bar(s), (static_cast<uint32_t>(g / STAGES) & 1u) ^ 1u, s_abort, DEV_TIMEOUT_PRODUCER, p.spin_limit))
                {
                    goto produced;
                }
                if (g == p.withhold && blockIdx.x == 0)
                {
                    continue;
                }
                // boxes of scale tiles are whole: behind the last tile of a row they read the next row's, which no MMA uses
                const uint32_t bar = map_to_cta(full_bar(s), 0);
                const uint32_t dst = s_stage + s * P::STAGE, sf = s_sf + s * P::SF_STAGE;
                const int      kt  = static_cast<int>(p.k_tiles), sf0 = c * F::kChunkTiles;
                if (el)
                {
                    const bool whole = item.half < 0;
                    if (rank == 0)
                    {
                        mbar_expect_tx(full_bar(s), whole ? 2 * (P::STAGE + P::SF_STAGE) : 2 * (kMxWBytes + kMxWBytes / 2 + 2 * F::kChunkScale));
                    }
                    tma_load_2d_pair(dst, &tmap_w, c * kMxChunkBytes, (wb * 2 + rank) * kMxRows, bar);
                    tma_load_2d_pair(sf, &tmap_wsf, 0, (wb * 2 + rank) * kt + sf0, bar);
                    if (whole)
                    {
                        tma_load_2d_pair(dst + kMxWBytes, &tmap_t, c * kMxChunkBytes, tb * kPairCols + rank * kMxRows, bar);
                        tma_load_2d_pair(sf + F::kChunkScale, &tmap_tsf, 0, tb * 2 * kt + sf0, bar);
                        tma_load_2d_pair(sf + 2 * F::kChunkScale, &tmap_tsf, 0, (tb * 2 + 1) * kt + sf0, bar);
                    }
                    else
                    {
                        tma_load_2d_pair(dst + kMxWBytes, &tmap_half, c * kMxChunkBytes, tb * kPairCols + item.half * kMxRows + rank * (kMxRows / 2), bar);
                        tma_load_2d_pair(sf + F::kChunkScale, &tmap_tsf, 0, (tb * 2 + item.half) * kt + sf0, bar);
                    }
                }
                __syncwarp();
            }
        }
    produced:
        issued = g;
    }
    else if (warp == kMmaWarp)
    {
        const bool el = elect_one();
        if (rank == 0)
        {
            int  g = 0, it = 0;
            bool ok = true;
            const uint32_t t_w = tmem_base + P::SF_COL, t_t = t_w + F::kChunkCols;
            for (int v = first; v < items && ok; v += stride, ++it)
            {
                const bool     whole = v < p.whole;
                const uint32_t idesc = whole ? p.idesc : p.idesc_half;
                ok = warp_wait(tempty, (static_cast<uint32_t>(it) & 1u) ^ 1u, s_abort, DEV_TIMEOUT_MMA, p.spin_limit);
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + (it & 1) * (kPairCols - kPairShared);
                for (int c = 0; c < chunks && ok; ++c, ++g)
                {
                    const int s = g % STAGES;
                    ok = warp_wait(full_bar(s), static_cast<uint32_t>(g / STAGES) & 1u, s_abort, DEV_TIMEOUT_MMA, p.spin_limit);
                    if (!ok) break;
                    tc_fence_after();
                    const int      steps  = min(kMxChunk / kMxStepK, (p.K - c * kMxChunk + kMxStepK - 1) / kMxStepK);
                    const uint64_t sf     = make_scale_desc(s_sf + s * P::SF_STAGE);
                    const uint64_t a_desc = make_kmajor_sw128_desc(s_stage + s * P::STAGE), b_desc = a_desc + (kMxWBytes >> 4);
                    if (el)
                    {
#pragma unroll
                        for (int t = 0; t < F::kChunkTiles; ++t) // a step's tokens: rows 0..127 in four columns, 128..255 in the next four
                        {
                            const uint64_t at = static_cast<uint64_t>(t * (kMxTileBytes >> 4));
                            tmem_copy_scales_pair(t_w + 4 * t, sf + at);
                            tmem_copy_scales_pair(t_t + 8 * t, sf + at + (F::kChunkScale >> 4));
                            if (whole) tmem_copy_scales_pair(t_t + 8 * t + 4, sf + at + 2 * (F::kChunkScale >> 4));
                        }
#pragma unroll
                        for (int k = 0; k < kMxChunk / kMxStepK; ++k)
                        {
                            if (k < steps)
                            {
                                umma_mx_pair<kFormat>(d_tmem, a_desc + 2u * k, b_desc + 2u * k, idesc | mx_scale_id<kFormat>(k),
                                                      t_w + 4 * mx_step_tile<kFormat>(k), t_t + 8 * mx_step_tile<kFormat>(k), (c | k) != 0 ? 1u : 0u);
                            }
                        }
                        umma_commit_pair(empty_bar(s)); // frees this stage in both CTAs
                    }
                    __syncwarp();
                }
                if (ok && el)
                {
                    umma_commit_pair(tfull_bar(it & 1));
                }
            }
        }
        __syncwarp();
    }
    else
    {
        // Two warps per lane quarter, which take turns with groups of 32 columns; the shared ones are the first two groups.
        const int      q = warp & 3, half = (warp - kFirstEpi) >> 2;
        const uint32_t release = map_to_cta(tempty, 0);
        int            it = 0;
        for (int v = first; v < items; v += stride, ++it)
        {
            const PairItem item = pair_item(v, p.whole);
            int            wb, tb;
            pair_tile(item.tile, w_blocks, t_blocks, wb, tb);
            const int   as = it & 1, n0 = (wb * 2 + rank) * kMxRows + q * 32;
            if (!warp_wait(tfull_bar(as), static_cast<uint32_t>(it >> 1) & 1u, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit))
            {
                break;
            }
            tc_fence_after();
            const int      m0   = tb * kPairCols + (item.half > 0 ? kMxRows : 0), cols = p.tokens - m0;
            const uint32_t acc  = tmem_base + as * (kPairCols - kPairShared) + (static_cast<uint32_t>(q * 32) << 16);
            float          bias[4] = {}; // kBulk = 2: of the fragments' rows, else of this lane's channel
            if (p.bias != nullptr)
            {
#pragma unroll
                for (int i = 0; i < (kBulk == 2 ? 4 : 1); ++i)
                {
                    const int n = n0 + (kBulk == 2 ? lane / 4 + 8 * i : lane);
                    bias[i]     = n < p.channels ? __ldg(p.bias + n) : 0.f;
                }
            }
#pragma unroll 1
            for (int i = 0; i < (item.half < 0 ? kPairCols / 64 : kMxRows / 64); ++i)
            {
                const int group = 2 * i + half;
                const int j     = as == 0 && item.half < 0 ? (group * 32 + kPairCols - kPairShared) % kPairCols : group * 32; // (a half has none of the first accumulator's shared columns)
                uint32_t  r[2][16];
                if constexpr (kBulk == 2)
                {
                    tmem_ld_frag32(acc + j, r[0]);
                    tmem_ld_frag32(acc + j + (16u << 16), r[1]);
                }
                else
                {
                    tmem_ld_x16(acc + j, r[0]);
                    tmem_ld_x16(acc + j + 16, r[1]);
                }
                tmem_ld_wait();
                if (i == 0)
                {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(release);
                }
                if constexpr (kBulk != 0)
                {
                    // two-byte results: two areas in turn; floats: one
                    const int      area  = (warp - kFirstEpi) * 4096 + (kBulk == 2 ? (i & 1) * 2048 : 0);
                    const uint32_t s_out = s_stage + P::OFF_OUT + area;
                    if (lane == 0) // the store that reads this area has done so
                    {
                        if (kBulk == 2) tma_store_wait_read_but_one();
                        else tma_store_wait_read();
                    }
                    __syncwarp();
                    if constexpr (kBulk == 4)
                    {
                        float *out = reinterpret_cast<float *>(smem + P::OFF_OUT + area) + lane;
#pragma unroll
                        for (int k = 0; k < 32; ++k) out[32 * k] = __fmaf_rn(__uint_as_float(r[k / 16][k % 16]), p.alpha, bias[0]);
                    }
                    else if (p.dtype == CUGL_F16) stage_block<__half>(s_out, lane, r[0], r[1], p.alpha, bias);
                    else stage_block<__nv_bfloat16>(s_out, lane, r[0], r[1], p.alpha, bias);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0)
                    {
                        if (j < cols && n0 < p.channels) tma_store_2d(&tmap_out, s_out, n0, m0 + j);
                        tma_store_commit();
                    }
                    __syncwarp();
                }
                else
                {
                    store_block(p, m0 + j, n0 + lane, r[0], cols - j, bias[0]);
                    store_block(p, m0 + j + 16, n0 + lane, r[1], cols - j - 16, bias[0]);
                }
            }
            tc_fence_before();
        }
        if (kBulk != 0 && lane == 0)
        {
            tma_store_wait_all(); // shared memory stays valid until the stores have read it
        }
    }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0)
    {
        st_cluster_u32(map_to_cta(smem_u32(s_peer), rank ^ 1), static_cast<uint32_t>(issued) | (*s_abort != 0 ? 0x80000000u : 0u));
    }
    __syncwarp();
    cluster_sync(); // neither CTA leaves (or frees tensor memory) while its peer may still touch it
    const uint32_t peer = *s_peer;
    if (*s_abort != 0 || (peer >> 31) != 0) // given up, here or there: the same in both CTAs
    {
        if (rank == 0 && warp == 0)
        {
            drain_pair_stages<STAGES>(
                bar_base, issued, static_cast<int>(peer & 0x7fffffffu), blockIdx.x == 0 ? p.withhold : -1, p.spin_limit, [&](int g) {
                    return first + static_cast<int64_t>(g / chunks) * stride < p.whole ? P::STAGE + P::SF_STAGE
                                                                                     : kMxWBytes + kMxWBytes / 2 + 2 * F::kChunkScale;
                });
        }
        if (rank == 0 && warp == kMmaWarp)
        {
            drain_mmas<true>(gone_bar, p.spin_limit);
        }
        cluster_sync();
    }
    if (warp == kMmaWarp)
    {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
    if (threadIdx.x == 0 && *s_abort != 0)
    {
        atomicCAS(p.status, 0, *s_abort);
    }
}

struct MxOperands
{
    const cugl_mx_gemm_desc *d;
    const void              *a, *b;
};

// dst in boxes of 32 tokens x 32 channels: rows of 64 bytes in the 64-byte swizzle, or of 128 bytes
bool encode_dst_map(CUtensorMap *map, const MxGemmParams &p)
{
    EncodeTiledFn    fn         = get_encode_fn();
    const cuuint64_t dims[2]    = {static_cast<cuuint64_t>(p.channels), static_cast<cuuint64_t>(p.tokens)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(p.ldd)};
    const cuuint32_t box[2]     = {32, 32};
    const cuuint32_t estr[2]    = {1, 1};
    return fn != nullptr && fn(map, p.dtype == CUGL_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, p.dst, dims, strides, box, estr,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, p.dtype == CUGL_F32 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kFormat, int NT, int STAGES, bool kSplit>
cugl_status launch_one(cugl_context *ctx, const MxOperands &op, MxGemmParams p, int ranks)
{
    using P = MxPlan<kFormat, NT, STAGES, kSplit>;
    CUtensorMap   map_w, map_t;
    const int64_t inner = (static_cast<int64_t>(p.K) + 1) / 2;
    if (!encode_packed_map(&map_w, op.b, p.channels, inner, op.d->ldb, kMxRows) || !encode_packed_map(&map_t, op.a, p.tokens, inner, op.d->lda, NT))
    {
        return fail(ctx, CUGL_RUNTIME_ERROR, "cuTensorMapEncodeTiled failed for a packed operand");
    }
    auto        kernel  = mx_gemm_kernel<kFormat, NT, STAGES, kSplit>;
    static std::atomic<bool> set[64] = {}; // per instantiation and device
    CUGL_TRY(allow_smem(ctx, kernel, P::DYN_BYTES, set));
    p.idesc             = mx_idesc(kFormat, kMxRows, NT);
    const int64_t tiles = static_cast<int64_t>((p.channels + kMxRows - 1) / kMxRows) * ((p.tokens + NT - 1) / NT);
    const int grid = kSplit ? static_cast<int>(tiles) * ranks : static_cast<int>(tiles < 2 * ctx->sm_count ? tiles : 2 * ctx->sm_count);
    CUGL_CUDA_TRY(ctx, launch_dependent_cluster(ctx, kernel, dim3(static_cast<unsigned>(grid)), P::THREADS, P::DYN_BYTES, kSplit ? ranks : 1,
                                                tiles, map_w, map_t, p));
    return CUGL_SUCCESS;
}

// as many stages as half an SM's shared memory holds
template <int kFormat, int NT>
cugl_status launch_tokens(cugl_context *ctx, const MxOperands &op, const MxGemmParams &p, int ranks)
{
    constexpr bool kSmall  = kFormat == CUGL_MXFP4; // half the scale bytes
    constexpr int  kStages = NT <= 32 || (NT == 64 && kSmall) ? 4 : 3, kShared = NT == 32 && !kSmall ? 3 : kStages;
    return ranks > 1 ? launch_one<kFormat, NT, kShared, true>(ctx, op, p, ranks) : launch_one<kFormat, NT, kStages, false>(ctx, op, p, 1);
}

template <int kFormat, int kBulk>
cugl_status launch_pair(cugl_context *ctx, const MxOperands &op, MxGemmParams p)
{
    using P = MxPairPlan<kFormat>;
    using F = MxTraits<kFormat>;
    CUtensorMap   map_w, map_t, map_half, map_wsf, map_tsf, map_out{};
    const int64_t inner = (static_cast<int64_t>(p.K) + 1) / 2;
    const int64_t w_tiles = (static_cast<int64_t>(p.channels) + 127) / 128 * p.k_tiles, t_tiles = (static_cast<int64_t>(p.tokens) + 127) / 128 * p.k_tiles;
    if (!encode_packed_map(&map_w, op.b, p.channels, inner, op.d->ldb, kMxRows) || !encode_packed_map(&map_t, op.a, p.tokens, inner, op.d->lda, kMxRows) ||
        !encode_packed_map(&map_half, op.a, p.tokens, inner, op.d->lda, kMxRows / 2) ||
        !encode_scale_map(&map_wsf, p.w_scales, w_tiles, F::kChunkTiles) || !encode_scale_map(&map_tsf, p.t_scales, t_tiles, F::kChunkTiles) ||
        (kBulk != 0 && !encode_dst_map(&map_out, p)))
    {
        return fail(ctx, CUGL_RUNTIME_ERROR, "cuTensorMapEncodeTiled failed for an operand");
    }
    auto        kernel  = mx_gemm_pair_kernel<kFormat, kBulk>;
    static std::atomic<bool> set[64] = {};
    CUGL_TRY(allow_smem(ctx, kernel, P::DYN_BYTES, set));
    p.idesc      = mx_idesc(kFormat, 2 * kMxRows, kPairCols);
    p.idesc_half = mx_idesc(kFormat, 2 * kMxRows, kPairCols / 2);
    const int tiles = static_cast<int>(static_cast<int64_t>((p.channels + 255) / 256) * ((p.tokens + 255) / 256)), pairs = ctx->sm_count / 2;
    const int tail  = tiles % pairs;
    p.whole         = tail > 0 && 2 * tail <= pairs ? tiles - tail : tiles;
    const int items = p.whole + 2 * (tiles - p.whole), grid = 2 * (items < pairs ? items : pairs);
    CUGL_CUDA_TRY(ctx, launch_dependent_cluster(ctx, kernel, dim3(static_cast<unsigned>(grid)), kPairThreads, P::DYN_BYTES, 2, 2ll * items, map_w, map_t, map_half,
                                                map_wsf, map_tsf, map_out, p));
    return CUGL_SUCCESS;
}

template <int kFormat>
cugl_status launch_product(cugl_context *ctx, const MxOperands &op, const MxGemmParams &p)
{
    const int nt     = p.tokens <= 16 ? 16 : p.tokens <= 32 ? 32 : p.tokens <= 64 ? 64 : 128;
    const int chunks = (p.K + kMxChunk - 1) / kMxChunk;
    const long long tiles = static_cast<long long>((p.channels + kMxRows - 1) / kMxRows) * ((p.tokens + nt - 1) / nt);
    if (tiles > INT32_MAX / 8)
    {
        return fail(ctx, CUGL_INVALID_ARGUMENT, "cugl_mx_gemm: more than 2^28 output tiles");
    }
    if (p.tokens > 128 && (tiles >= 128 || (tiles >= 64 && chunks >= 8)))
    {
        // us on one CTA per tile / an SM pair: 256 x 4096 x 4096 (64 tiles) 11.3 / 10.1, 256 x 7168 x 4096 12.5 / 11.0, 512 x 14336 x 4096
        // 23.2 / 18.7, 2048 x 4096 x 512 9.6 / 8.5; 1024 x 1024 x 1024 (64 tiles) 5.6 / 6.0, 150 x 2048 x 14336 (32 tiles, shared K)
        // 13.8 / 21.3.  Without bulk stores the pair's epilogue is the slower one unless K is long: 2048 x 4097 F32 NVFP4, K = 1024 13.7 / 16.5,
        // 2048 17.6 / 18.4, 3584 23.1 / 21.6, 4096 24.8 / 22.8, 8192 38.4 / 32.8; BF16 15.2 / 21.0, 19.7 / 23.0, 25.9 / 26.0, 26.0 / 25.1, 40.0 /
        // 34.5; MXFP4 BF16 13.7 / 19.2, 16.9 / 20.8, 22.2 / 23.5, 24.2 / 24.3, 36.6 / 32.7; 3000 x 6001 turns at K of 2048 to 3584.
        // A bulk store wants 16-byte aligned rows and clips at the end of a row in whole 16-byte units.
        const int  size = dtype_size(p.dtype);
        const bool bulk = ((reinterpret_cast<uintptr_t>(p.dst) | static_cast<uintptr_t>(p.ldd)) & 15) == 0 && p.channels * static_cast<int64_t>(size) % 16 == 0 &&
                          p.ldd < (1ll << 40);
        if (bulk)
        {
            return size == 4 ? launch_pair<kFormat, 4>(ctx, op, p) : launch_pair<kFormat, 2>(ctx, op, p);
        }
        if (tiles >= 2 * ctx->sm_count && chunks >= 16)
        {
            return launch_pair<kFormat, 0>(ctx, op, p);
        }
    }
    // Sharing K pays until the SMs are busy; the parts of 128 columns cost more to add up (64 KB per CTA).  us with 1 / 2 / 4 / 8
    // CTAs per tile: 1 x 4096 x 4096 (32 tiles) 7.8 / 5.8 / 4.9 / 5.7, 16 x 4096 x 14336 20.6 / 13.0 / 9.9 / 10.3, 64 x 4096 x 4096
    // 9.0 / 8.2 / 7.3 / 8.2, 100 x 4096 x 4096 10.1 / 9.5 / 8.9 / 9.9, 256 x 4096 x 4096 (64 tiles) 11.3 / 11.9 / 11.5 / 22.
    const int ranks = nt < 128 || tiles * 4 <= ctx->sm_count ? mx_split(tiles, chunks, 4) : 1;
    switch (nt)
    {
        case 16: return launch_tokens<kFormat, 16>(ctx, op, p, ranks);
        case 32: return launch_tokens<kFormat, 32>(ctx, op, p, ranks);
        case 64: return launch_tokens<kFormat, 64>(ctx, op, p, ranks);
        default: return launch_tokens<kFormat, 128>(ctx, op, p, ranks);
    }
}

const char *validate_gemm(const cugl_mx_gemm_desc *d)
{
    if (d == nullptr) return "descriptor is NULL";
    if (d->M < 0 || d->N < 1 || d->K < 1) return "M must not be negative, N and K must be positive";
    if (d->K > INT32_MAX - 1024 || d->N > INT32_MAX - 1024 || d->M > INT32_MAX - 1024) return "a dimension is too large";
    if (d->format != CUGL_MXFP4 && d->format != CUGL_NVFP4) return "format must be CUGL_MXFP4 or CUGL_NVFP4";
    if (!is_float_dtype(d->dst_dtype)) return "dst_dtype must be CUGL_F32, CUGL_F16 or CUGL_BF16";
    const int64_t row = (static_cast<int64_t>(d->K) + 1) / 2;
    if (d->lda < row || d->ldb < row || d->lda % 16 != 0 || d->ldb % 16 != 0) return "lda and ldb must hold a packed row and be multiples of 16";
    if (d->lda >= (1ll << 40) || d->ldb >= (1ll << 40)) return "lda and ldb must be below 2^40";
    const int size = dtype_size(d->dst_dtype);
    if (d->ldd < static_cast<int64_t>(d->N) * size || d->ldd % size != 0) return "ldd must hold a row of dst and be a multiple of its element size";
    if (!(d->alpha - d->alpha == 0.f)) return "alpha must be finite";
    return nullptr;
}
} // namespace
} // namespace cugl

using namespace cugl;

extern "C"
{
    cugl_status cugl_mx_gemm_validate(const cugl_mx_gemm_desc *desc, const char **reason)
    {
        const char *why = validate_gemm(desc);
        if (reason != nullptr)
        {
            *reason = why != nullptr ? why : "";
        }
        return why == nullptr ? CUGL_SUCCESS : CUGL_INVALID_ARGUMENT;
    }

    cugl_status cugl_mx_gemm(cugl_context *ctx, const cugl_mx_gemm_desc *desc, const void *d_a, const void *d_a_scales, const void *d_b,
                             const void *d_b_scales, const float *d_bias, void *d_dst)
    {
        if (ctx == nullptr)
        {
            return fail(nullptr, CUGL_INVALID_ARGUMENT, "context is NULL");
        }
        const char *why = validate_gemm(desc);
        if (why == nullptr && desc->M > 0)
        {
            const uintptr_t in = reinterpret_cast<uintptr_t>(d_a) | reinterpret_cast<uintptr_t>(d_a_scales) | reinterpret_cast<uintptr_t>(d_b) |
                                 reinterpret_cast<uintptr_t>(d_b_scales);
            if (d_a == nullptr || d_a_scales == nullptr || d_b == nullptr || d_b_scales == nullptr || d_dst == nullptr) why = "NULL pointer";
            else if ((desc->has_bias != 0) != (d_bias != nullptr)) why = "d_bias must be given exactly when has_bias is set";
            else if ((in & 15) != 0) why = "operands and scale tiles must be 16-byte aligned";
            else if (reinterpret_cast<uintptr_t>(d_dst) % static_cast<uintptr_t>(dtype_size(desc->dst_dtype)) != 0 || reinterpret_cast<uintptr_t>(d_bias) % 4 != 0)
                why = "dst or bias is not aligned to its elements";
        }
        if (why != nullptr)
        {
            return fail(ctx, CUGL_INVALID_ARGUMENT, std::string("cugl_mx_gemm: ") + why);
        }
        if (desc->M == 0) return CUGL_SUCCESS;
        const DeviceScope device(ctx);
        MxGemmParams      p{};
        p.w_scales   = static_cast<const uint8_t *>(d_b_scales);
        p.t_scales   = static_cast<const uint8_t *>(d_a_scales);
        p.dst        = static_cast<uint8_t *>(d_dst);
        p.bias       = d_bias;
        p.ldd        = desc->ldd;
        p.k_tiles    = mx_scale_tiles(desc->K, desc->format);
        p.tokens     = desc->M;
        p.channels   = desc->N;
        p.K          = desc->K;
        p.dtype      = desc->dst_dtype;
        p.alpha      = desc->alpha;
        p.pack_out   = ((reinterpret_cast<uintptr_t>(d_dst) | static_cast<uintptr_t>(desc->ldd)) & 3) == 0 && desc->N % 2 == 0;
        p.status     = ctx->d_status;
        p.spin_limit = ctx->spin_limit;
        p.withhold   = ctx->withhold_kb;
        ctx->withhold_kb = -1;
        const MxOperands op{desc, d_a, d_b};
        return desc->format == CUGL_NVFP4 ? launch_product<CUGL_NVFP4>(ctx, op, p) : launch_product<CUGL_MXFP4>(ctx, op, p);
    }
}
