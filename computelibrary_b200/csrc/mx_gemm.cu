// Product of two microscaled 4-bit matrices on the tensor cores: dst[m][n] = alpha * sum_k a[m][k] * b[n][k] + bias[n].
//
//   warp 0      TMA: 128 rows of weights (b) and NT rows of tokens (a), 128 bytes (256 elements) of each per stage, and the
//               scale tiles that belong to them as plain bulk copies
//   warp 1      one lane copies the stage's scales to tensor memory and issues its MMAs (M = 128, N = NT, K = 64)
//   warps 2..5  a tensor-memory lane quarter each: accumulator * alpha + bias, rounded once, stored as 32 consecutive
//               channels per token
//
// Every stage has scale columns of its own in tensor memory: they are written again only after the stage's MMAs have been
// committed, like its shared memory.
#include "mx_mma.cuh"

namespace cugl
{
namespace
{
constexpr int kMmaWarp  = 1;
constexpr int kFirstEpi = 2;
constexpr int kThreads  = 192;

struct MxGemmParams
{
    const uint8_t *w_scales, *t_scales;
    uint8_t       *dst;
    const float   *bias;
    int64_t        ldd;
    int64_t        k_tiles; // scale tiles along K
    int            tokens, channels, K;
    int            dtype;
    float          alpha;
    uint32_t       idesc;
    int32_t       *status;
    long long      spin_limit;
    int            withhold; // see cugl_context_withhold_copy_once
};

template <int kFormat, int NT, int STAGES, bool kSplit>
struct MxPlan
{
    using F                          = MxTraits<kFormat>;
    static constexpr int T_BYTES     = NT * kMxChunkBytes;
    static constexpr int STAGE       = kMxWBytes + T_BYTES;
    static constexpr int SF_STAGE    = 2 * F::kChunkScale;
    static constexpr int OFF_SF      = STAGES * STAGE;
    static constexpr int OFF_BAR     = OFF_SF + STAGES * SF_STAGE;
    static constexpr int OFF_MISC    = OFF_BAR + (2 * STAGES + 4) * 8;
    static constexpr int DYN_BYTES   = OFF_MISC + 16 + 1024;
    static constexpr int ACC         = kSplit ? 1 : 2;
    static constexpr int SF_COLS     = 2 * F::kChunkCols; // per stage
    static constexpr int COLS        = ACC * NT + STAGES * SF_COLS;
    static constexpr int TMEM_COLS   = COLS <= 32 ? 32 : COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    static_assert(COLS <= 512 && DYN_BYTES <= 232448, "tensor and shared memory of an SM");
    static_assert(!kSplit || STAGES * STAGE >= NT * kMxRows * 4, "the partial sums of a cluster fit where the stages were");
};

// Sixteen tokens of one channel.
template <typename T>
__device__ __forceinline__ void store_tokens(uint8_t *dst, int64_t ldd, const float (&v)[16], int tokens)
{
#pragma unroll
    for (int j = 0; j < 16; ++j)
    {
        if (j < tokens)
        {
            *reinterpret_cast<T *>(dst + j * ldd) = from_float<T>(v[j]);
        }
    }
}
__device__ __forceinline__ void store_tokens(const MxGemmParams &p, int m, int n, const float (&v)[16])
{
    uint8_t *dst = p.dst + static_cast<int64_t>(m) * p.ldd;
    if (p.dtype == CUGL_F32) store_tokens<float>(dst + 4ll * n, p.ldd, v, p.tokens - m);
    else if (p.dtype == CUGL_F16) store_tokens<__half>(dst + 2ll * n, p.ldd, v, p.tokens - m);
    else store_tokens<__nv_bfloat16>(dst + 2ll * n, p.ldd, v, p.tokens - m);
}

template <int kFormat, int NT, int STAGES, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_t, const __grid_constant__ MxGemmParams p)
{
    using P = MxPlan<kFormat, NT, STAGES, kSplit>;
    using F = MxTraits<kFormat>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t       *smem      = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t s_stage   = smem_u32(smem);
    const uint32_t s_sf      = smem_u32(smem + P::OFF_SF);
    const uint32_t bar_base  = smem_u32(smem + P::OFF_BAR);
    auto           full_bar  = [&](int s) { return bar_base + 8u * s; };
    auto           empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto           tfull_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
    auto           tempty_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + 2 + a); };
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
    const int per_rank    = (chunks + ranks - 1) / ranks;
    const int c_begin     = min(chunks, rank * per_rank);
    const int c_end       = min(chunks, c_begin + per_rank);

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
            mbar_init(tempty_bar(a), 4);
        }
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp)
    {
        tmem_alloc(smem_u32(s_tmem), P::TMEM_COLS);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *s_tmem;
    griddep_launch_dependents();
    griddep_wait(); // the prologue above touched no global memory

    if (warp == 0)
    {
        if (lane == 0)
        {
            int g = 0;
            for (int tile = first_tile; tile < tiles; tile += tile_stride)
            {
                const int      wb = tile % w_blocks, tb = tile / w_blocks;
                const uint8_t *w_sf = p.w_scales + static_cast<int64_t>(wb) * p.k_tiles * kMxTileBytes;
                const uint8_t *t_sf = p.t_scales + static_cast<int64_t>(tb) * p.k_tiles * kMxTileBytes; // NT < 128: one block only
                for (int c = c_begin; c < c_end; ++c, ++g)
                {
                    const int s = g % STAGES;
                    if (!mbar_wait(empty_bar(s), (static_cast<uint32_t>(g / STAGES) & 1u) ^ 1u, s_abort, DEV_TIMEOUT_PRODUCER, p.spin_limit))
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
                    mbar_expect_tx(full_bar(s), P::STAGE + 2 * bytes);
                    tma_load_2d(dst, &tmap_w, c * kMxChunkBytes, wb * kMxRows, full_bar(s));
                    tma_load_2d(dst + kMxWBytes, &tmap_t, c * kMxChunkBytes, tb * NT, full_bar(s));
                    bulk_load(sf, w_sf + static_cast<int64_t>(first) * kMxTileBytes, bytes, full_bar(s));
                    bulk_load(sf + F::kChunkScale, t_sf + static_cast<int64_t>(first) * kMxTileBytes, bytes, full_bar(s));
                }
            }
        produced:
            if (*s_abort != 0)
            {
                for (int i = max(0, g - STAGES); i < g; ++i)
                {
                    if (!(i == p.withhold && blockIdx.x == 0)) mbar_drain(full_bar(i % STAGES), static_cast<uint32_t>(i / STAGES) & 1u, p.spin_limit);
                }
            }
        }
        __syncwarp();
    }
    else if (warp == kMmaWarp)
    {
        if (lane == 0)
        {
            int  g = 0, it = 0;
            bool ok = true;
            for (int tile = first_tile; tile < tiles && ok; tile += tile_stride, ++it)
            {
                const int as = it % P::ACC;
                ok = mbar_wait(tempty_bar(as), (static_cast<uint32_t>(it / P::ACC) & 1u) ^ 1u, s_abort, DEV_TIMEOUT_MMA, p.spin_limit);
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + as * NT;
                for (int c = c_begin; c < c_end && ok; ++c, ++g)
                {
                    const int s = g % STAGES;
                    ok = mbar_wait(full_bar(s), static_cast<uint32_t>(g / STAGES) & 1u, s_abort, DEV_TIMEOUT_MMA, p.spin_limit);
                    if (!ok) break;
                    tc_fence_after();
                    const int      n     = min(F::kChunkTiles, static_cast<int>(p.k_tiles) - c * F::kChunkTiles);
                    const int      steps = min(kMxChunk / kMxStepK, (p.K - c * kMxChunk + kMxStepK - 1) / kMxStepK);
                    const uint32_t t_w   = tmem_base + P::ACC * NT + s * P::SF_COLS, t_t = t_w + F::kChunkCols;
                    const uint32_t sf    = s_sf + s * P::SF_STAGE;
                    mx_chunk_scales<kFormat>(t_w, sf, n);
                    mx_chunk_scales<kFormat>(t_t, sf + F::kChunkScale, n);
                    mx_chunk<kFormat>(d_tmem, s_stage + s * P::STAGE, s_stage + s * P::STAGE + kMxWBytes, t_w, t_t, p.idesc, steps, c == c_begin);
                    umma_commit(empty_bar(s));
                }
                if (ok)
                {
                    umma_commit(tfull_bar(as));
                }
            }
        }
        __syncwarp();
    }
    else if (!kSplit)
    {
        const int q  = warp & 3;
        int       it = 0;
        for (int tile = first_tile; tile < tiles; tile += tile_stride, ++it)
        {
            const int   wb = tile % w_blocks, tb = tile / w_blocks;
            const int   as = it % P::ACC;
            const int   n  = wb * kMxRows + q * 32 + lane;
            const float b  = p.bias != nullptr && n < p.channels ? __ldg(p.bias + n) : 0.f;
            if (!__all_sync(0xffffffffu, mbar_wait(tfull_bar(as), static_cast<uint32_t>(it / P::ACC) & 1u, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit)))
            {
                break;
            }
            tc_fence_after();
            const int cols = min(NT, p.tokens - tb * NT);
            for (int j = 0; j < cols; j += 16)
            {
                uint32_t r[16];
                tmem_ld_x16(tmem_base + as * NT + j + (static_cast<uint32_t>(q * 32) << 16), r);
                tmem_ld_wait();
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __fmaf_rn(__uint_as_float(r[i]), p.alpha, b);
                if (n < p.channels) store_tokens(p, tb * NT + j, n, v);
                __syncwarp();
            }
            tc_fence_before();
            if (lane == 0) mbar_arrive(tempty_bar(as));
        }
    }

    if constexpr (kSplit)
    {
        // Partial sums of the cluster: token j belongs to rank j % ranks; every CTA writes its part of the column (128
        // channels) into the owner's shared memory, where the stages were, and the owner adds them up in the order of the
        // ranks -- the same order every time.
        const int  tile = first_tile, wb = tile % w_blocks, tb = tile / w_blocks;
        const int  cols = min(NT, p.tokens - tb * NT);
        const int  q = warp & 3, ch = q * 32 + lane;
        bool       ok = true;
        if (warp >= kFirstEpi)
        {
            ok = __all_sync(0xffffffffu, mbar_wait(tfull_bar(0), 0, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit));
            tc_fence_after();
        }
        __syncthreads();
        cluster_sync(); // every CTA's MMAs have read their last stage
        const int per_owner = (NT + ranks - 1) / ranks;
        if (warp >= kFirstEpi && ok)
        {
            for (int j = 0; j < cols; j += 16)
            {
                uint32_t r[16];
                tmem_ld_x16(tmem_base + j + (static_cast<uint32_t>(q * 32) << 16), r);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    if (j + i < cols)
                    {
                        const float v = c_begin < c_end ? __uint_as_float(r[i]) : 0.f; // a rank without chunks has no accumulator
                        st_cluster_f32(map_to_cta(s_stage, (j + i) % ranks) + 4u * ((rank * per_owner + (j + i) / ranks) * kMxRows + ch), v);
                    }
                }
            }
        }
        cluster_sync();
        if (warp >= kFirstEpi && ok)
        {
            const int    n    = wb * kMxRows + ch;
            const float  b    = p.bias != nullptr && n < p.channels ? __ldg(p.bias + n) : 0.f;
            const float *part = reinterpret_cast<const float *>(smem);
            for (int i = 0; i * ranks + rank < cols; ++i)
            {
                float sum = 0.f;
                for (int src = 0; src < ranks; ++src) sum += part[(src * per_owner + i) * kMxRows + ch];
                if (n < p.channels)
                {
                    const float v   = __fmaf_rn(sum, p.alpha, b);
                    uint8_t    *dst = p.dst + static_cast<int64_t>(tb * NT + i * ranks + rank) * p.ldd;
                    if (p.dtype == CUGL_F32) reinterpret_cast<float *>(dst)[n] = v;
                    else if (p.dtype == CUGL_F16) reinterpret_cast<__half *>(dst)[n] = from_float<__half>(v);
                    else reinterpret_cast<__nv_bfloat16 *>(dst)[n] = from_float<__nv_bfloat16>(v);
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp)
    {
        tc_fence_after();
        tmem_dealloc(tmem_base, P::TMEM_COLS);
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
    auto        kernel       = mx_gemm_kernel<kFormat, NT, STAGES, kSplit>;
    static bool attr_set[64] = {}; // per instantiation and device
    if (!attr_set[ctx->device & 63])
    {
        CUGL_CUDA_TRY(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P::DYN_BYTES));
        attr_set[ctx->device & 63] = true;
    }
    p.idesc             = mx_idesc(kFormat, kMxRows, NT);
    const int64_t tiles = static_cast<int64_t>((p.channels + kMxRows - 1) / kMxRows) * ((p.tokens + NT - 1) / NT);
    if (tiles > INT32_MAX / 8)
    {
        return fail(ctx, CUGL_INVALID_ARGUMENT, "cugl_mx_gemm: more than 2^28 output tiles");
    }
    const int grid = kSplit ? static_cast<int>(tiles) * ranks : static_cast<int>(tiles < ctx->sm_count ? tiles : ctx->sm_count);
    CUGL_CUDA_TRY(ctx, launch_dependent_cluster(ctx, kernel, dim3(static_cast<unsigned>(grid)), kThreads, P::DYN_BYTES, kSplit ? ranks : 1,
                                                tiles, map_w, map_t, p));
    return CUGL_SUCCESS;
}

template <int kFormat>
cugl_status launch_product(cugl_context *ctx, const MxOperands &op, const MxGemmParams &p)
{
    const int nt     = p.tokens <= 16 ? 16 : p.tokens <= 32 ? 32 : p.tokens <= 64 ? 64 : 128;
    const int chunks = (p.K + kMxChunk - 1) / kMxChunk;
    const long long tiles = static_cast<long long>((p.channels + kMxRows - 1) / kMxRows) * ((p.tokens + nt - 1) / nt);
    int ranks = 1; // CTAs that share a tile's K: as many as leave no SM idle and every CTA a chunk
    while (ranks < 8 && tiles * ranks * 2 <= ctx->sm_count && ranks * 2 <= chunks) ranks *= 2;
    if (ranks > 1)
    {
        switch (nt)
        {
            case 16: return launch_one<kFormat, 16, 8, true>(ctx, op, p, ranks);
            case 32: return launch_one<kFormat, 32, 8, true>(ctx, op, p, ranks);
            case 64: return launch_one<kFormat, 64, 7, true>(ctx, op, p, ranks);
            default: return launch_one<kFormat, 128, 6, true>(ctx, op, p, ranks);
        }
    }
    switch (nt)
    {
        case 16: return launch_one<kFormat, 16, 8, false>(ctx, op, p, 1);
        case 32: return launch_one<kFormat, 32, 8, false>(ctx, op, p, 1);
        case 64: return launch_one<kFormat, 64, 7, false>(ctx, op, p, 1);
        default: return launch_one<kFormat, 128, 6, false>(ctx, op, p, 1);
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
        p.status     = ctx->d_status;
        p.spin_limit = ctx->spin_limit;
        p.withhold   = ctx->withhold_kb;
        ctx->withhold_kb = -1;
        const MxOperands op{desc, d_a, d_b};
        return desc->format == CUGL_NVFP4 ? launch_product<CUGL_NVFP4>(ctx, op, p) : launch_product<CUGL_MXFP4>(ctx, op, p);
    }
}
