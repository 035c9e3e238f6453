// Products of groups of microscaled 4-bit rows, each group with a weight matrix of its own (an expert's):
//   dst[r][n] = alpha_g * sum_k a[r][k] * b[g][n][k] + bias[g][n]                             r a row of group g
//   dst[r][n] = silu(alpha_g * sum_k a[r][k] * b[g][n][k]) * (up_alpha_g * sum_k a[r][k] * up[g][n][k])
//
// Where the groups lie is known on the device only: (start, count) pairs, starts at multiples of 128 rows, so that the scale tiles of
// a group are its own.  Every CTA adds up how many tiles of tokens the groups before each one have (a scan over at most 512 of
// them) and finds the tile behind an item's number by a binary search; nothing is launched per group and nothing is read back.
//
// Operand roles as in the plain product: weights are the rows of an MMA, tokens its columns, as many as a tile holds (a multiple of
// 16 or 32): a group of three rows costs sixteen columns.  Rows behind a group's end are columns that nothing reads: they may hold
// anything, and their rows of dst are left as they were.
//
// Two kernels.  Few rows a group: one CTA per SM, 128 channels x up to 128 tokens, a long ring of weights, two accumulators in turn.  Many:
// SM pairs, 256 channels x 256 tokens, or 256 channels x 128 tokens of both products of SwiGLU.
#include "mx_mma.cuh"

#include <cstring>

namespace cugl
{
namespace
{
constexpr int kMmaWarp   = 1;
constexpr int kFirstEpi  = 2;
constexpr int kFewEpi      = 8;  // epilogue warps, two per tensor-memory lane quarter
constexpr int kFewThreads  = 32 * (kFirstEpi + kFewEpi);
constexpr int kMaxGroups = 512;
constexpr int kSlab      = 128; // rows at whose multiples groups start

struct GroupedParams
{
    const int2    *groups;
    const uint8_t *b_scales, *up_scales, *a_scales;
    uint8_t       *dst;
    const float   *bias;              // [groups][channels]
    const float   *b_alpha, *up_alpha; // [groups]
    int64_t        ldd;
    int64_t        k_tiles;      // scale tiles along K
    int64_t        group_tiles;  // scale tiles of one group's weights
    int            n_groups, rows, channels, K, dtype;
    int            pack_out;     // two-byte results: rows of dst are words (4-byte aligned, an even number of channels)
    int            vec_out;      // rows of dst are 16-byte aligned and whole 16-byte units long
    float          alpha, up_scale;
    uint32_t       idesc;        // of one column: add columns / 8 << 17
    int32_t       *status;
    long long      spin_limit;
    int            withhold;     // see cugl_context_withhold_copy_once
};

// ---- where the groups lie ------------------------------------------------------------------------------------
// A group that does not start at a multiple of 128 or does not lie within the rows counts as empty and is reported.
__device__ __forceinline__ int2 load_group(const GroupedParams &p, int g, bool &bad)
{
    int2 v = p.groups[g];
    bad    = v.y < 0 || (v.y > 0 && (v.x < 0 || v.x % kSlab != 0 || v.x > p.rows || v.y > p.rows - v.x));
    if (bad || v.y <= 0) v = make_int2(0, 0);
    return v;
}
// before[g]: tiles of kTile rows of the groups before g; returns those of all.  Called by all threads.  Groups that do not overlap have no
// more tiles than the rows have slabs; more are reported and none of them is worked on, so that items stay countable.  Sums stop at kMostTiles.
constexpr int kMostTiles = 1 << 28;
template <int kTile>
__device__ __forceinline__ int scan_groups(const GroupedParams &p, int *before)
{
    for (int g = threadIdx.x; g < p.n_groups; g += static_cast<int>(blockDim.x))
    {
        bool       bad;
        const int2 v  = load_group(p, g, bad);
        before[g + 1] = (v.y + kTile - 1) / kTile;
        if (bad && blockIdx.x == 0) atomicExch(p.status + STATUS_GROUP, DEV_BAD_GROUP);
    }
    if (threadIdx.x == 0) before[0] = 0;
    __syncthreads();
    if (threadIdx.x < 32)
    {
        const int per = (p.n_groups + 31) / 32, first = 1 + static_cast<int>(threadIdx.x) * per;
        int       sum = 0;
        for (int i = first; i < min(first + per, p.n_groups + 1); ++i) sum += before[i];
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (static_cast<int>(threadIdx.x) >= o) incl = min(incl + v, kMostTiles);
        }
        int at = incl - sum;
        for (int i = first; i < min(first + per, p.n_groups + 1); ++i)
        {
            at        = min(at + before[i], kMostTiles);
            before[i] = at;
        }
    }
    __syncthreads();
    const int tiles = before[p.n_groups];
    if (tiles > (p.rows + kSlab - 1) / kSlab)
    {
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicExch(p.status + STATUS_GROUP, DEV_BAD_GROUP);
        return 0;
    }
    return tiles;
}

// An item: 128 (or 256) channels of a tile of tokens of a group.
struct Item
{
    int group, wb;
    int row, count; // first row, rows of the tile that belong to the group
};
// Channel blocks change fastest, in strips of kStrip: consecutive items share the tokens, those of a strip the weights.
constexpr int kStrip = 4;
template <int kTile>
__device__ __forceinline__ Item find_item(const GroupedParams &p, const int *before, int w_blocks, int item)
{
    const int tile = item / w_blocks;
    int       lo = 0, hi = p.n_groups; // before[lo] <= tile < before[hi]
    while (hi - lo > 1)
    {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= tile) lo = mid;
        else hi = mid;
    }
    Item it;
    it.group         = lo;
    const int tiles  = before[lo + 1] - before[lo], in = item - before[lo] * w_blocks;
    const int strip  = in / (kStrip * tiles), at = in - strip * kStrip * tiles;
    const int width  = min(kStrip, w_blocks - strip * kStrip);
    const int tb     = at / width;
    it.wb            = strip * kStrip + at - tb * width;
    const int2 v     = p.groups[lo];
    it.row           = v.x + tb * kTile;
    it.count         = min(kTile, v.y - tb * kTile);
    return it;
}

// The first items of a CTA, found once, side by side, at the start: a search is a thousand clocks of dependent instructions, which every
// role would otherwise run through at every item (and the MMAs wait for).  Later ones, of a CTA with many items, are searched for.
constexpr int kListed = 128;
struct ListedItem
{
    uint32_t group_count; // count << 16 | group
    int      wb, row;
};
template <int kTile>
__device__ __forceinline__ void list_items(const GroupedParams &p, const int *before, ListedItem *list, int w_blocks, int first, int stride, int items)
{
    const int i = static_cast<int>(threadIdx.x);
    if (i < kListed && static_cast<int64_t>(i) * stride + first < items)
    {
        const Item it = find_item<kTile>(p, before, w_blocks, first + i * stride);
        list[i]       = ListedItem{static_cast<uint32_t>(it.count) << 16 | static_cast<uint32_t>(it.group), it.wb, it.row};
    }
    __syncthreads();
}
template <int kTile>
__device__ __forceinline__ Item get_item(const GroupedParams &p, const int *before, const ListedItem *list, int w_blocks, int i, int item)
{
    if (i >= kListed) return find_item<kTile>(p, before, w_blocks, item);
    const ListedItem l = list[i];
    return Item{static_cast<int>(l.group_count & 0xffffu), l.wb, l.row, static_cast<int>(l.group_count >> 16)};
}

// ---- what happens to sums ------------------------------------------------------------------------------------
// silu(g) * u.  16-bit results take 2^x of the rounded product -g log2(e): off by 2^-20 + |g| 2^-23 of the result, where half a step of
// theirs is 2^-11 or 2^-8; eight instructions instead of seventeen (768 channels, K = 2048, 512 rows a group: 67 -> 64 us).  For gates
// from kSiluTail up.
template <bool kShort>
__device__ __forceinline__ float swiglu(float g, float u)
{
    if constexpr (kShort)
    {
        float e, q;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.442695041f));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + e));
        return g * q * u;
    }
    return __fdividef(g, 1.f + expf(-g)) * u;
}
// (Plain loads, here and wherever a kernel reads what a launch ahead may have written: read-only ones assume that nothing writes while the
// kernel runs, and it has run since before griddepcontrol.wait.)
struct Factors
{
    float alpha, up;
};
__device__ __forceinline__ Factors group_factors(const GroupedParams &p, int g)
{
    Factors f{p.alpha, p.up_scale};
    if (p.b_alpha != nullptr) f.alpha *= p.b_alpha[g];
    if (p.up_alpha != nullptr) f.up *= p.up_alpha[g];
    return f;
}
__device__ __forceinline__ float group_bias(const GroupedParams &p, int g, int n)
{
    return p.bias != nullptr && n < p.channels ? p.bias[static_cast<int64_t>(g) * p.channels + n] : 0.f;
}
// Sixteen sums (of both products) to results; bias(i): of the i-th.  Gates in silu's tail are rare: one test for all of them, and the
// whole sixteen once more where there is one.
template <bool kSwiglu, bool kShort, typename Bias>
__device__ __forceinline__ void finish_as(const uint32_t (&a)[16], const uint32_t (&u)[16], const Factors &f, Bias bias, float (&x)[16])
{
    if constexpr (kSwiglu)
    {
        float top = 0.f; // of the gates' magnitudes: one instruction for two
#pragma unroll
        for (int i = 0; i < 16; i += 2) asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(top) : "f"(top), "f"(__uint_as_float(a[i])), "f"(__uint_as_float(a[i + 1])));
        if (top * fabsf(f.alpha) <= -kSiluTail)
        {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = swiglu<kShort>(__uint_as_float(a[i]) * f.alpha, __uint_as_float(u[i]) * f.up);
        }
        else
        {
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                const float g = __uint_as_float(a[i]) * f.alpha, v = __uint_as_float(u[i]) * f.up;
                x[i]          = g < kSiluTail ? swiglu_tail(g, v) : swiglu<kShort>(g, v);
            }
        }
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = __fmaf_rn(__uint_as_float(a[i]), f.alpha, bias(i));
    }
}

// The same function for a type in every kernel: a result does not depend on which one a rule chose.
template <bool kSwiglu, typename Bias>
__device__ __forceinline__ void finish(const GroupedParams &p, const uint32_t (&a)[16], const uint32_t (&u)[16], const Factors &f, Bias bias, float (&x)[16])
{
    if (kSwiglu && p.dtype != CUGL_F32) finish_as<kSwiglu, true>(a, u, f, bias, x);
    else finish_as<kSwiglu, false>(a, u, f, bias, x);
}

// Sixteen tokens (rows m and up, `cols` of them valid) of a lane's channel n to dst.  Two-byte results of neighbouring channels leave
// as one word: lanes exchange a column each, after which the even lane of a pair holds both channels of the first token and the
// odd lane those of the second.
template <typename T>
__device__ __forceinline__ void store_tokens(const GroupedParams &p, int m, int n, const float (&v)[16], int cols)
{
    uint8_t *dst = p.dst + static_cast<int64_t>(m) * p.ldd + static_cast<int64_t>(n) * static_cast<int>(sizeof(T));
    if (sizeof(T) == 2 && p.pack_out != 0)
    {
        const int odd = n & 1;
        dst += odd != 0 ? p.ldd - 2 : 0;
#pragma unroll
        for (int j = 0; j < 16; j += 2)
        {
            const float got    = __shfl_xor_sync(0xffffffffu, odd != 0 ? v[j] : v[j + 1], 1);
            T           two[2] = {from_float<T>(odd != 0 ? got : v[j]), from_float<T>(odd != 0 ? v[j + 1] : got)};
            if (j + odd < cols && n < p.channels)
            {
                uint32_t w;
                memcpy(&w, two, 4);
                *reinterpret_cast<uint32_t *>(dst + j * p.ldd) = w;
            }
        }
        __syncwarp(); // aligned loads of tensor memory may be next
        return;
    }
    if (n < p.channels)
    {
#pragma unroll
        for (int j = 0; j < 16; ++j)
        {
            if (j < cols) *reinterpret_cast<T *>(dst + j * p.ldd) = from_float<T>(v[j]);
        }
    }
    __syncwarp();
}
__device__ __forceinline__ void store_tokens(const GroupedParams &p, int m, int n, const float (&v)[16], int cols)
{
    if (p.dtype == CUGL_F32) store_tokens<float>(p, m, n, v, cols);
    else if (p.dtype == CUGL_F16) store_tokens<__half>(p, m, n, v, cols);
    else store_tokens<__nv_bfloat16>(p, m, n, v, cols);
}

// ---- few rows a group ----------------------------------------------------------------------------------------
// One CTA per SM works through items of 128 channels x up to 128 tokens.  What bounds it: the weights' bytes, hence a ring that keeps
// 96 KB (plain) or 128 KB (SwiGLU) of them in flight per SM.  The token boxes have four heights, the MMAs as many columns as rows
// there are, in steps of sixteen.
//
// Tensor memory: two halves of 128 columns for sums and the scale columns of every stage.  A plain tile takes a half in turn; SwiGLU
// takes one where its gate and up sums fit there (64 tokens), else both.
template <int kFormat, bool kSwiglu>
struct FewPlan
{
    using F                        = MxTraits<kFormat>;
    static constexpr int WEIGHTS   = kSwiglu ? 2 : 1;
    static constexpr int STAGES    = kSwiglu ? 4 : 6;
    static constexpr int STAGE     = (WEIGHTS + 1) * kMxWBytes; // weights, tokens
    static constexpr int SF_STAGE  = (WEIGHTS + 1) * F::kChunkScale;
    static constexpr int SF_COLS   = (WEIGHTS + 1) * F::kChunkCols;
    static constexpr int OFF_SF    = STAGES * STAGE;
    static constexpr int OFF_BAR   = OFF_SF + STAGES * SF_STAGE;
    static constexpr int OFF_MISC  = OFF_BAR + (2 * STAGES + 5) * 8;
    static constexpr int OFF_SCAN  = OFF_MISC + 16;
    static constexpr int OFF_LIST  = OFF_SCAN + (kMaxGroups + 1) * 4;
    static constexpr int DYN_BYTES = OFF_LIST + kListed * static_cast<int>(sizeof(ListedItem)) + 1024;
    static constexpr int SF_COL    = 256;
    static_assert(SF_COL + STAGES * SF_COLS <= 512 && DYN_BYTES <= 232448, "tensor and shared memory of an SM");
};
struct TokenMaps
{
    CUtensorMap rows[4]; // boxes of 16, 32, 64, 128 rows
};
__device__ __forceinline__ int token_box(int count)
{
    return count <= 16 ? 0 : count <= 32 ? 1 : count <= 64 ? 2 : 3;
}

// The halves of tensor memory that consecutive tiles take, and how often each has been used: the same sequence for every role.
template <bool kSwiglu>
struct Halves
{
    int next = 0, used[2] = {0, 0};
    int first = 0;    // of the current tile
    bool both = false;
    __device__ __forceinline__ void take(int cols)
    {
        both  = kSwiglu && cols > 64;
        first = both ? 0 : next;
        next  = both ? 0 : next ^ 1;
    }
    __device__ __forceinline__ void done()
    {
        if (both || first == 0) ++used[0];
        if (both || first == 1) ++used[1];
    }
};

template <int kFormat, bool kSwiglu>
__global__ void __launch_bounds__(kFewThreads, 1)
    mx_grouped_few_kernel(const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_up, const __grid_constant__ TokenMaps tmap_a,
                          const __grid_constant__ GroupedParams p)
{
    using P = FewPlan<kFormat, kSwiglu>;
    using F = MxTraits<kFormat>;
    constexpr int STAGES = P::STAGES, W = P::WEIGHTS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t       *smem      = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t s_stage   = smem_u32(smem);
    const uint32_t s_sf      = smem_u32(smem + P::OFF_SF);
    const uint32_t bar_base  = smem_u32(smem + P::OFF_BAR);
    auto           full_bar  = [&](int s) { return bar_base + 8u * s; };
    auto           empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto           tfull_bar = [&](int h) { return bar_base + 8u * (2 * STAGES + h); };
    auto           tempty_bar = [&](int h) { return bar_base + 8u * (2 * STAGES + 2 + h); };
    const uint32_t gone_bar  = bar_base + 8u * (2 * STAGES + 4); // see drain_mmas
    uint32_t      *s_tmem    = reinterpret_cast<uint32_t *>(smem + P::OFF_MISC);
    volatile int  *s_abort   = reinterpret_cast<volatile int *>(smem + P::OFF_MISC + 4);
    int           *before    = reinterpret_cast<int *>(smem + P::OFF_SCAN);
    ListedItem    *list      = reinterpret_cast<ListedItem *>(smem + P::OFF_LIST);
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int      w_blocks = (p.channels + kMxRows - 1) / kMxRows;
    const int      chunks   = (p.K + kMxChunk - 1) / kMxChunk;

    if (threadIdx.x == 0)
    {
        for (int s = 0; s < STAGES; ++s)
        {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int h = 0; h < 2; ++h)
        {
            mbar_init(tfull_bar(h), 1);
            mbar_init(tempty_bar(h), kFewEpi);
        }
        mbar_init(gone_bar, 1);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp)
    {
        tmem_alloc(smem_u32(s_tmem), 512);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *s_tmem;
    griddep_launch_dependents();
    griddep_wait(); // the groups come from a kernel ahead
    const int items = scan_groups<kSlab>(p, before) * w_blocks;
    list_items<kSlab>(p, before, list, w_blocks, static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x), items);

    int issued = 0; // stages that the producer has filled
    if (warp == 0)
    {
        const bool el = elect_one();
        int        g = 0, n = 0;
        for (int v = blockIdx.x; v < items; v += gridDim.x, ++n)
        {
            const Item     it   = get_item<kSlab>(p, before, list, w_blocks, n, v);
            const int      box  = token_box(it.count);
            const int      w_row = it.group * p.channels + it.wb * kMxRows;
            const int64_t  w_sf = it.group * p.group_tiles + it.wb * p.k_tiles, a_sf = it.row / kSlab * p.k_tiles;
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
                const int      first = c * F::kChunkTiles;
                const uint32_t bytes = static_cast<uint32_t>(min(F::kChunkTiles, static_cast<int>(p.k_tiles) - first)) * kMxTileBytes;
                const uint32_t dst   = s_stage + s * P::STAGE, sf = s_sf + s * P::SF_STAGE;
                if (el)
                {
                    mbar_expect_tx(full_bar(s), static_cast<uint32_t>(W * kMxWBytes + (16 << box) * kMxChunkBytes) + (W + 1) * bytes);
                    tma_load_2d(dst, &tmap_b, c * kMxChunkBytes, w_row, full_bar(s));
                    bulk_load(sf, p.b_scales + (w_sf + first) * kMxTileBytes, bytes, full_bar(s));
                    if constexpr (kSwiglu)
                    {
                        tma_load_2d(dst + kMxWBytes, &tmap_up, c * kMxChunkBytes, w_row, full_bar(s));
                        bulk_load(sf + F::kChunkScale, p.up_scales + (w_sf + first) * kMxTileBytes, bytes, full_bar(s));
                    }
                    tma_load_2d(dst + W * kMxWBytes, &tmap_a.rows[box], c * kMxChunkBytes, it.row, full_bar(s));
                    bulk_load(sf + W * F::kChunkScale, p.a_scales + (a_sf + first) * kMxTileBytes, bytes, full_bar(s));
                }
                __syncwarp();
            }
        }
    produced:
        issued = g;
    }
    else if (warp == kMmaWarp)
    {
        const bool      el = elect_one();
        int             g = 0, n_item = 0;
        bool            ok = true;
        Halves<kSwiglu> half;
        for (int v = blockIdx.x; v < items && ok; v += gridDim.x, ++n_item)
        {
            const Item     it    = get_item<kSlab>(p, before, list, w_blocks, n_item, v);
            const int      cols  = (it.count + 15) & ~15;
            const uint32_t idesc = p.idesc | (static_cast<uint32_t>(cols >> 3) << 17);
            half.take(it.count);
            for (int h = 0; h < 2 && ok; ++h)
            {
                if (half.both || half.first == h)
                {
                    ok = warp_wait(tempty_bar(h), (static_cast<uint32_t>(half.used[h]) & 1u) ^ 1u, s_abort, DEV_TIMEOUT_MMA, p.spin_limit);
                }
            }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + half.first * 128, d_up = d_tmem + (half.both ? 128 : 64);
            for (int c = 0; c < chunks && ok; ++c, ++g)
            {
                const int s = g % STAGES;
                ok = warp_wait(full_bar(s), static_cast<uint32_t>(g / STAGES) & 1u, s_abort, DEV_TIMEOUT_MMA, p.spin_limit);
                if (!ok) break;
                tc_fence_after();
                const int      n     = min(F::kChunkTiles, static_cast<int>(p.k_tiles) - c * F::kChunkTiles);
                const int      steps = min(kMxChunk / kMxStepK, (p.K - c * kMxChunk + kMxStepK - 1) / kMxStepK);
                const uint32_t t_w   = tmem_base + P::SF_COL + s * P::SF_COLS, t_t = t_w + W * F::kChunkCols;
                const uint32_t sf    = s_sf + s * P::SF_STAGE, st = s_stage + s * P::STAGE;
                if (el)
                {
#pragma unroll
                    for (int w = 0; w <= W; ++w) mx_chunk_scales<kFormat>(t_w + w * F::kChunkCols, sf + w * F::kChunkScale, n);
                    mx_chunk<kFormat>(d_tmem, st, st + W * kMxWBytes, t_w, t_t, idesc, steps, c == 0);
                    if constexpr (kSwiglu) mx_chunk<kFormat>(d_up, st + kMxWBytes, st + W * kMxWBytes, t_w + F::kChunkCols, t_t, idesc, steps, c == 0);
                    umma_commit(empty_bar(s));
                }
                __syncwarp();
            }
            if (ok && el)
            {
                if (half.both || half.first == 0) umma_commit(tfull_bar(0));
                if (half.both || half.first == 1) umma_commit(tfull_bar(1));
            }
            half.done();
        }
        __syncwarp();
    }
    else
    {
        const int       q = warp & 3, turn = (warp - kFirstEpi) >> 2;
        Halves<kSwiglu> half;
        bool            ok = true;
        int             n_item = 0;
        for (int v = blockIdx.x; v < items && ok; v += gridDim.x, ++n_item)
        {
            const Item    it = get_item<kSlab>(p, before, list, w_blocks, n_item, v);
            const int     n  = it.wb * kMxRows + q * 32 + lane;
            const Factors f  = group_factors(p, it.group);
            const float   b  = group_bias(p, it.group, n);
            half.take(it.count);
            for (int h = 0; h < 2 && ok; ++h)
            {
                if (half.both || half.first == h)
                {
                    ok = warp_wait(tfull_bar(h), static_cast<uint32_t>(half.used[h]) & 1u, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit);
                }
            }
            if (!ok) break;
            tc_fence_after();
            const uint32_t acc = tmem_base + half.first * 128 + (static_cast<uint32_t>(q * 32) << 16), up = acc + (half.both ? 128 : 64);
            for (int j = 16 * turn; j < it.count; j += 32)
            {
                uint32_t r[16], u[16];
                tmem_ld_x16(acc + j, r);
                if constexpr (kSwiglu) tmem_ld_x16(up + j, u);
                tmem_ld_wait();
                float x[16];
                finish<kSwiglu>(p, r, u, f, [&](int) { return b; }, x);
                store_tokens(p, it.row + j, n, x, it.count - j);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
            {
                if (half.both || half.first == 0) mbar_arrive(tempty_bar(0));
                if (half.both || half.first == 1) mbar_arrive(tempty_bar(1));
            }
            __syncwarp();
            half.done();
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
        tmem_dealloc(tmem_base, 512);
    }
    if (threadIdx.x == 0 && *s_abort != 0)
    {
        atomicCAS(p.status, 0, *s_abort);
    }
}

// ---- many rows a group: SM pairs -----------------------------------------------------------------------------
// 256 channels x 256 tokens per cluster of two CTAs as in the plain product's pair kernel, or, for SwiGLU, 256 channels of both weight
// matrices x 128 tokens: the same 256 accumulator columns, the first half of them the gate's sums.  A tile's MMAs have as many
// columns as it has rows, in steps of 32 (sixteen staged by each CTA).  The boxes of tokens are whole, so that every stage counts
// the same bytes.
//
// Tensor memory: two accumulators that share 64 columns (0 .. 255 and 192 .. 447), the rest holds the scales of one chunk; a chunk's
// scales overwrite those of the chunk before behind the MMAs that read them (one thread's copies and MMAs go through one queue).  The
// epilogue drains the shared columns first.
constexpr int kPairCols   = 256;
constexpr int kPairShared = 64;
constexpr int kStaging    = 2048;
template <int kFormat, bool kSwiglu>
struct PairPlan
{
    using F                        = MxTraits<kFormat>;
    static constexpr int WEIGHTS   = kSwiglu ? 2 : 1;
    static constexpr int TILE      = kSwiglu ? 128 : 256; // tokens
    // Epilogue warps, two or four per tensor-memory lane quarter.  us sustained with eight / sixteen, 4096 tokens, top 8 of 64, NVFP4 to BF16:
    // SwiGLU 2048 -> 768 72.1 / 74.9 (power is what bounds it), 768 -> 2048 52.8 / 51.6.
    static constexpr int EPI       = kSwiglu ? 8 : 16;
    static constexpr int THREADS   = 32 * (kFirstEpi + EPI);
    static constexpr int STAGES    = kSwiglu ? 4 : 5;
    static constexpr int T_BYTES   = TILE / 2 * kMxChunkBytes;
    static constexpr int STAGE     = WEIGHTS * kMxWBytes + T_BYTES;
    static constexpr int SF_PARTS  = WEIGHTS + TILE / 128;
    static constexpr int SF_STAGE  = SF_PARTS * F::kChunkScale;
    static constexpr int OFF_OUT   = STAGES * STAGE; // staging: 2 KB per epilogue warp
    static constexpr int OFF_SF    = OFF_OUT + EPI * kStaging;
    static constexpr int OFF_BAR   = OFF_SF + STAGES * SF_STAGE;
    static constexpr int OFF_MISC  = OFF_BAR + (2 * STAGES + 4) * 8;
    static constexpr int OFF_SCAN  = OFF_MISC + 16;
    static constexpr int OFF_LIST  = OFF_SCAN + (kMaxGroups + 1) * 4;
    static constexpr int DYN_BYTES = OFF_LIST + kListed * static_cast<int>(sizeof(ListedItem)) + 1024;
    static constexpr int SF_COL    = 2 * kPairCols - kPairShared;
    static_assert(SF_COL + SF_PARTS * F::kChunkCols <= 512 && DYN_BYTES <= 232448, "tensor and shared memory of an SM");
    static_assert(STAGE % 1024 == 0, "operands start at multiples of the swizzle's period");
};

// 32 channels x 32 tokens of results (two halves of 16 lanes as fragments) to a staging area of 32 rows of 64 bytes in the 64-byte
// swizzle; r: neighbours of a row as words, the lower half's eight first.
__device__ __forceinline__ void stage_results(uint32_t s_out, int lane, const uint32_t (&r)[2][8])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) // eight tokens: matrix m holds channels 8 m .. 8 m + 7
    {
        const int      row  = 8 * i + (lane & 7), chunk = lane >> 3;
        const uint32_t addr = s_out + static_cast<uint32_t>(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
        stmatrix_x4_trans(addr, r[0][2 * i], r[0][2 * i + 1], r[1][2 * i], r[1][2 * i + 1]);
    }
}
template <typename T>
__device__ __forceinline__ uint32_t pack_two(float a, float b)
{
    const T  two[2] = {from_float<T>(a), from_float<T>(b)};
    uint32_t w;
    memcpy(&w, two, 4);
    return w;
}
// The first `cols` rows of a staging area to rows m and up of dst, channels n0 and up.  Bulk stores write whole boxes: this is for the one
// that a group's end cuts.
__device__ __forceinline__ void store_staged(const GroupedParams &p, const uint8_t *area, int lane, int m, int n0, int cols)
{
    const int units = min(4, (p.channels - n0) / 8); // of 16 bytes; rows are whole units long
    for (int i = lane; i < cols * 4; i += 32)
    {
        const int row = i / 4, unit = i % 4;
        if (unit < units)
        {
            *reinterpret_cast<uint4 *>(p.dst + static_cast<int64_t>(m + row) * p.ldd + static_cast<int64_t>(n0) * 2 + unit * 16) =
                *reinterpret_cast<const uint4 *>(area + row * 64 + ((unit ^ ((row >> 1) & 3)) << 4));
        }
    }
}

template <int kFormat, bool kBulk, bool kSwiglu>
__global__ void __launch_bounds__((PairPlan<kFormat, kSwiglu>::THREADS), 1)
    mx_grouped_pair_kernel(const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_up, const __grid_constant__ CUtensorMap tmap_a,
                           const __grid_constant__ CUtensorMap tmap_bsf, const __grid_constant__ CUtensorMap tmap_upsf,
                           const __grid_constant__ CUtensorMap tmap_asf, const __grid_constant__ CUtensorMap tmap_out,
                           const __grid_constant__ GroupedParams p)
{
    using P = PairPlan<kFormat, kSwiglu>;
    using F = MxTraits<kFormat>;
    constexpr int STAGES = P::STAGES, W = P::WEIGHTS, TILE = P::TILE;
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
    int           *before    = reinterpret_cast<int *>(smem + P::OFF_SCAN);
    ListedItem    *list      = reinterpret_cast<ListedItem *>(smem + P::OFF_LIST);
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int      rank     = static_cast<int>(cluster_ctarank());
    const int      w_blocks = (p.channels + 2 * kMxRows - 1) / (2 * kMxRows);
    const int      chunks   = (p.K + kMxChunk - 1) / kMxChunk;
    const int      first    = static_cast<int>(cluster_id_x());
    const int      stride   = static_cast<int>(num_clusters_x());

    if (threadIdx.x == 0)
    {
        for (int s = 0; s < STAGES; ++s)
        {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(tfull_bar(0), 1);
        mbar_init(tfull_bar(1), 1);
        mbar_init(tempty, 2 * P::EPI);
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
    griddep_wait(); // the groups come from a kernel ahead
    const int items = scan_groups<TILE>(p, before) * w_blocks;
    list_items<TILE>(p, before, list, w_blocks, first, stride, items);

    int issued = 0; // stages that the producer has filled
    if (warp == 0)
    {
        const bool el = elect_one();
        int        g = 0, n_item = 0;
        const int  kt = static_cast<int>(p.k_tiles);
        for (int v = first; v < items; v += stride, ++n_item)
        {
            const Item it    = get_item<TILE>(p, before, list, w_blocks, n_item, v);
            const int  w_row = it.group * p.channels + (it.wb * 2 + rank) * kMxRows;
            const int  w_sf  = static_cast<int>(it.group * p.group_tiles) + (it.wb * 2 + rank) * kt, a_sf = it.row / kSlab * kt;
            const int  a_row = it.row + rank * (((it.count + 31) & ~31) >> 1); // this CTA's half of the MMAs' columns
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
                const int      sf0 = c * F::kChunkTiles;
                if (el)
                {
                    if (rank == 0) mbar_expect_tx(full_bar(s), 2 * (P::STAGE + P::SF_STAGE));
                    tma_load_2d_pair(dst, &tmap_b, c * kMxChunkBytes, w_row, bar);
                    tma_load_2d_pair(sf, &tmap_bsf, 0, w_sf + sf0, bar);
                    if constexpr (kSwiglu)
                    {
                        tma_load_2d_pair(dst + kMxWBytes, &tmap_up, c * kMxChunkBytes, w_row, bar);
                        tma_load_2d_pair(sf + F::kChunkScale, &tmap_upsf, 0, w_sf + sf0, bar);
                    }
                    tma_load_2d_pair(dst + W * kMxWBytes, &tmap_a, c * kMxChunkBytes, a_row, bar);
#pragma unroll
                    for (int t = 0; t < TILE / 128; ++t) tma_load_2d_pair(sf + (W + t) * F::kChunkScale, &tmap_asf, 0, a_sf + t * kt + sf0, bar);
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
            int            g = 0, it = 0;
            bool           ok  = true;
            const uint32_t t_w = tmem_base + P::SF_COL, t_t = t_w + W * F::kChunkCols;
            constexpr int  kStepCols = 4 * (TILE / 128); // scale columns of a step's tokens
            for (int v = first; v < items && ok; v += stride, ++it)
            {
                const Item     item  = get_item<TILE>(p, before, list, w_blocks, it, v);
                const int      cols  = (item.count + 31) & ~31;
                const uint32_t idesc = p.idesc | (static_cast<uint32_t>(cols >> 3) << 17);
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
                    const uint64_t a_desc = make_kmajor_sw128_desc(s_stage + s * P::STAGE), b_desc = a_desc + (W * kMxWBytes >> 4);
                    if (el)
                    {
#pragma unroll
                        for (int t = 0; t < F::kChunkTiles; ++t) // a step's tokens: rows 0..127 in four columns, 128..255 in the next four
                        {
                            const uint64_t at = sf + static_cast<uint64_t>(t * (kMxTileBytes >> 4));
#pragma unroll
                            for (int w = 0; w < W; ++w) tmem_copy_scales_pair(t_w + w * F::kChunkCols + 4 * t, at + w * (F::kChunkScale >> 4));
                            tmem_copy_scales_pair(t_t + kStepCols * t, at + W * (F::kChunkScale >> 4));
                            if (TILE > 128 && cols > 128) tmem_copy_scales_pair(t_t + kStepCols * t + 4, at + (W + 1) * (F::kChunkScale >> 4));
                        }
#pragma unroll
                        for (int w = 0; w < W; ++w)
                        {
#pragma unroll
                            for (int k = 0; k < kMxChunk / kMxStepK; ++k)
                            {
                                if (k < steps)
                                {
                                    umma_mx_pair<kFormat>(d_tmem + 128 * w, a_desc + w * (kMxWBytes >> 4) + 2u * k, b_desc + 2u * k, idesc | mx_scale_id<kFormat>(k),
                                                          t_w + w * F::kChunkCols + 4 * mx_step_tile<kFormat>(k), t_t + kStepCols * mx_step_tile<kFormat>(k),
                                                          (c | k) != 0 ? 1u : 0u);
                                }
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
        // Two or four warps per lane quarter, which take turns with groups of 32 tokens; those in the shared columns are the first two groups.
        constexpr int  kTurns = P::EPI / 4;
        const int      q = warp & 3, turn = (warp - kFirstEpi) >> 2;
        const uint32_t release = map_to_cta(tempty, 0);
        uint8_t       *out     = smem + P::OFF_OUT + (warp - kFirstEpi) * kStaging;
        const uint32_t s_out   = s_stage + P::OFF_OUT + (warp - kFirstEpi) * kStaging;
        int            it = 0;
        for (int v = first; v < items; v += stride, ++it)
        {
            const Item    item = get_item<TILE>(p, before, list, w_blocks, it, v);
            const int     as = it & 1, n0 = (item.wb * 2 + rank) * kMxRows + q * 32;
            const Factors f  = group_factors(p, item.group);
            float         bias[4] = {}; // kBulk: of the fragments' rows, else of this lane's channel
            if (!kSwiglu && p.bias != nullptr)
            {
#pragma unroll
                for (int i = 0; i < (kBulk ? 4 : 1); ++i) bias[i] = group_bias(p, item.group, n0 + (kBulk ? lane / 4 + 8 * i : lane));
            }
            if (!warp_wait(tfull_bar(as), static_cast<uint32_t>(it >> 1) & 1u, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit))
            {
                break;
            }
            tc_fence_after();
            const uint32_t acc = tmem_base + as * (kPairCols - kPairShared) + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
            for (int i = 0; i < TILE / (32 * kTurns); ++i)
            {
                const int  group = kTurns * i + turn;
                const int  j     = as == 0 ? (group * 32 + TILE - kPairShared) % TILE : group * 32;
                const bool any   = j < item.count && n0 < p.channels; // the same for the warp
                auto       drained = [&]() { // the shared columns have been read
                    if (i == 0)
                    {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster_no_writes(release);
                        __syncwarp(); // aligned loads of tensor memory may be next
                    }
                };
                if (!any)
                {
                    drained();
                    continue;
                }
                const int m = item.row + j, cols = item.count - j;
                uint32_t  r[2][16], u[2][16]; // all of it first: the next tile's MMAs wait for the shared columns
#pragma unroll
                for (int h = 0; h < 2; ++h)
                {
                    if constexpr (kBulk)
                    {
                        tmem_ld_frag32(acc + j + (static_cast<uint32_t>(16 * h) << 16), r[h]);
                        if constexpr (kSwiglu) tmem_ld_frag32(acc + 128 + j + (static_cast<uint32_t>(16 * h) << 16), u[h]);
                    }
                    else
                    {
                        tmem_ld_x16(acc + j + 16 * h, r[h]);
                        if constexpr (kSwiglu) tmem_ld_x16(acc + 128 + j + 16 * h, u[h]);
                    }
                }
                tmem_ld_wait();
                drained();
                if constexpr (kBulk)
                {
                    uint32_t packed[2][8];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                    {
                        float x[16]; // elements 4 i + 0, 1 belong to row lane / 4, 4 i + 2, 3 to row lane / 4 + 8
                        finish_as<kSwiglu, true>(r[h], u[h], f, [&](int k) { return bias[2 * h + ((k >> 1) & 1)]; }, x);
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                        {
                            packed[h][k] = p.dtype == CUGL_F16 ? pack_two<__half>(x[2 * k], x[2 * k + 1]) : pack_two<__nv_bfloat16>(x[2 * k], x[2 * k + 1]);
                        }
                    }
                    if (lane == 0) tma_store_wait_read(); // the store that reads this area has done so
                    __syncwarp();
                    stage_results(s_out, lane, packed);
                    if (cols >= 32)
                    {
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) tma_store_2d(&tmap_out, s_out, n0, m);
                    }
                    else
                    {
                        __syncwarp();
                        store_staged(p, out, lane, m, n0, cols);
                    }
                    if (lane == 0) tma_store_commit();
                    __syncwarp();
                }
                else
                {
#pragma unroll
                    for (int h = 0; h < 2; ++h) // sixteen tokens
                    {
                        float x[16];
                        finish<kSwiglu>(p, r[h], u[h], f, [&](int) { return bias[0]; }, x);
                        const int left = cols - 16 * h;
                        store_tokens(p, m + 16 * h, n0 + lane, x, left);
                    }
                }
            }
            tc_fence_before();
        }
        if (kBulk && lane == 0)
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
            drain_pair_stages<STAGES>(bar_base, issued, static_cast<int>(peer & 0x7fffffffu), blockIdx.x == 0 ? p.withhold : -1, p.spin_limit,
                                      [](int) { return static_cast<uint32_t>(P::STAGE + P::SF_STAGE); });
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

// ---- host ----------------------------------------------------------------------------------------------------
struct GroupedOperands
{
    const cugl_mx_grouped_gemm_desc *d;
    const void                      *a, *b, *up;
};

template <int kFormat, bool kSwiglu>
cugl_status launch_few(cugl_context *ctx, const GroupedOperands &op, GroupedParams p, long long items)
{
    using P = FewPlan<kFormat, kSwiglu>;
    CUtensorMap   map_b, map_up{};
    TokenMaps     map_a;
    const int64_t inner = (static_cast<int64_t>(p.K) + 1) / 2, weights = static_cast<int64_t>(p.n_groups) * p.channels;
    bool          ok = encode_packed_map(&map_b, op.b, weights, inner, op.d->ldb, kMxRows) && (!kSwiglu || encode_packed_map(&map_up, op.up, weights, inner, op.d->ldb, kMxRows));
    for (int i = 0; i < 4; ++i) ok = ok && encode_packed_map(&map_a.rows[i], op.a, p.rows, inner, op.d->lda, 16 << i);
    if (!ok)
    {
        return fail(ctx, CUGL_RUNTIME_ERROR, "cuTensorMapEncodeTiled failed for a packed operand");
    }
    auto                     kernel  = mx_grouped_few_kernel<kFormat, kSwiglu>;
    static std::atomic<bool> set[64] = {};
    CUGL_TRY(allow_smem(ctx, kernel, P::DYN_BYTES, set));
    p.idesc        = mx_idesc(kFormat, kMxRows, 0);
    const int grid = static_cast<int>(items < ctx->sm_count ? items : ctx->sm_count);
    CUGL_CUDA_TRY(ctx, launch_dependent(ctx, kernel, dim3(static_cast<unsigned>(grid)), kFewThreads, P::DYN_BYTES, items, map_b, map_up, map_a, p));
    return CUGL_SUCCESS;
}

// 16-bit dst in boxes of 32 rows x 32 channels, in the 64-byte swizzle
bool encode_results_map(CUtensorMap *map, const GroupedParams &p)
{
    EncodeTiledFn    fn         = get_encode_fn();
    const cuuint64_t dims[2]    = {static_cast<cuuint64_t>(p.channels), static_cast<cuuint64_t>(p.rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(p.ldd)};
    const cuuint32_t box[2]     = {32, 32};
    const cuuint32_t estr[2]    = {1, 1};
    return fn != nullptr && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, p.dst, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                               CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kFormat, bool kBulk, bool kSwiglu>
cugl_status launch_pair(cugl_context *ctx, const GroupedOperands &op, GroupedParams p, long long items)
{
    using P = PairPlan<kFormat, kSwiglu>;
    using F = MxTraits<kFormat>;
    CUtensorMap   map_b, map_up{}, map_a, map_bsf, map_upsf{}, map_asf, map_out{};
    const int64_t inner = (static_cast<int64_t>(p.K) + 1) / 2, weights = static_cast<int64_t>(p.n_groups) * p.channels;
    const int64_t w_tiles = p.n_groups * p.group_tiles, a_tiles = (static_cast<int64_t>(p.rows) + kSlab - 1) / kSlab * p.k_tiles;
    if (!encode_packed_map(&map_b, op.b, weights, inner, op.d->ldb, kMxRows) || !encode_packed_map(&map_a, op.a, p.rows, inner, op.d->lda, P::TILE / 2) ||
        !encode_scale_map(&map_bsf, p.b_scales, w_tiles, F::kChunkTiles) || !encode_scale_map(&map_asf, p.a_scales, a_tiles, F::kChunkTiles) ||
        (kSwiglu && (!encode_packed_map(&map_up, op.up, weights, inner, op.d->ldb, kMxRows) || !encode_scale_map(&map_upsf, p.up_scales, w_tiles, F::kChunkTiles))) ||
        (kBulk && !encode_results_map(&map_out, p)))
    {
        return fail(ctx, CUGL_RUNTIME_ERROR, "cuTensorMapEncodeTiled failed for an operand");
    }
    auto                     kernel  = mx_grouped_pair_kernel<kFormat, kBulk, kSwiglu>;
    static std::atomic<bool> set[64] = {};
    CUGL_TRY(allow_smem(ctx, kernel, P::DYN_BYTES, set));
    p.idesc         = mx_idesc(kFormat, 2 * kMxRows, 0);
    const int pairs = ctx->sm_count / 2, grid = 2 * static_cast<int>(items < pairs ? items : pairs);
    CUGL_CUDA_TRY(ctx, launch_dependent_cluster(ctx, kernel, dim3(static_cast<unsigned>(grid)), P::THREADS, P::DYN_BYTES, 2, 2 * items, map_b, map_up, map_a, map_bsf,
                                                map_upsf, map_asf, map_out, p));
    return CUGL_SUCCESS;
}

template <int kFormat, bool kSwiglu>
cugl_status launch_grouped(cugl_context *ctx, const GroupedOperands &op, const GroupedParams &p)
{
    // tiles that the rows make at most (for the size of the grid): every group may end in one that is not full
    const long long expected = op.d->expected_rows > 0 ? op.d->expected_rows : p.rows;
    auto            items    = [&](int rows, int channels) {
        const long long tiles = (expected + rows - 1) / rows + (expected < p.n_groups ? expected : p.n_groups);
        return tiles * ((p.channels + channels - 1) / channels);
    };
    // us on one CTA per SM / SM pairs at 48, 64, 96, 128 rows a group, NVFP4.  64 groups, 2048 -> 768 SwiGLU to BF16 25.0 / 26.4, 25.4 / 26.9,
    // 30.3 / 27.6, 33.0 / 29.0; 64 groups, 768 -> 2048 to BF16 14.9 / 15.4, 15.3 / 15.3, 17.7 / 16.2, 21.0 / 17.8; 8 groups, 4096 -> 4096 to BF16
    // 16.0 / 16.4, 16.2 / 16.4, 17.2 / 16.6, 17.6 / 17.5.  Floats leave from registers either way: at 96, 128, 160, 256 rows 8 groups, 4096 -> 4096
    // 17.4 / 17.6, 18.3 / 18.7, 27.5 / 21.1, 30.2 / 26.5; 64 groups, 1024 -> 1024 14.4 / 15.5, 15.3 / 16.6, 21.3 / 19.6, 24.8 / 25.6.
    if (expected < (p.dtype == CUGL_F32 ? 130ll : 72ll) * p.n_groups)
    {
        return launch_few<kFormat, kSwiglu>(ctx, op, p, items(kSlab, kMxRows));
    }
    const long long n = items(PairPlan<kFormat, kSwiglu>::TILE, 2 * kMxRows);
    return p.vec_out != 0 && p.dtype != CUGL_F32 ? launch_pair<kFormat, true, kSwiglu>(ctx, op, p, n) : launch_pair<kFormat, false, kSwiglu>(ctx, op, p, n);
}

const char *validate_grouped(const cugl_mx_grouped_gemm_desc *d)
{
    if (d == nullptr) return "descriptor is NULL";
    if (d->groups < 1 || d->groups > kMaxGroups) return "groups must lie within 1 .. 512";
    if (d->rows < 0 || d->N < 1 || d->K < 1) return "rows must not be negative, N and K must be positive";
    if (d->rows > INT32_MAX - 1024 || d->N > INT32_MAX - 1024 || d->K > INT32_MAX - 1024) return "a dimension is too large";
    if (d->expected_rows < 0) return "expected_rows must not be negative";
    if (d->format != CUGL_MXFP4 && d->format != CUGL_NVFP4) return "format must be CUGL_MXFP4 or CUGL_NVFP4";
    if (!is_float_dtype(d->dst_dtype)) return "dst_dtype must be CUGL_F32, CUGL_F16 or CUGL_BF16";
    if (d->swiglu != 0 && d->has_bias != 0) return "a bias is for the plain product";
    const int64_t row = (static_cast<int64_t>(d->K) + 1) / 2;
    if (d->lda < row || d->ldb < row || d->lda % 16 != 0 || d->ldb % 16 != 0) return "lda and ldb must hold a packed row and be multiples of 16";
    if (d->lda >= (1ll << 40) || d->ldb >= (1ll << 40) || d->ldd >= (1ll << 40)) return "lda, ldb and ldd must be below 2^40";
    const int size = dtype_size(d->dst_dtype);
    if (d->ldd < static_cast<int64_t>(d->N) * size || d->ldd % size != 0) return "ldd must hold a row of dst and be a multiple of its element size";
    if (!(d->alpha - d->alpha == 0.f) || !(d->up_alpha - d->up_alpha == 0.f)) return "alpha and up_alpha must be finite";
    // coordinates of tiles and items are 32-bit numbers
    const int64_t k_tiles = mx_scale_tiles(d->K, d->format);
    if (d->groups * ((static_cast<int64_t>(d->N) + 255) / 128) * k_tiles > INT32_MAX / 2 || (static_cast<int64_t>(d->rows) / kSlab + 2) * k_tiles > INT32_MAX / 2 ||
        static_cast<int64_t>(d->groups) * d->N > INT32_MAX - 1024)
        return "weights or rows of more than 2^30 scale tiles";
    if ((static_cast<int64_t>(d->rows) / kSlab + d->groups) * ((static_cast<int64_t>(d->N) + 127) / 128) > INT32_MAX / 8) return "more than 2^28 output tiles";
    return nullptr;
}
} // namespace
} // namespace cugl

using namespace cugl;

extern "C"
{
    int64_t cugl_mx_group_rows(int32_t groups, int64_t rows)
    {
        if (groups < 0 || rows < 0 || rows > (1ll << 40))
        {
            return 0;
        }
        return (rows + (kSlab - 1) * (groups < rows ? groups : rows)) / kSlab * kSlab;
    }

    cugl_status cugl_mx_grouped_gemm_validate(const cugl_mx_grouped_gemm_desc *desc, const char **reason)
    {
        const char *why = validate_grouped(desc);
        if (reason != nullptr)
        {
            *reason = why != nullptr ? why : "";
        }
        return why == nullptr ? CUGL_SUCCESS : CUGL_INVALID_ARGUMENT;
    }

    cugl_status cugl_mx_grouped_gemm(cugl_context *ctx, const cugl_mx_grouped_gemm_desc *desc, const void *d_a, const void *d_a_scales,
                                     const int32_t *d_groups, const void *d_b, const void *d_b_scales, const float *d_b_alpha, const void *d_up,
                                     const void *d_up_scales, const float *d_up_alpha, const float *d_bias, void *d_dst)
    {
        if (ctx == nullptr)
        {
            return fail(nullptr, CUGL_INVALID_ARGUMENT, "context is NULL");
        }
        const char *why = validate_grouped(desc);
        if (why == nullptr && desc->rows > 0)
        {
            auto            bits = [](const void *q) { return reinterpret_cast<uintptr_t>(q); };
            const uintptr_t in   = bits(d_a) | bits(d_a_scales) | bits(d_b) | bits(d_b_scales) | bits(d_up) | bits(d_up_scales);
            if (d_a == nullptr || d_a_scales == nullptr || d_groups == nullptr || d_b == nullptr || d_b_scales == nullptr || d_dst == nullptr) why = "NULL pointer";
            else if ((desc->has_bias != 0) != (d_bias != nullptr)) why = "d_bias must be given exactly when has_bias is set";
            else if ((desc->swiglu != 0) != (d_up != nullptr) || (desc->swiglu != 0) != (d_up_scales != nullptr))
                why = "d_up and d_up_scales must be given exactly when swiglu is set";
            else if (desc->swiglu == 0 && d_up_alpha != nullptr) why = "d_up_alpha is for swiglu";
            else if ((in & 15) != 0) why = "operands and scale tiles must be 16-byte aligned";
            else if (bits(d_groups) % 8 != 0) why = "groups must be 8-byte aligned";
            else if (bits(d_dst) % static_cast<uintptr_t>(dtype_size(desc->dst_dtype)) != 0 || (bits(d_bias) | bits(d_b_alpha) | bits(d_up_alpha)) % 4 != 0)
                why = "dst, bias or factors are not aligned to their elements";
        }
        if (why != nullptr)
        {
            return fail(ctx, CUGL_INVALID_ARGUMENT, std::string("cugl_mx_grouped_gemm: ") + why);
        }
        if (desc->rows == 0) return CUGL_SUCCESS;
        const DeviceScope device(ctx);
        const int         size = dtype_size(desc->dst_dtype);
        const uintptr_t   out  = reinterpret_cast<uintptr_t>(d_dst) | static_cast<uintptr_t>(desc->ldd);
        GroupedParams     p{};
        p.groups      = reinterpret_cast<const int2 *>(d_groups);
        p.a_scales    = static_cast<const uint8_t *>(d_a_scales);
        p.b_scales    = static_cast<const uint8_t *>(d_b_scales);
        p.up_scales   = static_cast<const uint8_t *>(d_up_scales);
        p.dst         = static_cast<uint8_t *>(d_dst);
        p.bias        = d_bias;
        p.b_alpha     = d_b_alpha;
        p.up_alpha    = d_up_alpha;
        p.ldd         = desc->ldd;
        p.k_tiles     = mx_scale_tiles(desc->K, desc->format);
        p.group_tiles = (static_cast<int64_t>(desc->N) + 127) / 128 * p.k_tiles;
        p.n_groups    = desc->groups;
        p.rows        = desc->rows;
        p.channels    = desc->N;
        p.K           = desc->K;
        p.dtype       = desc->dst_dtype;
        p.pack_out    = (out & 3) == 0 && desc->N % 2 == 0;
        p.vec_out     = (out & 15) == 0 && desc->N * static_cast<int64_t>(size) % 16 == 0;
        p.alpha       = desc->alpha;
        p.up_scale    = desc->up_alpha;
        p.status      = ctx->d_status;
        p.spin_limit  = ctx->spin_limit;
        p.withhold    = ctx->withhold_kb;
        ctx->withhold_kb = -1;
        const GroupedOperands op{desc, d_a, d_b, d_up};
        if (desc->format == CUGL_NVFP4)
        {
            return desc->swiglu != 0 ? launch_grouped<CUGL_NVFP4, true>(ctx, op, p) : launch_grouped<CUGL_NVFP4, false>(ctx, op, p);
        }
        return desc->swiglu != 0 ? launch_grouped<CUGL_MXFP4, true>(ctx, op, p) : launch_grouped<CUGL_MXFP4, false>(ctx, op, p);
    }
}
