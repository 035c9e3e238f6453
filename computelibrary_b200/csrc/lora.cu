// Low-rank adapters of many requests at once, beside a projection that all of them share:
//   dst[t] = base[t] + scale_a * (x[t] . A_a^T) . B_a^T          a: the adapter of the request that token t belongs to
//
// Two launches.  The first makes v = x . A^T: a tile of up to 64 tokens of one request per cluster, whose CTAs share K; their sums are added
// up in a fixed order through distributed shared memory.  The second adds scale * v . B^T to base, 256 channels x a tile of tokens per
// CTA.  Which tiles there are is known on the device only (the requests' lengths): every CTA counts them (a scan over the requests)
// and takes the one with its number; the grid is the most that there can be.
//
// What bounds it: bytes.  x, base and dst pass once, the adapters once per tile of tokens; with ranks up to 128 the products are short
// work (4096 tokens, 4096 -> 4096, rank 64: 2 x 2.1 GFLOP beside 170 MB).  Hence mma.sync, whose accumulators are the registers that
// base is added to: nothing of a matrix unit's rate is missing, and no operand waits in shared memory.
//
// Fragments.  Sums do not care in which order their terms come, as long as both operands agree: a lane takes 8 consecutive elements of
// K (16 bytes) as the four pairs that two steps of the matrix instruction want from it, and 4 consecutive ranks as the two pairs of
// one step.  Channels likewise: the four 8-column tiles of a warp's 32 channels are dealt out so that a lane's results are 8 consecutive
// channels of a row.
//
// v is kept as two 16-bit parts, v = high + low (three where bf16 adapters add to 32-bit results): 16 (bf16) or 22 (f16) bits of it
// count, 24 with three parts, so rounding v costs less than rounding the result.  f16 parts would leave that type's range: a token's
// v is first divided by a power of two that brings its largest rank into [1, 2).
#include "mx.cuh"
#include "sm100.cuh"

#include <atomic>
#include <cmath>
#include <cstring>

namespace cugl
{
namespace
{
constexpr int kThreads  = 256;
constexpr int kWarps    = kThreads / 32;
constexpr int kChannels = 32 * kWarps; // of a CTA of the second launch
constexpr int kMaxRank  = 128;
constexpr int kMaxSplit = 8;

struct LoraParams
{
    const uint8_t *x, *a, *b, *base;
    uint8_t       *dst;
    const int32_t *starts, *adapters, *ranks;
    const float   *scales;
    uint16_t      *v;      // [parts][tokens][padded rank]
    float         *factor; // [tokens]
    int64_t        ld_x, ld_a, ld_b, ld_base, ld_dst; // bytes
    int            tokens, requests, n_adapters, max_rank, K, N, parts, tile;
};

// ---- which tokens a tile holds -------------------------------------------------------------------------------
struct Tile
{
    int first, count; // tokens; count 0: there is no such tile
    int adapter;      // -1: none
    int rank;
};
// Loads that may come ahead of griddepcontrol.wait, of what was complete before the launch ahead passed its own wait: from L2, where a line
// that an earlier kernel left in this SM's L1 does not count.
__device__ __forceinline__ int load_l2(const int32_t *p)
{
    return __ldcg(p);
}
// A request's tokens are [starts[i], starts[i + 1]), cut to those there are.  Called by all threads.
__device__ __forceinline__ Tile find_tile(const LoraParams &p, int wanted)
{
    __shared__ Tile found;
    __shared__ int  sums[kWarps];
    const int       lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) found = Tile{0, 0, -1, 0};
    int before = 0;
    for (int r0 = 0; r0 < p.requests; r0 += kThreads)
    {
        const int r = r0 + static_cast<int>(threadIdx.x);
        int       begin = 0, end = 0;
        if (r < p.requests)
        {
            begin = min(max(load_l2(p.starts + r), 0), p.tokens);
            end   = min(max(load_l2(p.starts + r + 1), begin), p.tokens);
        }
        const int tiles = (end - begin + p.tile - 1) / p.tile;
        int       incl  = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const int n = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += n;
        }
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        int at = before, all = before;
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
        {
            if (w < warp) at += sums[w];
            all += sums[w];
        }
        at += incl - tiles;
        if (wanted >= at && wanted < at + tiles)
        {
            const int first = begin + (wanted - at) * p.tile;
            int       a     = load_l2(p.adapters + r), rank = 0;
            if (a >= 0 && a < p.n_adapters) rank = p.ranks != nullptr ? min(max(load_l2(p.ranks + a), 0), p.max_rank) : p.max_rank;
            found = Tile{first, min(p.tile, end - first), rank > 0 ? a : -1, rank};
        }
        before = all;
        __syncthreads();
        if (wanted < before) break; // the same for all
    }
    __syncthreads();
    return found;
}

// ---- matrix instruction --------------------------------------------------------------------------------------
// D (+)= A . B, 16 x 8 x 16: rows lane / 4 and lane / 4 + 8, columns 2 (lane % 4) and the next
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<T, __half>::value)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    else
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

// eight 16-bit elements of a row from column k on, zeros behind `cols`
template <bool kVec>
__device__ __forceinline__ uint4 load_eight(const uint8_t *row, int k, int cols)
{
    const uint16_t *src = reinterpret_cast<const uint16_t *>(row) + k;
    if (kVec && k + 8 <= cols) return __ldg(reinterpret_cast<const uint4 *>(src));
    uint16_t e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = k + i < cols ? __ldg(src + i) : static_cast<uint16_t>(0);
    uint4 v;
    memcpy(&v, e, 16);
    return v;
}

// ---- first launch: v = x . A^T -------------------------------------------------------------------------------
// A warp multiplies 16 kMt tokens with all ranks over a share of K; tiles of more tokens take two warps side by side.  The loads of two
// blocks of 32 columns are in flight per warp.
template <int kRank>
struct Shrink
{
    static constexpr int kMt     = kRank == 128 ? 1 : 2; // 16-row tiles of a warp
    static constexpr int kRows   = 16 * kMt;
    static constexpr int kTile   = 2 * kRows;
    static constexpr int kPitch  = kRank + 8; // floats: rows in different banks
    static constexpr int kSmem   = kWarps * kRows * kPitch * 4;
    static_assert(kTile * kPitch <= kWarps * kRows * kPitch, "sums fit where the warps' shares were");
};
__device__ __forceinline__ float load_cluster(uint32_t addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

template <typename T, int kRank, bool kVec>
__global__ void __launch_bounds__(kThreads, 2) lora_shrink_kernel(const __grid_constant__ LoraParams p)
{
    using S = Shrink<kRank>;
    constexpr int kNt = kRank / 8;
    extern __shared__ __align__(16) float share[]; // [warp][row][rank], then [token][rank]
    griddep_wait();
    griddep_launch_dependents(); // whatever ran before has completed: the second launch may read it
    const int ranks = static_cast<int>(gridDim.x / num_clusters_x());
    const int rank  = static_cast<int>(cluster_ctarank());
    const Tile t    = find_tile(p, static_cast<int>(cluster_id_x()));
    if (t.count == 0 || t.adapter < 0)
    {
        return; // the same for the cluster
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int halves = t.count > S::kRows ? 2 : 1, subs = kWarps / halves;
    const int half = warp & (halves - 1), sub = halves == 2 ? warp >> 1 : warp;
    // blocks of 32 columns, shared by the CTAs of the cluster and their warps
    const int blocks = (p.K + 31) / 32, parts = ranks * subs, part = rank * subs + sub;
    const int k_begin = static_cast<int>(static_cast<int64_t>(blocks) * part / parts), k_end = static_cast<int>(static_cast<int64_t>(blocks) * (part + 1) / parts);
    const int row0 = half * S::kRows, left = t.count - row0; // tokens of this warp
    const uint8_t *x = p.x + static_cast<int64_t>(t.first + row0) * p.ld_x;
    const uint8_t *a = p.a + static_cast<int64_t>(t.adapter) * p.max_rank * p.ld_a;
    float          acc[S::kMt][kNt][4] = {};
    const uint4    zero = make_uint4(0, 0, 0, 0);
#pragma unroll 2
    for (int kb = k_begin; kb < k_end; ++kb)
    {
        const int k = kb * 32 + c * 8;
        uint4     xv[S::kMt][2];
#pragma unroll
        for (int m = 0; m < S::kMt; ++m)
        {
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                const int r = m * 16 + h * 8 + g;
                xv[m][h]    = r < left ? load_eight<kVec>(x + r * p.ld_x, k, p.K) : zero;
            }
        }
#pragma unroll
        for (int n = 0; n < kNt; ++n)
        {
            if (n * 8 < t.rank)
            {
                const int   r  = n * 8 + g;
                const uint4 av = r < t.rank ? load_eight<kVec>(a + r * p.ld_a, k, p.K) : zero;
#pragma unroll
                for (int m = 0; m < S::kMt; ++m)
                {
                    if (m * 16 < left)
                    {
                        mma<T>(acc[m][n], xv[m][0].x, xv[m][1].x, xv[m][0].y, xv[m][1].y, av.x, av.y);
                        mma<T>(acc[m][n], xv[m][0].z, xv[m][1].z, xv[m][0].w, xv[m][1].w, av.z, av.w);
                    }
                }
            }
        }
    }
    float *mine = share + static_cast<int>(warp) * S::kRows * S::kPitch;
#pragma unroll
    for (int m = 0; m < S::kMt; ++m)
    {
#pragma unroll
        for (int n = 0; n < kNt; ++n)
        {
            float *at = mine + (m * 16 + g) * S::kPitch + n * 8 + 2 * c;
            *reinterpret_cast<float2 *>(at)                 = make_float2(acc[m][n][0], acc[m][n][1]);
            *reinterpret_cast<float2 *>(at + 8 * S::kPitch) = make_float2(acc[m][n][2], acc[m][n][3]);
        }
    }
    __syncthreads();
    // the warps' shares, in their order, to where the first of them was (a thread adds up what it writes to; with two halves the second
    // half's sums go to the second warp's place)
    for (int i = threadIdx.x; i < t.count * kRank; i += kThreads)
    {
        const int tok = i / kRank, r = i % kRank, h = tok / S::kRows, row = tok % S::kRows;
        float    *at = share + (h * S::kRows + row) * S::kPitch + r;
        float     sum = *at;
        for (int s = 1; s < subs; ++s) sum += at[s * halves * S::kRows * S::kPitch];
        *at = sum;
    }
    if (ranks > 1) cluster_sync();
    else __syncthreads();
    // the CTAs' sums, in their order: a warp per token
    for (int tok = rank * kWarps + warp; tok < t.count; tok += ranks * kWarps)
    {
        constexpr int  kPer = (kRank + 31) / 32;
        const uint32_t at   = smem_u32(share + tok * S::kPitch); // rows of both halves follow each other
        float          v[kPer];
        float          top = 0.f;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
        {
            const int r = i * 32 + lane;
            v[i]        = 0.f;
            if (r < kRank)
            {
                for (int q = 0; q < ranks; ++q) v[i] += load_cluster(map_to_cta(at + 4u * r, static_cast<uint32_t>(q)));
            }
            if (fabsf(v[i]) < INFINITY) top = fmaxf(top, fabsf(v[i]));
        }
        float factor = __ldg(p.scales + t.adapter);
        float mul    = 1.f;
        if constexpr (std::is_same<T, __half>::value)
        {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
            if (e > -126 && e < 127) // zero and subnormal sums stay as they are
            {
                mul = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                factor *= __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            }
        }
        uint16_t *out = p.v + static_cast<int64_t>(t.first + tok) * kRank;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
        {
            const int r = i * 32 + lane;
            if (r < kRank)
            {
                float rest = v[i] * mul;
                for (int q = 0; q < p.parts; ++q)
                {
                    const T part = from_float<T>(rest);
                    uint16_t bits;
                    memcpy(&bits, &part, 2);
                    out[static_cast<int64_t>(q) * p.tokens * kRank + r] = bits;
                    const float f = to_float(part);
                    rest          = fabsf(f) < INFINITY ? rest - f : 0.f; // an infinity or NaN is whole in the first part
                }
            }
        }
        if (lane == 0) p.factor[t.first + tok] = factor;
    }
    if (ranks > 1) cluster_sync(); // nobody leaves while others read its sums
}

// ---- second launch: dst = base + factor * v . B^T --------------------------------------------------------------
template <typename TD, bool kVec>
__device__ __forceinline__ void load_base(const uint8_t *row, int n, int cols, float (&v)[8])
{
    TD        e[8];
    const TD *src = reinterpret_cast<const TD *>(row) + n;
    if constexpr (kVec)
    {
        uint4 q[sizeof(TD) / 2];
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(TD)) / 2; ++i) q[i] = __ldcg(reinterpret_cast<const uint4 *>(src) + i);
        memcpy(e, q, sizeof(e));
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            e[i] = from_float<TD>(0.f);
            if (n + i < cols) e[i] = __ldcg(src + i);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float(e[i]);
}
template <typename TD, bool kVec>
__device__ __forceinline__ void store_row(uint8_t *row, int n, int cols, const float (&v)[8])
{
    TD  e[8];
    TD *dst = reinterpret_cast<TD *>(row) + n;
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_float<TD>(v[i]);
    if constexpr (kVec)
    {
        uint4 q[sizeof(TD) / 2];
        memcpy(q, e, sizeof(e));
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(TD)) / 2; ++i) reinterpret_cast<uint4 *>(dst)[i] = q[i];
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            if (n + i < cols) dst[i] = e[i];
        }
    }
}

// A warp: 32 channels, the tokens of a tile sixteen at a time.  Lane (g, c) of the results: rows g and g + 8, channels 8 c .. 8 c + 7.
template <typename T, typename TD, int kRank, bool kVec>
__global__ void __launch_bounds__(kThreads, 2) lora_expand_kernel(const __grid_constant__ LoraParams p)
{
    constexpr int kSteps = kRank / 16;
    constexpr int kParts = std::is_same<T, __nv_bfloat16>::value && sizeof(TD) == 4 ? 3 : 2;
    griddep_launch_dependents();
    // the launch ahead let this one start after its own wait: all but v is as it will be
    const Tile t = find_tile(p, static_cast<int>(blockIdx.y));
    if (t.count == 0)
    {
        griddep_wait();
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int n0 = static_cast<int>(blockIdx.x) * kChannels + warp * 32, n = n0 + 8 * c;
    uint2     b[4][kSteps];
    if (t.adapter >= 0)
    {
        const uint8_t *rows = p.b + static_cast<int64_t>(t.adapter) * p.N * p.ld_b;
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            // column g of the i-th tile of eight: the lane that gets its results has c = g / 2, as its elements 2 i and 2 i + 1
            const int ch = n0 + 8 * (g >> 1) + 2 * i + (g & 1);
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
            {
                const int r = s * 16 + 4 * c;
                b[i][s]     = make_uint2(0, 0);
                if (ch < p.N && r < t.rank)
                {
                    b[i][s] = __ldcg(reinterpret_cast<const uint2 *>(rows + ch * p.ld_b + r * 2));
                    // what lies behind the adapter's rank counts nothing, whatever it is
                    if (t.rank - r < 4) b[i][s].y = t.rank - r == 3 ? b[i][s].y & 0xffffu : 0u;
                    if (t.rank - r == 1) b[i][s].x &= 0xffffu;
                }
            }
        }
    }
    bool waited = false;
    for (int m = 0; m < t.count; m += 16)
    {
        float base[2][8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            const int row = m + h * 8 + g;
            if (row < t.count && n < p.N) load_base<TD, kVec>(p.base + static_cast<int64_t>(t.first + row) * p.ld_base, n, p.N, base[h]);
        }
        if (!waited)
        {
            griddep_wait();
            waited = true;
        }
        if (t.adapter >= 0)
        {
            float acc[4][4] = {};
#pragma unroll
            for (int q = kParts - 1; q >= 0; --q) // small parts first
            {
                const uint16_t *v = p.v + (static_cast<int64_t>(q) * p.tokens + t.first + m) * kRank;
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
                {
                    if (s * 16 < t.rank)
                    {
                        uint2 lo = make_uint2(0, 0), hi = make_uint2(0, 0);
                        if (m + g < t.count) lo = *reinterpret_cast<const uint2 *>(v + g * kRank + s * 16 + 4 * c);
                        if (m + g + 8 < t.count) hi = *reinterpret_cast<const uint2 *>(v + (g + 8) * kRank + s * 16 + 4 * c);
#pragma unroll
                        for (int i = 0; i < 4; ++i) mma<T>(acc[i], lo.x, hi.x, lo.y, hi.y, b[i][s].x, b[i][s].y);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                const int   row = m + h * 8 + g;
                const float f   = row < t.count ? p.factor[t.first + row] : 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
                    base[h][2 * i]     = fmaf(acc[i][2 * h], f, base[h][2 * i]);
                    base[h][2 * i + 1] = fmaf(acc[i][2 * h + 1], f, base[h][2 * i + 1]);
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            const int row = m + h * 8 + g;
            if (row < t.count && n < p.N) store_row<TD, kVec>(p.dst + static_cast<int64_t>(t.first + row) * p.ld_dst, n, p.N, base[h]);
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------
int padded_rank(int r)
{
    return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : 128;
}
int tile_tokens(int r)
{
    return padded_rank(r) == 128 ? Shrink<128>::kTile : Shrink<64>::kTile;
}
int v_parts(const cugl_lora_desc &d)
{
    return d.dtype == CUGL_BF16 && d.dst_dtype == CUGL_F32 ? 3 : 2;
}
int64_t most_tiles(const cugl_lora_desc &d) // of a request, all but the last are full
{
    const int64_t tile = tile_tokens(d.max_rank), some = d.requests < d.tokens ? d.requests : d.tokens;
    return (d.tokens - some) / tile + some;
}

template <typename T, int kRank, bool kVec>
cugl_status launch_shrink(cugl_context *ctx, const LoraParams &p, int64_t tiles)
{
    using S                          = Shrink<kRank>;
    auto                     kernel  = lora_shrink_kernel<T, kRank, kVec>;
    static std::atomic<bool> set[64] = {};
    if (!set[ctx->device & 63].load(std::memory_order_acquire))
    {
        CUGL_CUDA_TRY(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
        set[ctx->device & 63].store(true, std::memory_order_release);
    }
    // CTAs that share a tile's K: until there are two for every SM, each with a block of 32 columns per warp at least
    int split = 1;
    while (split < kMaxSplit && tiles * split < 2 * ctx->sm_count && p.K >= 2 * split * 32 * kWarps) split *= 2;
    CUGL_CUDA_TRY(ctx, launch_dependent_cluster(ctx, kernel, dim3(static_cast<unsigned>(tiles * split)), kThreads, S::kSmem, split, tiles * split, p));
    return CUGL_SUCCESS;
}
template <typename T, typename TD, int kRank>
cugl_status launch_lora(cugl_context *ctx, const LoraParams &p, int64_t tiles, bool vec_in, bool vec_out)
{
    CUGL_TRY((vec_in ? launch_shrink<T, kRank, true>(ctx, p, tiles) : launch_shrink<T, kRank, false>(ctx, p, tiles)));
    const dim3 grid(static_cast<unsigned>((p.N + kChannels - 1) / kChannels), static_cast<unsigned>(tiles));
    const long long units = static_cast<long long>(grid.x) * grid.y;
    CUGL_CUDA_TRY(ctx, vec_out ? launch_dependent(ctx, lora_expand_kernel<T, TD, kRank, true>, grid, kThreads, 0, units, p)
                               : launch_dependent(ctx, lora_expand_kernel<T, TD, kRank, false>, grid, kThreads, 0, units, p));
    return CUGL_SUCCESS;
}
template <typename T, typename TD>
cugl_status launch_lora(cugl_context *ctx, const LoraParams &p, int64_t tiles, bool vec_in, bool vec_out)
{
    switch (padded_rank(p.max_rank))
    {
        case 16: return launch_lora<T, TD, 16>(ctx, p, tiles, vec_in, vec_out);
        case 32: return launch_lora<T, TD, 32>(ctx, p, tiles, vec_in, vec_out);
        case 64: return launch_lora<T, TD, 64>(ctx, p, tiles, vec_in, vec_out);
        default: return launch_lora<T, TD, 128>(ctx, p, tiles, vec_in, vec_out);
    }
}

const char *validate_lora(const cugl_lora_desc *d)
{
    if (d == nullptr) return "descriptor is NULL";
    if (d->tokens < 0 || d->requests < 0) return "tokens and requests must not be negative";
    if (d->adapters < 1) return "adapters must be positive";
    if (d->max_rank < 1 || d->max_rank > kMaxRank) return "max_rank must lie within 1 .. 128";
    if (d->N < 1 || d->K < 1) return "N and K must be positive";
    if (d->N > INT32_MAX - 1024 || d->K > INT32_MAX - 1024 || d->tokens > INT32_MAX - 1024) return "a dimension is too large";
    if (d->dtype != CUGL_F16 && d->dtype != CUGL_BF16) return "dtype must be CUGL_F16 or CUGL_BF16";
    if (d->dst_dtype != d->dtype && d->dst_dtype != CUGL_F32) return "dst_dtype must be dtype or CUGL_F32";
    const int size = dtype_size(d->dst_dtype);
    if (d->ld_x < 2ll * d->K || d->ld_x % 2 != 0 || d->ld_a < 2ll * d->K || d->ld_a % 2 != 0) return "ld_x and ld_a must hold a row and be multiples of 2";
    if (d->ld_b < 2ll * d->max_rank || d->ld_b % 16 != 0) return "ld_b must hold a row and be a multiple of 16";
    if (d->ld_base < static_cast<int64_t>(d->N) * size || d->ld_base % size != 0 || d->ld_dst < static_cast<int64_t>(d->N) * size || d->ld_dst % size != 0)
        return "ld_base and ld_dst must hold a row and be multiples of the element size";
    if (most_tiles(*d) > 65535) return "more than 65535 tiles of tokens";
    return nullptr;
}
} // namespace
} // namespace cugl

using namespace cugl;

extern "C"
{
    cugl_status cugl_lora_validate(const cugl_lora_desc *desc, const char **reason)
    {
        const char *why = validate_lora(desc);
        if (reason != nullptr)
        {
            *reason = why != nullptr ? why : "";
        }
        return why == nullptr ? CUGL_SUCCESS : CUGL_INVALID_ARGUMENT;
    }

    size_t cugl_lora_workspace_bytes(const cugl_lora_desc *desc)
    {
        if (validate_lora(desc) != nullptr)
        {
            return 0;
        }
        return 16 + static_cast<size_t>(desc->tokens) * (static_cast<size_t>(padded_rank(desc->max_rank)) * 2 * static_cast<size_t>(v_parts(*desc)) + 4);
    }

    cugl_status cugl_lora(cugl_context *ctx, const cugl_lora_desc *desc, const void *d_x, const int32_t *d_starts, const int32_t *d_request_adapters,
                          const int32_t *d_ranks, const float *d_scales, const void *d_a, const void *d_b, const void *d_base, void *d_dst,
                          void *d_workspace, size_t workspace_bytes)
    {
        if (ctx == nullptr)
        {
            return fail(nullptr, CUGL_INVALID_ARGUMENT, "context is NULL");
        }
        const char *why = validate_lora(desc);
        if (why == nullptr && desc->tokens > 0 && desc->requests > 0)
        {
            auto            bits = [](const void *q) { return reinterpret_cast<uintptr_t>(q); };
            const uintptr_t size = static_cast<uintptr_t>(dtype_size(desc->dst_dtype));
            if (d_x == nullptr || d_starts == nullptr || d_request_adapters == nullptr || d_scales == nullptr || d_a == nullptr || d_b == nullptr || d_base == nullptr ||
                d_dst == nullptr || d_workspace == nullptr)
                why = "NULL pointer";
            else if (bits(d_b) % 16 != 0 || bits(d_workspace) % 16 != 0) why = "b and the workspace must be 16-byte aligned";
            else if ((bits(d_x) | bits(d_a)) % 2 != 0 || (bits(d_base) | bits(d_dst)) % size != 0 ||
                     (bits(d_starts) | bits(d_request_adapters) | bits(d_ranks) | bits(d_scales)) % 4 != 0)
                why = "a buffer is not aligned to its elements";
            else if (d_dst == d_base && desc->ld_dst != desc->ld_base) why = "in place, ld_dst must be ld_base";
            else if (workspace_bytes < cugl_lora_workspace_bytes(desc)) why = "the workspace is too small";
        }
        if (why != nullptr)
        {
            return fail(ctx, CUGL_INVALID_ARGUMENT, std::string("cugl_lora: ") + why);
        }
        if (desc->tokens == 0 || desc->requests == 0) return CUGL_SUCCESS;
        const DeviceScope device(ctx);
        LoraParams        p{};
        p.x          = static_cast<const uint8_t *>(d_x);
        p.a          = static_cast<const uint8_t *>(d_a);
        p.b          = static_cast<const uint8_t *>(d_b);
        p.base       = static_cast<const uint8_t *>(d_base);
        p.dst        = static_cast<uint8_t *>(d_dst);
        p.starts     = d_starts;
        p.adapters   = d_request_adapters;
        p.ranks      = d_ranks;
        p.scales     = d_scales;
        p.ld_x       = desc->ld_x;
        p.ld_a       = desc->ld_a;
        p.ld_b       = desc->ld_b;
        p.ld_base    = desc->ld_base;
        p.ld_dst     = desc->ld_dst;
        p.tokens     = desc->tokens;
        p.requests   = desc->requests;
        p.n_adapters = desc->adapters;
        p.max_rank   = desc->max_rank;
        p.K          = desc->K;
        p.N          = desc->N;
        p.parts      = v_parts(*desc);
        p.tile       = tile_tokens(desc->max_rank);
        p.v          = static_cast<uint16_t *>(d_workspace);
        p.factor     = reinterpret_cast<float *>(static_cast<uint8_t *>(d_workspace) + static_cast<size_t>(p.tokens) * padded_rank(p.max_rank) * 2 * p.parts);
        auto       even = [](const void *q, int64_t ld) { return ((reinterpret_cast<uintptr_t>(q) | static_cast<uintptr_t>(ld)) & 15) == 0; };
        const bool vec_in  = even(d_x, desc->ld_x) && even(d_a, desc->ld_a);
        const bool vec_out = even(d_base, desc->ld_base) && even(d_dst, desc->ld_dst) && desc->N % 8 == 0;
        const int64_t tiles = most_tiles(*desc);
        if (desc->dtype == CUGL_F16)
        {
            return desc->dst_dtype == CUGL_F32 ? launch_lora<__half, float>(ctx, p, tiles, vec_in, vec_out) : launch_lora<__half, __half>(ctx, p, tiles, vec_in, vec_out);
        }
        return desc->dst_dtype == CUGL_F32 ? launch_lora<__nv_bfloat16, float>(ctx, p, tiles, vec_in, vec_out)
                                           : launch_lora<__nv_bfloat16, __nv_bfloat16>(ctx, p, tiles, vec_in, vec_out);
    }
}
