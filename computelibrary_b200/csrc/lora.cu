// Low-rank adapters of many requests at once, beside a projection that all of them share:
//   dst[t] = base[t] + scale_a * (x[t] . A_a^T) . B_a^T          a: the adapter of the request that token t belongs to
//
// Long requests take two launches, short ones have one that does the same for tiles of 16 tokens (lora_few_kernel: 24 requests of a token,
// 4096 -> 14336, rank 16, BF16 9.3 us, in two launches 13.3).  The first makes v = x . A^T: a tile of up to 64 tokens of one request per
// cluster, whose CTAs share K; their sums are added up in a fixed order through distributed shared memory.  The second adds
// scale * v . B^T to base, 256 channels x a tile of tokens per item.  Which tiles there are is known on the device only (the requests'
// lengths): every CTA counts them (a scan over the requests) and takes the one with its number, or every gridDim.x-th item; the grid is the
// most that there can be.
//
// What bounds it: bytes.  x, base and dst pass once, the adapters once per tile of tokens.  The first product is one for tcgen05.mma (K is
// long, its sums few); the second has K of at most 128 ranks, and all the rest of its time goes to base and dst, hence mma.sync, whose
// accumulators are the registers that base is added to.
//
// Fragments.  Sums do not care in which order their terms come, as long as both operands agree: a lane of the second launch takes 4
// consecutive ranks as the two pairs that a step of the matrix instruction wants from it.  Channels likewise: the four 8-column tiles
// of a warp's 32 channels are dealt out so that a lane's results are whole 16-byte pieces of a row.
//
// v is kept as two 16-bit parts, v = high + low (three where bf16 adapters add to 32-bit results): 16 (bf16) or 22 (f16) bits of it
// count, 24 with three parts, so rounding v costs less than rounding the result (prompts, K = 4096, ranks up to 64, F16 to F32: 1.7e-8 of it
// beside 2.5e-8).  f16 parts would leave that type's range: a token's
// v is first divided by a power of two that brings its largest rank into [1, 2).
#include "mx_mma.cuh"

#include <algorithm>
#include <cmath>
#include <cstring>

namespace cugl
{
namespace
{
constexpr int kThreads  = 256;
constexpr int kWarps    = kThreads / 32;
constexpr int kMaxRank  = 128;
constexpr int kMaxSplit = 8;
constexpr int kFewRank  = 64; // largest padded rank of the single launch

struct LoraParams
{
    const uint8_t *x, *a, *b, *base;
    uint8_t       *dst;
    const int32_t *starts, *adapters, *ranks;
    const float   *scales;
    uint16_t      *v; // [parts][tokens][padded rank + 8]: the first part's last eight elements hold the token's factor (a float)
    int64_t        ld_x, ld_a, ld_b, ld_base, ld_dst; // bytes
    int            tokens, requests, n_adapters, max_rank, K, N, parts, tile;
    int            tiles; // at most
    int            chains; // accumulators of a sum on tcgen05.mma: 1 or kChains
    uint32_t       idesc; // of no columns
    int32_t       *status;
    long long      spin_limit;
    int            withhold; // see cugl_context_withhold_copy_once
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
// A request's tokens are [starts[i], starts[i + 1]), cut to those there are.
struct Request
{
    int begin, end, adapter, rank; // adapter and rank as they were read
};
__device__ __forceinline__ Request load_request(const LoraParams &p, int r)
{
    Request q{0, 0, -1, 0};
    if (r < p.requests)
    {
        const int begin = load_l2(p.starts + r), end = load_l2(p.starts + r + 1);
        q.adapter       = load_l2(p.adapters + r);
        q.rank          = p.max_rank;
        if (p.ranks != nullptr && q.adapter >= 0 && q.adapter < p.n_adapters) q.rank = load_l2(p.ranks + q.adapter); // on its way during the scan
        q.begin = min(max(begin, 0), p.tokens);
        q.end   = min(max(end, q.begin), p.tokens);
    }
    return q;
}
// Tiles of a request.  Starts that are not in order may give more of them than there can be: none of it runs out of range, and nothing
// behind p.tiles is worked on.
__device__ __forceinline__ int request_tiles(const LoraParams &p, const Request &q)
{
    return min((q.end - q.begin + p.tile - 1) / p.tile, p.tiles);
}
// tile `i` of a request
__device__ __forceinline__ Tile request_tile(const LoraParams &p, const Request &q, int i)
{
    const int first = q.begin + i * p.tile, rank = min(max(q.rank, 0), p.max_rank);
    return Tile{first, min(p.tile, q.end - first), q.adapter >= 0 && q.adapter < p.n_adapters && rank > 0 ? q.adapter : -1, rank};
}
struct ScanShared
{
    int sums[2][kWarps];
};
// The tiles of kThreads requests: a thread's own come behind `at` others, `all` are there.  By all threads; turn: alternately 0 and 1.
__device__ __forceinline__ void scan_tiles(ScanShared &s, int turn, int tiles, int &at, int &all)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int       incl = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const int n = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += n;
    }
    if (lane == 31) s.sums[turn][warp] = incl;
    __syncthreads();
    at = incl - tiles;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
    {
        if (w < warp) at += s.sums[turn][w];
        all += s.sums[turn][w];
    }
}
// Tile number `wanted`.  By all threads.
__device__ __forceinline__ Tile find_tile(const LoraParams &p, int wanted)
{
    __shared__ Tile       found;
    __shared__ ScanShared scan;
    if (threadIdx.x == 0) found = Tile{0, 0, -1, 0};
    int before = 0, turn = 0;
    for (int r0 = 0; r0 < p.requests && before <= wanted; r0 += kThreads, turn ^= 1)
    {
        const Request q     = load_request(p, r0 + static_cast<int>(threadIdx.x));
        const int     tiles = request_tiles(p, q);
        int           at, all;
        scan_tiles(scan, turn, tiles, at, all);
        const int i = wanted - before - at;
        if (i >= 0 && i < tiles) found = request_tile(p, q, i);
        before = min(before + all, p.tiles);
    }
    __syncthreads();
    return found;
}

// ---- matrix instruction --------------------------------------------------------------------------------------
// D (+)= A . B, 16 x 8 x 16: rows lane / 4 and lane / 4 + 8, columns 2 (lane % 4) and the next
template <typename T, bool kFirst = false>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    const float c0 = kFirst ? 0.f : d[0], c1 = kFirst ? 0.f : d[1], c2 = kFirst ? 0.f : d[2], c3 = kFirst ? 0.f : d[3];
    if constexpr (std::is_same<T, __half>::value)
    {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
    }
    else
    {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
    }
}

// ---- asynchronous copies -------------------------------------------------------------------------------------
// 16 bytes to shared memory, those from `valid` on as zeros; past L1
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, int valid)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
}
__device__ __forceinline__ void copy_commit()
{
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int kPending>
__device__ __forceinline__ void copy_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void store_word(uint32_t dst, uint32_t v)
{
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst), "r"(v) : "memory");
}
// where the share of part i of n equal ones begins
__device__ __forceinline__ int share_begin(int total, int i, int n)
{
    const int each = total / n;
    return i * each + min(i, total - each * n);
}
// How rows of x and A start: at multiples of 16 bytes, of 4 (and K is even), or anywhere.
enum RowsIn
{
    kUnits16,
    kWords,
    kAnywhere
};

// ---- first launch: v = x . A^T -------------------------------------------------------------------------------
// A CTA takes a share of K of a tile, in blocks of 64 columns; rows of 128 bytes whose 16-byte units are exchanged by row.
template <int kRank>
struct Shrink
{
    static constexpr int kMt    = kRank == 128 ? 1 : 2; // 16-row tiles of a warp
    static constexpr int kRows  = 16 * kMt;
    static constexpr int kTile  = 2 * kRows;
    static constexpr int kStage = (kTile + kRank) * 128; // bytes; two of them
    static constexpr int kPitch = kRank + 8;             // floats: rows in different banks
    static constexpr int kSums  = kWarps * kRows * kPitch * 4;
    static constexpr int kSmem  = 2 * kStage > kSums ? 2 * kStage : kSums;
};
__device__ __forceinline__ float load_cluster(uint32_t addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// Where rank r stands in a row of v: of sixteen, lane c of the second launch wants 4 c and the next as the matrix instruction's columns 2 c
// and the next, 4 c + 2 and the next as 2 c + 8 and the next.
__device__ __forceinline__ int v_place(int r)
{
    return (r & ~15) + ((r >> 1) & 6) + ((r & 2) << 2) + (r & 1);
}

// v of a token: the CTAs' sums of x . A^T ([token][rank] in the shared memory of each), added up in the order of the CTAs, its parts to
// put(part, place, bits); returns the token's factor.  By a warp.
template <typename T, int kRank, typename Put>
__device__ __forceinline__ float token_v(const LoraParams &p, const Tile &t, const float *share, int pitch, int ranks, int tok, Put put)
{
    constexpr int  kPer = (kRank + 31) / 32;
    const int      lane = threadIdx.x & 31;
    const uint32_t at   = smem_u32(share + tok * pitch);
    float          v[kPer], parts[kPer][kMaxSplit];
    float          top = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) // all of them under way before the first is added
    {
        const int r = min(i * 32 + lane, kRank - 1);
#pragma unroll
        for (int q = 0; q < kMaxSplit; ++q)
        {
            parts[i][q] = 0.f;
            if (q < ranks) parts[i][q] = load_cluster(map_to_cta(at + 4u * r, static_cast<uint32_t>(q)));
        }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
    {
        v[i] = parts[i][0];
#pragma unroll
        for (int q = 1; q < kMaxSplit; ++q) v[i] += parts[i][q];
        if (fabsf(v[i]) < INFINITY) top = fmaxf(top, fabsf(v[i]));
    }
    float factor = p.scales[t.adapter];
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
#pragma unroll
    for (int i = 0; i < kPer; ++i)
    {
        const int r = i * 32 + lane;
        if (r < kRank)
        {
            float rest = v[i] * mul;
            for (int q = 0; q < p.parts; ++q)
            {
                const T  part = from_float<T>(rest);
                uint16_t bits;
                memcpy(&bits, &part, 2);
                put(q, v_place(r), bits);
                const float f = to_float(part);
                rest          = fabsf(f) < INFINITY ? rest - f : 0.f; // an infinity or NaN is whole in the first part
            }
        }
    }
    return factor;
}
// v of a tile's tokens to memory, shared by the CTAs of the cluster: a warp per token.  By all threads of the cluster.
template <typename T, int kRank>
__device__ __forceinline__ void finish_v(const LoraParams &p, const Tile &t, const float *share, int pitch, int rank, int ranks)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (ranks > 1) cluster_sync();
    else __syncthreads();
    for (int tok = rank * kWarps + warp; tok < t.count; tok += ranks * kWarps)
    {
        uint16_t   *out    = p.v + static_cast<int64_t>(t.first + tok) * (kRank + 8);
        const float factor = token_v<T, kRank>(p, t, share, pitch, ranks, tok, [&](int part, int place, uint16_t bits) {
            out[static_cast<int64_t>(part) * p.tokens * (kRank + 8) + place] = bits;
        });
        if (lane == 0) *reinterpret_cast<float *>(out + kRank) = factor;
    }
    // Nobody leaves while others read its sums: they have what they read.  (A releasing arrival would wait for the stores of v.)
    __syncwarp();
    if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- first launch, rows of x and A at multiples of 16 bytes --------------------------------------------------
// Ranks are the rows of a tcgen05.mma, tokens its columns, blocks of 64 columns of K come by TMA.  A CTA's sums stay in tensor memory
// until its share of K is done: no adding up of warps, and the stream of blocks from L2 bounds it, where the warps' own matrix
// instructions took twice as long (prompts of 4096 tokens, K = 4096, ranks up to 64: 20.6 -> 14.2 us under ncu).  Of the 128 rows of an MMA only
// the adapter's count; the others are whatever shared memory holds behind them.  Rows of x behind the tile belong to other requests:
// columns that nobody reads.
//
// An accumulator in tensor memory is cut to 24 bits at every step, not rounded, and v's error grows with their number.  Where results have 32
// bits, four of them take the blocks of K in turn and are added up as floats (prompts of 4096 tokens, K = 4096, ranks up to 64, F16 to
// F32, relative error against 64 bits: one 4.9e-7, four 1.6e-7, the plain 32-bit form 2.1e-7; 42.8 -> 43.1 us, 24 requests of a token at rank 16 6.9 -> 7.2); 16-bit results
// have one.
constexpr int kChains = 4;
// The sums of sixteen columns of `chains` accumulators, `gap` columns apart.  (One at a time: registers that the first launch needs more than
// 64 of keep the second from starting beside it, 11.2 -> 12.7 us for 8 requests of 32 tokens at rank 128.)
__device__ __forceinline__ void add_chains(uint32_t tmem, int gap, int chains, float (&sum)[16])
{
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = 0.f;
#pragma unroll 1
    for (int q = 0; q < chains; ++q)
    {
        uint32_t v[16];
        tmem_ld_x16(tmem + q * gap, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[i] += __uint_as_float(v[i]);
    }
}
template <int kRank>
struct ShrinkMma
{
    static constexpr int kTile   = Shrink<kRank>::kTile;
    static constexpr int kStages = kRank == 128 ? 4 : kRank == 64 ? 6 : 8;
    static constexpr int kA      = kRank * 128, kX = kTile * 128, kStage = kA + kX; // bytes
    static constexpr int kPitch  = kRank + 1;                                       // floats of a token's sums
    static constexpr int kOffBar = (kStages - 1) * kStage + (kStage > 16384 ? kStage : 16384); // an MMA reads 16 KB from a stage's start on
    static constexpr int kSmem   = kOffBar + (2 * kStages + 2) * 8 + 16 + 1024;
    __host__ __device__ static constexpr int columns(int chains) { return chains * kTile; } // of tensor memory; see Few::kSmem
    static_assert(kTile * kPitch * 4 <= kOffBar && columns(kChains) <= 256, "sums fit where the stages were, and in tensor memory");
};
inline uint32_t f16_idesc(bool bf16) // float sums, 128 rows; add columns / 8 << 17
{
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((128u >> 4) << 24);
}
// D[tmem] (+)= sum over 16 elements
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t"
                 ".reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
                 "}"
                 :
                 : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
                 : "memory");
}

template <typename T, int kRank>
__global__ void __launch_bounds__(kThreads, 2)
    lora_shrink_mma_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_few,
                           const __grid_constant__ LoraParams p)
{
    using S = ShrinkMma<kRank>;
    constexpr int STAGES = S::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t       *smem      = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t s_stage   = smem_u32(smem), bar_base = smem_u32(smem + S::kOffBar);
    auto           full_bar  = [&](int s) { return bar_base + 8u * s; };
    auto           empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    const uint32_t done_bar  = bar_base + 8u * (2 * STAGES), gone_bar = done_bar + 8;
    uint32_t      *s_tmem    = reinterpret_cast<uint32_t *>(smem + S::kOffBar + (2 * STAGES + 2) * 8);
    volatile int  *s_abort   = reinterpret_cast<volatile int *>(s_tmem + 1);
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0)
    {
        for (int s = 0; s < STAGES; ++s)
        {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
        mbar_init(gone_bar, 1);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1)
    {
        tmem_alloc(smem_u32(s_tmem), static_cast<uint32_t>(S::columns(p.chains)));
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    griddep_wait();
    griddep_launch_dependents(); // whatever ran before has completed: the second launch may read it
    const int  ranks = static_cast<int>(gridDim.x / num_clusters_x()), rank = static_cast<int>(cluster_ctarank());
    const Tile t     = find_tile(p, static_cast<int>(cluster_id_x()));
    if (t.count == 0 || t.adapter < 0) // the same for the cluster
    {
        if (warp == 1) tmem_dealloc(tmem, static_cast<uint32_t>(S::columns(p.chains)));
        return;
    }
    const int blocks = (p.K + 63) / 64; // of 64 columns, shared by the CTAs of the cluster
    const int first  = share_begin(blocks, rank, ranks), n_blocks = share_begin(blocks, rank + 1, ranks) - first;
    int       issued = 0; // stages that the producer has filled
    if (warp == 0)
    {
        const bool el  = elect_one(), few = t.count <= 16;
        const int  a_row = t.adapter * p.max_rank;
        int        g = 0;
        for (; g < n_blocks; ++g)
        {
            const int s = g % STAGES;
            if (!warp_wait(empty_bar(s), (static_cast<uint32_t>(g / STAGES) & 1u) ^ 1u, s_abort, DEV_TIMEOUT_PRODUCER, p.spin_limit)) break;
            if (g == p.withhold && blockIdx.x == 0) continue;
            if (el)
            {
                const uint32_t dst = s_stage + s * S::kStage;
                mbar_expect_tx(full_bar(s), static_cast<uint32_t>(S::kA + (few ? 16 * 128 : S::kX)));
                tma_load_2d(dst, &tmap_a, (first + g) * 64, a_row, full_bar(s));
                tma_load_2d(dst + S::kA, few ? &tmap_few : &tmap_x, (first + g) * 64, t.first, full_bar(s));
            }
            __syncwarp();
        }
        issued = g;
    }
    else if (warp == 1)
    {
        const bool     el    = elect_one();
        const uint32_t idesc = p.idesc | (static_cast<uint32_t>((t.count + 15) >> 4) << 18); // columns / 8
        bool           ok    = true;
        for (int g = 0; g < n_blocks && ok; ++g)
        {
            const int s = g % STAGES;
            ok = warp_wait(full_bar(s), static_cast<uint32_t>(g / STAGES) & 1u, s_abort, DEV_TIMEOUT_MMA, p.spin_limit);
            if (!ok) break;
            tc_fence_after();
            const uint64_t a_desc = make_kmajor_sw128_desc(s_stage + s * S::kStage), b_desc = make_kmajor_sw128_desc(s_stage + s * S::kStage + S::kA);
            if (el)
            {
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_f16(tmem + (g & (p.chains - 1)) * S::kTile, a_desc + 2u * k, b_desc + 2u * k, idesc, g >= p.chains || k != 0 ? 1u : 0u);
                umma_commit(empty_bar(s));
            }
            __syncwarp();
        }
        if (ok && el) umma_commit(done_bar);
        __syncwarp();
    }
    // sums to shared memory, [token][rank]: a lane has a rank, warps 4 .. 7 the upper half of the tokens
    const bool ok    = warp_wait(done_bar, 0, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit);
    float     *share = reinterpret_cast<float *>(smem);
    const int  r = (warp & 3) * 32 + lane, c0 = (warp >> 2) * 32;
    __syncthreads(); // every warp's waits are over; the MMAs have read the stages
    if (ok && *s_abort == 0 && (warp & 3) * 32 < kRank && c0 < t.count)
    {
        tc_fence_after();
#pragma unroll 1
        for (int c = c0; c < min(c0 + 32, t.count); c += 16)
        {
            float v[16];
            add_chains(tmem + c + (static_cast<uint32_t>((warp & 3) * 32) << 16), S::kTile, min(n_blocks, p.chains), v);
            if (r < kRank)
            {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    if (c + i < t.count) share[(c + i) * S::kPitch + r] = r < t.rank ? v[i] : 0.f; // behind the adapter's ranks: zeros
                }
            }
            __syncwarp(); // aligned loads are next
        }
    }
    tc_fence_before();
    __syncthreads();
    const bool gone = *s_abort != 0;
    if (warp == 0 && gone)
    {
        drain_stages<STAGES>(bar_base, issued, blockIdx.x == 0 ? p.withhold : -1, p.spin_limit);
    }
    if (warp == 1)
    {
        if (gone) drain_mmas<false>(gone_bar, p.spin_limit);
        tc_fence_after();
        tmem_dealloc(tmem, static_cast<uint32_t>(S::columns(p.chains)));
    }
    if (threadIdx.x == 0 && gone)
    {
        atomicCAS(p.status, 0, *s_abort);
    }
    finish_v<T, kRank>(p, t, share, S::kPitch, rank, ranks); // (of a CTA that has given up: nothing of use)
}

// ---- first launch, other rows ----------------------------------------------------------------------------------
// Rows that are not 16-byte aligned: a warp takes a row, a lane two of its columns.  A block passes through registers, asked for before
// the one ahead of it is multiplied by the warps' own matrix instructions: a warp takes 16 columns of a block and 32 (16) tokens; tiles of
// few tokens leave every other block to the other half of the warps.  What bounds it: one block of K in flight per CTA (404 tokens, K = 6319,
// 25 us); and at ranks 64 and 128 rows that start anywhere take two registers a pair of columns and spill 192 and 372 bytes.
template <typename T, int kRank, int kIn>
__global__ void __launch_bounds__(kThreads, 2) lora_shrink_kernel(const __grid_constant__ LoraParams p)
{
    using S = Shrink<kRank>;
    constexpr int kNt = kRank / 8;
    extern __shared__ __align__(128) float share[]; // stages, then sums [warp][row][rank], then [token][rank]
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
    const int blocks = (p.K + 63) / 64; // of 64 columns, shared by the CTAs of the cluster
    const int first = share_begin(blocks, rank, ranks), n_blocks = share_begin(blocks, rank + 1, ranks) - first;
    const int x_rows = (t.count + 15) & ~15, a_rows = (t.rank + 15) & ~15; // those that the matrix instructions read
    const uint8_t *x = p.x + static_cast<int64_t>(t.first) * p.ld_x;
    const uint8_t *a = p.a + static_cast<int64_t>(t.adapter) * p.max_rank * p.ld_a;
    const uint32_t s_base = smem_u32(share);
    float     acc[S::kMt][kNt][4] = {};
    const int step = halves == 2 ? sub : sub & 3; // 16 columns of a stage
    // rows 16 m + lane % 16 of x, rows 8 n + .. of A: their numbers modulo 8, and so the places of their units, do not depend on m and n
    const uint32_t x_at = s_base + static_cast<uint32_t>((half * S::kRows + (lane & 15)) * 128 + (((2 * step + (lane >> 4)) ^ (lane & 7)) << 4));
    const uint32_t a_at = s_base + static_cast<uint32_t>((S::kTile + (lane & 7) + ((lane >> 4) << 3)) * 128 + (((2 * step + ((lane >> 3) & 1)) ^ (lane & 7)) << 4));
    auto           multiply = [&](int i, uint32_t st) { // block i, in the stage at st
        if (halves == 1 && (i & 1) != (sub >> 2)) return;
        uint32_t xv[S::kMt][4];
#pragma unroll
        for (int m = 0; m < S::kMt; ++m)
        {
            if (half * S::kRows + m * 16 < t.count) ldmatrix_x4(x_at + st + m * 16 * 128, xv[m]);
        }
#pragma unroll
        for (int n = 0; n < kNt; n += 2)
        {
            if (n * 8 < t.rank)
            {
                uint32_t av[4];
                ldmatrix_x4(a_at + st + n * 8 * 128, av);
#pragma unroll
                for (int m = 0; m < S::kMt; ++m)
                {
                    if (half * S::kRows + m * 16 < t.count)
                    {
                        mma<T>(acc[m][n], xv[m][0], xv[m][1], xv[m][2], xv[m][3], av[0], av[1]);
                        mma<T>(acc[m][n + 1], xv[m][0], xv[m][1], xv[m][2], xv[m][3], av[2], av[3]);
                    }
                }
            }
        }
    };
    // (Nothing may use a value between the loads: each would then wait for its own.)
    constexpr int  kEach = (S::kTile + kRank) / kWarps;
    constexpr bool kWord = kIn == kWords;
    uint32_t       low[kEach], high[kWord ? 1 : kEach];
    auto           fetch = [&](int block) {
        const int k = (first + block) * 64 + 2 * lane, k0 = min(k, kWord ? p.K - 2 : p.K - 1), k1 = min(k + 1, p.K - 1);
#pragma unroll
        for (int j = 0; j < kEach; ++j)
        {
            const int i = warp + j * kWarps, row = i < S::kTile ? i : i - S::kTile; // (whole groups of eight rows lie before A's)
            if (row < (i < S::kTile ? t.count : t.rank))
            {
                const uint8_t *src = i < S::kTile ? x + row * p.ld_x : a + row * p.ld_a;
                if constexpr (kWord) low[j] = *reinterpret_cast<const uint32_t *>(src + static_cast<int64_t>(k0) * 2);
                else
                {
                    low[j]  = reinterpret_cast<const uint16_t *>(src)[k0];
                    high[j] = reinterpret_cast<const uint16_t *>(src)[k1];
                }
            }
        }
    };
    fetch(0);
    for (int i = 0; i < n_blocks; ++i)
    {
        const uint32_t st = (i & 1) != 0 ? S::kStage : 0u;
        const int      k  = (first + i) * 64 + 2 * lane;
#pragma unroll
        for (int j = 0; j < kEach; ++j)
        {
            const int at = warp + j * kWarps, row = at < S::kTile ? at : at - S::kTile;
            uint32_t  w = 0; // rows behind the last and columns behind K: zeros
            if (row < (at < S::kTile ? t.count : t.rank))
            {
                if constexpr (kWord) w = k < p.K ? low[j] : 0u;
                else w = (k < p.K ? low[j] : 0u) | (k + 1 < p.K ? high[j] << 16 : 0u);
            }
            if (row < (at < S::kTile ? x_rows : a_rows))
                store_word(s_base + st + static_cast<uint32_t>(at * 128 + (((lane >> 2) ^ (at & 7)) << 4) + (lane & 3) * 4), w);
        }
        __syncthreads(); // (the stage of the block before is the other one)
        if (i + 1 < n_blocks) fetch(i + 1);
        multiply(i, st);
    }
    __syncthreads(); // the stages are free
    float *mine = share + warp * S::kRows * S::kPitch;
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
    // the warps' sums, in their order, to where the first of them was (a thread adds up what it writes to; with two halves the second
    // half's sums go to the second warp's place)
    for (int i = threadIdx.x; i < t.count * kRank; i += kThreads)
    {
        const int tok = i / kRank, r = i % kRank;
        float    *at = share + tok * S::kPitch + r; // rows of both halves follow each other
        float     part[kWarps];
#pragma unroll
        for (int s = 0; s < kWarps; ++s) part[s] = s < subs ? at[s * halves * S::kRows * S::kPitch] : 0.f;
        float sum = part[0];
#pragma unroll
        for (int s = 1; s < kWarps; ++s) sum += part[s];
        *at = sum;
    }
    finish_v<T, kRank>(p, t, share, S::kPitch, rank, ranks);
}

// ---- second launch: dst = base + factor * v . B^T --------------------------------------------------------------
// An item is 256 channels of a tile.  Every CTA takes every gridDim.x-th of them, so that tiles of high and of low rank, which are not
// equally much work, are spread over all (prompts of 4096 tokens with ranks of 16 to 64, both launches: consecutive shares 46.8 us,
// this 45.5 when it was taken).  A warp has 32 channels, the tokens of the tile sixteen at a time.  What it needs next is under way
// while it works: units of 16 tokens x 32 channels of base pass through a ring of four slots of its own, the next item's v waits in the other half of its buffer, and its B
// in registers where there are enough of them.  Of a unit's results lane (g, c) has rows g and g + 8, and of each the channels that it stores as 16-byte pieces:
//   two-byte results  8 c .. 8 c + 7
//   floats            4 c .. 4 c + 3 and 16 + 4 c .. 16 + 4 c + 3, so that a store of four lanes covers whole sectors
constexpr int kListed = 256; // items of a CTA at most
struct Item
{
    Tile tile;
    int  n; // first channel
};
template <typename T, typename TD, int kRank>
struct Expand
{
    static constexpr int kSteps   = kRank / 16;
    static constexpr bool kAhead  = kRank <= 32;          // the next item's B in registers
    static constexpr int kParts   = std::is_same<T, __nv_bfloat16>::value && sizeof(TD) == 4 ? 3 : 2;
    static constexpr int kTile    = Shrink<kRank>::kTile;
    static constexpr int kPitch   = kRank * 2 + 16; // bytes of a row of v, its factor included: eight rows in different banks
    static constexpr int kV       = kParts * kTile * kPitch;
    static constexpr int kRow     = 32 * static_cast<int>(sizeof(TD)); // bytes of a row of a unit
    static constexpr int kSlots   = 4;
    static constexpr int kOffBase = 2 * kV;
    static constexpr int kSmem    = kOffBase + kWarps * kSlots * 16 * kRow;
    // CTAs per SM: as many as shared memory holds with the list, the scan and the 1 KB that goes with a CTA.  Rank 64 in three parts is one (a
    // grid and registers for two of them, which ran one after the other: 4096 tokens of 7 requests, 4096 -> 4096, bf16 to F32 57 us, this 53).
    static constexpr int kWhole   = kSmem + kListed * static_cast<int>(sizeof(Item)) + static_cast<int>(sizeof(ScanShared)) + 1024;
    static constexpr int kCtas    = kRank == 128 || 2 * kWhole > 228 * 1024 ? 1 : 2;
    static_assert(kWhole <= 228 * 1024 && kListed * sizeof(Item) <= 8192, "shared memory of an SM");
};
// the first channel of a lane's piece of 16 bytes
template <typename TD>
__device__ __forceinline__ int piece_channel(int piece, int c)
{
    return sizeof(TD) == 4 ? piece * 16 + 4 * c : 8 * c;
}

// B of an item, as fragments; what lies behind the adapter's rank counts nothing, whatever it is.  Channels behind the last one are read
// as the last one: nobody stores their results.
template <typename TD, int kSteps>
__device__ __forceinline__ void load_b(const LoraParams &p, const Tile &t, int n, int lane, uint2 (&b)[4][kSteps])
{
    constexpr int  kPer = 16 / static_cast<int>(sizeof(TD));
    const int      g = lane >> 2, c = lane & 3;
    const uint8_t *row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        // column j = g of the i-th tile of eight: the lane that gets its results has c = j / 2, as its elements 2 i + j % 2
        const int el = 2 * i + (g & 1), ch = n + piece_channel<TD>(el / kPer, g >> 1) + el % kPer;
        row[i]       = p.b + (static_cast<int64_t>(max(t.adapter, 0)) * p.N + min(ch, p.N - 1)) * p.ld_b + 8 * c;
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
    {
        if (t.adapter >= 0 && s * 16 < t.rank)
        {
            const int left = t.rank - s * 16 - 4 * c; // ranks of this lane's four
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                b[i][s] = make_uint2(0, 0);
                if (left > 0) b[i][s] = __ldcg(reinterpret_cast<const uint2 *>(row[i] + s * 32));
            }
        }
    }
    if ((t.rank & 3) != 0)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
        {
            const int left = t.rank - s * 16 - 4 * c;
            if (left > 0 && left < 4)
            {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
                    b[i][s].y = left == 3 ? b[i][s].y & 0xffffu : 0u;
                    if (left == 1) b[i][s].x &= 0xffffu;
                }
            }
        }
    }
}

template <typename T, typename TD, int kRank, bool kVec>
__global__ void __launch_bounds__(kThreads, (Expand<T, TD, kRank>::kCtas)) lora_expand_kernel(const __grid_constant__ LoraParams p)
{
    using E = Expand<T, TD, kRank>;
    constexpr int kPieces = static_cast<int>(sizeof(TD)) / 2, kPer = 8 / kPieces; // 16-byte pieces of a lane's row, elements of one
    extern __shared__ __align__(128) uint8_t smem[]; // v of two tiles, then the slots
    __shared__ Item       list[kListed];
    __shared__ ScanShared scan;
    griddep_launch_dependents();
    // the launch ahead let this one start after its own wait: all but v is as it will be
    const int blocks = (p.N + 32 * kWarps - 1) / (32 * kWarps); // of channels
    const int grid = static_cast<int>(gridDim.x), own = static_cast<int>(blockIdx.x);
    int       before = 0, turn = 0; // tiles of the requests so far
    for (int r0 = 0; r0 < p.requests; r0 += kThreads, turn ^= 1)
    {
        const Request q     = load_request(p, r0 + static_cast<int>(threadIdx.x));
        const int     tiles = request_tiles(p, q);
        int           at, all;
        scan_tiles(scan, turn, tiles, at, all);
        const int first = min(before + at, p.tiles) * blocks, end = min(before + at + tiles, p.tiles) * blocks; // the request's items
        if (first < end)
        {
            for (int i = max(first - own + grid - 1, 0) / grid; i < kListed && own + i * grid < end; ++i)
            {
                const int in = own + i * grid - first;
                list[i]      = Item{request_tile(p, q, in / blocks), in % blocks * 32 * kWarps};
            }
        }
        before = min(before + all, p.tiles);
    }
    const int items = min(max(before * blocks - own + grid - 1, 0) / grid, kListed);
    if (items == 0)
    {
        griddep_wait();
        return;
    }
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const uint32_t slots = smem_u32(smem) + E::kOffBase + static_cast<uint32_t>(warp) * E::kSlots * 16 * E::kRow;
    const int warp_n = warp * 32; // the warp's channels of an item
    // The ring: units in the order in which they are worked on.  16-byte pieces are exchanged by row where a row has eight of them
    // (reading two rows side by side hits all banks once).  A lane copies one piece of every kStep-th row.
    constexpr int  kUnit = E::kRow / 16, kStep = 32 / kUnit; // pieces of a row, rows that the warp copies at a time
    const int      copy_row = lane / kUnit, copy_ch = warp_n + lane % kUnit * (16 / static_cast<int>(sizeof(TD)));
    const uint32_t copy_to  = slots + static_cast<uint32_t>(copy_row * E::kRow + ((kUnit == 8 ? (lane % kUnit) ^ ((copy_row & 1) << 2) : lane % kUnit) << 4));
    int            ahead = 0, ahead_rows = 0, ahead_units = 0; // the next item; rows of this lane and units of the present one that are still to come
    uint32_t       ahead_slot = 0;
    const uint8_t *ahead_src  = nullptr;
    const int64_t  copy_step  = kStep * p.ld_base;
    TD             held[kVec ? 1 : 16]; // rows that start anywhere: the next unit's values of this lane's channel, on their way
    auto           load_unit  = [&]() {
        if (ahead_units == 0)
        {
            while (ahead < items && list[ahead].n + warp_n >= p.N) ++ahead; // nothing for this warp there
            if (ahead < items)
            {
                const Tile &t  = list[ahead].tile;
                const int   ch = list[ahead].n + (kVec ? copy_ch : warp_n + lane), row = kVec ? copy_row : 0;
                ahead_units    = (t.count + 15) >> 4;
                ahead_rows     = ch < p.N ? t.count - row : 0; // pieces lie before the last channel or behind it
                ahead_src      = p.base + static_cast<int64_t>(t.first + row) * p.ld_base + static_cast<int64_t>(ch) * static_cast<int>(sizeof(TD));
                ++ahead;
            }
        }
        if (ahead_units > 0)
        {
            if constexpr (kVec)
            {
#pragma unroll
                for (int j = 0; j < 16 / kStep; ++j, ahead_src += copy_step)
                {
                    if (j * kStep < ahead_rows) copy16(copy_to + ahead_slot + j * kStep * E::kRow, ahead_src, 16); // rows behind the last: never stored
                }
            }
            else
            {
#pragma unroll
                for (int j = 0; j < 16; ++j, ahead_src += p.ld_base)
                {
                    held[j] = from_float<TD>(0.f);
                    if (j < ahead_rows) held[j] = __ldcg(reinterpret_cast<const TD *>(ahead_src));
                }
            }
            ahead_rows -= 16;
            --ahead_units;
            ahead_slot = ahead_slot == (E::kSlots - 1) * 16 * E::kRow ? 0u : ahead_slot + 16 * E::kRow;
        }
        copy_commit();
    };
    // v of a tile to one half of its buffer, by all threads
    auto load_v = [&](const Tile &t, int half) {
        if (t.adapter < 0) return;
        constexpr int kUnits = kRank / 8 + 1; // 16-byte units of a row
        const int     rows   = (t.count + 15) & ~15;
        for (int i = threadIdx.x; i < rows * kUnits; i += kThreads)
        {
            const int       row = i / kUnits, unit = i % kUnits;
            const uint16_t *src = p.v + static_cast<int64_t>(t.first + min(row, t.count - 1)) * (kRank + 8) + unit * 8;
            const uint32_t  dst = smem_u32(smem) + static_cast<uint32_t>(half * E::kV + row * E::kPitch + unit * 16);
#pragma unroll
            for (int part = 0; part < E::kParts; ++part)
            {
                copy16(dst + part * E::kTile * E::kPitch, src + static_cast<int64_t>(part) * p.tokens * (kRank + 8), row < t.count ? 16 : 0);
            }
        }
    };
#pragma unroll
    for (int u = 0; u < (kVec ? E::kSlots : 1); ++u) load_unit();
    // Rows that start anywhere pass through one slot, in and out: a lane's channel of all rows on the one side, its pieces on the other.
    TD *const column = reinterpret_cast<TD *>(smem + E::kOffBase + warp * E::kSlots * 16 * E::kRow);
    auto      place  = [&](int row) {
        const int at = lane * static_cast<int>(sizeof(TD)), unit = at >> 4;
        return (row * E::kRow + ((kUnit == 8 ? unit ^ ((row & 1) << 2) : unit) << 4) + (at & 15)) / static_cast<int>(sizeof(TD));
    };
    uint2 b[4][E::kSteps], next[E::kAhead ? 4 : 1][E::kSteps];
    if constexpr (E::kAhead) load_b<TD>(p, list[0].tile, list[0].n + warp_n, lane, next);
    griddep_wait();
    load_v(list[0].tile, 0);
    copy_commit();
    // a lane's pieces of a unit, in the slot that is next
    const uint8_t *piece[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
        piece[i] = smem + E::kOffBase + warp * E::kSlots * 16 * E::kRow + g * E::kRow + 16 * (kPieces == 2 ? (4 * i + c) ^ ((g & 1) << 2) : c);
    int slot = 0, units = 0; // units: groups of copies since the one that brought this item's v
    for (int item = 0; item < items; ++item)
    {
        const Tile t    = list[item].tile;
        const int  n    = list[item].n + warp_n, half = item & 1;
        if constexpr (E::kAhead)
        {
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
#pragma unroll
                for (int s = 0; s < E::kSteps; ++s) b[i][s] = next[i][s];
            }
            if (item + 1 < items) load_b<TD>(p, list[item + 1].tile, list[item + 1].n + warp_n, lane, next);
        }
        else
        {
            load_b<TD>(p, t, n, lane, b);
        }
        if (units == 0) copy_wait<0>();
        else if (units == 1) copy_wait<1>();
        else if (units == 2) copy_wait<2>();
        else if (units == 3) copy_wait<3>();
        else copy_wait<4>();
        __syncthreads(); // v is there, and all warps have done with the item before
        if (item + 1 < items) load_v(list[item + 1].tile, half ^ 1);
        copy_commit();
        units = 0;
        if (n >= p.N) continue; // the same for the warp
        units = (t.count + 15) >> 4;
        const uint32_t v_at    = smem_u32(smem) + static_cast<uint32_t>(half * E::kV + (lane & 15) * E::kPitch + (lane >> 4) * 16);
        uint8_t       *dst_row = p.dst + static_cast<int64_t>(t.first + g) * p.ld_dst + static_cast<int64_t>(n) * static_cast<int>(sizeof(TD));
        const uint8_t *v_row   = smem + half * E::kV + g * E::kPitch;
        const int64_t  low_row = 8 * p.ld_dst;
        for (int m = 0; m < t.count; m += 16, dst_row += 2 * low_row, v_row += 16 * E::kPitch)
        {
            if constexpr (kVec) copy_wait<E::kSlots - 1>();
            else
            {
#pragma unroll
                for (int j = 0; j < 16; ++j) column[place(j)] = held[j];
            }
            __syncwarp();
            float base[2][8];
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                TD e[8];
#pragma unroll
                for (int i = 0; i < kPieces; ++i)
                {
                    const uint4 v = *reinterpret_cast<const uint4 *>(piece[i] + slot + h * 8 * E::kRow);
                    memcpy(e + i * kPer, &v, 16);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) base[h][i] = to_float(e[i]);
            }
            __syncwarp();
            load_unit(); // to the slot that the warp has read
            if constexpr (kVec) slot = slot == (E::kSlots - 1) * 16 * E::kRow ? 0 : slot + 16 * E::kRow;
            if (t.adapter >= 0)
            {
                float acc[4][4];
#pragma unroll
                for (int part = E::kParts - 1; part >= 0; --part) // small parts first
                {
#pragma unroll
                    for (int s = 0; s < E::kSteps; ++s)
                    {
                        if (s * 16 < t.rank)
                        {
                            uint32_t v[4];
                            ldmatrix_x4(v_at + static_cast<uint32_t>(m * E::kPitch + part * E::kTile * E::kPitch + s * 32), v);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                            {
                                if (part == E::kParts - 1 && s == 0) mma<T, true>(acc[i], v[0], v[1], v[2], v[3], b[i][s].x, b[i][s].y);
                                else mma<T>(acc[i], v[0], v[1], v[2], v[3], b[i][s].x, b[i][s].y);
                            }
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
                {
                    const float f = *reinterpret_cast<const float *>(v_row + h * 8 * E::kPitch + kRank * 2);
#pragma unroll
                    for (int i = 0; i < 8; ++i) base[h][i] = fmaf(acc[i >> 1][2 * h + (i & 1)], f, base[h][i]);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                TD  e[8];
                TD *dst = reinterpret_cast<TD *>(h == 0 ? dst_row : dst_row + low_row);
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = from_float<TD>(base[h][i]);
#pragma unroll
                for (int i = 0; i < kPieces; ++i)
                {
                    uint4 v;
                    memcpy(&v, e + i * kPer, 16);
                    if constexpr (kVec)
                    {
                        const int ch = piece_channel<TD>(i, c);
                        if (m + h * 8 + g < t.count && n + ch < p.N) *reinterpret_cast<uint4 *>(dst + ch) = v;
                    }
                    else
                    {
                        *reinterpret_cast<uint4 *>(const_cast<uint8_t *>(piece[i]) + h * 8 * E::kRow) = v;
                    }
                }
            }
            if constexpr (!kVec)
            {
                __syncwarp();
                TD *dst = reinterpret_cast<TD *>(dst_row - g * p.ld_dst) + lane;
                if (n + lane < p.N)
                {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                    {
                        if (m + j < t.count) *reinterpret_cast<TD *>(reinterpret_cast<uint8_t *>(dst) + j * p.ld_dst) = column[place(j)];
                    }
                }
                __syncwarp();
            }
        }
    }
    copy_wait<0>();
}

// ---- few tiles: both products in one launch ---------------------------------------------------------------------
// Tiles of up to 16 tokens, a cluster each.  Its CTAs share K as above, every one of them adds up all of v for itself, and takes every
// ranks-th block of 256 channels.  What bounds it is the chain requests -> tile (2 us) -> x and A -> sums (4 us) -> results (3 us, 24 requests
// of a token, 14336 channels), and in the last part its instructions: addresses that are kept, v in registers at 16 ranks and no work for
// rows that are not there took 10.8 to 9.3 us.  B and base of a warp's first blocks are on their way before the sums are there, those of the
// blocks to come while others are multiplied (at rank 16 and 32-bit results 128 registers are 40 bytes too few).
template <typename T, typename TD, int kRank>
struct Few
{
    static constexpr int kTile    = 16;
    static constexpr int kSteps   = kRank / 16;
    static constexpr int kParts   = std::is_same<T, __nv_bfloat16>::value && sizeof(TD) == 4 ? 3 : 2;
    static constexpr int kDepth   = kRank == 16 ? 3 : kRank == 32 ? 2 : 1; // blocks whose B and base a warp has in registers
    static constexpr bool kKept   = kRank == 16;                           // v in registers
    static constexpr int kStages  = kRank == 64 ? 6 : 8;
    static constexpr int kA       = kRank * 128, kX = kTile * 128, kStage = kA + kX;
    static constexpr int kShare   = kRank + 1;                                                   // floats of a token's sums
    static constexpr int kOffV    = (kStages - 1) * kStage + (kStage > 16384 ? kStage : 16384);  // an MMA reads 16 KB from a stage's start on
    static constexpr int kPitch   = kRank * 2 + 16;                                              // bytes of a row of v, its factor included
    static constexpr int kOffBar  = kOffV + kParts * kTile * kPitch;
    // Allocating columns of tensor memory waits until there are enough of them, and a CTA of a cluster that waits keeps the others of its
    // cluster where they are: were there more CTAs on an SM than its tensor memory holds, of calls on two streams for instance, they could wait
    // for each other.  So this CTA takes shared memory enough not to fit beside two that have half of tensor memory each (ShrinkMma's with four
    // chains, 90 KB, and the products' and the expert layer's, 88 KB or more).
    static constexpr int kNeeded  = kOffBar + (2 * kStages + 2) * 8 + 16 + 1024;
    static constexpr int kSmem    = kNeeded > 57344 ? kNeeded : 57344;
    static constexpr int kChained = sizeof(TD) == 4 ? kChains : 1; // see add_chains
    static constexpr int kColumns = kChained == 1 ? 32 : kChained * kTile;
    static_assert(kSmem + 2 * 88176 > 228 * 1024 - 1024 && kSmem + 2 * (ShrinkMma<16>::kSmem + 1024) > 228 * 1024 - 1024, "no room beside two halves of tensor memory");
    static_assert(kTile * kShare * 4 <= kOffV && kStage % 1024 == 0, "sums fit where the stages were");
};
template <typename T, typename TD, int kRank, bool kVec>
__global__ void __launch_bounds__(kThreads, 2)
    lora_few_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ LoraParams p)
{
    using S = Few<T, TD, kRank>;
    constexpr int STAGES = S::kStages, kPieces = static_cast<int>(sizeof(TD)) / 2, kPer = 8 / kPieces; // 16-byte pieces of a lane's row, elements of one
    extern __shared__ uint8_t smem_raw[];
    uint8_t       *smem      = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t s_stage   = smem_u32(smem), bar_base = smem_u32(smem + S::kOffBar);
    auto           full_bar  = [&](int s) { return bar_base + 8u * s; };
    auto           empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    const uint32_t done_bar  = bar_base + 8u * (2 * STAGES), gone_bar = done_bar + 8;
    uint32_t      *s_tmem    = reinterpret_cast<uint32_t *>(smem + S::kOffBar + (2 * STAGES + 2) * 8);
    volatile int  *s_abort   = reinterpret_cast<volatile int *>(s_tmem + 1);
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    if (threadIdx.x == 0)
    {
        for (int s = 0; s < STAGES; ++s)
        {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
        mbar_init(gone_bar, 1);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1)
    {
        tmem_alloc(smem_u32(s_tmem), S::kColumns);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    griddep_launch_dependents();
    griddep_wait();
    const int  ranks = static_cast<int>(gridDim.x / num_clusters_x()), rank = static_cast<int>(cluster_ctarank());
    const Tile t     = find_tile(p, static_cast<int>(cluster_id_x()));
    if (t.count == 0) // the same for the cluster, as is whether there is an adapter
    {
        if (warp == 1) tmem_dealloc(tmem, S::kColumns);
        return;
    }
    const bool adds   = t.adapter >= 0;
    const int  blocks = (p.K + 63) / 64; // of 64 columns, shared by the CTAs of the cluster
    const int  first  = share_begin(blocks, rank, ranks), n_blocks = adds ? share_begin(blocks, rank + 1, ranks) - first : 0;
    int        issued = 0; // stages that the producer has filled
    auto       produce = [&](int end) { // by warp 0
        const bool el    = elect_one();
        const int  a_row = max(t.adapter, 0) * p.max_rank;
        for (; issued < end; ++issued)
        {
            const int s = issued % STAGES;
            if (!warp_wait(empty_bar(s), (static_cast<uint32_t>(issued / STAGES) & 1u) ^ 1u, s_abort, DEV_TIMEOUT_PRODUCER, p.spin_limit)) break;
            if (issued == p.withhold && blockIdx.x == 0) continue;
            if (el)
            {
                const uint32_t dst = s_stage + s * S::kStage;
                mbar_expect_tx(full_bar(s), static_cast<uint32_t>(S::kStage));
                tma_load_2d(dst, &tmap_a, (first + issued) * 64, a_row, full_bar(s));
                tma_load_2d(dst + S::kA, &tmap_x, (first + issued) * 64, t.first, full_bar(s));
            }
            __syncwarp();
        }
    };
    if (warp == 0) produce(min(n_blocks, STAGES));
    // B and base of the warp's first blocks of channels, ahead of its part in the sums
    const int wide = (p.N + 32 * kWarps - 1) / (32 * kWarps);
    uint2     b[S::kDepth][4][S::kSteps] = {};
    uint4     base[S::kDepth][2][kPieces];
    // A lane's places in the warp's next block to load and to store: row of B of its first column (see load_b), piece of rows g of base and dst.
    const int      n_first   = rank * 32 * kWarps + warp * 32;
    const uint8_t *b_lane    = p.b + (static_cast<int64_t>(max(t.adapter, 0)) * p.N + n_first + piece_channel<TD>(0, g >> 1) + (g & 1)) * p.ld_b + 8 * c;
    const uint8_t *base_lane = p.base + static_cast<int64_t>(t.first + g) * p.ld_base + static_cast<int64_t>(n_first) * static_cast<int>(sizeof(TD)) + 16 * c;
    uint8_t       *dst_lane  = p.dst + static_cast<int64_t>(t.first + g) * p.ld_dst + static_cast<int64_t>(n_first) * static_cast<int>(sizeof(TD)) + 16 * c;
    const int64_t  b_step    = static_cast<int64_t>(ranks) * 32 * kWarps * p.ld_b, step = static_cast<int64_t>(ranks) * 32 * kWarps * static_cast<int>(sizeof(TD));
    const bool     plain     = kVec && adds && (t.rank & 3) == 0; // whole blocks need no tests
    auto load_block = [&](int block, uint2 (&to)[4][S::kSteps], uint4 (&rows)[2][kPieces]) { // blocks one after the other
        if (block >= wide) return;
        const int n = block * 32 * kWarps + warp * 32;
        if (n >= p.N) return; // the same for the warp
        if (plain && n + 32 <= p.N)
        {
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const int ch = sizeof(TD) == 2 ? 2 * i : 16 * (i >> 1) + 2 * (i & 1);
#pragma unroll
                for (int s = 0; s < S::kSteps; ++s)
                {
                    if (s * 16 + 4 * c < t.rank) to[i][s] = __ldcg(reinterpret_cast<const uint2 *>(b_lane + ch * p.ld_b + s * 32)); // else: zeros, as they were
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                if (h * 8 + g < t.count)
                {
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) rows[h][i] = __ldcg(reinterpret_cast<const uint4 *>(base_lane + h * 8 * p.ld_base + 64 * i));
                }
            }
            b_lane += b_step;
            base_lane += step;
            return;
        }
        load_b<TD>(p, t, n, lane, to);
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            const int row = h * 8 + g;
            if (row >= t.count) continue;
            const uint8_t *src = p.base + static_cast<int64_t>(t.first + row) * p.ld_base;
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
            {
                const int ch = n + piece_channel<TD>(i, c);
                if constexpr (kVec)
                {
                    if (ch < p.N) rows[h][i] = __ldcg(reinterpret_cast<const uint4 *>(src + static_cast<int64_t>(ch) * static_cast<int>(sizeof(TD))));
                }
                else
                {
                    TD e[kPer];
#pragma unroll
                    for (int k = 0; k < kPer; ++k)
                    {
                        e[k] = from_float<TD>(0.f);
                        if (ch + k < p.N) e[k] = __ldcg(reinterpret_cast<const TD *>(src) + ch + k);
                    }
                    memcpy(&rows[h][i], e, 16);
                }
            }
        }
    };
#pragma unroll
    for (int d = 0; d < S::kDepth; ++d) load_block(rank + d * ranks, b[d], base[d]);
    __syncwarp();
    if (warp == 0)
    {
        produce(n_blocks);
    }
    else if (warp == 1)
    {
        const bool     el    = elect_one();
        const uint32_t idesc = p.idesc | (2u << 17); // 16 columns
        bool           ok    = true;
        for (int i = 0; i < n_blocks && ok; ++i)
        {
            const int s = i % STAGES;
            ok = warp_wait(full_bar(s), static_cast<uint32_t>(i / STAGES) & 1u, s_abort, DEV_TIMEOUT_MMA, p.spin_limit);
            if (!ok) break;
            tc_fence_after();
            const uint64_t a_desc = make_kmajor_sw128_desc(s_stage + s * S::kStage), b_desc = make_kmajor_sw128_desc(s_stage + s * S::kStage + S::kA);
            if (el)
            {
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_f16(tmem + i % S::kChained * S::kTile, a_desc + 2u * k, b_desc + 2u * k, idesc, i >= S::kChained || k != 0 ? 1u : 0u);
                umma_commit(empty_bar(s));
            }
            __syncwarp();
        }
        if (ok && el && adds) umma_commit(done_bar);
        __syncwarp();
    }
    uint8_t *const area = smem + S::kOffV; // v: [part][token][rank], the factor behind a token's first part
    if (adds)
    {
        const bool ok    = warp_wait(done_bar, 0, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit);
        float     *share = reinterpret_cast<float *>(smem);
        const int  r     = warp * 32 + lane;
        __syncthreads(); // every warp's waits are over; the MMAs have read the stages
        if (ok && *s_abort == 0 && warp * 32 < kRank) // sums to shared memory, [token][rank]: a lane has a rank
        {
            tc_fence_after();
            float v[16];
            add_chains(tmem + (static_cast<uint32_t>(warp * 32) << 16), S::kTile, min(n_blocks, S::kChained), v);
            if (r < kRank)
            {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    if (i < t.count) share[i * S::kShare + r] = r < t.rank ? v[i] : 0.f; // behind the adapter's ranks: zeros
                }
            }
        }
        tc_fence_before();
        __syncthreads();
        const bool gone = *s_abort != 0;
        if (warp == 0 && gone)
        {
            drain_stages<STAGES>(bar_base, issued, blockIdx.x == 0 ? p.withhold : -1, p.spin_limit);
        }
        if (warp == 1 && gone)
        {
            drain_mmas<false>(gone_bar, p.spin_limit);
        }
        if (threadIdx.x == 0 && gone)
        {
            atomicCAS(p.status, 0, *s_abort);
        }
        __syncwarp();
        if (ranks > 1) cluster_sync();
        else __syncthreads();
        for (int tok = warp; tok < t.count; tok += kWarps) // (of a CTA that has given up: nothing of use)
        {
            uint8_t *const row    = area + tok * S::kPitch;
            const float    factor = token_v<T, kRank>(p, t, share, S::kShare, ranks, tok, [&](int part, int place, uint16_t bits) {
                *reinterpret_cast<uint16_t *>(row + part * S::kTile * S::kPitch + place * 2) = bits;
            });
            if (lane == 0) *reinterpret_cast<float *>(row + kRank * 2) = factor;
        }
        __syncwarp();
        if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); // this warp has read the others' sums
        __syncthreads();
    }
    if (warp == 1)
    {
        tc_fence_after();
        tmem_dealloc(tmem, S::kColumns);
    }
    float f[2] = {};
    if (adds)
    {
#pragma unroll
        for (int h = 0; h < 2; ++h) f[h] = *reinterpret_cast<const float *>(area + (h * 8 + g) * S::kPitch + kRank * 2); // rows behind the last: not stored
    }
    const uint32_t v_at = smem_u32(area) + static_cast<uint32_t>((lane & 15) * S::kPitch + (lane >> 4) * 16);
    auto           load_v = [&](int part, int s, uint32_t (&v)[4]) { ldmatrix_x4(v_at + static_cast<uint32_t>(part * S::kTile * S::kPitch + s * 32), v); };
    uint32_t       kept[S::kKept ? S::kParts : 1][4];
    if (S::kKept && adds)
    {
#pragma unroll
        for (int part = 0; part < S::kParts; ++part) load_v(part, 0, kept[S::kKept ? part : 0]);
    }
    for (int block = rank; block < wide; block += S::kDepth * ranks)
    {
#pragma unroll
        for (int d = 0; d < S::kDepth; ++d)
        {
            const int at = block + d * ranks, n = at < wide ? at * 32 * kWarps + warp * 32 : p.N;
            if (n < p.N) // the same for the warp
            {
                float acc[4][4];
                __syncwarp();
                if (adds)
                {
#pragma unroll
                    for (int part = S::kParts - 1; part >= 0; --part) // small parts first
                    {
#pragma unroll
                        for (int s = 0; s < S::kSteps; ++s)
                        {
                            if (s * 16 < t.rank)
                            {
                                uint32_t own[4];
                                if (!S::kKept) load_v(part, s, own);
                                const uint32_t(&v)[4] = S::kKept ? kept[S::kKept ? part : 0] : own;
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                {
                                    if (part == S::kParts - 1 && s == 0) mma<T, true>(acc[i], v[0], v[1], v[2], v[3], b[d][i][s].x, b[d][i][s].y);
                                    else mma<T>(acc[i], v[0], v[1], v[2], v[3], b[d][i][s].x, b[d][i][s].y);
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
                {
                    if (h * 8 >= t.count) break; // the same for the block
                    TD e[8];
                    memcpy(e, base[d][h], 16 * kPieces);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                    {
                        if (adds) e[i] = from_float<TD>(fmaf(acc[i >> 1][2 * h + (i & 1)], f[h], to_float(e[i])));
                    }
                    const int row = h * 8 + g;
                    if (plain && n + 32 <= p.N)
                    {
                        uint4 v[kPieces];
                        memcpy(v, e, sizeof(v));
                        if (row < t.count)
                        {
#pragma unroll
                            for (int i = 0; i < kPieces; ++i)
                                *reinterpret_cast<uint4 *>(dst_lane + h * 8 * p.ld_dst + 64 * i) = v[i];
                        }
                    }
                    else if (row < t.count)
                    {
                        TD *dst = reinterpret_cast<TD *>(p.dst + static_cast<int64_t>(t.first + row) * p.ld_dst);
#pragma unroll
                        for (int i = 0; i < kPieces; ++i)
                        {
                            const int ch = n + piece_channel<TD>(i, c);
                            if constexpr (kVec)
                            {
                                uint4 v;
                                memcpy(&v, e + i * kPer, 16);
                                if (ch < p.N) *reinterpret_cast<uint4 *>(dst + ch) = v;
                            }
                            else
                            {
#pragma unroll
                                for (int k = 0; k < kPer; ++k)
                                {
                                    if (ch + k < p.N) dst[ch + k] = e[i * kPer + k];
                                }
                            }
                        }
                    }
                }
            }
            dst_lane += step;
            load_block(at + S::kDepth * ranks, b[d], base[d]);
        }
    }
    __syncwarp();
    if (adds && ranks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); // nobody leaves while others read its sums
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
int64_t most_tiles(const cugl_lora_desc &d, int64_t tile) // of a request, all but the last are full
{
    const int64_t some = d.requests < d.tokens ? d.requests : d.tokens;
    return (d.tokens - some) / tile + some;
}

// CTAs that share a tile's K: as many as run at once, two to an SM, with two blocks of 64 columns each at least
int shrink_split(const cugl_context *ctx, const LoraParams &p, int64_t tiles)
{
    int split = 1;
    while (split < kMaxSplit && tiles * split * 2 <= 2 * ctx->sm_count && p.K >= 2 * split * 128) split *= 2;
    return split;
}
// rows of 16-bit elements; box = 64 columns x box_rows in the 128-byte swizzle, what lies outside reads as 0
bool encode_rows_map(CUtensorMap *map, const void *base, int64_t rows, int cols, int64_t ld, int box_rows)
{
    EncodeTiledFn    fn         = get_encode_fn();
    const cuuint64_t dims[2]    = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
    const cuuint32_t box[2]     = {64, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estr[2]    = {1, 1};
    return fn != nullptr && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
template <typename T, int kRank>
cugl_status launch_shrink_mma(cugl_context *ctx, const LoraParams &p, int64_t tiles)
{
    using S = ShrinkMma<kRank>;
    CUtensorMap map_a, map_x, map_few;
    if (!encode_rows_map(&map_a, p.a, static_cast<int64_t>(p.n_adapters) * p.max_rank, p.K, p.ld_a, kRank) || !encode_rows_map(&map_x, p.x, p.tokens, p.K, p.ld_x, S::kTile) ||
        !encode_rows_map(&map_few, p.x, p.tokens, p.K, p.ld_x, 16))
    {
        return fail(ctx, CUGL_RUNTIME_ERROR, "cuTensorMapEncodeTiled failed for x or A");
    }
    auto                     kernel  = lora_shrink_mma_kernel<T, kRank>;
    static std::atomic<bool> set[64] = {};
    CUGL_TRY(allow_smem(ctx, kernel, S::kSmem, set));
    const int split = shrink_split(ctx, p, tiles);
    CUGL_CUDA_TRY(ctx, launch_dependent_cluster(ctx, kernel, dim3(static_cast<unsigned>(tiles * split)), kThreads, S::kSmem, split, tiles * split, map_a, map_x, map_few, p));
    return CUGL_SUCCESS;
}
template <typename T, int kRank, int kIn>
cugl_status launch_shrink(cugl_context *ctx, const LoraParams &p, int64_t tiles)
{
    using S                          = Shrink<kRank>;
    auto                     kernel  = lora_shrink_kernel<T, kRank, kIn>;
    static std::atomic<bool> set[64] = {};
    CUGL_TRY(allow_smem(ctx, kernel, S::kSmem, set));
    const int split = shrink_split(ctx, p, tiles);
    CUGL_CUDA_TRY(ctx, launch_dependent_cluster(ctx, kernel, dim3(static_cast<unsigned>(tiles * split)), kThreads, S::kSmem, split, tiles * split, p));
    return CUGL_SUCCESS;
}
template <typename T, typename TD, int kRank, bool kVec>
cugl_status launch_expand(cugl_context *ctx, LoraParams p, int64_t tiles)
{
    using E                          = Expand<T, TD, kRank>;
    auto                     kernel  = lora_expand_kernel<T, TD, kRank, kVec>;
    static std::atomic<bool> set[64] = {};
    CUGL_TRY(allow_smem(ctx, kernel, E::kSmem, set));
    // one CTA or two to an SM; more only where there are more items than these list
    const int64_t items = (static_cast<int64_t>(p.N) + 32 * kWarps - 1) / (32 * kWarps) * tiles, most = std::max<int64_t>(E::kCtas * ctx->sm_count, (items + kListed - 1) / kListed);
    const int64_t grid  = items < most ? items : most;
    CUGL_CUDA_TRY(ctx, launch_dependent(ctx, kernel, dim3(static_cast<unsigned>(grid)), kThreads, E::kSmem, grid, p));
    return CUGL_SUCCESS;
}
// CTAs of a cluster that works on both products in one launch; 0: two launches.  One launch where requests are short, and are eight at least or
// have little to add (few channels, low ranks).  us in two / in one, K = 4096, requests x tokens.  Rank 16, N = 14336, BF16: 1 x 1 6.7 / 7.9,
// 8 x 1 8.5 / 8.4, 24 x 1 13.3 / 9.4, 148 x 1 47 / 26, 24 x 8 13.8 / 10.5, 24 x 16 15.7 / 14.2, 256 x 4 78 / 50.  Rank 64, N = 4096, BF16: 1 x 1
// 7.2 / 7.8, 8 x 1 8.6 / 8.5, 24 x 8 13.8 / 12.1, 8 x 16 9.1 / 12.0.  Rank 16, N = 4096, F16 to F32: 1 x 1 6.6 / 6.3, 24 x 8 9.3 / 7.7.  Rank 128,
// N = 4096, BF16: 1 x 1 8.7 / 11.6, 24 x 1 20.4 / 20.3.
int few_split(const LoraParams &p, int padded)
{
    const int64_t some = std::min(p.requests, p.tokens), wide = (static_cast<int64_t>(p.N) + 32 * kWarps - 1) / (32 * kWarps);
    if (padded > kFewRank || p.tokens > 8 * some || (some < 8 && wide * padded > 256)) return 0;
    // as many as run at once (see mx_split).  us with eight / four / two / one CTA, rank 16, N = 14336, requests of a token: 30 9.5 / 13.9 / 22 / 40,
    // 40 17.1 / 14.7 / 24 / 41, 60 19 / 15.0 / 25 / 42, 74 27 / 26 / 23 / 41, 148 47 / 41 / 26 / 42, 160 48 / 43 / 48 / 46
    return some <= 33 ? 8 : some <= 71 ? 4 : some <= 148 ? 2 : 1;
}
template <typename T, typename TD, int kRank>
cugl_status launch_few(cugl_context *ctx, LoraParams p, int64_t tiles, int split, bool vec_out)
{
    using S = Few<T, TD, kRank>;
    CUtensorMap map_a, map_x;
    if (!encode_rows_map(&map_a, p.a, static_cast<int64_t>(p.n_adapters) * p.max_rank, p.K, p.ld_a, kRank) || !encode_rows_map(&map_x, p.x, p.tokens, p.K, p.ld_x, S::kTile))
    {
        return fail(ctx, CUGL_RUNTIME_ERROR, "cuTensorMapEncodeTiled failed for x or A");
    }
    p.tile  = S::kTile;
    p.tiles = static_cast<int>(tiles);
    static std::atomic<bool> set[2][64] = {};
    auto                     kernel     = vec_out ? lora_few_kernel<T, TD, kRank, true> : lora_few_kernel<T, TD, kRank, false>;
    CUGL_TRY(allow_smem(ctx, kernel, S::kSmem, set[vec_out ? 1 : 0]));
    CUGL_CUDA_TRY(ctx, launch_dependent_cluster(ctx, kernel, dim3(static_cast<unsigned>(tiles * split)), kThreads, S::kSmem, split, tiles * split, map_a, map_x, p));
    return CUGL_SUCCESS;
}
template <typename T, typename TD, int kRank>
cugl_status launch_lora(cugl_context *ctx, const LoraParams &p, int64_t tiles, int64_t few_tiles, int rows_in, bool vec_out)
{
    if constexpr (kRank <= kFewRank)
    {
        const int split = rows_in == kUnits16 ? few_split(p, kRank) : 0;
        if (split > 0) return launch_few<T, TD, kRank>(ctx, p, few_tiles, split, vec_out);
    }
    CUGL_TRY((rows_in == kUnits16 ? launch_shrink_mma<T, kRank>(ctx, p, tiles)
              : rows_in == kWords ? launch_shrink<T, kRank, kWords>(ctx, p, tiles)
                                  : launch_shrink<T, kRank, kAnywhere>(ctx, p, tiles)));
    return vec_out ? launch_expand<T, TD, kRank, true>(ctx, p, tiles) : launch_expand<T, TD, kRank, false>(ctx, p, tiles);
}
template <typename T, typename TD>
cugl_status launch_lora(cugl_context *ctx, const LoraParams &p, int64_t tiles, int64_t few_tiles, int rows_in, bool vec_out)
{
    switch (padded_rank(p.max_rank))
    {
        case 16: return launch_lora<T, TD, 16>(ctx, p, tiles, few_tiles, rows_in, vec_out);
        case 32: return launch_lora<T, TD, 32>(ctx, p, tiles, few_tiles, rows_in, vec_out);
        case 64: return launch_lora<T, TD, 64>(ctx, p, tiles, few_tiles, rows_in, vec_out);
        default: return launch_lora<T, TD, 128>(ctx, p, tiles, few_tiles, rows_in, vec_out);
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
    const int64_t tiles = most_tiles(*d, tile_tokens(d->max_rank));
    if (tiles > 65535) return "more than 65535 tiles of tokens";
    if (tiles * ((static_cast<int64_t>(d->N) + 32 * kWarps - 1) / (32 * kWarps)) > INT32_MAX / 2) return "more than 2^30 tiles of tokens and channels";
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
        return static_cast<size_t>(desc->tokens) * static_cast<size_t>(padded_rank(desc->max_rank) + 8) * 2 * static_cast<size_t>(v_parts(*desc)) + 16;
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
        auto       even = [](const void *q, int64_t ld) { return ((reinterpret_cast<uintptr_t>(q) | static_cast<uintptr_t>(ld)) & 15) == 0; };
        const bool words = ((reinterpret_cast<uintptr_t>(d_x) | reinterpret_cast<uintptr_t>(d_a) | static_cast<uintptr_t>(desc->ld_x) | static_cast<uintptr_t>(desc->ld_a)) & 3) == 0;
        const bool mapped  = desc->ld_x < (1ll << 40) && desc->ld_a < (1ll << 40) && static_cast<int64_t>(desc->adapters) * desc->max_rank < (1ll << 31);
        const int  rows_in = even(d_x, desc->ld_x) && even(d_a, desc->ld_a) && mapped ? kUnits16 : words && desc->K % 2 == 0 ? kWords : kAnywhere;
        const bool vec_out = even(d_base, desc->ld_base) && even(d_dst, desc->ld_dst) && desc->N % 8 == 0;
        const int64_t tiles = most_tiles(*desc, p.tile), few_tiles = most_tiles(*desc, 16);
        p.tiles             = static_cast<int>(tiles);
        p.chains            = desc->dst_dtype == CUGL_F32 ? kChains : 1;
        p.idesc             = f16_idesc(desc->dtype == CUGL_BF16);
        p.status            = ctx->d_status;
        p.spin_limit        = ctx->spin_limit;
        p.withhold          = ctx->withhold_kb;
        ctx->withhold_kb    = -1;
        if (desc->dtype == CUGL_F16)
        {
            return desc->dst_dtype == CUGL_F32 ? launch_lora<__half, float>(ctx, p, tiles, few_tiles, rows_in, vec_out) : launch_lora<__half, __half>(ctx, p, tiles, few_tiles, rows_in, vec_out);
        }
        return desc->dst_dtype == CUGL_F32 ? launch_lora<__nv_bfloat16, float>(ctx, p, tiles, few_tiles, rows_in, vec_out)
                                           : launch_lora<__nv_bfloat16, __nv_bfloat16>(ctx, p, tiles, few_tiles, rows_in, vec_out);
    }
}
