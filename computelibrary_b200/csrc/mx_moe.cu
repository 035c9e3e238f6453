// Mixture-of-experts layer for a few tokens with microscaled 4-bit weights:
//   p      = softmax over the token's top_k largest logits (or over all of them)
//   x'     = quantise(x)
//   h[e]   = quantise(p[e] * silu(x' . Wg[e]^T) * (x' . Wu[e]^T))       for every expert e that some token chose
//   y      = sum_e h[e] . Wd[e]^T
// The weights of the chosen experts are all there is to read, each of them once; everything else is small.  So every product
// runs over ALL tokens as MMA columns (an MMA with 128 columns still takes less time than its weights take to arrive): no
// gathering of tokens, and because the gate's weight is folded into h before it is stored -- 0 for a token that did not
// choose the expert -- the down product is one long sum over (expert, intermediate) in the accumulator: no combining pass, no
// atomics, the same order every time.
//
// Three launches, overlapped by programmatic dependent launch: gate + quantisation of x, gate/up products + SwiGLU +
// quantisation, down product.  The second lets the third start only after its own wait, i.e. when the first has completed: so
// the third knows the experts and loads its first weights while the second is still running.
//
// us (floor: the chosen experts' weights at the copy rate), hidden 2048, intermediate 768, 64 experts: 1 token, top 8, NVFP4 14.5
// (3.3), three launches of little else than latency; 48 tokens, top 4, MXFP4 40 (24); 128 tokens, top 8, NVFP4 56 (26), MXFP4
// 51 (25), where the exchange of the down product's partial sums (64 KB per CTA) and an epilogue that no MMA overlaps are next.
#include "mx_mma.cuh"

#include <cmath>
#include <initializer_list>

namespace cugl
{
namespace
{
constexpr int kMmaWarp  = 1;
constexpr int kFirstEpi = 2;
// epilogue warps: two per tensor-memory lane quarter for gate and up (SwiGLU and the re-quantisation are long chains of
// dependent instructions), one for down
constexpr int kUpEpi = 8, kDownEpi = 4;
constexpr int kUpThreads = 32 * (kFirstEpi + kUpEpi), kDownThreads = 32 * (kFirstEpi + kDownEpi);
constexpr int kMaxTokens = 128, kMaxExperts = 512, kMaxTopK = 16;
constexpr int kWithholdDown = 1 << 16; // ordinals of cugl_context_withhold_copy_once from here on: the third launch's

struct MoeParams
{
    const uint8_t *x;
    const float   *logits;
    const uint8_t *gate_scales, *up_scales, *down_scales;
    uint8_t       *dst;
    int32_t       *ids; // [tokens][top_k] chosen experts, -1: none
    float         *p;   // [tokens][top_k]
    uint8_t       *xq, *xs, *hq, *hs;
    int64_t        ld_x, ld_logits, ld_dst, ld_xq, ld_hq; // bytes
    int64_t        h_tiles, f_tiles;                      // scale tiles along hidden / intermediate
    int            tokens, hidden, inner, experts, top_k, renormalize, dtype;
    int            vec_x;
    int            route_blocks, quant_x;                 // first launch: blocks of the gate; blocks along a row of x
    float          x_mul, h_mul;                          // 2^-exponent of x and h
    float          gate_alpha, up_alpha, down_alpha;      // tensor exponents included
    uint32_t       idesc;
    int32_t       *status;
    long long      spin_limit;
    int            withhold_up, withhold_down; // see cugl_context_withhold_copy_once
};

// ---- first launch ----------------------------------------------------------------------------------------
// The gate: a warp per token.  Logits become unsigned keys in their order (0: not to be chosen: NaN and -infinity, or chosen
// already); a choice is the largest key, the lowest index among equal ones.
template <int kPer> // experts per lane
__device__ __forceinline__ void route_token(const MoeParams &p, int t, int lane)
{
    const float *row = reinterpret_cast<const float *>(reinterpret_cast<const uint8_t *>(p.logits) + t * p.ld_logits);
    uint32_t     key[kPer];
    float        top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
    {
        const int   e = i * 32 + lane;
        const float v = e < p.experts ? __ldg(row + e) : -INFINITY;
        const uint32_t b = __float_as_uint(v + 0.f); // -0 and 0 are equal logits
        key[i] = v > -INFINITY ? ((b >> 31) != 0 ? ~b : b | 0x80000000u) : 0u;
        if (v > top) top = v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float all = 0.f;
    if (p.renormalize == 0)
    {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
        {
            const int e = i * 32 + lane;
            if (e < p.experts && key[i] != 0) all += expf(__ldg(row + e) - top);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    int   mine = -1; // lane j keeps the j-th choice
    float weight = 0.f, sum = 0.f;
    for (int j = 0; j < p.top_k; ++j)
    {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) best = max(best, key[i]);
        best = __reduce_max_sync(0xffffffffu, best);
        int at = kMaxExperts;
#pragma unroll
        for (int i = kPer - 1; i >= 0; --i)
        {
            if (best != 0 && key[i] == best) at = i * 32 + lane;
        }
        at = __reduce_min_sync(0xffffffffu, at);
        if (best == 0) break;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
        {
            if (at == i * 32 + lane) key[i] = 0;
        }
        const float w = expf(__uint_as_float((best >> 31) != 0 ? best & 0x7fffffffu : ~best) - top);
        sum += w;
        if (lane == j)
        {
            mine   = at;
            weight = w;
        }
    }
    if (lane < p.top_k)
    {
        p.ids[t * p.top_k + lane] = mine;
        p.p[t * p.top_k + lane]   = weight / (p.renormalize != 0 ? sum : all);
    }
}

// x to codes and scales (the rounding of mx.cuh), sixteen columns per lane.
template <typename T, int kFormat>
__device__ __forceinline__ void quantize_tokens(const MoeParams &p, int block, int warp, int lane)
{
    constexpr int kLanesPerBlock = kFormat == CUGL_NVFP4 ? 1 : 2;
    const int     row = (block / p.quant_x) * 8 + warp, chunk = (block % p.quant_x) * 32 + lane, c0 = chunk * 16;
    if (row >= p.tokens)
    {
        return;
    }
    const T *src  = reinterpret_cast<const T *>(p.x + row * p.ld_x) + c0;
    float    v[16];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.f;
    if (c0 < p.hidden) // a multiple of 16
    {
        if (p.vec_x != 0)
        {
            uint4 q[2] = {__ldg(reinterpret_cast<const uint4 *>(src)), __ldg(reinterpret_cast<const uint4 *>(src) + 1)};
            const T *e = reinterpret_cast<const T *>(q);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = to_float(e[i]);
        }
        else
        {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = to_float(src[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
    if (kLanesPerBlock == 2)
    {
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    }
    const MxScale s    = mx_scale_of<kFormat>(amax, p.x_mul);
    uint32_t      word = s.byte << (8 * ((lane / kLanesPerBlock) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, kLanesPerBlock);
    word |= __shfl_xor_sync(0xffffffffu, word, 2 * kLanesPerBlock);
    const int block_of_k = chunk / kLanesPerBlock;
    if ((chunk & (4 * kLanesPerBlock - 1)) == 0 && block_of_k < p.h_tiles * 4)
    {
        *reinterpret_cast<uint32_t *>(p.xs + mx_scale_offset(row, block_of_k, p.h_tiles)) = word;
    }
    if (c0 < p.hidden)
    {
        scale_to_codes<kFormat, false>(v, s);
        *reinterpret_cast<uint2 *>(p.xq + row * p.ld_xq + c0 / 2) = make_uint2(pack_e2m1x8(v), pack_e2m1x8(v + 8));
    }
}

template <typename T, int kFormat>
__global__ void __launch_bounds__(256) moe_route_kernel(const __grid_constant__ MoeParams p)
{
    dependent_prologue();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, block = static_cast<int>(blockIdx.x);
    if (block < p.route_blocks)
    {
        const int t = block * 8 + warp;
        if (t < p.tokens)
        {
            if (p.experts <= 64) route_token<2>(p, t, lane);
            else if (p.experts <= 128) route_token<4>(p, t, lane);
            else route_token<kMaxExperts / 32>(p, t, lane);
        }
        return;
    }
    quantize_tokens<T, kFormat>(p, block - p.route_blocks, warp, lane);
}

// ---- what the two product launches share ---------------------------------------------------------------------
// A choice as the first launch left it.  kEarly: read ahead of griddepcontrol.wait, by the third launch.  The first launch had
// completed before the second let the third start, so its writes are performed on the device; but nothing makes a line that an
// earlier call left in this SM's L1 stale, and a workspace has the same addresses every time.  Hence a load at device scope, which
// goes to L2 (and, unlike acquiring ones, does not hold up the next).
template <bool kEarly>
__device__ __forceinline__ int chosen_id(const int32_t *at)
{
    if constexpr (!kEarly) return *at;
    int32_t v;
    asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(at) : "memory");
    return v;
}
// Experts that some token chose, in order.  list: [kMaxExperts], bits: [kMaxExperts / 32] in shared memory.
template <bool kEarly>
__device__ __forceinline__ int active_experts(const MoeParams &p, uint16_t *list, uint32_t *bits)
{
    if (threadIdx.x < kMaxExperts / 32) bits[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < p.tokens * p.top_k; i += static_cast<int>(blockDim.x))
    {
        const int e = chosen_id<kEarly>(p.ids + i);
        if (e >= 0) atomicOr(&bits[e >> 5], 1u << (e & 31));
    }
    __syncthreads();
    int total = 0;
    for (int w = 0; w < kMaxExperts / 32; ++w) total += __popc(bits[w]);
    for (int e = threadIdx.x; e < p.experts; e += static_cast<int>(blockDim.x))
    {
        if ((bits[e >> 5] >> (e & 31)) & 1u)
        {
            int at = __popc(bits[e >> 5] & ((1u << (e & 31)) - 1u));
            for (int w = 0; w < (e >> 5); ++w) at += __popc(bits[w]);
            list[at] = static_cast<uint16_t>(e);
        }
    }
    __syncthreads();
    return total;
}

// The gate's weight of expert e for token t; kNotChosen where the token did not choose it.
constexpr float kNotChosen = -1.f;
__device__ __forceinline__ float gate_weight(const MoeParams &p, int t, int e)
{
    float w = kNotChosen;
    for (int j = 0; j < p.top_k; ++j)
    {
        if (p.ids[t * p.top_k + j] == e) w = p.p[t * p.top_k + j];
    }
    return w;
}
// While a unit's MMAs run, the epilogue warps fill a table of its gate weights, a token per thread, and write the zeros of the
// tokens that did not choose the expert.  They agree on carrying on: a warp that gave up says so here instead of leaving the
// others at the barrier.
template <int kFormat>
__device__ __forceinline__ bool begin_unit(const MoeParams &p, float *table, int a, int e, int f0, bool ok)
{
    const int t = threadIdx.x - 32 * kFirstEpi;
    if (t < p.tokens)
    {
        const float w = gate_weight(p, t, e);
        table[t]      = w;
        if (w == kNotChosen)
        {
            uint2 *codes = reinterpret_cast<uint2 *>(p.hq + (static_cast<int64_t>(a) * p.tokens + t) * p.ld_hq + f0 / 2);
            for (int i = 0; i < min(kMxRows, p.inner - f0) / 16; ++i) codes[i] = make_uint2(0, 0);
            constexpr int kTiles = kMxRows / (4 * (kFormat == CUGL_NVFP4 ? 16 : 32)); // scale tiles along a unit
            uint8_t      *scales = p.hs + static_cast<int64_t>(a) * p.f_tiles * kMxTileBytes;
            for (int i = f0 / kMxRows * kTiles; i < min(f0 / kMxRows * kTiles + kTiles, static_cast<int>(p.f_tiles)); ++i)
            {
                *reinterpret_cast<uint32_t *>(scales + mx_scale_offset(t, 4 * i, p.f_tiles)) = 0;
            }
        }
    }
    __syncwarp(); // the barrier is an aligned one
    uint32_t r;
    asm volatile("{\n\t"
                 ".reg .pred p, q;\n\t"
                 "setp.ne.u32 q, %1, 0;\n\t"
                 "bar.red.and.pred p, 1, %2, q;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t"
                 "}"
                 : "=r"(r)
                 : "r"(static_cast<uint32_t>(ok)), "n"(32 * kUpEpi)
                 : "memory");
    return r != 0;
}

// Sums g and u of four tokens at a warp's 32 consecutive f to h, its codes and scales; valid: bit i, token t[i] is to be stored.
// Four at a time because each is one long chain of dependent instructions.
template <int kFormat>
__device__ __forceinline__ void store_hidden(const MoeParams &p, int a, const int (&t)[4], int f, int lane, const float (&g)[4], const float (&u)[4],
                                             const float *weight, uint32_t valid)
{
    constexpr int kBlock = kFormat == CUGL_NVFP4 ? 16 : 32;
    float         h[4];
    uint32_t      amax[4], w[4];
    MxScale       s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const float x = g[i] * p.gate_alpha;
        const float v = weight[t[i]] * __fdividef(x, 1.f + expf(-x)) * (u[i] * p.up_alpha); // SwiGLU, the gate's weight folded in
        h[i]          = f < p.inner ? v : 0.f;
        amax[i]       = __float_as_uint(h[i]) & 0x7fffffffu;
    }
    if (kFormat == CUGL_MXFP4)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) amax[i] = __reduce_max_sync(0xffffffffu, amax[i]);
    }
    else
    {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
        {
#pragma unroll
            for (int i = 0; i < 4; ++i) amax[i] = max(amax[i], __shfl_xor_sync(0xffffffffu, amax[i], o));
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        s[i] = mx_scale_of<kFormat, false, false>(amax[i], p.h_mul); // h carries the error of float sums: no exact quotients
        w[i] = (static_cast<uint32_t>(__nv_cvt_float_to_fp4(h[i] * s[i].mul, __NV_E2M1, cudaRoundNearest)) & 15u) << (4 * (lane & 7));
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] |= __shfl_xor_sync(0xffffffffu, w[i], o);
    }
    uint8_t *codes  = p.hq + static_cast<int64_t>(a) * p.tokens * p.ld_hq + f / 2;
    uint8_t *scales = p.hs + static_cast<int64_t>(a) * p.f_tiles * kMxTileBytes;
    const bool code_lane = (lane & 7) == 0 && f < p.inner, scale_lane = (lane & (kBlock - 1)) == 0 && f / kBlock < p.f_tiles * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        if ((valid >> i) & 1u)
        {
            if (code_lane) *reinterpret_cast<uint32_t *>(codes + t[i] * p.ld_hq) = w[i];
            if (scale_lane) scales[mx_scale_offset(t[i], f / kBlock, p.f_tiles)] = static_cast<uint8_t>(s[i].byte);
        }
    }
    __syncwarp(); // aligned loads of tensor memory may be next
}

// kOperands: weight matrices that share a stage's tokens (2: gate and up, 1: down).  Up to 64 tokens two CTAs share an SM.
template <int kFormat, int NT, int STAGES, int kOperands, bool kSplit, int kAcc>
struct MoePlan
{
    using F                         = MxTraits<kFormat>;
    static constexpr int T_BYTES    = NT * kMxChunkBytes;
    static constexpr int STAGE      = kOperands * kMxWBytes + T_BYTES;
    static constexpr int SF_STAGE   = (kOperands + 1) * F::kChunkScale;
    static constexpr int OFF_SF     = STAGES * STAGE;
    // the partial sums of a cluster: an area of their own where there is room, else where the stages were
    static constexpr int  PART      = kOperands * NT * kMxRows * 4;
    static constexpr bool OWN_PART  = PART <= 16384;
    [[maybe_unused]] static constexpr int OFF_PART   = OWN_PART ? OFF_SF + STAGES * SF_STAGE : 0;
    static constexpr int OFF_BAR    = OFF_SF + STAGES * SF_STAGE + (kSplit && OWN_PART ? PART : 0);
    static constexpr int OFF_MISC   = OFF_BAR + (2 * STAGES + 6) * 8;
    static constexpr int OFF_BITS   = OFF_MISC + 16;
    static constexpr int OFF_LIST   = OFF_BITS + kMaxExperts / 8;
    static constexpr int OFF_WEIGHT = OFF_LIST + kMaxExperts * 2;
    static constexpr int DYN_BYTES  = OFF_WEIGHT + (kOperands == 2 ? 2 * kMaxTokens * 4 : 0) + 1024; // two tables
    static constexpr int ACC_COLS   = kOperands * NT;
    static constexpr int SF_COLS    = (kOperands + 1) * F::kChunkCols;
    static constexpr int COLS       = kAcc * ACC_COLS + STAGES * SF_COLS;
    static constexpr int TMEM_COLS  = COLS <= 32 ? 32 : COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    static constexpr int PER_SM     = TMEM_COLS <= 256 && DYN_BYTES <= 115200 ? 2 : 1;
    static_assert(COLS <= 512 && DYN_BYTES <= 232448, "tensor and shared memory of an SM");
    static_assert(STAGES * STAGE >= PART, "the partial sums of a cluster fit where the stages were");
};

// ---- second launch -------------------------------------------------------------------------------------------
// Unit of work: 128 rows of one active expert's gate and up matrices, over all tokens.  kSplit: the CTAs of a cluster share a
// unit's K (few units); else a CTA works through its units, the stages of the next one arriving during the epilogue.
template <int kFormat, int NT, int STAGES, bool kSplit, int kAcc>
__global__ void __launch_bounds__(kUpThreads, MoePlan<kFormat, NT, STAGES, 2, kSplit, kAcc>::PER_SM)
    moe_gate_up_kernel(const __grid_constant__ CUtensorMap tmap_g, const __grid_constant__ CUtensorMap tmap_u, const __grid_constant__ CUtensorMap tmap_x,
                       const __grid_constant__ MoeParams p)
{
    using P = MoePlan<kFormat, NT, STAGES, 2, kSplit, kAcc>;
    using F = MxTraits<kFormat>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t       *smem       = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t s_stage    = smem_u32(smem);
    const uint32_t s_sf       = smem_u32(smem + P::OFF_SF);
    const uint32_t bar_base   = smem_u32(smem + P::OFF_BAR);
    auto           full_bar   = [&](int s) { return bar_base + 8u * s; };
    auto           empty_bar  = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto           tfull_bar  = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
    auto           tempty_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + 2 + a); };
    const uint32_t part_bar   = bar_base + 8u * (2 * STAGES + 4);
    const uint32_t gone_bar   = bar_base + 8u * (2 * STAGES + 5); // see drain_mmas
    uint32_t      *s_tmem     = reinterpret_cast<uint32_t *>(smem + P::OFF_MISC);
    volatile int  *s_abort    = reinterpret_cast<volatile int *>(smem + P::OFF_MISC + 4);
    uint32_t      *s_bits     = reinterpret_cast<uint32_t *>(smem + P::OFF_BITS);
    uint16_t      *s_list     = reinterpret_cast<uint16_t *>(smem + P::OFF_LIST);
    float         *s_weight   = reinterpret_cast<float *>(smem + P::OFF_WEIGHT);
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int      rank  = kSplit ? static_cast<int>(cluster_ctarank()) : 0;
    const int      ranks = kSplit ? static_cast<int>(gridDim.x) / static_cast<int>(num_clusters_x()) : 1;

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
            mbar_init(tempty_bar(a), kUpEpi);
        }
        mbar_init(part_bar, partial_arrivals(31 - __clz(ranks), kUpEpi));
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
    griddep_wait(); // the prologue above touched no global memory
    griddep_launch_dependents();

    const int active      = active_experts<false>(p, s_list, s_bits);
    const int blocks      = (p.inner + kMxRows - 1) / kMxRows;
    const int units       = active * blocks;
    const int chunks      = (p.hidden + kMxChunk - 1) / kMxChunk;
    const int first_unit  = kSplit ? static_cast<int>(cluster_id_x()) : static_cast<int>(blockIdx.x);
    const int unit_stride = kSplit ? max(units, 1) : static_cast<int>(gridDim.x);
    const int c_begin     = chunk_share(chunks, rank, ranks);
    const int c_end       = chunk_share(chunks, rank + 1, ranks);
    int       issued      = 0; // stages that the producer has filled

    if (warp == 0)
    {
        const bool el = elect_one();
        const int  withheld = blockIdx.x == 0 ? p.withhold_up : -1;
        int        g = 0;
        for (int unit = first_unit; unit < units; unit += unit_stride)
        {
            const int      e = s_list[unit / blocks], fb = unit % blocks;
            const int64_t  sf_at = (static_cast<int64_t>(e) * blocks + fb) * p.h_tiles * kMxTileBytes;
            const int      row = e * p.inner + fb * kMxRows;
            for (int c = c_begin; c < c_end; ++c, ++g)
            {
                const int s = g % STAGES;
                if (!warp_wait(empty_bar(s), (static_cast<uint32_t>(g / STAGES) & 1u) ^ 1u, s_abort, DEV_TIMEOUT_PRODUCER, p.spin_limit))
                {
                    goto produced;
                }
                const int      first = c * F::kChunkTiles;
                const int      n     = min(F::kChunkTiles, static_cast<int>(p.h_tiles) - first);
                const uint32_t bytes = static_cast<uint32_t>(n) * kMxTileBytes;
                const int64_t  at    = static_cast<int64_t>(first) * kMxTileBytes;
                const uint32_t dst   = s_stage + s * P::STAGE, sf = s_sf + s * P::SF_STAGE;
                if (el && g != withheld)
                {
                    mbar_expect_tx(full_bar(s), P::STAGE + 3 * bytes);
                    tma_load_2d(dst, &tmap_g, c * kMxChunkBytes, row, full_bar(s));
                    tma_load_2d(dst + kMxWBytes, &tmap_u, c * kMxChunkBytes, row, full_bar(s));
                    tma_load_2d(dst + 2 * kMxWBytes, &tmap_x, c * kMxChunkBytes, 0, full_bar(s));
                    bulk_load(sf, p.gate_scales + sf_at + at, bytes, full_bar(s));
                    bulk_load(sf + F::kChunkScale, p.up_scales + sf_at + at, bytes, full_bar(s));
                    bulk_load(sf + 2 * F::kChunkScale, p.xs + at, bytes, full_bar(s));
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
        for (int unit = first_unit; unit < units && ok; unit += unit_stride, ++it)
        {
            const int as = it % kAcc;
            ok = warp_wait(tempty_bar(as), (static_cast<uint32_t>(it / kAcc) & 1u) ^ 1u, s_abort, DEV_TIMEOUT_MMA, p.spin_limit);
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + as * P::ACC_COLS;
            for (int c = c_begin; c < c_end && ok; ++c, ++g)
            {
                const int s = g % STAGES;
                ok = warp_wait(full_bar(s), static_cast<uint32_t>(g / STAGES) & 1u, s_abort, DEV_TIMEOUT_MMA, p.spin_limit);
                if (!ok) break;
                tc_fence_after();
                const int      n     = min(F::kChunkTiles, static_cast<int>(p.h_tiles) - c * F::kChunkTiles);
                const int      steps = min(kMxChunk / kMxStepK, (p.hidden - c * kMxChunk + kMxStepK - 1) / kMxStepK);
                const uint32_t t_g   = tmem_base + kAcc * P::ACC_COLS + s * P::SF_COLS, t_u = t_g + F::kChunkCols, t_x = t_u + F::kChunkCols;
                const uint32_t sf = s_sf + s * P::SF_STAGE, st = s_stage + s * P::STAGE;
                if (el)
                {
                    mx_chunk_scales<kFormat>(t_x, sf + 2 * F::kChunkScale, n);
                    mx_chunk_scales<kFormat>(t_g, sf, n);
                    mx_chunk_scales<kFormat>(t_u, sf + F::kChunkScale, n);
                    mx_chunk<kFormat>(d_tmem, st, st + 2 * kMxWBytes, t_g, t_x, p.idesc, steps, c == c_begin);
                    mx_chunk<kFormat>(d_tmem + NT, st + kMxWBytes, st + 2 * kMxWBytes, t_u, t_x, p.idesc, steps, c == c_begin);
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
        bool      ok = true;
        for (int unit = first_unit; unit < units; unit += unit_stride, ++it)
        {
            const int a = unit / blocks, f0 = (unit % blocks) * kMxRows, f = f0 + q * 32 + lane;
            const int as = it % kAcc;
            float    *weight = s_weight + (it & 1) * kMaxTokens; // the other table may still be read by a slower warp
            if (!begin_unit<kFormat>(p, weight, a, s_list[a], f0, ok)) break;
            ok = warp_wait(tfull_bar(as), static_cast<uint32_t>(it / kAcc) & 1u, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit);
            if (!ok) continue; // the next barrier ends it for all eight warps
            tc_fence_after();
            // The tokens that chose the expert, four at a time; the two warps of a lane quarter take turns.  (Four neighbours of which
            // one or more chose it: 128 tokens 65 us instead of 56.)
            const uint32_t acc  = tmem_base + as * P::ACC_COLS + (static_cast<uint32_t>(q * 32) << 16);
            int            turn = 0;
            for (int w = 0; w < p.tokens; w += 32)
            {
                uint32_t left = __ballot_sync(0xffffffffu, w + lane < p.tokens && weight[min(w + lane, kMaxTokens - 1)] != kNotChosen);
                for (; left != 0; ++turn)
                {
                    int      t[4];
                    uint32_t valid = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                    {
                        t[i] = left != 0 ? w + __ffs(left) - 1 : t[0];
                        valid |= left != 0 ? 1u << i : 0u;
                        left &= left - 1;
                    }
                    if ((turn & 1) != half) continue;
                    uint32_t g[4], u[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                    {
                        tmem_ld_x1(acc + t[i], g[i]);
                        tmem_ld_x1(acc + NT + t[i], u[i]);
                    }
                    tmem_ld_wait();
                    const float g4[4] = {__uint_as_float(g[0]), __uint_as_float(g[1]), __uint_as_float(g[2]), __uint_as_float(g[3])};
                    const float u4[4] = {__uint_as_float(u[0]), __uint_as_float(u[1]), __uint_as_float(u[2]), __uint_as_float(u[3])};
                    store_hidden<kFormat>(p, a, t, f, lane, g4, u4, weight, valid);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty_bar(as));
        }
    }

    if constexpr (kSplit)
    {
        const bool work = first_unit < units; // the same in the whole cluster
        const int  q = warp & 3, half = (warp - kFirstEpi) >> 2, shift = 31 - __clz(ranks);
        const int  a = work ? first_unit / blocks : 0;
        bool       ok = work;
        if (warp >= kFirstEpi && work)
        {
            (void)begin_unit<kFormat>(p, s_weight, a, s_list[a], first_unit % blocks * kMxRows, true);
            ok = warp_wait(tfull_bar(0), 0, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit);
            tc_fence_after();
        }
        if (!P::OWN_PART)
        {
            __syncthreads();
            cluster_sync(); // every CTA's MMAs have read their last stage
        }
        if (warp >= kFirstEpi && ok)
        {
            const int      ch = q * 32 + lane;
            const uint32_t to = partial_address(smem_u32(smem + P::OFF_PART), ch, rank, shift, 2 * NT);
            for (int j = 16 * half; j < p.tokens; j += 4 * kUpEpi)
            {
                uint32_t g[16], u[16];
                tmem_ld_x16(tmem_base + j + (static_cast<uint32_t>(q * 32) << 16), g);
                tmem_ld_x16(tmem_base + NT + j + (static_cast<uint32_t>(q * 32) << 16), u);
                tmem_ld_wait();
                send_partial(to + static_cast<uint32_t>(j) * (4u * kMxRows >> shift), shift, g, p.tokens - j, c_begin < c_end);
                send_partial(to + static_cast<uint32_t>(NT + j) * (4u * kMxRows >> shift), shift, u, p.tokens - j, c_begin < c_end);
            }
            arrive_partial(part_bar, ch, shift);
            ok = __all_sync(0xffffffffu, mbar_wait_cluster(part_bar, 0, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit));
        }
        if (warp >= kFirstEpi && ok)
        {
            // a warp takes 32 consecutive channels of four tokens at a time: a rank owns at least 32 (launch_layers)
            const int    own = kMxRows >> shift;
            const float *part = reinterpret_cast<const float *>(smem + P::OFF_PART);
            for (int at = (warp - kFirstEpi) * 32 + lane; at - lane < (p.tokens + 3) / 4 * own; at += 32 * kUpEpi)
            {
                const int    t0 = (at >> (7 - shift)) * 4, f = (first_unit % blocks) * kMxRows + rank * own + (at & (own - 1));
                const uint32_t chosen = __ballot_sync(0xffffffffu, lane < 4 && t0 + lane < p.tokens && s_weight[t0 + lane] != kNotChosen);
                if (chosen != 0)
                {
                    const float4 g4 = sum_partial(part, at, shift, 2 * NT), u4 = sum_partial(part + NT * own, at, shift, 2 * NT);
                    const float  g[4] = {g4.x, g4.y, g4.z, g4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w};
                    const int    t[4] = {t0, t0 + 1, t0 + 2, t0 + 3};
                    store_hidden<kFormat>(p, a, t, f, lane, g, u, s_weight, chosen);
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 0 && *s_abort != 0)
    {
        drain_stages<STAGES>(bar_base, issued, blockIdx.x == 0 ? p.withhold_up : -1, p.spin_limit);
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

// ---- third launch --------------------------------------------------------------------------------------------
// Unit of work: 128 output channels; K is (active expert, intermediate), shared by the CTAs of a cluster.
template <int kFormat, int NT, int STAGES>
__global__ void __launch_bounds__(kDownThreads, 2)
    moe_down_kernel(const __grid_constant__ CUtensorMap tmap_d, const __grid_constant__ CUtensorMap tmap_h, const __grid_constant__ MoeParams p)
{
    using P = MoePlan<kFormat, NT, STAGES, 1, true, 1>;
    static_assert(P::PER_SM == 2, "two CTAs share an SM");
    using F = MxTraits<kFormat>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t       *smem      = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t s_stage   = smem_u32(smem);
    const uint32_t s_sf      = smem_u32(smem + P::OFF_SF);
    const uint32_t bar_base  = smem_u32(smem + P::OFF_BAR);
    auto           full_bar  = [&](int s) { return bar_base + 8u * s; };
    auto           empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    const uint32_t tfull     = bar_base + 8u * (2 * STAGES), part_bar = bar_base + 8u * (2 * STAGES + 4);
    const uint32_t gone_bar  = bar_base + 8u * (2 * STAGES + 5); // see drain_mmas
    uint32_t      *s_tmem    = reinterpret_cast<uint32_t *>(smem + P::OFF_MISC);
    volatile int  *s_abort   = reinterpret_cast<volatile int *>(smem + P::OFF_MISC + 4);
    uint32_t      *s_bits    = reinterpret_cast<uint32_t *>(smem + P::OFF_BITS);
    uint16_t      *s_list    = reinterpret_cast<uint16_t *>(smem + P::OFF_LIST);
    const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int      rank  = static_cast<int>(cluster_ctarank());
    const int      ranks = static_cast<int>(gridDim.x) / static_cast<int>(num_clusters_x());

    if (threadIdx.x == 0)
    {
        for (int s = 0; s < STAGES; ++s)
        {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(tfull, 1);
        mbar_init(part_bar, partial_arrivals(31 - __clz(ranks), kDownEpi));
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
    cluster_sync(); // every CTA runs and has its barriers before anything is sent to it
    tc_fence_after();
    const uint32_t tmem_base = *s_tmem;
    griddep_launch_dependents();

    // before the wait for the second launch: what the first one wrote, and the weights
    const int active     = active_experts<true>(p, s_list, s_bits);
    const int per_expert = (p.inner + kMxChunk - 1) / kMxChunk;
    const int chunks     = active * per_expert;
    const int blocks     = (p.hidden + kMxRows - 1) / kMxRows;
    const int block      = static_cast<int>(cluster_id_x());
    const int c_begin    = chunk_share(chunks, rank, ranks);
    const int c_end      = chunk_share(chunks, rank + 1, ranks);
    int       issued     = 0; // stages that the producer has filled

    if (warp == 0)
    {
        const bool el = elect_one();
        const int  withheld = blockIdx.x == 0 ? p.withhold_down : -1;
        auto load_weights = [&](int g) {
            const int      i = c_begin + g, s = g % STAGES, a = i / per_expert, c = i - a * per_expert, e = s_list[a], first = c * F::kChunkTiles;
            const uint32_t bytes = static_cast<uint32_t>(min(F::kChunkTiles, static_cast<int>(p.f_tiles) - first)) * kMxTileBytes;
            if (el && g != withheld)
            {
                mbar_expect_tx(full_bar(s), P::STAGE + 2 * bytes);
                tma_load_2d(s_stage + s * P::STAGE, &tmap_d, c * kMxChunkBytes, e * p.hidden + block * kMxRows, full_bar(s));
                bulk_load(s_sf + s * P::SF_STAGE, p.down_scales + ((static_cast<int64_t>(e) * blocks + block) * p.f_tiles + first) * kMxTileBytes, bytes,
                          full_bar(s));
            }
            __syncwarp();
        };
        auto load_tokens = [&](int g) {
            const int      i = c_begin + g, s = g % STAGES, a = i / per_expert, c = i - a * per_expert, first = c * F::kChunkTiles;
            const uint32_t bytes = static_cast<uint32_t>(min(F::kChunkTiles, static_cast<int>(p.f_tiles) - first)) * kMxTileBytes;
            if (el && g != withheld)
            {
                tma_load_2d(s_stage + s * P::STAGE + kMxWBytes, &tmap_h, c * kMxChunkBytes, a * p.tokens, full_bar(s));
                bulk_load(s_sf + s * P::SF_STAGE + F::kChunkScale, p.hs + (static_cast<int64_t>(a) * p.f_tiles + first) * kMxTileBytes, bytes, full_bar(s));
            }
            __syncwarp();
        };
        const int mine = c_end - c_begin, early = min(mine, STAGES);
        int       g = 0;
        for (; g < early; ++g) load_weights(g);
        griddep_wait();
        for (int i = 0; i < early; ++i) load_tokens(i);
        for (; g < mine; ++g)
        {
            const int s = g % STAGES;
            if (!warp_wait(empty_bar(s), (static_cast<uint32_t>(g / STAGES) & 1u) ^ 1u, s_abort, DEV_TIMEOUT_PRODUCER, p.spin_limit))
            {
                break;
            }
            load_weights(g);
            load_tokens(g);
        }
        issued = g;
    }
    else if (warp == kMmaWarp)
    {
        griddep_wait(); // the tokens' half of a stage comes after the second launch, whose time is not to count in this one's waits
        const bool el = elect_one();
        int  g  = 0;
        bool ok = true;
        for (int i = c_begin; i < c_end && ok; ++i, ++g)
        {
            const int s = g % STAGES;
            ok = warp_wait(full_bar(s), static_cast<uint32_t>(g / STAGES) & 1u, s_abort, DEV_TIMEOUT_MMA, p.spin_limit);
            if (!ok) break;
            tc_fence_after();
            const int      c     = i % per_expert;
            const int      n     = min(F::kChunkTiles, static_cast<int>(p.f_tiles) - c * F::kChunkTiles);
            const int      steps = min(kMxChunk / kMxStepK, (p.inner - c * kMxChunk + kMxStepK - 1) / kMxStepK);
            const uint32_t t_w   = tmem_base + NT + s * P::SF_COLS, t_t = t_w + F::kChunkCols;
            const uint32_t sf    = s_sf + s * P::SF_STAGE, st = s_stage + s * P::STAGE;
            if (el)
            {
                mx_chunk_scales<kFormat>(t_w, sf, n);
                mx_chunk_scales<kFormat>(t_t, sf + F::kChunkScale, n);
                mx_chunk<kFormat>(tmem_base, st, st + kMxWBytes, t_w, t_t, p.idesc, steps, i == c_begin);
                umma_commit(empty_bar(s));
            }
            __syncwarp();
        }
        if (ok && el)
        {
            umma_commit(tfull);
        }
        __syncwarp();
    }

    const int q = warp & 3, shift = 31 - __clz(ranks);
    bool      ok = true;
    if (warp >= kFirstEpi)
    {
        griddep_wait(); // nothing is written before the launches ahead have completed
        ok = warp_wait(tfull, 0, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit);
        tc_fence_after();
    }
    if (!P::OWN_PART)
    {
        __syncthreads();
        cluster_sync(); // every CTA's MMAs have read their last stage
    }
    if (warp >= kFirstEpi && ok)
    {
        const int      ch = q * 32 + lane;
        const uint32_t to = partial_address(smem_u32(smem + P::OFF_PART), ch, rank, shift, NT);
        for (int j = 0; j < p.tokens; j += 16)
        {
            uint32_t r[16];
            tmem_ld_x16(tmem_base + j + (static_cast<uint32_t>(q * 32) << 16), r);
            tmem_ld_wait();
            send_partial(to + static_cast<uint32_t>(j) * (4u * kMxRows >> shift), shift, r, p.tokens - j, c_begin < c_end);
        }
        arrive_partial(part_bar, ch, shift);
        ok = __all_sync(0xffffffffu, mbar_wait_cluster(part_bar, 0, s_abort, DEV_TIMEOUT_EPILOGUE, p.spin_limit));
    }
    if (warp >= kFirstEpi && ok)
    {
        const int    own = kMxRows >> shift, et = threadIdx.x - 32 * kFirstEpi;
        const int    n = block * kMxRows + rank * own + (et & (own - 1));
        const float *part = reinterpret_cast<const float *>(smem + P::OFF_PART);
        if (n < p.hidden)
        {
            for (int at = et; at < (p.tokens + 3) / 4 * own; at += 32 * kDownEpi)
            {
                const int    j  = (at >> (7 - shift)) * 4;
                const float4 v4 = sum_partial(part, at, shift, NT);
                const float  v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
                    if (j + i < p.tokens)
                    {
                        uint8_t *dst = p.dst + static_cast<int64_t>(j + i) * p.ld_dst;
                        if (p.dtype == CUGL_F16) reinterpret_cast<__half *>(dst)[n] = from_float<__half>(v[i] * p.down_alpha);
                        else reinterpret_cast<__nv_bfloat16 *>(dst)[n] = from_float<__nv_bfloat16>(v[i] * p.down_alpha);
                    }
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 0 && *s_abort != 0)
    {
        drain_stages<STAGES>(bar_base, issued, blockIdx.x == 0 ? p.withhold_down : -1, p.spin_limit);
    }
    if (warp == kMmaWarp)
    {
        if (*s_abort != 0) drain_mmas<false>(gone_bar, p.spin_limit);
        tc_fence_after();
        tmem_dealloc(tmem_base, P::TMEM_COLS);
    }
    if (*s_abort != 0)
    {
        cluster_sync(); // this CTA may not have received all parts: it stays until the others have left or given up too
    }
    if (threadIdx.x == 0 && *s_abort != 0)
    {
        atomicCAS(p.status, 0, *s_abort);
    }
}

// ---- host ----------------------------------------------------------------------------------------------------
struct MoeBuffers // offsets into the workspace
{
    size_t  ids, p, xq, xs, hq, hs, total;
    int64_t ld_xq, ld_hq;
    int     most_active;
};
MoeBuffers moe_buffers(const cugl_mx_moe_desc &d)
{
    MoeBuffers b{};
    size_t     at  = 0;
    auto       add = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const int64_t pairs = static_cast<int64_t>(d.tokens) * d.top_k;
    b.most_active = static_cast<int>(pairs < d.experts ? pairs : d.experts);
    b.ld_xq       = (static_cast<int64_t>(d.hidden) + 31) / 32 * 16;
    b.ld_hq       = (static_cast<int64_t>(d.intermediate) + 31) / 32 * 16;
    b.ids         = add(static_cast<size_t>(pairs) * 4);
    b.p           = add(static_cast<size_t>(pairs) * 4);
    b.xq          = add(static_cast<size_t>(d.tokens) * b.ld_xq);
    b.xs          = add(static_cast<size_t>(mx_scale_tiles(d.hidden, d.format)) * kMxTileBytes);
    b.hq          = add(static_cast<size_t>(b.most_active) * d.tokens * b.ld_hq);
    b.hs          = add(static_cast<size_t>(b.most_active) * mx_scale_tiles(d.intermediate, d.format) * kMxTileBytes);
    b.total       = at;
    return b;
}

const char *validate_moe(const cugl_mx_moe_desc *d)
{
    if (d == nullptr) return "descriptor is NULL";
    if (d->tokens < 0 || d->tokens > kMaxTokens) return "tokens must lie within 0 .. 128";
    if (d->hidden < 16 || d->intermediate < 16 || d->hidden % 16 != 0 || d->intermediate % 16 != 0 || d->hidden > (1 << 20) || d->intermediate > (1 << 20))
        return "hidden and intermediate must be multiples of 16 up to 2^20";
    if (d->experts < 1 || d->experts > kMaxExperts) return "experts must lie within 1 .. 512";
    if (d->top_k < 1 || d->top_k > kMaxTopK || d->top_k > d->experts) return "top_k must lie within 1 .. 16 and not exceed experts";
    if (static_cast<int64_t>(d->experts) * (d->hidden > d->intermediate ? d->hidden : d->intermediate) > INT32_MAX - 1024) return "too many weight rows";
    if (d->format != CUGL_MXFP4 && d->format != CUGL_NVFP4) return "format must be CUGL_MXFP4 or CUGL_NVFP4";
    if (d->dtype != CUGL_F16 && d->dtype != CUGL_BF16) return "dtype must be CUGL_F16 or CUGL_BF16";
    if (d->ld_x < 2ll * d->hidden || d->ld_dst < 2ll * d->hidden || d->ld_x % 2 != 0 || d->ld_dst % 2 != 0) return "ld_x and ld_dst must hold a row and be even";
    if (d->ld_logits < 4ll * d->experts || d->ld_logits % 4 != 0) return "ld_logits must hold a row and be a multiple of 4";
    if (d->ld_gate_up < d->hidden / 2 || d->ld_down < d->intermediate / 2 || d->ld_gate_up % 16 != 0 || d->ld_down % 16 != 0 ||
        d->ld_gate_up >= (1ll << 40) || d->ld_down >= (1ll << 40))
        return "ld_gate_up and ld_down must hold a packed row and be multiples of 16 below 2^40";
    if (d->format == CUGL_MXFP4 && (d->x_exponent != 0 || d->h_exponent != 0)) return "x_exponent and h_exponent are for CUGL_NVFP4";
    if (d->x_exponent < -64 || d->x_exponent > 64 || d->h_exponent < -64 || d->h_exponent > 64) return "x_exponent and h_exponent must lie within -64 .. 64";
    for (const float v : {std::ldexp(d->gate_alpha, d->x_exponent), std::ldexp(d->up_alpha, d->x_exponent), std::ldexp(d->down_alpha, d->h_exponent)})
    {
        if (!(v - v == 0.f)) return "an alpha times 2 to its operand's exponent must be finite";
    }
    return nullptr;
}

struct MoeMaps
{
    CUtensorMap gate, up, x, down, h;
};

template <int kFormat, int NT, int STAGES, bool kSplit, int kAcc>
cugl_status launch_gate_up(cugl_context *ctx, const MoeMaps &m, const MoeParams &p, int most_units, int ranks)
{
    using P     = MoePlan<kFormat, NT, STAGES, 2, kSplit, kAcc>;
    auto kernel = moe_gate_up_kernel<kFormat, NT, STAGES, kSplit, kAcc>;
    static std::atomic<bool> set[64] = {};
    CUGL_TRY(allow_smem(ctx, kernel, P::DYN_BYTES, set));
    const int slots = P::PER_SM * ctx->sm_count;
    const int grid  = kSplit ? most_units * ranks : (most_units < slots ? most_units : slots);
    CUGL_CUDA_TRY(ctx, launch_dependent_cluster(ctx, kernel, dim3(static_cast<unsigned>(grid)), kUpThreads, P::DYN_BYTES, kSplit ? ranks : 1, most_units,
                                                m.gate, m.up, m.x, p));
    return CUGL_SUCCESS;
}

template <int kFormat, int NT, int kUpStages, int kUpAcc, int kDownStages>
cugl_status launch_layers(cugl_context *ctx, const MoeMaps &m, const MoeParams &p, int most_active)
{
    const int most_units = most_active * ((p.inner + kMxRows - 1) / kMxRows);
    const int chunks     = (p.hidden + kMxChunk - 1) / kMxChunk;
    // at most four: a rank then owns 32 channels of a unit, one MXFP4 block; and only where two CTAs share an SM (mx_split)
    int ranks = NT <= 64 ? mx_split(most_units, chunks, 4) : 1;
    // Up to eight tokens and twelve chunks: one CTA per SM instead of two.  us with 2 / 4 CTAs per unit, 48 units: hidden 1536, 1 token NVFP4
    // 13.2 / 14.3, 2048 14.1 / 15.1 and MXFP4 13.3 / 14.5, 2560 14.7 / 15.5, 13.7 / 14.9, 2880 15.1 / 16.0, 14.7 / 15.4, 3584 16.1 / 16.5 (8 tokens
    // 16.9 / 16.5), 4096 17.5 / 16.9, 16.4 / 16.1, 6144 20.5 / 19.1, 8192 26.2 / 22.6; 16 tokens, hidden 2048, 16.3 / 15.9.
    if (ranks == 4 && most_units * 4 > ctx->sm_count && chunks <= 12 && p.tokens <= 8) ranks = 2;
    if constexpr (NT <= 64)
    {
        if (ranks > 1) CUGL_TRY((launch_gate_up<kFormat, NT, kUpStages, true, 1>(ctx, m, p, most_units, ranks)));
    }
    if (ranks == 1)
    {
        CUGL_TRY((launch_gate_up<kFormat, NT, kUpStages, false, kUpAcc>(ctx, m, p, most_units, 1)));
    }
    using P     = MoePlan<kFormat, NT, kDownStages, 1, true, 1>;
    auto kernel = moe_down_kernel<kFormat, NT, kDownStages>;
    static std::atomic<bool> set[64] = {};
    CUGL_TRY(allow_smem(ctx, kernel, P::DYN_BYTES, set));
    const int blocks = (p.hidden + kMxRows - 1) / kMxRows, most_chunks = most_active * ((p.inner + kMxChunk - 1) / kMxChunk);
    ranks = mx_split(blocks, most_chunks, 8);
    // One CTA per SM instead of two where that leaves no more than a quarter of them idle: fewer parts to exchange, and room beside
    // the second launch.  Few chunks per CTA gain by it, 1 token, hidden 4096, intermediate 2048, top 2, NVFP4 (16 chunks) 15.9 -> 14.5
    // us, intermediate 1536, top 8 (48) 23.7 -> 22.9; many lose, 48 tokens, intermediate 768, 64 experts (192) 71 -> 76; but the parts
    // of 128 columns are the greater cost: 100 tokens, intermediate 512, 4 experts 34 -> 28, 128 tokens, 1536, 64 experts 158 -> 148.
    // Half the SMs idle: 128 tokens, hidden 2560 (20 blocks) 41.7 -> 46;
    // two parts of 128 columns instead of four, hidden 8192: 43.7 -> 46.3 (1 token, 8 chunks: 16.0 -> 15.3).
    // Ten layers (hidden 1024 .. 8192, 4 .. 64 experts) with 1, 8, 48, 100 and 128 tokens in both formats: within 5 % of the best of 2, 4 and 8
    // parts, but for MXFP4, hidden 4096, intermediate 1536, 64 experts and 48 tokens (eight 130, four 119).
    while (ranks > 2 && blocks * ranks > ctx->sm_count && blocks * ranks / 2 >= ctx->sm_count * 3 / 4 &&
           (NT == 128 ? ranks == 8 : most_chunks <= 6 * ranks))
    {
        ranks /= 2;
    }
    CUGL_CUDA_TRY(ctx, launch_dependent_cluster(ctx, kernel, dim3(static_cast<unsigned>(blocks * ranks)), kDownThreads, P::DYN_BYTES, ranks, blocks * ranks,
                                                m.down, m.h, p));
    return CUGL_SUCCESS;
}

template <int kFormat>
cugl_status launch_moe(cugl_context *ctx, const MoeMaps &m, MoeParams p, int nt, int most_active)
{
    const int blocks = p.route_blocks + p.quant_x * ((p.tokens + 7) / 8);
    if (p.dtype == CUGL_F16)
    {
        CUGL_CUDA_TRY(ctx, launch_dependent(ctx, moe_route_kernel<__half, kFormat>, dim3(static_cast<unsigned>(blocks)), 256, 0, blocks, p));
    }
    else
    {
        CUGL_CUDA_TRY(ctx, launch_dependent(ctx, moe_route_kernel<__nv_bfloat16, kFormat>, dim3(static_cast<unsigned>(blocks)), 256, 0, blocks, p));
    }
    p.idesc = mx_idesc(kFormat, kMxRows, nt);
    switch (nt)
    {
        case 16: return launch_layers<kFormat, 16, 2, 2, 4>(ctx, m, p, most_active);
        case 32: return launch_layers<kFormat, 32, 2, 2, kFormat == CUGL_MXFP4 ? 4 : 3>(ctx, m, p, most_active);
        case 64: return launch_layers<kFormat, 64, 2, 1, kFormat == CUGL_MXFP4 ? 4 : 3>(ctx, m, p, most_active);
        default: return launch_layers<kFormat, 128, 4, 1, 3>(ctx, m, p, most_active);
    }
}
} // namespace
} // namespace cugl

using namespace cugl;

extern "C"
{
    cugl_status cugl_mx_moe_validate(const cugl_mx_moe_desc *desc, const char **reason)
    {
        const char *why = validate_moe(desc);
        if (reason != nullptr)
        {
            *reason = why != nullptr ? why : "";
        }
        return why == nullptr ? CUGL_SUCCESS : CUGL_INVALID_ARGUMENT;
    }

    size_t cugl_mx_moe_workspace_bytes(const cugl_mx_moe_desc *desc)
    {
        return validate_moe(desc) == nullptr ? moe_buffers(*desc).total : 0;
    }

    cugl_status cugl_mx_moe(cugl_context *ctx, const cugl_mx_moe_desc *desc, const void *d_x, const float *d_logits, const void *d_gate,
                            const void *d_gate_scales, const void *d_up, const void *d_up_scales, const void *d_down, const void *d_down_scales,
                            void *d_dst, void *d_workspace, size_t workspace_bytes)
    {
        if (ctx == nullptr)
        {
            return fail(nullptr, CUGL_INVALID_ARGUMENT, "context is NULL");
        }
        const char *why = validate_moe(desc);
        MoeBuffers  b{};
        if (why == nullptr && desc->tokens > 0)
        {
            b                    = moe_buffers(*desc);
            const void *const in[] = {d_gate, d_gate_scales, d_up, d_up_scales, d_down, d_down_scales};
            uintptr_t         bits = 0;
            bool              null = d_x == nullptr || d_logits == nullptr || d_dst == nullptr || d_workspace == nullptr;
            for (const void *q : in)
            {
                bits |= reinterpret_cast<uintptr_t>(q);
                null |= q == nullptr;
            }
            if (null) why = "NULL pointer";
            else if ((bits & 15) != 0) why = "weights and scale tiles must be 16-byte aligned";
            else if (((reinterpret_cast<uintptr_t>(d_x) | reinterpret_cast<uintptr_t>(d_dst)) & 1) != 0 || (reinterpret_cast<uintptr_t>(d_logits) & 3) != 0)
                why = "x, logits or dst is not aligned to its elements";
            else if ((reinterpret_cast<uintptr_t>(d_workspace) & 255) != 0) why = "the workspace must be 256-byte aligned";
            else if (workspace_bytes < b.total) why = "the workspace is too small (cugl_mx_moe_workspace_bytes)";
        }
        if (why != nullptr)
        {
            return fail(ctx, CUGL_INVALID_ARGUMENT, std::string("cugl_mx_moe: ") + why);
        }
        if (desc->tokens == 0) return CUGL_SUCCESS;
        const DeviceScope device(ctx);
        uint8_t          *ws = static_cast<uint8_t *>(d_workspace);
        MoeParams         p{};
        p.x            = static_cast<const uint8_t *>(d_x);
        p.logits       = d_logits;
        p.gate_scales  = static_cast<const uint8_t *>(d_gate_scales);
        p.up_scales    = static_cast<const uint8_t *>(d_up_scales);
        p.down_scales  = static_cast<const uint8_t *>(d_down_scales);
        p.dst          = static_cast<uint8_t *>(d_dst);
        p.ids          = reinterpret_cast<int32_t *>(ws + b.ids);
        p.p            = reinterpret_cast<float *>(ws + b.p);
        p.xq           = ws + b.xq;
        p.xs           = ws + b.xs;
        p.hq           = ws + b.hq;
        p.hs           = ws + b.hs;
        p.ld_x         = desc->ld_x;
        p.ld_logits    = desc->ld_logits;
        p.ld_dst       = desc->ld_dst;
        p.ld_xq        = b.ld_xq;
        p.ld_hq        = b.ld_hq;
        p.h_tiles      = mx_scale_tiles(desc->hidden, desc->format);
        p.f_tiles      = mx_scale_tiles(desc->intermediate, desc->format);
        p.tokens       = desc->tokens;
        p.hidden       = desc->hidden;
        p.inner        = desc->intermediate;
        p.experts      = desc->experts;
        p.top_k        = desc->top_k;
        p.renormalize  = desc->renormalize;
        p.dtype        = desc->dtype;
        p.vec_x        = (reinterpret_cast<uintptr_t>(d_x) & 15) == 0 && desc->ld_x % 16 == 0;
        p.route_blocks = (desc->tokens + 7) / 8;
        p.quant_x      = static_cast<int>((p.h_tiles * 4 * mx_block(desc->format) / 16 + 31) / 32);
        p.x_mul        = std::ldexp(1.f, -desc->x_exponent);
        p.h_mul        = std::ldexp(1.f, -desc->h_exponent);
        p.gate_alpha   = std::ldexp(desc->gate_alpha, desc->x_exponent);
        p.up_alpha     = std::ldexp(desc->up_alpha, desc->x_exponent);
        p.down_alpha   = std::ldexp(desc->down_alpha, desc->h_exponent);
        p.status       = ctx->d_status;
        p.spin_limit   = ctx->spin_limit;
        p.withhold_up   = ctx->withhold_kb < kWithholdDown ? ctx->withhold_kb : -1;
        p.withhold_down = ctx->withhold_kb >= kWithholdDown ? ctx->withhold_kb - kWithholdDown : -1;
        ctx->withhold_kb = -1;
        const int nt   = desc->tokens <= 16 ? 16 : desc->tokens <= 32 ? 32 : desc->tokens <= 64 ? 64 : 128;
        const int64_t rows_f = static_cast<int64_t>(desc->experts) * desc->intermediate, rows_h = static_cast<int64_t>(desc->experts) * desc->hidden;
        MoeMaps       m;
        if (!encode_packed_map(&m.gate, d_gate, rows_f, desc->hidden / 2, desc->ld_gate_up, kMxRows) ||
            !encode_packed_map(&m.up, d_up, rows_f, desc->hidden / 2, desc->ld_gate_up, kMxRows) ||
            !encode_packed_map(&m.x, p.xq, desc->tokens, desc->hidden / 2, b.ld_xq, nt) ||
            !encode_packed_map(&m.down, d_down, rows_h, desc->intermediate / 2, desc->ld_down, kMxRows) ||
            !encode_packed_map(&m.h, p.hq, static_cast<int64_t>(b.most_active) * desc->tokens, desc->intermediate / 2, b.ld_hq, nt))
        {
            return fail(ctx, CUGL_RUNTIME_ERROR, "cuTensorMapEncodeTiled failed for a packed operand");
        }
        return desc->format == CUGL_NVFP4 ? launch_moe<CUGL_NVFP4>(ctx, m, p, nt, b.most_active) : launch_moe<CUGL_MXFP4>(ctx, m, p, nt, b.most_active);
    }
}
