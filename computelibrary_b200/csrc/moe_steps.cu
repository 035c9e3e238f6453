// The steps of an expert layer around its products: the gate, which also gives every choice a row of a group, and the combination of a
// token's rows.
#include "mx.cuh"

#include <algorithm>
#include <cmath>
#include <cstring>

namespace cugl
{
namespace
{
constexpr int kMaxExperts = 512, kMaxTopK = 16;
constexpr int kSlab = 128; // rows at whose multiples groups start

// ---- the gate ------------------------------------------------------------------------------------------------
// A warp chooses for a token; a block takes a chunk of consecutive tokens.  The rows of a group are in the order of the tokens, so a
// choice's row is its group's start, the choices of that expert in the chunks before, and those of the tokens before it in its own
// chunk (bits of a mask per expert, 128 tokens at a time).  One chunk: one launch.  Several: the first launch leaves the number of
// choices per chunk and expert, the second adds up those of the chunks before (no block waits for another one, nothing depends on the
// order of atomics).  There are at most 256 chunks, which every block of the second launch reads.
//
// What bounds it: the instructions of the choices, top_k of which follow each other, and two launches.  8192 tokens, 128 experts, top 8:
// 13 us, 0.5 at the copy rate.
constexpr int kRouteWarps  = 32;
constexpr int kRouteSingle = 32;  // tokens of a single block, and of a block at least where there are several
constexpr int kRouteChunks = 256; // at most
constexpr int kRoutePart   = 128; // tokens at a time
constexpr int kMaskWords   = kRoutePart / 32;

struct RouteParams
{
    const uint8_t *logits;
    int32_t       *ids, *slots;
    float         *weights;
    int2          *groups;
    int32_t       *counts; // [chunks][experts]
    int64_t        ld;
    int            tokens, experts, top_k, renormalize, chunk, chunks;
    int            vec; // rows of the logits are 16-byte aligned
};

// Logits become unsigned keys in their order (0: not to be chosen: NaN and -infinity, or chosen already).  A lane holds kPer experts that
// follow each other, and knows its largest key, the first among equal ones: up to four are sorted at the start and move up when one is
// taken, more are searched through.  A choice is the lowest lane with the largest key of all.  16-bit logits leave the lowest 13 bits of a
// 32-bit key alone: nine of them hold the expert's number, the lowest one largest, and the largest key is the choice, with nothing to
// look up.  All lanes run the same instructions: the winner's part under a branch cost twice as many.  Lane j returns the j-th choice
// (-1: none) and its weight.
constexpr uint32_t kNumberBits = kMaxExperts - 1;
template <bool kPacked>
__device__ __forceinline__ uint32_t logit_key(float v, int e)
{
    const uint32_t b = __float_as_uint(v + 0.f); // -0 and 0 are equal logits
    uint32_t       k = (b >> 31) != 0 ? ~b : b | 0x80000000u;
    if constexpr (kPacked) k = (k & ~kNumberBits) | (kNumberBits - static_cast<uint32_t>(e));
    return v > -INFINITY ? k : 0u;
}
template <bool kPacked>
__device__ __forceinline__ float key_logit(uint32_t key)
{
    if constexpr (kPacked) key = (key >> 31) != 0 ? key & ~kNumberBits : key | kNumberBits;
    return __uint_as_float((key >> 31) != 0 ? key & 0x7fffffffu : ~key);
}
template <typename T, int kPer> // experts per lane
__device__ __forceinline__ int route_token(const RouteParams &p, int t, int lane, float &weight)
{
    constexpr bool kPacked = sizeof(T) == 2;
    const T *row = reinterpret_cast<const T *>(p.logits + t * p.ld) + lane * kPer;
    uint32_t key[kPer];
    constexpr int kBytes = kPer * static_cast<int>(sizeof(T)), kUnit = kBytes >= 16 ? 16 : kBytes;
    if (p.vec != 0 && (lane + 1) * kPer <= p.experts)
    {
        alignas(16) T e[kPer];
#pragma unroll
        for (int i = 0; i < kBytes / kUnit; ++i)
        {
            if constexpr (kUnit == 16) reinterpret_cast<uint4 *>(e)[i] = reinterpret_cast<const uint4 *>(row)[i];
            else if constexpr (kUnit == 8) reinterpret_cast<uint2 *>(e)[i] = reinterpret_cast<const uint2 *>(row)[i];
            else reinterpret_cast<uint32_t *>(e)[i] = reinterpret_cast<const uint32_t *>(row)[i];
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) key[i] = logit_key<kPacked>(to_float(e[i]), lane * kPer + i);
    }
    else
    {
#pragma unroll
        for (int i = 0; i < kPer; ++i) key[i] = lane * kPer + i < p.experts ? logit_key<kPacked>(to_float(row[i]), lane * kPer + i) : 0u;
    }
    float    top = 0.f, all = 0.f;
    uint32_t own = 0;
    int      mine = -1, index[kPacked ? 1 : kPer];
    constexpr bool kSorted = kPer <= 4;
    if constexpr (!kPacked)
    {
#pragma unroll
        for (int i = 0; i < kPer; ++i) index[i] = lane * kPer + i;
    }
    if constexpr (kSorted)
    {
        // neighbours change places, equal ones do not: stable
#pragma unroll
        for (int round = 0; round < kPer; ++round)
        {
#pragma unroll
            for (int i = round & 1; i + 1 < kPer; i += 2)
            {
                const bool     swap = key[i + 1] > key[i];
                const uint32_t k    = key[i];
                key[i]              = swap ? key[i + 1] : k;
                key[i + 1]          = swap ? k : key[i + 1];
                if constexpr (!kPacked)
                {
                    const int n  = index[i];
                    index[i]     = swap ? index[i + 1] : n;
                    index[i + 1] = swap ? n : index[i + 1];
                }
            }
        }
    }
    for (int j = 0; j < p.top_k; ++j)
    {
        uint32_t head = key[0];
        int      at   = kPacked ? 0 : index[0];
        if constexpr (!kSorted)
        {
#pragma unroll
            for (int i = 1; i < kPer; ++i)
            {
                const bool more = key[i] > head;
                head            = more ? key[i] : head;
                if constexpr (!kPacked) at = more ? index[i] : at;
            }
        }
        const uint32_t best = __reduce_max_sync(0xffffffffu, head);
        if (best == 0) break;
        own      = lane == j ? best : own;
        bool won = head == best;
        if constexpr (!kPacked) // several lanes may hold it
        {
            const int winner = __ffs(__ballot_sync(0xffffffffu, won)) - 1;
            const int e      = __shfl_sync(0xffffffffu, at, winner);
            mine             = lane == j ? e : mine;
            won              = lane == winner;
        }
        if (j == 0)
        {
            top = key_logit<kPacked>(best);
            if (p.renormalize == 0)
            {
#pragma unroll
                for (int i = 0; i < kPer; ++i) all += key[i] != 0 ? expf(key_logit<kPacked>(key[i]) - top) : 0.f;
            }
        }
        if constexpr (kSorted)
        {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
            {
                key[i] = won ? (i + 1 < kPer ? key[i + 1] : 0u) : key[i];
                if constexpr (!kPacked) index[i] = won && i + 1 < kPer ? index[i + 1] : index[i];
            }
        }
        else
        {
#pragma unroll
            for (int i = 0; i < kPer; ++i) key[i] = won && (kPacked ? key[i] == best : index[kPacked ? 0 : i] == at) ? 0u : key[i];
        }
    }
    if constexpr (kPacked) mine = own != 0 ? static_cast<int>(kNumberBits - (own & kNumberBits)) : -1;
    const float w = mine >= 0 ? expf(key_logit<kPacked>(own) - top) : 0.f;
    if (p.renormalize != 0) all = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    weight = mine >= 0 ? w / all : 0.f;
    return mine;
}
template <typename T>
__device__ __forceinline__ int route_any(const RouteParams &p, int t, int lane, float &weight)
{
    if (p.experts <= 64) return route_token<T, 2>(p, t, lane, weight);
    if (p.experts <= 128) return route_token<T, 4>(p, t, lane, weight);
    if (p.experts <= 256) return route_token<T, 8>(p, t, lane, weight);
    return route_token<T, kMaxExperts / 32>(p, t, lane, weight);
}

struct RouteShared
{
    uint32_t mask[kMaxExperts][kMaskWords]; // tokens of the chunk that chose an expert
    int      start[kMaxExperts];            // the group's first row, then the chunk's first row of it
    int      scan[kMaxExperts];
    int      before[kMaxExperts];
    int      total[kMaxExperts / 32];
};
// Starts of the groups from the choices per expert in `scan` (which is left as it is): every group takes whole slabs.  By all threads; warp w
// adds up the experts from 32 w on.
__device__ __forceinline__ void group_starts(const RouteParams &p, RouteShared &s)
{
    const int lane = threadIdx.x & 31, warps = static_cast<int>(blockDim.x) >> 5;
    for (int w = static_cast<int>(threadIdx.x) >> 5; w < (p.experts + 31) / 32; w += warps)
    {
        const int e    = w * 32 + lane;
        const int room = e < p.experts ? (s.scan[e] + kSlab - 1) / kSlab * kSlab : 0;
        int       incl = room;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (e < p.experts) s.start[e] = incl - room;
        if (lane == 31) s.total[w] = incl;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.experts; e += static_cast<int>(blockDim.x))
    {
        int start = s.start[e];
        for (int w = 0; w < (e >> 5); ++w) start += s.total[w];
        if (blockIdx.x == 0) p.groups[e] = make_int2(start, s.scan[e]);
        s.start[e] = start + s.before[e];
    }
}
// The mask of a part's choices: read back where another launch made them.
__device__ __forceinline__ void clear_mask(const RouteParams &p, RouteShared &s)
{
    for (int i = threadIdx.x; i < p.experts * kMaskWords; i += static_cast<int>(blockDim.x)) (&s.mask[0][0])[i] = 0;
}
__device__ __forceinline__ void set_mask(const RouteParams &p, RouteShared &s, int t0, int tokens)
{
    for (int i = threadIdx.x; i < tokens * p.top_k; i += static_cast<int>(blockDim.x))
    {
        const int e = p.ids[static_cast<int64_t>(t0) * p.top_k + i], t = i / p.top_k;
        if (e >= 0) atomicOr(&s.mask[e][t >> 5], 1u << (t & 31));
    }
}
__device__ __forceinline__ int mask_count(const RouteShared &s, int e)
{
    int n = 0;
#pragma unroll
    for (int w = 0; w < kMaskWords; ++w) n += __popc(s.mask[e][w]);
    return n;
}
// rows of the choices of a part's tokens, from the mask and the part's first rows
__device__ __forceinline__ void place_choices(const RouteParams &p, const RouteShared &s, int t0, int tokens)
{
    for (int i = threadIdx.x; i < tokens * p.top_k; i += static_cast<int>(blockDim.x))
    {
        const int t = i / p.top_k, e = p.ids[static_cast<int64_t>(t0) * p.top_k + i];
        int       row = -1;
        if (e >= 0)
        {
            row = s.start[e];
            for (int w = 0; w < (t >> 5); ++w) row += __popc(s.mask[e][w]);
            row += __popc(s.mask[e][t >> 5] & ((1u << (t & 31)) - 1u));
        }
        p.slots[static_cast<int64_t>(t0) * p.top_k + i] = row;
    }
}

// kStep 0: all of it in one block; 1: choices of a chunk; 2: their rows
template <typename T, int kStep>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const __grid_constant__ RouteParams p)
{
    __shared__ RouteShared s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = static_cast<int>(blockDim.x) >> 5;
    const int t0 = static_cast<int>(blockIdx.x) * p.chunk, end = t0 + min(p.chunk, p.tokens - t0); // (t0 + chunk may pass 32 bits)
    clear_mask(p, s);
    for (int e = threadIdx.x; e < p.experts; e += static_cast<int>(blockDim.x)) s.scan[e] = s.before[e] = 0;
    dependent_prologue();
    __syncthreads();
    if constexpr (kStep != 2)
    {
        for (int part = t0; part < end; part += kRoutePart)
        {
            const int tokens = min(kRoutePart, end - part);
            for (int t = warp; t < tokens; t += warps)
            {
                float     weight;
                const int e = route_any<T>(p, part + t, lane, weight);
                if (lane < p.top_k)
                {
                    const int64_t at = static_cast<int64_t>(part + t) * p.top_k + lane;
                    p.ids[at]        = e;
                    p.weights[at]    = weight;
                    if (e >= 0) atomicOr(&s.mask[e][t >> 5], 1u << (t & 31));
                }
            }
            __syncthreads();
            for (int e = threadIdx.x; e < p.experts; e += static_cast<int>(blockDim.x)) s.scan[e] += mask_count(s, e);
            if (part + kRoutePart < end)
            {
                __syncthreads();
                clear_mask(p, s);
                __syncthreads();
            }
        }
        if constexpr (kStep == 1)
        {
            for (int e = threadIdx.x; e < p.experts; e += static_cast<int>(blockDim.x)) // (written by the same thread)
            {
                p.counts[static_cast<int64_t>(blockIdx.x) * p.experts + e] = s.scan[e];
            }
            return;
        }
    }
    else
    {
        // choices of all chunks and of those before this one: slices of chunks per expert, eight loads in flight per thread
        const int slices = max(1, static_cast<int>(blockDim.x) / p.experts);
        for (int i = threadIdx.x; i < slices * p.experts; i += static_cast<int>(blockDim.x))
        {
            const int e = i % p.experts, slice = i / p.experts;
            int       all = 0, own = 0;
            for (int c = slice; c < p.chunks; c += 8 * slices)
            {
                int n[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) n[k] = c + k * slices < p.chunks ? p.counts[static_cast<int64_t>(c + k * slices) * p.experts + e] : 0;
#pragma unroll
                for (int k = 0; k < 8; ++k)
                {
                    all += n[k];
                    own += c + k * slices < static_cast<int>(blockIdx.x) ? n[k] : 0;
                }
            }
            atomicAdd(&s.scan[e], all); // whole numbers: the same sum in any order
            atomicAdd(&s.before[e], own);
        }
        set_mask(p, s, t0, min(kRoutePart, end - t0));
    }
    __syncthreads();
    group_starts(p, s);
    __syncthreads();
    for (int part = t0; part < end; part += kRoutePart)
    {
        place_choices(p, s, part, min(kRoutePart, end - part));
        if (part + kRoutePart < end)
        {
            __syncthreads();
            for (int e = threadIdx.x; e < p.experts; e += static_cast<int>(blockDim.x)) s.start[e] += mask_count(s, e);
            __syncthreads();
            clear_mask(p, s);
            __syncthreads();
            set_mask(p, s, part + kRoutePart, min(kRoutePart, end - part - kRoutePart));
            __syncthreads();
        }
    }
}

// ---- combination ---------------------------------------------------------------------------------------------
// dst[t] = sum_j weights[t][j] * src[slots[t][j]], in the order of j, in float, rounded once.  Eight columns of a token per thread: all
// its slots and weights are asked for together, then all its rows, before the first is used (slot by slot 29.6 us, this 27.8: 4096 x
// 2048 BF16, eight choices, 84 % of the copy rate).  The bytes bound it.
struct CombineParams
{
    const uint8_t *src;
    const int32_t *slots;
    const float   *weights;
    uint8_t       *dst;
    int64_t        ld_src, ld_dst;
    int            tokens, top_k, cols, rows, units; // units: of a row, eight columns a thread or 256 a warp
};

template <typename TS>
__device__ __forceinline__ void widen8(const uint4 *raw, float (&v)[8])
{
    TS e[8];
    memcpy(e, raw, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float(e[i]);
}

template <typename TS, typename TD, bool kVec>
__global__ void __launch_bounds__(256) combine_kernel(const __grid_constant__ CombineParams p)
{
    dependent_prologue();
    // kVec: a thread has eight columns that follow each other; else its warp has 256 and the thread every 32nd of them
    constexpr int kColumns = kVec ? 8 : 256, kGap = kVec ? 1 : 32;
    const int     lane = threadIdx.x & 31;
    const int64_t own = kVec ? static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x : static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int64_t total = static_cast<int64_t>(p.tokens) * p.units, step = static_cast<int64_t>(gridDim.x) * (kVec ? 256 : 8);
    for (int64_t i = own; i < total; i += step)
    {
        const int t = static_cast<int>(i / p.units), c0 = static_cast<int>(i - static_cast<int64_t>(t) * p.units) * kColumns + (kVec ? 0 : lane), n = p.cols - c0;
        const int32_t *slots   = p.slots + static_cast<int64_t>(t) * p.top_k;
        const float   *weights = p.weights + static_cast<int64_t>(t) * p.top_k;
        float          sum[8] = {};
        constexpr int  kBatch = sizeof(TS) == 4 ? 4 : 8, kLoads = sizeof(TS) / 2;
        for (int j0 = 0; j0 < p.top_k; j0 += kBatch)
        {
            uint4 raw[kBatch][kLoads];
            float w[kBatch];
            int   row[kBatch];
            bool  has[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
            {
                row[j] = -1;
                w[j]   = 0.f;
                if (j0 + j < p.top_k)
                {
                    row[j] = slots[j0 + j];
                    w[j]   = weights[j0 + j];
                }
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
            {
                has[j] = row[j] >= 0 && row[j] < p.rows;
                if (has[j])
                {
                    const TS *src = reinterpret_cast<const TS *>(p.src + row[j] * p.ld_src) + c0;
                    if constexpr (kVec)
                    {
#pragma unroll
                        for (int l = 0; l < kLoads; ++l) raw[j][l] = __ldcg(reinterpret_cast<const uint4 *>(src) + l);
                    }
                    else
                    {
                        TS e[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                        {
                            e[k] = from_float<TS>(0.f);
                            if (k * kGap < n) e[k] = src[k * kGap];
                        }
                        memcpy(raw[j], e, sizeof(e));
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
            {
                if (has[j])
                {
                    float v[8];
                    widen8<TS>(raw[j], v);
#pragma unroll
                    for (int k = 0; k < 8; ++k) sum[k] = fmaf(w[j], v[k], sum[k]);
                }
            }
        }
        TD  out[8];
        TD *dst = reinterpret_cast<TD *>(p.dst + t * p.ld_dst) + c0;
#pragma unroll
        for (int k = 0; k < 8; ++k) out[k] = from_float<TD>(sum[k]);
        if constexpr (kVec)
        {
            uint4 q[sizeof(TD) / 2];
            memcpy(q, out, sizeof(out));
#pragma unroll
            for (int l = 0; l < static_cast<int>(sizeof(TD)) / 2; ++l) reinterpret_cast<uint4 *>(dst)[l] = q[l];
        }
        else
        {
#pragma unroll
            for (int k = 0; k < 8; ++k)
            {
                if (k * kGap < n) dst[k * kGap] = out[k];
            }
        }
    }
}

template <typename TS, typename TD>
cudaError_t launch_combine(cugl_context *ctx, CombineParams p, bool vec)
{
    p.units              = vec ? p.cols / 8 : (p.cols + 255) / 256;
    const int64_t each   = vec ? 256 : 8;
    const int64_t blocks = (static_cast<int64_t>(p.tokens) * p.units + each - 1) / each, most = static_cast<int64_t>(ctx->sm_count) * 64;
    const unsigned grid  = static_cast<unsigned>(blocks < most ? blocks : most);
    return vec ? launch_dependent(ctx, combine_kernel<TS, TD, true>, dim3(grid), 256, 0, blocks, p)
               : launch_dependent(ctx, combine_kernel<TS, TD, false>, dim3(grid), 256, 0, blocks, p);
}
template <typename TS>
cudaError_t launch_combine(cugl_context *ctx, int dst_dtype, const CombineParams &p, bool vec)
{
    return dst_dtype == CUGL_F32 ? launch_combine<TS, float>(ctx, p, vec)
           : dst_dtype == CUGL_F16 ? launch_combine<TS, __half>(ctx, p, vec)
                                   : launch_combine<TS, __nv_bfloat16>(ctx, p, vec);
}

bool aligned(const void *p, uintptr_t n)
{
    return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

const char *validate_route(const cugl_moe_route_desc *d)
{
    if (d == nullptr) return "descriptor is NULL";
    if (d->tokens < 0) return "tokens must not be negative";
    if (d->experts < 1 || d->experts > kMaxExperts) return "experts must lie within 1 .. 512";
    if (d->top_k < 1 || d->top_k > kMaxTopK || d->top_k > d->experts) return "top_k must lie within 1 .. 16 and not exceed experts";
    if (!is_float_dtype(d->dtype)) return "dtype must be CUGL_F32, CUGL_F16 or CUGL_BF16";
    if (d->ld_logits < static_cast<int64_t>(d->experts) * dtype_size(d->dtype) || d->ld_logits % dtype_size(d->dtype) != 0)
        return "ld_logits must hold a row and be a multiple of the element size";
    if (static_cast<int64_t>(d->tokens) * d->top_k + static_cast<int64_t>(kSlab) * d->experts > INT32_MAX - 1024) return "more rows than 32 bits count";
    return nullptr;
}
int route_chunk(int tokens) // tokens of a block; 148, the SMs of a B200: the workspace's size follows from it, and asking for that names no device
{
    // one token a warp while there is an SM for every block: 8192 tokens, 128 experts, 256 blocks of 32 17.2 us, 128 of 64 13.3
    if (tokens <= 148 * kRouteSingle) return kRouteSingle;
    const int least = (tokens + kRouteChunks - 1) / kRouteChunks;
    return least <= 2 * kRouteSingle ? 2 * kRouteSingle : (least + kRoutePart - 1) / kRoutePart * kRoutePart;
}
int route_chunks(int tokens)
{
    const int chunk = route_chunk(tokens);
    return tokens <= chunk ? 1 : tokens / chunk + (tokens % chunk != 0 ? 1 : 0); // (tokens + chunk may pass 32 bits)
}

const char *validate_combine(const cugl_moe_combine_desc *d)
{
    if (d == nullptr) return "descriptor is NULL";
    if (d->tokens < 0 || d->cols < 1 || d->rows < 0) return "tokens and rows must not be negative, cols must be positive";
    if (d->cols > INT32_MAX - 1024) return "cols is too large";
    if (d->top_k < 1 || d->top_k > kMaxTopK) return "top_k must lie within 1 .. 16";
    if (!is_float_dtype(d->src_dtype) || !is_float_dtype(d->dst_dtype)) return "dtypes must be CUGL_F32, CUGL_F16 or CUGL_BF16";
    const int ss = dtype_size(d->src_dtype), ds = dtype_size(d->dst_dtype);
    if (d->ld_src < static_cast<int64_t>(d->cols) * ss || d->ld_src % ss != 0 || d->ld_dst < static_cast<int64_t>(d->cols) * ds || d->ld_dst % ds != 0)
        return "ld_src and ld_dst must hold a row and be multiples of their element sizes";
    return nullptr;
}

cugl_status told(const char *why, const char **reason)
{
    if (reason != nullptr)
    {
        *reason = why != nullptr ? why : "";
    }
    return why == nullptr ? CUGL_SUCCESS : CUGL_INVALID_ARGUMENT;
}
} // namespace
} // namespace cugl

using namespace cugl;

extern "C"
{
    cugl_status cugl_moe_route_validate(const cugl_moe_route_desc *desc, const char **reason)
    {
        return told(validate_route(desc), reason);
    }

    size_t cugl_moe_route_workspace_bytes(const cugl_moe_route_desc *desc)
    {
        if (validate_route(desc) != nullptr)
        {
            return 0;
        }
        const int chunks = route_chunks(desc->tokens);
        return chunks == 1 ? 16 : static_cast<size_t>(chunks) * static_cast<size_t>(desc->experts) * 4;
    }

    cugl_status cugl_moe_route(cugl_context *ctx, const cugl_moe_route_desc *desc, const void *d_logits, int32_t *d_ids, float *d_weights,
                               int32_t *d_slots, int32_t *d_groups, void *d_workspace, size_t workspace_bytes)
    {
        if (ctx == nullptr)
        {
            return fail(nullptr, CUGL_INVALID_ARGUMENT, "context is NULL");
        }
        const char *why = validate_route(desc);
        if (why == nullptr)
        {
            const bool some = desc->tokens > 0;
            if (d_groups == nullptr || (some && (d_logits == nullptr || d_ids == nullptr || d_weights == nullptr || d_slots == nullptr || d_workspace == nullptr)))
                why = "NULL pointer";
            else if (!aligned(d_groups, 8)) why = "groups must be 8-byte aligned";
            else if (some && (!aligned(d_logits, static_cast<uintptr_t>(dtype_size(desc->dtype))) || !aligned(d_ids, 4) || !aligned(d_weights, 4) || !aligned(d_slots, 4) ||
                              !aligned(d_workspace, 16)))
                why = "a buffer is not aligned to its elements (the workspace: 16 bytes)";
            else if (some && workspace_bytes < cugl_moe_route_workspace_bytes(desc)) why = "the workspace is too small";
        }
        if (why != nullptr)
        {
            return fail(ctx, CUGL_INVALID_ARGUMENT, std::string("cugl_moe_route: ") + why);
        }
        const DeviceScope device(ctx);
        RouteParams       p{};
        p.logits      = static_cast<const uint8_t *>(d_logits);
        p.ids         = d_ids;
        p.slots       = d_slots;
        p.weights     = d_weights;
        p.groups      = reinterpret_cast<int2 *>(d_groups);
        p.counts      = static_cast<int32_t *>(d_workspace);
        p.ld          = desc->ld_logits;
        p.tokens      = desc->tokens;
        p.experts     = desc->experts;
        p.top_k       = desc->top_k;
        p.renormalize = desc->renormalize;
        p.chunks      = route_chunks(desc->tokens);
        p.chunk       = route_chunk(desc->tokens);
        p.vec         = aligned(d_logits, 16) && desc->ld_logits % 16 == 0;
        auto run      = [&](auto element) -> cugl_status {
            using T = decltype(element);
            if (p.chunks == 1)
            {
                const int threads = 32 * std::min(kRouteWarps, std::max(4, p.tokens));
                CUGL_CUDA_TRY(ctx, launch_dependent(ctx, route_kernel<T, 0>, dim3(1), threads, 0, 1, p));
                return CUGL_SUCCESS;
            }
            const dim3 grid(static_cast<unsigned>(p.chunks));
            CUGL_CUDA_TRY(ctx, launch_dependent(ctx, route_kernel<T, 1>, grid, kRouteWarps * 32, 0, p.chunks, p));
            CUGL_CUDA_TRY(ctx, launch_dependent(ctx, route_kernel<T, 2>, grid, kRouteWarps * 32, 0, p.chunks, p));
            return CUGL_SUCCESS;
        };
        return desc->dtype == CUGL_F32 ? run(float{}) : desc->dtype == CUGL_F16 ? run(__half{}) : run(__nv_bfloat16{});
    }

    cugl_status cugl_moe_combine_validate(const cugl_moe_combine_desc *desc, const char **reason)
    {
        return told(validate_combine(desc), reason);
    }

    cugl_status cugl_moe_combine(cugl_context *ctx, const cugl_moe_combine_desc *desc, const void *d_src, const int32_t *d_slots, const float *d_weights,
                                 void *d_dst)
    {
        if (ctx == nullptr)
        {
            return fail(nullptr, CUGL_INVALID_ARGUMENT, "context is NULL");
        }
        const char *why = validate_combine(desc);
        if (why == nullptr && desc->tokens > 0)
        {
            if ((d_src == nullptr && desc->rows > 0) || d_slots == nullptr || d_weights == nullptr || d_dst == nullptr) why = "NULL pointer";
            else if (!aligned(d_src, static_cast<uintptr_t>(dtype_size(desc->src_dtype))) || !aligned(d_dst, static_cast<uintptr_t>(dtype_size(desc->dst_dtype))) ||
                     !aligned(d_slots, 4) || !aligned(d_weights, 4))
                why = "a buffer is not aligned to its elements";
        }
        if (why != nullptr)
        {
            return fail(ctx, CUGL_INVALID_ARGUMENT, std::string("cugl_moe_combine: ") + why);
        }
        if (desc->tokens == 0) return CUGL_SUCCESS;
        const DeviceScope device(ctx);
        CombineParams     p{};
        p.src     = static_cast<const uint8_t *>(d_src);
        p.slots   = d_slots;
        p.weights = d_weights;
        p.dst     = static_cast<uint8_t *>(d_dst);
        p.ld_src  = desc->ld_src;
        p.ld_dst  = desc->ld_dst;
        p.tokens  = desc->tokens;
        p.top_k   = desc->top_k;
        p.cols    = desc->cols;
        p.rows    = desc->rows;
        const bool vec = desc->cols % 8 == 0 && aligned(d_src, 16) && aligned(d_dst, 16) && desc->ld_src % 16 == 0 && desc->ld_dst % 16 == 0;
        CUGL_CUDA_TRY(ctx, desc->src_dtype == CUGL_F32 ? launch_combine<float>(ctx, desc->dst_dtype, p, vec)
                           : desc->src_dtype == CUGL_F16 ? launch_combine<__half>(ctx, desc->dst_dtype, p, vec)
                                                         : launch_combine<__nv_bfloat16>(ctx, desc->dst_dtype, p, vec));
        return CUGL_SUCCESS;
    }
}
