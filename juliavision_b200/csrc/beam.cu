// Beam search's choice: of the K V continuations of a search's beams,
//     c[k, v] = score[k] + x[k, v] - log sum_u exp x[k, u],
// the N largest, in order, ties to the lowest k V + v.  An ended beam has one continuation, the padding token at its own score.
//
// Bandwidth-bound: every logit is read once.  Within a beam the order is that of the logits, so the first launch needs no sums to choose by:
// a warp walks a share of a row, keeps sums of exponentials relative to each lane's running maximum, and the share's N largest, one a lane,
// as 64-bit keys (the logit's bits in order, then the index from above) of which no two are alike.  Almost every tile of 32 lanes' elements
// is done with after one comparison a lane, of its maximum against the Nth; the first tile gets a bound from the Nth largest of the lanes' maxima.
// Lists are merged in the block.  The second launch, a block a search, merges a row's lists, takes log sums and scores in fp64 and merges the rows'.
#include <cuda_fp16.h>

#include "internal.h"
#include "ptx.cuh"

namespace b200 {

constexpr int BM_WARPS = 8;          // of a scanning block
constexpr int BM_MOST = 32;          // beams, and results: one a lane

struct BeamParams {
    const void* x;
    int64_t ldk, ldb;                // elements between beams, between searches
    const float* score;
    const int32_t* ended;            // or null
    float* best;
    int32_t *parents, *tokens;
    unsigned long long* keys;        // [rows][parts][N]
    float2* sums;                    // [rows][parts]: maximum, sum of exponentials relative to it
    int64_t V;
    int K, N, parts, pad;
    int64_t share;                   // vectors of a warp
};

__device__ __forceinline__ uint32_t bm_order(float x) {          // bits whose order is that of the numbers, -0 and 0 alike
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float bm_number(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ unsigned long long bm_key(float x, uint32_t index) { return (unsigned long long)bm_order(x) << 32 | (uint32_t)~index; }
__device__ __forceinline__ unsigned long long bm_other(unsigned long long a, int lane_mask) { return __shfl_xor_sync(0xffffffffu, a, lane_mask); }

// A warp's keys, one a lane, sorted from the largest down; `bitonic`: they rise and fall once.
template <bool BITONIC> __device__ __forceinline__ unsigned long long bm_sort(unsigned long long a) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = BITONIC ? 32 : 2; size <= 32; size *= 2)
#pragma unroll
        for (int d = size / 2; d > 0; d /= 2) {
            const unsigned long long b = bm_other(a, d);
            const bool high = ((lane & size) == 0 || size == 32) == ((lane & d) == 0);     // the larger belongs here
            a = (a > b) == high ? a : b;
        }
    return a;
}
// The 32 largest of two sorted lists, sorted.
__device__ __forceinline__ unsigned long long bm_merge(unsigned long long a, unsigned long long b) {
    b = __shfl_sync(0xffffffffu, b, 31 - (threadIdx.x & 31));
    return bm_sort<true>(a > b ? a : b);
}
__device__ __forceinline__ float bm_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T> struct BmVec;
template <> struct BmVec<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(float* v, uint4 r) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ float one(const void* x, int64_t i) { return __half2float(((const __half*)x)[i]); }
};
template <> struct BmVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(float* v, uint4 r) {
        v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ float one(const void* x, int64_t i) { return ((const float*)x)[i]; }
};

template <typename T>
__global__ void __launch_bounds__(32 * BM_WARPS)
beam_scan_kernel(const BeamParams p) {
    using Vec = BmVec<T>;
    constexpr int U = 4, E = U * Vec::N;             // vectors and elements of a lane's tile
    __shared__ unsigned long long lists[BM_WARPS][32];
    __shared__ float2 sums[BM_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x / p.parts, part_of_row = blockIdx.x - row * p.parts;
    grid_dep_wait();
    grid_dep_launch();
    const T* x = (const T*)p.x + row / p.K * p.ldb + row % p.K * p.ldk;
    // vectors from the 16-byte boundary at or below the row's first element; what is not of the row is left out
    const int skew = (int)((uintptr_t)x % 16 / sizeof(T));
    const uint4* base = reinterpret_cast<const uint4*>(x - skew);
    const int64_t end = (p.V + skew + Vec::N - 1) / Vec::N;
    int64_t at = (part_of_row * BM_WARPS + warp) * p.share;
    const int64_t stop = at + p.share < end ? at + p.share : end;
    unsigned long long list = 0;                     // no element's key is 0
    float bound = -INFINITY, m = -INFINITY, s = 0.f;
    bool first = true;
    for (; at < stop; at += 32 * U) {
        float v[E];
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (at + u * 32 + lane < stop) raw[u] = __ldg(base + at + u * 32 + lane);
        uint32_t some = 0;                           // bit e: element e is one of the row's
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = (at + u * 32 + lane) * Vec::N - skew;         // its first element's index
            Vec::load(v + u * Vec::N, raw[u]);
            if (at + u * 32 + lane >= stop || i < 0 || i + Vec::N > p.V) {
#pragma unroll
                for (int k = 0; k < Vec::N; ++k) {
                    const bool in = at + u * 32 + lane < stop && i + k >= 0 && i + k < p.V;
                    some |= (uint32_t)in << (u * Vec::N + k);
                    if (!in) v[u * Vec::N + k] = -INFINITY;
                }
            } else {
                some |= ((1u << Vec::N) - 1) << (u * Vec::N);
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) top = fmaxf(top, v[e]);
        // the sum of exponentials, relative to the lane's maximum so far; differences first: their error is theirs, not the logit's
        const float high = fmaxf(m, top), ref = high == -INFINITY ? 0.f : high;
        uint64_t part = pack2(0.f, 0.f);
        const uint64_t less = pack2(-ref, -ref), unit = pack2(1.4426950408889634f, 1.4426950408889634f);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            float a, b;
            unpack2(mul2(add2(pack2(v[e], v[e + 1]), less), unit), a, b);
            part = add2(part, pack2(bm_ex2(a), bm_ex2(b)));
        }
        float a, b;
        unpack2(part, a, b);
        s = s * (m == high ? 1.f : bm_ex2((m - ref) * 1.4426950408889634f)) + (a + b);
        m = high;
        // candidates
        uint32_t hits = 0;
        if (first) {
            // the Nth largest of the lanes' maxima: at least N elements are as large
            const unsigned long long sorted = bm_sort<false>((unsigned long long)bm_order(top) << 32);
            bound = bm_number((uint32_t)(__shfl_sync(0xffffffffu, sorted, p.N - 1) >> 32));
#pragma unroll
            for (int e = 0; e < E; ++e) hits |= (uint32_t)(v[e] >= bound) << e;
            hits &= some;
            first = false;
        } else if (__any_sync(0xffffffffu, top > bound)) {
#pragma unroll
            for (int e = 0; e < E; ++e) hits |= (uint32_t)(v[e] > bound) << e;
        }
        while (__any_sync(0xffffffffu, hits != 0)) {         // a candidate a lane at a time
            unsigned long long key = 0;
            if (hits) {
                const int e = __ffs(hits) - 1;
                hits &= hits - 1;
                const int64_t i = (at + e / Vec::N * 32 + lane) * Vec::N + e % Vec::N - skew;
                key = bm_key(Vec::one(x, i), (uint32_t)i);
            }
            list = bm_merge(list, bm_sort<false>(key));
            const unsigned long long nth = __shfl_sync(0xffffffffu, list, p.N - 1);
            if (nth) bound = bm_number((uint32_t)(nth >> 32));
        }
    }
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const float om = __shfl_xor_sync(0xffffffffu, m, d), os = __shfl_xor_sync(0xffffffffu, s, d), high = fmaxf(m, om);
        const float ref = high == -INFINITY ? 0.f : high;
        // the same on both sides of a pair
        const float mine = s * (m == high ? 1.f : bm_ex2((m - ref) * 1.4426950408889634f)), others = os * (om == high ? 1.f : bm_ex2((om - ref) * 1.4426950408889634f));
        s = mine + others;
        m = high;
    }
    lists[warp][lane] = list;
    if (lane == 0) sums[warp] = make_float2(m, s);
#pragma unroll
    for (int d = BM_WARPS / 2; d > 0; d /= 2) {
        __syncthreads();
        if (warp < d) {
            list = bm_merge(list, lists[warp + d][lane]);
            lists[warp][lane] = list;
        }
    }
    if (warp == 0) {
        const int64_t place = blockIdx.x;
        if (lane < p.N) p.keys[place * p.N + lane] = list;
        if (lane == 0) {
            float high = -INFINITY, total = 0.f;
            for (int w = 0; w < BM_WARPS; ++w) high = fmaxf(high, sums[w].x);
            const float ref = high == -INFINITY ? 0.f : high;
            for (int w = 0; w < BM_WARPS; ++w) total += sums[w].y * (sums[w].x == high ? 1.f : bm_ex2((sums[w].x - ref) * 1.4426950408889634f));
            p.sums[place] = make_float2(high, total);
        }
    }
}

// A candidate of the search: its score's bits in order, and from above (beam, place in the beam's list), which is the order of ties.
struct BmCandidate {
    unsigned long long score;
    uint32_t tie, token;
    __device__ __forceinline__ bool above(const BmCandidate& o) const { return score != o.score ? score > o.score : tie > o.tie; }
};
__device__ __forceinline__ BmCandidate bm_pick(const BmCandidate& a, const BmCandidate& b, bool first) { return first ? a : b; }
__device__ __forceinline__ BmCandidate bm_merge(BmCandidate a, BmCandidate b) {
    const int lane = threadIdx.x & 31;
    b.score = __shfl_sync(0xffffffffu, b.score, 31 - lane);
    b.tie = __shfl_sync(0xffffffffu, b.tie, 31 - lane);
    b.token = __shfl_sync(0xffffffffu, b.token, 31 - lane);
    a = bm_pick(a, b, a.above(b));
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        BmCandidate o;
        o.score = bm_other(a.score, d);
        o.tie = __shfl_xor_sync(0xffffffffu, a.tie, d);
        o.token = __shfl_xor_sync(0xffffffffu, a.token, d);
        a = bm_pick(a, o, a.above(o) == ((lane & d) == 0));
    }
    return a;
}

__global__ void __launch_bounds__(32 * BM_MOST)
beam_pick_kernel(const BeamParams p) {
    __shared__ BmCandidate lists[BM_MOST][32];
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;        // a warp a beam
    const int64_t search = blockIdx.x, row = search * p.K + k;
    grid_dep_wait();
    grid_dep_launch();
    BmCandidate c = {0, 0, 0};                                      // below every candidate
    if (k < p.K) {
        unsigned long long list = 0;
        float m = -INFINITY;
        double s = 0;
        for (int i = 0; i < p.parts; ++i) {
            const unsigned long long next = lane < p.N ? p.keys[(row * p.parts + i) * p.N + lane] : 0;
            list = i ? bm_merge(list, next) : next;
        }
        for (int i = lane; i < p.parts; i += 32) m = fmaxf(m, p.sums[row * p.parts + i].x);
#pragma unroll
        for (int d = 1; d < 32; d *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        for (int i = lane; i < p.parts; i += 32) {
            const float2 x = p.sums[row * p.parts + i];
            if (m > -INFINITY) s += (double)x.y * exp((double)x.x - (double)m);
        }
#pragma unroll
        for (int d = 1; d < 32; d *= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
        const double score = (double)p.score[row], sum = (double)m + log(s);
        const bool ended = p.ended != nullptr && p.ended[row] != 0;
        const bool over = !(score < INFINITY && score > -INFINITY);
        double value = -INFINITY;
        uint32_t token = (uint32_t)lane;                            // of a beam that offers nothing: the first tokens
        bool some = lane < p.V;
        if (ended) {
            token = lane == 0 ? (uint32_t)p.pad : (uint32_t)(lane - 1 + (lane - 1 >= p.pad));
            if (lane == 0 && !over) value = score;
            if (over) token = (uint32_t)lane;
        } else if (!over && sum < INFINITY && sum > -INFINITY) {
            some = list != 0;
            token = ~(uint32_t)list;
            value = score + ((double)bm_number((uint32_t)(list >> 32)) - sum);
        }
        if (some && lane < p.N) {
            const unsigned long long b = (unsigned long long)__double_as_longlong(value + 0.0);
            c.score = b >> 63 ? ~b : b | 1ull << 63;
            c.tie = ~(uint32_t)(k * 32 + lane);
            c.token = token;
        }
    }
    lists[k][lane] = c;
    int n = 1;
    while (n < p.K) n *= 2;
    for (int d = n / 2; d > 0; d /= 2) {
        __syncthreads();
        if (k < d && k + d < p.K) {
            c = bm_merge(c, lists[k + d][lane]);
            lists[k][lane] = c;
        }
    }
    if (k == 0 && lane < p.N) {
        const unsigned long long b = c.score >> 63 ? c.score & ~(1ull << 63) : ~c.score;
        const int64_t to = search * p.N + lane;
        p.best[to] = (float)__longlong_as_double((long long)b);
        p.parents[to] = (int32_t)(~c.tie >> 5);
        p.tokens[to] = (int32_t)c.token;
    }
}

} // namespace b200

using namespace b200;

extern "C" {

int b200_beam_select(b200_ctx* ctx, int64_t V, int64_t K, int64_t B, int64_t N, const void* logits, int dtype, int64_t ldk, int64_t ldb,
                     const float* scores, const int32_t* ended, int64_t pad, float* best, int32_t* parents, int32_t* tokens) {
    B200_REQUIRE(ctx, B200_EINVAL, "beam_select: null argument");
    B200_REQUIRE(V >= 0 && K >= 0 && B >= 0 && N >= 0, B200_EINVAL, "beam_select: V=%lld K=%lld B=%lld N=%lld", (long long)V, (long long)K, (long long)B,
                 (long long)N);
    B200_REQUIRE(dtype == B200_F16 || dtype == B200_F32, B200_DECLINE_ELTYPE, "beam_select: logits of type %d", dtype);
    B200_REQUIRE(K <= BM_MOST && N <= BM_MOST, B200_DECLINE_EXTENT, "beam_select: %lld beams, %lld results (at most %d)", (long long)K, (long long)N, BM_MOST);
    B200_REQUIRE(V < (1ll << 31) && B < (1ll << 25), B200_DECLINE_EXTENT, "beam_select: V=%lld B=%lld", (long long)V, (long long)B);
    if (N == 0 || B == 0) return B200_OK;
    B200_REQUIRE(N <= K * V, B200_DECLINE_EXTENT, "beam_select: %lld results of %lld", (long long)N, (long long)(K * V));
    B200_REQUIRE(logits && scores && best && parents && tokens, B200_EINVAL, "beam_select: null array");
    B200_REQUIRE(ended == nullptr || (pad >= 0 && pad < V), B200_EINVAL, "beam_select: padding token %lld of %lld", (long long)pad, (long long)V);
    B200_CUDA(cudaSetDevice(ctx->device));
    BeamParams p = {};
    p.x = logits, p.ldk = ldk, p.ldb = ldb, p.score = scores, p.ended = ended;
    p.best = best, p.parents = parents, p.tokens = tokens;
    p.V = V, p.K = (int)K, p.N = (int)N, p.pad = (int)pad;
    const int per = dtype == B200_F16 ? 8 : 4, tile = 32 * 4;     // elements of a vector, vectors of a warp's tile
    const int64_t rows = B * K, tiles = cdiv(cdiv(V + per - 1, per), tile), sms = ctx->prop.multiProcessorCount;
    // Tiles of a warp: as many as leave some six blocks an SM, and one at least.
    int64_t each = tiles * rows / (6 * sms * BM_WARPS);
    each = each < 1 ? 1 : each;
    p.share = each * tile;
    p.parts = (int)cdiv(tiles, each * BM_WARPS);
    B200_REQUIRE(rows * p.parts < (1ll << 31), B200_DECLINE_EXTENT, "beam_select: %lld beams of %lld in all", (long long)rows, (long long)V);
    void* ws = nullptr;
    int rc = ws_scratch(ctx, (size_t)(rows * p.parts) * (N * sizeof(unsigned long long) + sizeof(float2)), &ws);
    if (rc) return rc;
    p.keys = (unsigned long long*)ws;
    p.sums = (float2*)(p.keys + rows * p.parts * N);
    const dim3 grid((unsigned)(rows * p.parts)), block(32 * BM_WARPS);
    B200_CUDA(dtype == B200_F16 ? launch_dep(beam_scan_kernel<__half>, grid, block, 0, ctx->stream, 1, p)
                                : launch_dep(beam_scan_kernel<float>, grid, block, 0, ctx->stream, 1, p));
    B200_CUDA(launch_dep(beam_pick_kernel, dim3((unsigned)B), dim3((unsigned)(32 * K)), 0, ctx->stream, 1, p));
    ctx->launches += 2;
    return B200_OK;
}

} // extern "C"
