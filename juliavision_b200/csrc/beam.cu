// Beam search's choice: of the K V continuations of a search's beams,
//     c[k, v] = score[k] + x[k, v] - log sum_u exp x[k, u],
// the N largest, in order, ties to the lowest k V + v.  An ended beam has one continuation, the padding token at its own score.
//
// Every logit is read once: 64 searches of 8 beams of 131072 halves are 134 MB, 20.5 us at the copy's rate, and take 37.5 (3.6 TB/s; 1 x 5 x 51865:
// 8.4, two launches).  What bounds it is instructions: an exponential, its conversion, difference, product and sum are five issues a lane for two
// elements and two of the exponential unit's turns (18 us of them), and the rest goes into finding candidates.  Within a beam the order is that
// of the logits, so the first launch needs no sums to choose by, and one pass does.
//
// A block walks a share of a row, a tile of 4 or 8 vectors a lane at a time; a lane keeps the sum of exponentials relative to its own running
// maximum, in fp32.  The choice goes by a bound that at least N elements of the block reach: in each of W warps the ceil(N / W)th largest of the
// lanes' running maxima, and the least of those over the warps; some two or three times N elements of the first tile do.  Vectors whose maximum
// reaches it are looked at again, and those elements are set down as 64-bit keys (the logit's bits in order, then the index from above), of
// which no two are alike, in shared memory; the block sorts what is there at the end.  (A list a warp, into which each candidate was put in
// order, took 57 us.)  Rows with more candidates than there is room, ties of thousands or logits that rise all along, put the others into
// a list of the warp's 32 largest, one a lane.  The second launch, a block a search, merges a row's parts, takes log sums and scores in fp64
// and merges the rows'.
#include <cfloat>
#include <cuda_fp16.h>

#include "internal.h"
#include "ptx.cuh"

namespace b200 {

constexpr int BM_WARPS = 8;          // of a scanning block
constexpr int BM_FOUND = 1024;      // candidates that a block sets down
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
    int K, N, parts, pad, tiles;     // tiles of a block
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

// One key into the list.
__device__ __forceinline__ void bm_insert(unsigned long long& list, unsigned long long key) {
    const int lane = threadIdx.x & 31, at = __popc(__ballot_sync(0xffffffffu, list > key));
    const unsigned long long before = __shfl_up_sync(0xffffffffu, list, 1);
    list = lane < at ? list : lane == at ? key : before;
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
    static __device__ __forceinline__ float one(const __half* x) { return __half2float(__ldg(x)); }
    static __device__ __forceinline__ float most(uint4 r) {        // the largest that is a number
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
        const __half2* h = reinterpret_cast<const __half2*>(w);
        const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return __half2float(__hmax(__low2half(m), __high2half(m)));
    }
    static __device__ __forceinline__ uint4 none() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }      // -inf
    static __device__ __forceinline__ void drop(uint4& r, int i) {
        uint32_t& w = i < 4 ? (i < 2 ? r.x : r.y) : (i < 6 ? r.z : r.w);
        w = i & 1 ? (w & 0xffffu) | 0xfc000000u : (w & 0xffff0000u) | 0xfc00u;
    }
};
template <> struct BmVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(float* v, uint4 r) {
        v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ float one(const float* x) { return __ldg(x); }
    static __device__ __forceinline__ float most(uint4 r) {
        return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
    }
    static __device__ __forceinline__ uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
    static __device__ __forceinline__ void drop(uint4& r, int i) { (i < 2 ? (i ? r.y : r.x) : (i < 3 ? r.z : r.w)) = 0xff800000u; }
};

// 2^((x - ref) log2 e): the difference first, whose error is its own and not the logit's.
__device__ __forceinline__ float bm_weight(float x, float ref) { return bm_ex2((x - ref) * 1.4426950408889634f); }

template <typename T, int U>       // vectors of a lane's tile
__global__ void __launch_bounds__(32 * BM_WARPS, 4)
beam_scan_kernel(const BeamParams p) {
    using Vec = BmVec<T>;
    __shared__ unsigned long long found[BM_FOUND], lists[BM_WARPS][32];
    __shared__ float2 sums[BM_WARPS];
    __shared__ volatile uint32_t bounds[BM_WARPS];     // in order
    __shared__ uint32_t count;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x / p.parts, part_of_row = blockIdx.x - row * p.parts;
    grid_dep_wait();
    grid_dep_launch();
    const T* x = (const T*)p.x + row / p.K * p.ldb + row % p.K * p.ldk;
    // vectors from the 16-byte boundary at or below the row's first element; what is not of the row is taken as -inf
    const int skew = (int)((uintptr_t)x % 16 / sizeof(T));
    const uint4* base = reinterpret_cast<const uint4*>(x - skew);
    constexpr int TILE = BM_WARPS * 32 * U;
    const int end = (int)((p.V + skew + Vec::N - 1) / Vec::N), block0 = (int)part_of_row * (p.tiles * TILE);
    const int stop = block0 + p.tiles * TILE < end ? block0 + p.tiles * TILE : end;
    unsigned long long list = 0;                     // no element's key is 0
    float m = -INFINITY, s = 0.f;
    if (threadIdx.x == 0) count = 0;                 // read behind a barrier, of a block behind the row's end too
    const int full = (end - block0) / (32 * U), warps = full < BM_WARPS ? full : BM_WARPS;      // warps with an element in every lane
#pragma unroll 1
    for (int tile = block0; tile < stop; tile += TILE) {
        const int at = tile + warp * (32 * U);
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            raw[u] = Vec::none();
            if (at + u * 32 + lane < end) raw[u] = __ldg(base + at + u * 32 + lane);
        }
        if (at == 0 || at + 32 * U > end - 1) {      // a row's first and last vectors
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t i = (int64_t)(at + u * 32 + lane) * Vec::N - skew;
                if (i < 0 || i + Vec::N > p.V)
#pragma unroll
                    for (int k = 0; k < Vec::N; ++k)
                        if (i + k < 0 || i + k >= p.V) Vec::drop(raw[u], k);
            }
        }
        float most[U], high = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            most[u] = Vec::most(raw[u]);
            high = fmaxf(high, most[u]);
        }
        // the sum
        {
            const float ref = high == -INFINITY ? 0.f : high;
            const uint64_t less = pack2(-ref, -ref), unit = pack2(1.4426950408889634f, 1.4426950408889634f);
            uint64_t sum0 = pack2(m == high ? s : s * bm_weight(m, ref), 0.f), sum1 = pack2(0.f, 0.f);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float v[Vec::N];
                Vec::load(v, raw[u]);
#pragma unroll
                for (int e = 0; e < Vec::N; e += 2) {
                    float a, b;
                    unpack2(mul2(add2(pack2(v[e], v[e + 1]), less), unit), a, b);
                    uint64_t& sum = (e >> 1) & 1 ? sum1 : sum0;
                    sum = add2(sum, pack2(bm_ex2(a), bm_ex2(b)));
                }
            }
            float a, b;
            unpack2(add2(sum0, sum1), a, b);
            s = a + b;
            m = high;
        }
        // the bound: what the others set down may be an older one, which holds as well
        if (warps > 0) {
            uint32_t left = bm_order(m), nth = 0;
            for (int q = (p.N + warps - 1) / warps; q > 0; --q) {
                nth = __reduce_max_sync(0xffffffffu, left);
                if (lane == __ffs(__ballot_sync(0xffffffffu, left == nth)) - 1) left = 0;
            }
            if (lane == 0) bounds[warp] = warp < warps ? nth : 0xffffffffu;
        }
        if (tile == block0) __syncthreads();
        // -inf is no candidate, however few others a row has: the second launch knows which tokens come then (1500 of 131072 allowed, 64 searches
        // of 8 beams: 60 us, 176 with all of them in lists)
        const float bound = fmaxf(warps > 0 ? bm_number(__reduce_min_sync(0xffffffffu, bounds[lane & (BM_WARPS - 1)])) : -INFINITY, -FLT_MAX);
        // the candidates
        uint32_t hits = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) hits |= (uint32_t)(most[u] >= bound) << u;
        while (__any_sync(0xffffffffu, hits != 0)) {
            uint32_t some = 0;
            int first = 0;                                  // the vector's first element; below 0 in a row's first vector, of a row that is not aligned
            if (hits) {
                const int at_vec = at + (__ffs(hits) - 1) * 32 + lane;
                hits &= hits - 1;
                if (at_vec < end) {
                    float v[Vec::N];
                    Vec::load(v, __ldg(base + at_vec));
#pragma unroll
                    for (int k = 0; k < Vec::N; ++k) some |= (uint32_t)(v[k] >= bound) << k;
                    const int64_t i = (int64_t)at_vec * Vec::N - skew;
                    first = (int)i;
                    if (i < 0) some &= ~0u << -first;
                    if (i + Vec::N > p.V) some &= (1u << (int)(p.V - i)) - 1;
                    uint32_t to = atomicAdd(&count, __popc(some));
                    for (; some && to < BM_FOUND; some &= some - 1) {
                        const int k = first + __ffs(some) - 1;
                        found[to++] = bm_key(Vec::one(x + k), (uint32_t)k);
                    }
                }
            }
            if (__any_sync(0xffffffffu, some != 0)) {       // no room: into the warp's list, if above its Nth
                unsigned long long most_key = 0;
                for (uint32_t c = some; c; c &= c - 1) {
                    const int k = first + __ffs(c) - 1;
                    const unsigned long long key = bm_key(Vec::one(x + k), (uint32_t)k);
                    most_key = key > most_key ? key : most_key;
                }
                unsigned long long nth = __shfl_sync(0xffffffffu, list, p.N - 1);
                if (!__any_sync(0xffffffffu, most_key > nth)) continue;
#pragma unroll 1
                for (int k = 0; k < Vec::N; ++k) {
                    unsigned long long key = some >> k & 1 ? bm_key(Vec::one(x + first + k), (uint32_t)(first + k)) : 0;
                    unsigned above;
                    while ((above = __ballot_sync(0xffffffffu, key > nth)) != 0) {       // one at a time
                        const int from = __ffs(above) - 1;
                        bm_insert(list, __shfl_sync(0xffffffffu, key, from));
                        nth = __shfl_sync(0xffffffffu, list, p.N - 1);
                        if (lane == from) key = 0;
                    }
                }
            }
        }
    }
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const float om = __shfl_xor_sync(0xffffffffu, m, d), os = __shfl_xor_sync(0xffffffffu, s, d), high = fmaxf(m, om);
        const float ref = high == -INFINITY ? 0.f : high;
        s = s * (m == high ? 1.f : bm_weight(m, ref)) + os * (om == high ? 1.f : bm_weight(om, ref));
        m = high;
    }
    if (lane == 0) sums[warp] = make_float2(m, s);
    __syncthreads();
    const int set = count < BM_FOUND ? count : BM_FOUND, busy = count > BM_FOUND ? BM_WARPS : (set + 31) / 32;      // warps with a list
    for (int c = warp * 32; c < set; c += BM_WARPS * 32) list = bm_merge(list, bm_sort<false>(c + lane < set ? found[c + lane] : 0));
    lists[warp][lane] = list;
#pragma unroll
    for (int d = BM_WARPS / 2; d > 0; d /= 2) {
        if (d >= busy) continue;
        __syncthreads();
        if (warp < d && warp + d < busy) {
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
            for (int w = 0; w < BM_WARPS; ++w) total += sums[w].y * (sums[w].x == high ? 1.f : bm_weight(sums[w].x, ref));
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
        const float score0 = p.score[row];
        const bool ended = p.ended != nullptr && p.ended[row] != 0;
        const float2 first = lane < p.parts ? p.sums[row * p.parts + lane] : make_float2(-INFINITY, 0.f);
        unsigned long long list = 0;
        float m = first.x;
        double s = 0;
        for (int i = 0; i < p.parts; i += 4) {
            unsigned long long next[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) next[j] = i + j < p.parts && lane < p.N ? p.keys[(row * p.parts + i + j) * p.N + lane] : 0;
            if (i + 2 < p.parts) list = bm_merge(list, bm_merge(bm_merge(next[0], next[1]), bm_merge(next[2], next[3])));
            else list = bm_merge(list, i + 1 < p.parts ? bm_merge(next[0], next[1]) : next[0]);
        }
        for (int i = lane + 32; i < p.parts; i += 32) m = fmaxf(m, p.sums[row * p.parts + i].x);
#pragma unroll
        for (int d = 1; d < 32; d *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        for (int i = lane; i < p.parts; i += 32) {
            const float2 x = i == lane ? first : p.sums[row * p.parts + i];
            if (m > -INFINITY) s += (double)x.y * exp((double)x.x - (double)m);
        }
#pragma unroll
        for (int d = 1; d < 32; d *= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
        const double score = (double)score0, sum = (double)m + log(s);
        const bool over = !(score < INFINITY && score > -INFINITY);
        double value = -INFINITY;
        uint32_t token = (uint32_t)lane;                            // of a beam that offers nothing: the first tokens
        bool some = lane < p.V;
        if (ended) {
            token = lane == 0 ? (uint32_t)p.pad : (uint32_t)(lane - 1 + (lane - 1 >= p.pad));
            if (lane == 0 && !over) value = score;
            if (over) token = (uint32_t)lane;
        } else if (!over && sum < INFINITY && sum > -INFINITY) {
            const int found = __popc(__ballot_sync(0xffffffffu, list != 0 && lane < p.N));
            token = ~(uint32_t)list;
            if (list != 0) value = score + ((double)bm_number((uint32_t)(list >> 32)) - sum);
            if (found < p.N) {              // then those at -inf, lowest first: the lane - found th that is not listed
                uint32_t t = (uint32_t)(lane - found);
                for (int round = 0; round < found; ++round) {
                    uint32_t below = 0;
                    for (int i = 0; i < found; ++i) below += __shfl_sync(0xffffffffu, token, i) <= t;
                    t = (uint32_t)(lane - found) + below;
                }
                if (lane >= found) token = t;
                some = lane < found || (int64_t)t < p.V;
            } else {
                some = true;
            }
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
    const int per = dtype == B200_F16 ? 8 : 4;
    const bool whole = ((uintptr_t)logits % 16 | (uint64_t)ldk % per | (uint64_t)ldb % per) == 0;      // rows start on 16-byte boundaries
    const int64_t rows = B * K, vectors = cdiv(whole ? V : V + per - 1, per), sms = ctx->prop.multiProcessorCount;
    // Tiles of 8 vectors a lane where that leaves two blocks an SM (512 rows of 131072 halves: 37.5 us, with 4 53), else of 4 (5 rows of 51865:
    // 8.4, with 2 9.7, with 1 11.7: the more parts, the longer the second launch).  As many tiles a block as leave six blocks an SM, four of
    // which are resident: each block's first tile gives candidates (512 rows: 4 tiles 37.5, 3 tiles 41).
    const int U = rows * cdiv(vectors, 32 * BM_WARPS * 8) >= 2 * sms ? 8 : 4;
    const int64_t tiles = cdiv(vectors, 32 * BM_WARPS * U), each = tiles * rows / (6 * sms);
    p.tiles = (int)(each < 1 ? 1 : each < tiles ? each : tiles);
    p.parts = (int)cdiv(tiles, p.tiles);
    B200_REQUIRE(rows * p.parts < (1ll << 31), B200_DECLINE_EXTENT, "beam_select: %lld beams of %lld in all", (long long)rows, (long long)V);
    void* ws = nullptr;
    int rc = ws_scratch(ctx, (size_t)(rows * p.parts) * (N * sizeof(unsigned long long) + sizeof(float2)), &ws);
    if (rc) return rc;
    p.keys = (unsigned long long*)ws;
    p.sums = (float2*)(p.keys + rows * p.parts * N);
    const dim3 grid((unsigned)(rows * p.parts)), block(32 * BM_WARPS);
    auto run = [&](auto kern) { return launch_dep(kern, grid, block, 0, ctx->stream, 1, p); };
    cudaError_t e;
    if (dtype == B200_F16) e = U == 8 ? run(beam_scan_kernel<__half, 8>) : run(beam_scan_kernel<__half, 4>);
    else e = U == 8 ? run(beam_scan_kernel<float, 8>) : run(beam_scan_kernel<float, 4>);
    B200_CUDA(e);
    B200_CUDA(launch_dep(beam_pick_kernel, dim3((unsigned)B), dim3((unsigned)(32 * K)), 0, ctx->stream, 1, p));
    ctx->launches += 2;
    return B200_OK;
}

} // extern "C"
