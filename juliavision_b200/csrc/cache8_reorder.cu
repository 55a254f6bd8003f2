// Beams of a search change places: beam s goes on from its parent's tokens.  Of those, whole pages change hands by their numbers, and stay
// where they are: column s of the table becomes its parent's up to the last full page.  The page that is not full is copied, its tokens and its
// maxima, from the one that the parent was writing to the one that s writes: a beam only ever writes pages of its own (`own`), one for every T
// tokens, so that no page is written that another beam reads.
//
// Bandwidth-bound: the tokens of a part-filled page, read and written, for every beam whose parent is another.  A thread takes the same 16
// bytes of all of a search's beams and reads them all before it writes any, so the beams may change places in any way without a second copy.
// 16 searches of 4 beams in 16 caches of 8 heads of 128, 55 MB in all, none of it in the L2 cache before: 16.0 us (3.4 TB/s; the copy's rate would
// give 8.3), of 5 beams in 32 caches of 20 heads of 64, 11 MB: 7.6 (6.0 with all of it there), of which a launch and three reads one after another
// are more than half: lengths, parents (which do not hang on lengths; the check of these stands between) and pages.
// A block takes a head of a cache's keys or values at a time, whatever is filled of the page, and goes on to another where there are more than 32
// blocks an SM: with 16 blocks 17.2 us, with 12 19.0; with what is moved in the L2 cache already 10.2, 10.9 and 12.5.  By 256 vectors over all
// heads, which costs three divisions a vector, 15.3 where this took 14.0; with a block for each 256 vectors of full pages 18.2 where that took 13.4.
#include "cache8.cuh"

namespace b200 {

constexpr int CR_CACHES = 128;       // of a launch
constexpr int CR_BEAMS = 32;         // of a search
constexpr int CR_THREADS = 128;

struct ReorderParams {
    uint8_t* data[2 * CR_CACHES];    // keys and values of a cache
    float* most[2 * CR_CACHES];
    CacheView c;                     // sizes and strides, the same for all; table unused
    int32_t* table;
    const int32_t *own, *parents, *lens;
    int64_t table_ld, own_ld;
    Divisor by_vectors;              // of a token and head
    int K, sides, tables;            // keys and values of all caches; whether this launch brings the table up to date
};

// What every block looks up of its search; whatever the arrays hold, it is inside the cache.
struct ReorderSearch {
    int full, kept;                  // whole pages, tokens of the next
    __device__ __forceinline__ ReorderSearch(const ReorderParams& p, int64_t search) {
        const int n = p.c.tokens((int)(search * p.K), p.lens);
        full = n >> p.c.logT;
        kept = n - (full << p.c.logT);
    }
};
__device__ __forceinline__ int cr_parent(const ReorderParams& p, int64_t search, int k) {
    const int s = p.parents[search * p.K + k];
    if (s >= 0 && s < p.K) return s;
    atomicCAS(p.c.d_status, 0, KST_BEAM_PARENT);
    return k;
}

template <int K>     // beams of a search at most
__global__ void __launch_bounds__(CR_THREADS, K <= 4 ? 12 : 1)        // 40 registers for 52: 16.5 us -> 16.0
cache_reorder_kernel(const __grid_constant__ ReorderParams p) {
    __shared__ int parent[CR_BEAMS];
    __shared__ int64_t page[CR_BEAMS], source[CR_BEAMS];          // that a beam writes, or -1; that it copies from, or -1
    const int tid = threadIdx.x;
    const int64_t search = blockIdx.y;
    grid_dep_wait();
    grid_dep_launch();
    const ReorderSearch s(p, search);
    if (tid < p.K) {
        const int from = cr_parent(p, search, tid);
        parent[tid] = from;
        int64_t pg = -1;
        if (s.kept > 0 && s.full < p.c.width) {
            pg = p.own[(search * p.K + tid) * p.own_ld + s.full];
            if (pg < 0 || pg >= p.c.P) {
                p.c.report(KST_CACHE_PAGE);
                pg = -1;
            }
        }
        page[tid] = pg;
        if (p.tables && blockIdx.x == 0 && p.lens[search * p.K + tid] != p.lens[search * p.K]) p.c.report(KST_CACHE_LENGTH);
    }
    __syncthreads();
    if (tid < p.K) source[tid] = parent[tid] != tid && page[tid] >= 0 ? page[parent[tid]] : -1;
    __syncthreads();
    if (blockIdx.x < (unsigned)p.tables) {       // the first block: the table
        for (int i = tid; i < p.c.width; i += CR_THREADS) {
            int32_t* at = p.table + search * p.K * p.table_ld + i;
            int32_t was[K];
#pragma unroll
            for (int k = 0; k < K; ++k) was[k] = k < p.K ? i < s.full ? at[parent[k] * p.table_ld] : p.own[(search * p.K + k) * p.own_ld + i] : 0;
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (k < p.K) at[k * p.table_ld] = was[k];
        }
        return;
    }
    if (s.kept == 0) return;
    const int row = s.kept * (p.c.E / 16), stride = gridDim.x - p.tables;        // vectors of a head
    for (int unit = blockIdx.x - p.tables; unit < p.sides * p.c.H; unit += stride) {
        const int side = unit / p.c.H, h = unit - side * p.c.H;
        const bool value = side & 1;
        uint8_t* head = p.data[side] + h * (value ? p.c.vH : p.c.kH);
        const int64_t pitch = value ? p.c.vP : p.c.kP, token = value ? p.c.vT : p.c.kT;
        for (int i = tid; i < row; i += CR_THREADS) {
            const int t = p.by_vectors.div(i);
            uint8_t* at = head + t * token + (i - t * (p.c.E / 16)) * 16;
            uint4 v[K];
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (k < p.K && source[k] >= 0) v[k] = *reinterpret_cast<const uint4*>(at + source[k] * pitch);
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (k < p.K && source[k] >= 0) *reinterpret_cast<uint4*>(at + page[k] * pitch) = v[k];
        }
        if (tid < 32) {              // the maxima: a lane a beam
            float* at = p.most[side] + h;
            const bool on = tid < p.K && source[tid] >= 0;
            const float v = on ? at[source[tid] * p.c.H] : 0.f;
            __syncwarp();
            if (on) at[page[tid] * p.c.H] = v;
        }
    }
}

// Whether two arrays of `columns` columns of `width` numbers have one in common.  With leading dimensions that differ, whether they lie in one another.
static bool cr_meet(const int32_t* a, int64_t a_ld, const int32_t* b, int64_t b_ld, int64_t columns, int64_t width) {
    const int64_t size = sizeof(int32_t), d = (int64_t)((uintptr_t)b - (uintptr_t)a), w = width * size;
    const int64_t a_span = (columns - 1) * a_ld * size + w, b_span = (columns - 1) * b_ld * size + w;
    if (d >= a_span || -d >= b_span) return false;
    if (columns == 1 || a_ld != b_ld) return true;
    const int64_t ld = a_ld * size, into = (d % ld + ld) % ld, apart = (d - into) / ld;       // b begins `into` bytes behind the start of a's column `apart`
    const auto inside = [&](int64_t c) { return c < columns && -c < columns; };
    return (into < w && inside(apart)) || (ld - into < w && inside(apart + 1));
}

} // namespace b200

using namespace b200;

extern "C" {

int b200_cache_reorder(b200_ctx* ctx, const b200_cache8* caches, int64_t n, int64_t K, int64_t B, int32_t* table, int64_t table_ld,
                       const int32_t* own, int64_t own_ld, int64_t width, const int32_t* parents, const int32_t* lens) {
    B200_REQUIRE(ctx && (caches || n <= 0), B200_EINVAL, "cache_reorder: null argument");
    B200_REQUIRE(n >= 1 && K >= 0 && B >= 0, B200_EINVAL, "cache_reorder: %lld caches, K=%lld B=%lld", (long long)n, (long long)K, (long long)B);
    B200_REQUIRE(K <= CR_BEAMS && B < 65536, B200_DECLINE_EXTENT, "cache_reorder: %lld beams (at most %d), %lld searches", (long long)K, CR_BEAMS, (long long)B);
    if (K == 0 || B == 0) return B200_OK;
    B200_REQUIRE(table && own && parents && lens, B200_EINVAL, "cache_reorder: null array");
    B200_REQUIRE(own_ld >= width, B200_DECLINE_EXTENT, "cache_reorder: leading dimension %lld of %lld pages", (long long)own_ld, (long long)width);
    ReorderParams p = {};
    for (int64_t i = 0; i < n; ++i) {            // all of them, before the first launch
        b200_cache8 c = caches[i];
        c.table = table, c.table_ld = table_ld, c.width = width;
        CacheView v;
        int rc = cache_view(ctx, &c, "cache_reorder", &v);
        if (rc) return rc;
        if (i == 0) p.c = v;
        B200_REQUIRE(v.E == p.c.E && v.T == p.c.T && v.H == p.c.H && v.P == p.c.P && v.kT == p.c.kT && v.kH == p.c.kH && v.kP == p.c.kP &&
                         v.vT == p.c.vT && v.vH == p.c.vH && v.vP == p.c.vP,
                     B200_DECLINE_EXTENT, "cache_reorder: cache %lld has other sizes or strides than the first", (long long)i);
        bool twice = c.k == c.v;                 // moved twice at the same time
        for (int64_t j = 0; j < i; ++j) twice |= caches[j].k == c.k || caches[j].v == c.v || caches[j].k == c.v || caches[j].v == c.k;
        B200_REQUIRE(!twice, B200_EINVAL, "cache_reorder: the array of cache %lld is given twice", (long long)i);
    }
    // A table over `own` would overwrite with the parents' pages what says which pages a beam writes; two beams could then write one.
    B200_REQUIRE(!cr_meet(table, table_ld, own, own_ld, K * B, width), B200_EINVAL, "cache_reorder: table and own share memory");
    p.by_vectors = Divisor::of(p.c.E / 16);
    B200_CUDA(cudaSetDevice(ctx->device));
    p.table = table, p.table_ld = table_ld, p.own = own, p.own_ld = own_ld;
    p.parents = parents, p.lens = lens;
    p.K = (int)K;
    for (int64_t at = 0; at < n; at += CR_CACHES) {
        const int count = (int)(n - at < CR_CACHES ? n - at : CR_CACHES);
        for (int i = 0; i < count; ++i) {
            const b200_cache8& c = caches[at + i];
            p.data[2 * i] = (uint8_t*)c.k, p.data[2 * i + 1] = (uint8_t*)c.v;
            p.most[2 * i] = c.kmax, p.most[2 * i + 1] = c.vmax;
        }
        p.tables = at == 0;
        p.sides = 2 * count;
        const int64_t share = cdiv(32 * (int64_t)ctx->prop.multiProcessorCount, B), units = p.sides * (int64_t)p.c.H;      // 32 blocks an SM
        const int64_t grid = p.tables + (units < share ? units : share);
        const dim3 g((unsigned)grid, (unsigned)B), b(CR_THREADS);
        auto run = [&](auto kern) { return launch_dep(kern, g, b, 0, ctx->stream, 1, p); };
        B200_CUDA(K <= 4 ? run(cache_reorder_kernel<4>) : K <= 8 ? run(cache_reorder_kernel<8>) : K <= 16 ? run(cache_reorder_kernel<16>)
                                                                                                        : run(cache_reorder_kernel<32>));
        ctx->launches++;
    }
    return B200_OK;
}

} // extern "C"
