// Writing tokens into the paged 8-bit cache and reading them back (cache8.cuh has the format).  Two bytes read and one written an
// element, or the reverse, so HBM is the floor; what comes first is instructions, 19 an element written.  13600 tokens of four
// sequences, 8 heads of 128: keys and values written in 21 us (3.9 TB/s), each read back as fp16 in 11.6 us (3.6 TB/s).
//
// Append: one block owns one (sequence, page, head) of the keys or of the values, so nothing is shared between blocks.  It holds
// the page's new elements in registers (up to 64 a thread), takes their largest magnitude as an integer maximum over the fp16
// bits, which a NaN or an infinity wins, and writes the quotients.  A page that holds earlier tokens keeps its m unless the
// new tokens exceed it; then the earlier values are brought to the larger m, a second rounding of at most half a step.  A page
// whose m is not finite is stored as zeros under a NaN, so that whoever attends to the page sees it.
#include <cuda_fp16.h>

#include "cache8.cuh"

namespace b200 {

constexpr int CA_THREADS = 256;

int cache_view(b200_ctx* ctx, const b200_cache8* c, const char* op, CacheView* out) {
    B200_REQUIRE(ctx && c, B200_EINVAL, "%s: null argument", op);
    B200_REQUIRE(c->kind == B200_I8 || c->kind == B200_E4M3, B200_DECLINE_ELTYPE, "%s: cache kind %d", op, c->kind);
    B200_REQUIRE(c->E >= 16 && c->E <= 128 && c->E % 16 == 0, B200_DECLINE_EXTENT, "%s: head dim %lld (a multiple of 16 up to 128)", op,
                 (long long)c->E);
    B200_REQUIRE(c->T >= 16 && c->T <= CACHE_MOST_T && (c->T & (c->T - 1)) == 0, B200_DECLINE_EXTENT,
                 "%s: %lld tokens a page (16, 32, 64 or 128)", op, (long long)c->T);
    B200_REQUIRE(c->H >= 1 && c->H < 65536 && c->P >= 1 && c->P < (1ll << 31), B200_DECLINE_EXTENT, "%s: %lld heads, %lld pages", op,
                 (long long)c->H, (long long)c->P);
    B200_REQUIRE(c->width >= 1 && c->width * c->T <= (1ll << 30) && c->table_ld >= c->width, B200_DECLINE_EXTENT,
                 "%s: a table of %lld pages a sequence, leading dimension %lld", op, (long long)c->width, (long long)c->table_ld);
    B200_REQUIRE(c->k && c->v && c->kmax && c->vmax && c->table, B200_EINVAL, "%s: null array", op);
    uint64_t odd = (uintptr_t)c->k | (uintptr_t)c->v;
    for (int i = 1; i < 4; ++i) odd |= (uint64_t)c->kstride[i] | (uint64_t)c->vstride[i];
    B200_REQUIRE(odd % 16 == 0 && c->kstride[0] == 1 && c->vstride[0] == 1, B200_DECLINE_ALIGN,
                 "%s: a page's rows must be contiguous and start on 16-byte boundaries", op);
    out->k = (uint8_t*)c->k, out->v = (uint8_t*)c->v;
    out->kT = c->kstride[1], out->kH = c->kstride[2], out->kP = c->kstride[3];
    out->vT = c->vstride[1], out->vH = c->vstride[2], out->vP = c->vstride[3];
    out->kmax = c->kmax, out->vmax = c->vmax;
    out->table = c->table;
    out->table_ld = c->table_ld, out->P = c->P;
    out->E = (int)c->E, out->T = (int)c->T, out->H = (int)c->H, out->width = (int)c->width;
    out->logT = 0;
    while ((1 << out->logT) < out->T) ++out->logT;
    out->d_status = ctx->d_status;
    return B200_OK;
}

struct AppendParams {
    CacheView c;
    const __half *k, *v;
    int64_t kL, kH, kB, vL, vH, vB;
    const int32_t *lens, *news;
    int L, blocks;   // pages a sequence's new tokens can touch
    int whole;       // rows of k and v start on 16-byte boundaries
    Divisor per;     // eights of a row
};

// a / m of two numbers, rounded to nearest, a exact: the product by r = 1 / m corrected once by its residual (Markstein).  Where
// a / m is a number of fp32 the residual is exact and so is the result.  Two at a time, since what an element costs here is
// instructions (28 M elements of keys and values: one at a time 24 us).
__device__ __forceinline__ float2 ca_quotients(float2 x, float f, float m, float r) {
    const uint64_t a = mul2(pack2(x.x, x.y), pack2(f, f)), r2 = pack2(r, r), t = mul2(a, r2);
    float2 q;
    unpack2(fma2(fma2(t, pack2(-m, -m), a), r2, t), q.x, q.y);
    return q;
}
__device__ __forceinline__ float2 ca_float2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
// four quotients as 8-bit values
template <bool FP8> __device__ __forceinline__ uint32_t ca_pack(float a, float b, float c, float d) {
    if constexpr (FP8) {
        uint32_t w;
        asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
            : "=r"(w) : "f"(a), "f"(b), "f"(c), "f"(d));
        return w;
    } else {   // 1.5 * 2^23 more: the sum's low byte is the nearest integer, ties to even
        const uint64_t one = pack2(12582912.f, 12582912.f);
        float x, y, z, w;
        unpack2(add2(pack2(a, b), one), x, y);
        unpack2(add2(pack2(c, d), one), z, w);
        return __byte_perm(__byte_perm(__float_as_uint(x), __float_as_uint(y), 0x0040), __byte_perm(__float_as_uint(z), __float_as_uint(w), 0x0040), 0x5410);
    }
}

// NV: vectors of eight elements a thread holds
template <bool FP8, int NV>
__global__ void __launch_bounds__(CA_THREADS)
cache_append_kernel(const AppendParams p) {
    __shared__ uint32_t tops[CA_THREADS / 32];
    const CacheView& c = p.c;
    const int tid = threadIdx.x, h = blockIdx.y, side = blockIdx.x & 1;
    const unsigned at = blockIdx.x >> 1;
    const int b = at / p.blocks, j = at - b * p.blocks;
    grid_dep_wait();
    grid_dep_launch();
    const int n = c.tokens(b, p.lens), m = c.fresh(b, p.news, p.L);
    const int start = n - m > 0 ? n - m : 0, first = start >> c.logT, blk = first + j;
    if (m == 0 || n == 0 || (blk << c.logT) >= n) return;   // uniform over the block
    const int64_t page = c.page(b, blk);
    if (page < 0) return;
    const int t0 = blk << c.logT, lo = start > t0 ? start - t0 : 0, hi = n - t0 < c.T ? n - t0 : c.T;
    const int64_t srcL = side ? p.vL : p.kL;
    // token t0 + row is row t0 + row - (n - m) of the new ones
    const __half* src = (side ? p.v + b * p.vB + h * p.vH : p.k + b * p.kB + h * p.kH) + (t0 - (n - m)) * srcL;
    const int64_t dstT = side ? c.vT : c.kT;
    uint8_t* dst = side ? c.v + page * c.vP + h * c.vH : c.k + page * c.kP + h * c.kH;
    float* top_at = (side ? c.vmax : c.kmax) + page * c.H + h;
    const int per = c.E / 8;
    uint4 x[NV];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = tid + i * CA_THREADS, r0 = p.per.div(at), row = lo + r0, e = (at - r0 * per) * 8;
        x[i] = make_uint4(0, 0, 0, 0);
        if (row < hi) {
            const __half* s = src + row * srcL + e;
            if (p.whole) {
                x[i] = __ldg(reinterpret_cast<const uint4*>(s));
            } else {
                const unsigned short* u = reinterpret_cast<const unsigned short*>(s);
                x[i] = make_uint4(u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t a = __vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu), d = __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu);
        top = __vmaxu2(top, __vmaxu2(a, d));
    }
    top = __reduce_max_sync(0xffffffffu, top >> 16 > (top & 0xffff) ? top >> 16 : top & 0xffff);
    if ((tid & 31) == 0) tops[tid >> 5] = top;
    const float was = lo > 0 ? *top_at : 0.f;
    __syncthreads();   // also: every thread has read m before one of them replaces it
#pragma unroll
    for (int i = 0; i < CA_THREADS / 32; ++i) top = max(top, tops[i]);
    float most = __half2float(__ushort_as_half((unsigned short)top));
    if (was > most || was != was) most = was;             // a NaN stays
    const bool finite = most < INFINITY;                  // false for a NaN
    const float r = finite && most > 0.f ? 1.f / most : 0.f;
    if (!finite) most = __int_as_float(0x7fffffff);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = tid + i * CA_THREADS, r0 = p.per.div(at), row = lo + r0, e = (at - r0 * per) * 8;
        if (row >= hi) continue;
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint2 q = make_uint2(0, 0);
        if (finite) {
            float2 f[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = ca_quotients(ca_float2(w[k]), cache_top<FP8>(), most, r);
            q = make_uint2(ca_pack<FP8>(f[0].x, f[0].y, f[1].x, f[1].y), ca_pack<FP8>(f[2].x, f[2].y, f[3].x, f[3].y));
        }
        *reinterpret_cast<uint2*>(dst + row * dstT + e) = q;
    }
    if (lo > 0 && !(most == was)) {   // the earlier tokens' values under the larger m
        for (int at = tid; at < lo * per; at += CA_THREADS) {
            uint2* d = reinterpret_cast<uint2*>(dst + at / per * dstT + at % per * 8);
            uint2 q = make_uint2(0, 0);
            if (finite) {
                const uint2 old = *d;
                const uint32_t w[2] = {old.x, old.y};
                uint32_t o[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t lo2, hi2;
                    cache_halves<FP8>(w[k], lo2, hi2);
                    const float2 g = ca_quotients(ca_float2(lo2), was, most, r), l = ca_quotients(ca_float2(hi2), was, most, r);
                    o[k] = ca_pack<FP8>(g.x, g.y, l.x, l.y);
                }
                q = make_uint2(o[0], o[1]);
            }
            *d = q;
        }
    }
    if (tid == 0) *top_at = most;
}

struct ReadParams {
    CacheView c;
    int side, L, rows, blocks;   // rows of a block, blocks of a sequence
    Divisor per, heads;          // sixteens of a head, heads of a row
    const int32_t *starts, *lens;
    void* out;
    int64_t oL, oH, oB;
    int whole;
};

template <bool FP8, typename OutT>
__global__ void __launch_bounds__(CA_THREADS)
cache_read_kernel(const ReadParams p) {
    const CacheView& c = p.c;
    grid_dep_wait();
    grid_dep_launch();
    const int per = c.E / 16, b = blockIdx.x / p.blocks, row0 = (blockIdx.x - b * p.blocks) * p.rows;
    const int rows = p.L - row0 < p.rows ? p.L - row0 : p.rows;
    const float inv = 1.f / cache_top<FP8>();
    const int n = c.tokens(b, p.lens), from = p.starts != nullptr ? p.starts[b] : 0;
    const int64_t first = (int64_t)from + row0;
    if (first >= n || first + rows <= 0) return;
    constexpr int AT_ONCE = 2;        // sixteens of elements a thread has on their way: each is two trips, for the page's number and for it
    const int all = rows * c.H * per;
    for (int i0 = threadIdx.x; i0 < all; i0 += AT_ONCE * CA_THREADS) {
        uint4 w4[AT_ONCE];
        float most[AT_ONCE];
        int64_t at[AT_ONCE];
        bool live[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int i = i0 + u * CA_THREADS, a = p.per.div(i), e = (i - a * per) * 16, r = p.heads.div(a), h = a - r * c.H;
            const int64_t token = first + r;
            live[u] = i < all && token >= 0 && token < n;
            const int64_t page = live[u] ? c.page(b, (int)(token >> c.logT)) : -1;
            live[u] = page >= 0;
            const int in = (int)token & (c.T - 1);
            at[u] = (int64_t)b * p.oB + (row0 + r) * p.oL + h * p.oH + e;
            w4[u] = make_uint4(0, 0, 0, 0);
            most[u] = 0.f;
            if (live[u]) {
                w4[u] = *reinterpret_cast<const uint4*>(p.side ? c.v + page * c.vP + h * c.vH + in * c.vT + e : c.k + page * c.kP + h * c.kH + in * c.kT + e);
                most[u] = (p.side ? c.vmax : c.kmax)[page * c.H + h];
            }
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            if (!live[u]) continue;
            const uint32_t w[4] = {w4[u].x, w4[u].y, w4[u].z, w4[u].w};
            OutT* o = (OutT*)p.out + at[u];
            float2 f[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t lo, hi;
                cache_halves<FP8>(w[k], lo, hi);
                f[2 * k] = ca_quotients(ca_float2(lo), most[u], cache_top<FP8>(), inv);
                f[2 * k + 1] = ca_quotients(ca_float2(hi), most[u], cache_top<FP8>(), inv);
            }
            if (sizeof(OutT) == 2 && p.whole) {
                uint32_t r[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const __half2 v = __floats2half2_rn(f[k].x, f[k].y);
                    r[k] = *reinterpret_cast<const uint32_t*>(&v);
                }
                reinterpret_cast<uint4*>(o)[0] = make_uint4(r[0], r[1], r[2], r[3]);
                reinterpret_cast<uint4*>(o)[1] = make_uint4(r[4], r[5], r[6], r[7]);
            } else if (p.whole) {
#pragma unroll
                for (int k = 0; k < 4; ++k) reinterpret_cast<float4*>(o)[k] = make_float4(f[2 * k].x, f[2 * k].y, f[2 * k + 1].x, f[2 * k + 1].y);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    o[2 * k] = (OutT)f[k].x;
                    o[2 * k + 1] = (OutT)f[k].y;
                }
            }
        }
    }
}

template <bool FP8>
static int append_launch(b200_ctx* ctx, const AppendParams& p, int64_t B) {
    const int64_t vectors = (int64_t)p.c.T * p.c.E / 8;
    const int64_t gx = 2 * B * p.blocks;
    B200_REQUIRE(gx < (1ll << 31), B200_DECLINE_EXTENT, "cache_append: %lld sequences of %d pages", (long long)B, p.blocks);
    auto kern = vectors <= CA_THREADS ? cache_append_kernel<FP8, 1> : vectors <= 2 * CA_THREADS ? cache_append_kernel<FP8, 2>
              : vectors <= 4 * CA_THREADS ? cache_append_kernel<FP8, 4> : cache_append_kernel<FP8, 8>;
    B200_CUDA(launch_dep(kern, dim3((unsigned)gx, (unsigned)p.c.H), dim3(CA_THREADS), 0, ctx->stream, 1, p));
    ctx->launches++;
    return B200_OK;
}

} // namespace b200

using namespace b200;

extern "C" {

int b200_cache_append(b200_ctx* ctx, const b200_cache8* cache, int64_t L, int64_t B, const b200_strided4* k, const b200_strided4* v,
                      const int32_t* lens, const int32_t* news) {
    AppendParams p = {};
    int rc = cache_view(ctx, cache, "cache_append", &p.c);
    if (rc) return rc;
    B200_REQUIRE(k && v, B200_EINVAL, "cache_append: null argument");
    B200_REQUIRE(L >= 0 && B >= 0 && L < (1ll << 30) && B < (1ll << 30), B200_EINVAL, "cache_append: L=%lld B=%lld", (long long)L, (long long)B);
    if (L == 0 || B == 0) return B200_OK;
    B200_REQUIRE(k->ptr && v->ptr && lens, B200_EINVAL, "cache_append: null array");
    B200_REQUIRE(k->stride[0] == 1 && v->stride[0] == 1, B200_DECLINE_ALIGN, "cache_append: E is not contiguous");
    p.k = (const __half*)k->ptr, p.v = (const __half*)v->ptr;
    p.kL = k->stride[1], p.kH = k->stride[2], p.kB = k->stride[3];
    p.vL = v->stride[1], p.vH = v->stride[2], p.vB = v->stride[3];
    p.lens = lens, p.news = news;
    p.L = (int)L;
    p.blocks = (int)((L + p.c.T - 2) / p.c.T + 1);
    if (p.blocks > p.c.width) p.blocks = p.c.width;
    uint64_t odd = ((uintptr_t)k->ptr | (uintptr_t)v->ptr) % 16;
    for (int i = 1; i < 4; ++i) odd |= ((uint64_t)k->stride[i] | (uint64_t)v->stride[i]) % 8;
    p.whole = odd == 0;
    p.per = Divisor::of(p.c.E / 8);
    B200_CUDA(cudaSetDevice(ctx->device));
    return cache->kind == B200_E4M3 ? append_launch<true>(ctx, p, B) : append_launch<false>(ctx, p, B);
}

int b200_cache_read(b200_ctx* ctx, const b200_cache8* cache, int values, int64_t L, int64_t B, const int32_t* starts, const int32_t* lens,
                    const b200_strided4* out, int out_dtype) {
    ReadParams p = {};
    int rc = cache_view(ctx, cache, "cache_read", &p.c);
    if (rc) return rc;
    B200_REQUIRE(out, B200_EINVAL, "cache_read: null argument");
    B200_REQUIRE(L >= 0 && B >= 0 && L < (1ll << 30) && B < (1ll << 30), B200_EINVAL, "cache_read: L=%lld B=%lld", (long long)L, (long long)B);
    B200_REQUIRE(out_dtype == B200_F16 || out_dtype == B200_F32, B200_DECLINE_ELTYPE, "cache_read: out dtype %d", out_dtype);
    if (L == 0 || B == 0) return B200_OK;
    B200_REQUIRE(out->ptr && lens, B200_EINVAL, "cache_read: null array");
    B200_REQUIRE(out->stride[0] == 1, B200_DECLINE_ALIGN, "cache_read: E is not contiguous");
    const int64_t size = out_dtype == B200_F16 ? 2 : 4;
    p.side = values != 0;
    p.L = (int)L;
    p.starts = starts, p.lens = lens;
    p.out = const_cast<void*>(out->ptr);
    p.oL = out->stride[1], p.oH = out->stride[2], p.oB = out->stride[3];
    p.whole = ((uintptr_t)out->ptr | (uint64_t)(out->stride[1] * size) | (uint64_t)(out->stride[2] * size) | (uint64_t)(out->stride[3] * size)) % 16 == 0;
    B200_CUDA(cudaSetDevice(ctx->device));
    // rows of a block: two steps a thread, as long as there are blocks for the GPU
    const int64_t per_row = (int64_t)p.c.H * (p.c.E / 16);
    int64_t rows = 1;
    while (rows * per_row < 2 * CA_THREADS && cdiv(L, 2 * rows) * B >= 4 * ctx->prop.multiProcessorCount) rows *= 2;
    p.rows = (int)rows;
    p.per = Divisor::of(p.c.E / 16);
    p.heads = Divisor::of(p.c.H);
    p.blocks = (int)cdiv(L, rows);
    B200_REQUIRE(p.blocks * B < (1ll << 31), B200_DECLINE_EXTENT, "cache_read: %lld rows of %lld sequences", (long long)L, (long long)B);
    auto kern = cache->kind == B200_E4M3 ? (size == 2 ? cache_read_kernel<true, __half> : cache_read_kernel<true, float>)
                                         : (size == 2 ? cache_read_kernel<false, __half> : cache_read_kernel<false, float>);
    B200_CUDA(launch_dep(kern, dim3((unsigned)(p.blocks * B)), dim3(CA_THREADS), 0, ctx->stream, 1, p));
    ctx->launches++;
    return B200_OK;
}

} // extern "C"
