// Rotary positions: pair i of a head, (u, w), is turned by the angle position * f_i,
//     (u, w) -> gain * (u cos - w sin, w cos + u sin),
// over the first `rot` elements of a head, the rest passed on; a pair is elements (2 i, 2 i + 1) or (i, i + rot / 2).
//
// Angles are kept as turns in 64-bit fixed point: f_i in units of 2^-64 turns, so that position * f_i modulo one turn is one
// integer product, exact for every 32-bit position, where an fp32 product of a position of 120000 is off by 0.004 radians.
// The fraction's top 32 bits become a float in [-1/2, 1/2), off by at most 2^-25 turns.  Sines and products are fp32; the
// result is rounded once.
//
// Bandwidth-bound: two bytes read and two written an element (14336 tokens, 40 heads of 128: 51 us a call, 5.8 TB/s; a step of 8 x 40 heads
// of 64 3 us, the launch).  A block takes whole rows (a token of a sequence) over all or
// some of the heads; a row's rot / 2 cosines and sines are computed once for them, into shared memory, since 40 instructions
// a pair would cost more than the pair's eight bytes take.
#include <cuda_fp16.h>

#include "internal.h"
#include "ptx.cuh"

namespace b200 {

constexpr int ROT_THREADS = 256;
constexpr int ROT_PAIRS = 512;     // cosines and sines a block holds: rows * rot / 2 at most

struct RotaryParams {
    const __half* x;
    __half* out;
    int64_t xL, xH, xB, oL, oH, oB;
    const unsigned long long* freq;
    const int32_t *positions, *lens, *news;
    int64_t posL, posB;
    float gain;
    int E, rot, L, H, heads, rows;   // heads of a block, rows of a block
    int64_t total;                   // rows in all: L * B
    Divisor per, per_heads;          // steps of a head, heads of a block
    int interleaved, moves;          // moves: out is not x, so the rest of a head is copied
};

__device__ __forceinline__ uint32_t rot_pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 rot_unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// VEC: 16 elements (8 pairs) a step as two aligned vectors; otherwise pair by pair, at any alignment.
template <bool VEC>
__global__ void __launch_bounds__(ROT_THREADS)
rotary_kernel(const RotaryParams p) {
    __shared__ __align__(16) float cs[ROT_PAIRS], sn[ROT_PAIRS];
    __shared__ int64_t xat[32], oat[32];
    __shared__ bool on[32];                   // false: a row that is left alone
    const int half = p.rot / 2, tid = threadIdx.x;
    const int64_t row0 = (int64_t)blockIdx.x * p.rows;
    const int rows = p.total - row0 < p.rows ? (int)(p.total - row0) : p.rows;
    const int h0 = blockIdx.y * p.heads, heads = p.H - h0 < p.heads ? p.H - h0 : p.heads;
    grid_dep_wait();
    grid_dep_launch();
    auto position = [&](int64_t l, int64_t b, bool& live) {
        if (p.positions != nullptr) {
            live = true;
            return p.positions[l * p.posL + b * p.posB];
        }
        const int m = p.news != nullptr ? p.news[b] : p.L;
        live = l < m;
        return (int)((unsigned)p.lens[b] - (unsigned)m + (unsigned)l);
    };
    if (tid < rows) {
        const int64_t row = row0 + tid, b = row / p.L, l = row - b * p.L;
        bool live;
        position(l, b, live);
        on[tid] = live;
        xat[tid] = l * p.xL + b * p.xB;
        oat[tid] = l * p.oL + b * p.oB;
    }
    for (int i = tid; i < rows * half; i += ROT_THREADS) {
        const int r = i / half, pair = i - r * half;
        const int64_t row = row0 + r, b = row / p.L, l = row - b * p.L;
        bool live;
        const int at = position(l, b, live);
        const unsigned long long turns = (unsigned long long)(long long)at * p.freq[pair];
        float s, c;
        sincospif((float)(int)(turns >> 32) * 0x1p-31f, &s, &c);
        cs[i] = c * p.gain;
        sn[i] = s * p.gain;
    }
    __syncthreads();
    if constexpr (VEC) {
        const int units = p.rot / 16, per = units + (p.moves ? (p.E - p.rot) / 16 : 0);
        const int n = rows * p.heads * per;
        for (int i = tid; i < n; i += ROT_THREADS) {
            const int rh = p.per.div(i), u = i - rh * per, r = p.per_heads.div(rh), h = rh - r * p.heads;
            if (h >= heads) continue;        // the last block of a row may have fewer
            if (!on[r]) continue;
            const __half* x = p.x + xat[r] + (h0 + h) * p.xH;
            __half* o = p.out + oat[r] + (h0 + h) * p.oH;
            if (u >= units) {   // past the turned part
                const int e = p.rot + (u - units) * 16;
                const uint4 a = *reinterpret_cast<const uint4*>(x + e), b = *reinterpret_cast<const uint4*>(x + e + 8);
                *reinterpret_cast<uint4*>(o + e) = a;
                *reinterpret_cast<uint4*>(o + e + 8) = b;
                continue;
            }
            const int e0 = p.interleaved ? u * 16 : u * 8, e1 = p.interleaved ? e0 + 8 : e0 + half;
            const uint4 a = *reinterpret_cast<const uint4*>(x + e0), b = *reinterpret_cast<const uint4*>(x + e1);
            const float* c = cs + r * half + u * 8;
            const float* s = sn + r * half + u * 8;
            float cv[8], sv[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                cv[j] = c[j];
                sv[j] = s[j];
            }
            const uint32_t va[4] = {a.x, a.y, a.z, a.w}, vb[4] = {b.x, b.y, b.z, b.w};
            uint32_t ra[4], rb[4];
            if (p.interleaved) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = rot_unpack(va[j]), g = rot_unpack(vb[j]);
                    ra[j] = rot_pack(f.x * cv[j] - f.y * sv[j], f.y * cv[j] + f.x * sv[j]);
                    rb[j] = rot_pack(g.x * cv[4 + j] - g.y * sv[4 + j], g.y * cv[4 + j] + g.x * sv[4 + j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = rot_unpack(va[j]), g = rot_unpack(vb[j]);
                    ra[j] = rot_pack(f.x * cv[2 * j] - g.x * sv[2 * j], f.y * cv[2 * j + 1] - g.y * sv[2 * j + 1]);
                    rb[j] = rot_pack(g.x * cv[2 * j] + f.x * sv[2 * j], g.y * cv[2 * j + 1] + f.y * sv[2 * j + 1]);
                }
            }
            *reinterpret_cast<uint4*>(o + e0) = make_uint4(ra[0], ra[1], ra[2], ra[3]);
            *reinterpret_cast<uint4*>(o + e1) = make_uint4(rb[0], rb[1], rb[2], rb[3]);
        }
    } else {
        const int per = half + (p.moves ? p.E - p.rot : 0);
        const int64_t n = (int64_t)rows * heads * per;
        for (int64_t i = tid; i < n; i += ROT_THREADS) {
            const int rh = (int)(i / per), u = (int)(i - (int64_t)rh * per), r = rh / heads, h = h0 + rh - r * heads;
            if (!on[r]) continue;
            const __half* x = p.x + xat[r] + h * p.xH;
            __half* o = p.out + oat[r] + h * p.oH;
            if (u >= half) {
                o[p.rot + u - half] = x[p.rot + u - half];
                continue;
            }
            const int e0 = p.interleaved ? 2 * u : u, e1 = p.interleaved ? e0 + 1 : u + half;
            const float f = __half2float(x[e0]), g = __half2float(x[e1]), c = cs[r * half + u], s = sn[r * half + u];
            o[e0] = __float2half_rn(f * c - g * s);
            o[e1] = __float2half_rn(g * c + f * s);
        }
    }
}

} // namespace b200

using namespace b200;

extern "C" {

int b200_rotary_f16(b200_ctx* ctx, int64_t E, int64_t L, int64_t H, int64_t B, const b200_strided4* x, const b200_strided4* out,
                    const uint64_t* freq, int64_t rot, int interleaved, float gain, const int32_t* positions, int64_t pos_l,
                    int64_t pos_b, const int32_t* lens, const int32_t* news) {
    B200_REQUIRE(ctx && x && out, B200_EINVAL, "rotary: null argument");
    B200_REQUIRE(E >= 0 && L >= 0 && H >= 0 && B >= 0, B200_EINVAL, "rotary: E=%lld L=%lld H=%lld B=%lld", (long long)E, (long long)L,
                 (long long)H, (long long)B);
    B200_REQUIRE(rot >= 0 && rot % 2 == 0 && rot <= E, B200_DECLINE_EXTENT, "rotary: %lld of %lld elements", (long long)rot, (long long)E);
    B200_REQUIRE(rot <= 2 * ROT_PAIRS && E <= 4096 && L < (1ll << 31) && H < 65536 && B < (1ll << 31), B200_DECLINE_EXTENT,
                 "rotary: E=%lld L=%lld H=%lld B=%lld rot=%lld", (long long)E, (long long)L, (long long)H, (long long)B, (long long)rot);
    B200_REQUIRE(E <= 1 || (x->stride[0] == 1 && out->stride[0] == 1), B200_DECLINE_ALIGN, "rotary: E is not contiguous");
    if (E == 0 || L == 0 || H == 0 || B == 0) return B200_OK;
    B200_REQUIRE(x->ptr && out->ptr && (rot == 0 || freq), B200_EINVAL, "rotary: null array");
    B200_REQUIRE(positions || lens, B200_EINVAL, "rotary: neither positions nor lens");
    B200_REQUIRE(!(positions && (lens || news)), B200_EINVAL, "rotary: positions as well as lens or news");
    B200_CUDA(cudaSetDevice(ctx->device));
    RotaryParams p = {};
    p.x = (const __half*)x->ptr;
    p.out = (__half*)const_cast<void*>(out->ptr);
    p.xL = x->stride[1], p.xH = x->stride[2], p.xB = x->stride[3];
    p.oL = out->stride[1], p.oH = out->stride[2], p.oB = out->stride[3];
    p.freq = (const unsigned long long*)freq;
    p.positions = positions, p.lens = lens, p.news = news;
    p.posL = pos_l, p.posB = pos_b;
    p.gain = gain;
    p.E = (int)E, p.rot = (int)rot, p.L = (int)L, p.H = (int)H;
    p.total = L * B;
    p.interleaved = interleaved;
    p.moves = x->ptr != out->ptr || x->stride[1] != out->stride[1] || x->stride[2] != out->stride[2] || x->stride[3] != out->stride[3];
    const auto whole = [&](const b200_strided4* a) {
        return ((uintptr_t)a->ptr % 16 | (uint64_t)a->stride[1] % 8 | (uint64_t)a->stride[2] % 8 | (uint64_t)a->stride[3] % 8) == 0;
    };
    const bool vec = rot % 16 == 0 && (E - rot) % 16 == 0 && whole(x) && whole(out);
    // Rows of a block: enough for four steps a thread, as long as the blocks fill the GPU four times over; then heads are
    // dealt out too until there are two blocks an SM.
    const int64_t per = vec ? E / 16 : (rot / 2 + E - rot), sms = ctx->prop.multiProcessorCount;
    int64_t rows = 1;
    while (rows < 32 && 2 * rows * (rot / 2) <= ROT_PAIRS && rows * H * per < 4 * ROT_THREADS && cdiv(p.total, 2 * rows) >= 8 * sms) rows *= 2;
    int64_t heads = H < 2048 ? H : 2048;   // what the divisions take
    while (heads > 1 && cdiv(p.total, rows) * cdiv(H, heads) < 2 * sms && heads * per * rows > ROT_THREADS / 2) heads = cdiv(heads, 2);
    p.rows = (int)rows;
    p.heads = (int)heads;
    p.per = Divisor::of(vec ? rot / 16 + (p.moves ? (E - rot) / 16 : 0) : 1);
    p.per_heads = Divisor::of(heads);
    const int64_t gx = cdiv(p.total, rows), gy = cdiv(H, heads);
    B200_REQUIRE(gx < (1ll << 31) && gy < 65536, B200_DECLINE_EXTENT, "rotary: %lld rows of %lld heads", (long long)p.total, (long long)H);
    B200_CUDA(launch_dep(vec ? rotary_kernel<true> : rotary_kernel<false>, dim3((unsigned)gx, (unsigned)gy), dim3(ROT_THREADS), 0, ctx->stream, 1, p));
    ctx->launches++;
    return B200_OK;
}

} // extern "C"
