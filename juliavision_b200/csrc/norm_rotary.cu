// Norms of queries and keys, a head at a time, and the position rotation behind them in the same pass:
//     z = x w / sqrt(mean x^2 + eps),   pair (u, v) of z's first `rot` elements -> gain (u cos - v sin, v cos + u sin),
// the rest of a head is z.  Sums, root and products are fp32; the result is rounded once.  Angles are those of rotary.cu.
//
// Bandwidth-bound: two bytes read and two written an element.  A warp takes one token and some or all of its heads.  It computes the
// token's cosines and sines once, a pair a lane, and hands them round through shared memory of its own; then a group of lanes takes a head,
// 16 elements a lane, so that both halves of a pair lie in one lane and the sum of squares is a few shuffles.  Nothing waits for another
// warp.  With nothing of it in the L2 cache 40 heads of 128 of 2 x 8192 tokens, 294 MB there and back: 52 us (5.65 TB/s; the copy's rate would give 45),
// 24 of 96 of 7 x 611, 31 MB: 11.3 (9.0 with all of it there), 40 of 64 of 8 tokens: 3.8, a launch.  What is under way at once bounds the large
// ones: 72 registers a lane leave 28 warps an SM.  One head of a group at a time 59.6 and 12.1, four 59.6 and 14.7.  With the turns in registers
// too, read once a token and not once a head, there are 24 warps (58.5 us for 55 in the same runs); arithmetic on one element at a time and
// not on two takes more registers and instructions (55.2 for 55); fewer registers by force spill (61 to 69).
#include <cuda_fp16.h>

#include "internal.h"
#include "ptx.cuh"
#include "rotary.cuh"

namespace b200 {

constexpr int NR_WARPS = 4;      // of a block

struct NormRotaryParams {
    const __half* x;
    __half* out;
    int64_t xL, xH, xB, oL, oH, oB;
    const void* weight;           // (E, columns), or null: ones
    int64_t weight_ld;
    int weight_f32, split;        // heads from `split` on take column 1, those before it column 0; -1: head h takes column h
    const unsigned long long* freq;
    RotPositions at;
    float gain, eps;
    int E, rot, L, H, heads;      // heads of a warp
    uint32_t chunks, units;       // warps of a token; warps in all
    int interleaved;
};

// The warp's token and first head; false where there is nothing to do.
struct NormRotaryWork {
    int64_t l, b;
    int h0, h1, position;
    __device__ __forceinline__ bool of(const NormRotaryParams& p) {
        const uint32_t unit = blockIdx.x * NR_WARPS + (threadIdx.x >> 5);
        if (unit >= p.units) return false;
        const uint32_t row = unit / p.chunks, at = row / (uint32_t)p.L;
        b = at, l = row - at * (uint32_t)p.L;
        h0 = (int)(unit - row * p.chunks) * p.heads;
        h1 = h0 + p.heads < p.H ? h0 + p.heads : p.H;
        bool live;
        position = p.at.at(l, b, live);
        return live;
    }
};

__device__ __forceinline__ int nr_column(const NormRotaryParams& p, int h) { return p.split < 0 ? h : h >= p.split; }

// G lanes a head, vectors of 16 bytes.  U heads of a group on their way at once.
template <int G, int U>
__global__ void __launch_bounds__(32 * NR_WARPS)
norm_rotary_kernel(const NormRotaryParams p) {
    __shared__ __align__(16) float turns[NR_WARPS][16 * G];      // cosines and sines of two pairs together, those of a lane G apart
    const int lane = threadIdx.x & 31, g = lane / G, u = lane % G, half = p.rot / 2, units = p.rot / 16;
    grid_dep_wait();
    grid_dep_launch();
    NormRotaryWork w;
    if (!w.of(p)) return;       // the same for the warp
    float* mine = turns[threadIdx.x >> 5];
    for (int i = lane; i < half; i += 32) {
        float s, c;
        rot_turn(w.position, p.freq[i], s, c);
        float* to = mine + ((i % 8 / 2) * G + i / 8) * 4 + i % 2;
        to[0] = c * p.gain, to[2] = s * p.gain;
    }
    __syncwarp();
    const bool on = u * 16 < p.E, turned = u < units;
    const int e0 = !turned || p.interleaved ? u * 16 : u * 8, e1 = turned && !p.interleaved ? e0 + half : e0 + 8;
    uint64_t wt[8];                          // of two elements
    const uint64_t minus = pack2(-1.f, -1.f);
#pragma unroll
    for (int j = 0; j < 8; ++j) wt[j] = pack2(1.f, 1.f);
    int have = -1;
    const __half* x = p.x + w.l * p.xL + w.b * p.xB;
    __half* o = p.out + w.l * p.oL + w.b * p.oB;
    const float each = 1.f / (float)p.E;
    constexpr int STEP = 32 / G;
    for (int h = w.h0 + g, n = (w.h1 - w.h0 + STEP - 1) / STEP; n > 0; n -= U, h += U * STEP) {
        uint4 a[U], b[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            a[k] = b[k] = make_uint4(0, 0, 0, 0);
            if (on && h + k * STEP < w.h1) {
                const __half* at = x + (h + k * STEP) * p.xH;
                a[k] = *reinterpret_cast<const uint4*>(at + e0);
                b[k] = *reinterpret_cast<const uint4*>(at + e1);
            }
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int head = h + k * STEP;
            const uint32_t raw[8] = {a[k].x, a[k].y, a[k].z, a[k].w, b[k].x, b[k].y, b[k].z, b[k].w};
            uint64_t v[8], squares = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float2 f = rot_unpack(raw[j]);
                v[j] = pack2(f.x, f.y);
                squares = fma2(v[j], v[j], squares);
            }
            float sum, odd;
            unpack2(squares, sum, odd);
            sum += odd;
#pragma unroll
            for (int d = 1; d < G; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (!on || head >= w.h1) continue;
            const int column = nr_column(p, head);
            if (p.weight != nullptr && column != have) {
                have = column;
                if (p.weight_f32) {
                    const float* q = (const float*)p.weight + column * p.weight_ld;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float4 f = __ldg(reinterpret_cast<const float4*>(q + (j < 2 ? e0 : e1) + (j & 1) * 4));
                        wt[2 * j] = pack2(f.x, f.y), wt[2 * j + 1] = pack2(f.z, f.w);
                    }
                } else {
                    const __half* q = (const __half*)p.weight + column * p.weight_ld;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint4 f = __ldg(reinterpret_cast<const uint4*>(q + (j ? e1 : e0)));
                        const uint32_t r[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 t = rot_unpack(r[i]);
                            wt[4 * j + i] = pack2(t.x, t.y);
                        }
                    }
                }
            }
            const float r = rsqrtf(fmaf(sum, each, p.eps));
            const uint64_t rr = pack2(r, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = mul2(mul2(v[j], rr), wt[j]);
            uint32_t to[8];
            auto rounded = [](uint64_t y) {
                float a, b;
                unpack2(y, a, b);
                return rot_pack(a, b);
            };
            auto turn = [&](int j) { return reinterpret_cast<const ulonglong2*>(mine)[j * G + u]; };
            if (!turned) {
#pragma unroll
                for (int j = 0; j < 8; ++j) to[j] = rounded(v[j]);
            } else if (p.interleaved) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float a, b, c[2], s[2];
                    unpack2(v[j], a, b), unpack2(turn(j / 2).x, c[0], c[1]), unpack2(turn(j / 2).y, s[0], s[1]);
                    to[j] = rot_pack(a * c[j & 1] - b * s[j & 1], b * c[j & 1] + a * s[j & 1]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const ulonglong2 y = turn(j);
                    to[j] = rounded(fma2(v[j], y.x, mul2(mul2(v[4 + j], minus), y.y)));
                    to[4 + j] = rounded(fma2(v[4 + j], y.x, mul2(v[j], y.y)));
                }
            }
            __half* q = o + head * p.oH;
            *reinterpret_cast<uint4*>(q + e0) = make_uint4(to[0], to[1], to[2], to[3]);
            *reinterpret_cast<uint4*>(q + e1) = make_uint4(to[4], to[5], to[6], to[7]);
        }
    }
}

// Any size, any alignment: a warp a head, element by element, the head read twice.
__global__ void __launch_bounds__(32 * NR_WARPS)
norm_rotary_any_kernel(const NormRotaryParams p) {
    __shared__ float2 turns[NR_WARPS][ROT_PAIRS];
    const int lane = threadIdx.x & 31, half = p.rot / 2;
    grid_dep_wait();
    grid_dep_launch();
    NormRotaryWork w;
    if (!w.of(p)) return;
    float2* mine = turns[threadIdx.x >> 5];
    for (int i = lane; i < half; i += 32) {
        float s, c;
        rot_turn(w.position, p.freq[i], s, c);
        mine[i] = make_float2(c * p.gain, s * p.gain);
    }
    __syncwarp();
    for (int h = w.h0; h < w.h1; ++h) {
        const __half* x = p.x + w.l * p.xL + w.b * p.xB + h * p.xH;
        __half* o = p.out + w.l * p.oL + w.b * p.oB + h * p.oH;
        const int64_t column = nr_column(p, h) * p.weight_ld;
        auto weight = [&](int e) {
            return p.weight == nullptr ? 1.f : p.weight_f32 ? ((const float*)p.weight)[column + e] : __half2float(((const __half*)p.weight)[column + e]);
        };
        float sum = 0.f;
        for (int e = lane; e < p.E; e += 32) {
            const float f = __half2float(x[e]);
            sum = fmaf(f, f, sum);
        }
#pragma unroll
        for (int d = 1; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);   // and every element has been read: out may be x
        const float r = rsqrtf(sum / (float)p.E + p.eps);
        for (int i = lane; i < half; i += 32) {
            const int e0 = p.interleaved ? 2 * i : i, e1 = p.interleaved ? e0 + 1 : i + half;
            const float a = __half2float(x[e0]) * r * weight(e0), b = __half2float(x[e1]) * r * weight(e1);
            const float2 t = mine[i];
            o[e0] = __float2half_rn(a * t.x - b * t.y);
            o[e1] = __float2half_rn(b * t.x + a * t.y);
        }
        for (int e = p.rot + lane; e < p.E; e += 32) o[e] = __float2half_rn(__half2float(x[e]) * r * weight(e));
    }
}

} // namespace b200

using namespace b200;

extern "C" {

int b200_norm_rotary_f16(b200_ctx* ctx, int64_t E, int64_t L, int64_t H, int64_t B, const b200_strided4* x, const b200_strided4* out,
                         const void* weight, int weight_dtype, int64_t weight_ld, int64_t split, float eps, const uint64_t* freq,
                         int64_t rot, int interleaved, float gain, const int32_t* positions, int64_t pos_l, int64_t pos_b,
                         const int32_t* lens, const int32_t* news) {
    B200_REQUIRE(ctx && x && out, B200_EINVAL, "norm_rotary: null argument");
    B200_REQUIRE(E >= 0 && L >= 0 && H >= 0 && B >= 0, B200_EINVAL, "norm_rotary: E=%lld L=%lld H=%lld B=%lld", (long long)E, (long long)L,
                 (long long)H, (long long)B);
    B200_REQUIRE(rot >= 0 && rot % 2 == 0 && rot <= E, B200_DECLINE_EXTENT, "norm_rotary: %lld of %lld elements", (long long)rot, (long long)E);
    B200_REQUIRE(rot <= 2 * ROT_PAIRS && E <= 4096 && L < (1ll << 31) && H < 65536 && B < (1ll << 31), B200_DECLINE_EXTENT,
                 "norm_rotary: E=%lld L=%lld H=%lld B=%lld rot=%lld", (long long)E, (long long)L, (long long)H, (long long)B, (long long)rot);
    B200_REQUIRE(E <= 1 || (x->stride[0] == 1 && out->stride[0] == 1), B200_DECLINE_ALIGN, "norm_rotary: E is not contiguous");
    B200_REQUIRE(weight == nullptr || weight_dtype == B200_F16 || weight_dtype == B200_F32, B200_DECLINE_ELTYPE, "norm_rotary: weight type %d",
                 weight_dtype);
    B200_REQUIRE(split >= -1 && split <= H, B200_EINVAL, "norm_rotary: split at %lld of %lld heads", (long long)split, (long long)H);
    B200_REQUIRE(eps >= 0.f && eps < INFINITY, B200_EINVAL, "norm_rotary: eps %g", eps);
    if (E == 0 || L == 0 || H == 0 || B == 0) return B200_OK;
    B200_REQUIRE(x->ptr && out->ptr && (rot == 0 || freq), B200_EINVAL, "norm_rotary: null array");
    B200_REQUIRE(positions || lens, B200_EINVAL, "norm_rotary: neither positions nor lens");
    B200_REQUIRE(!(positions && (lens || news)), B200_EINVAL, "norm_rotary: positions as well as lens or news");
    B200_CUDA(cudaSetDevice(ctx->device));
    NormRotaryParams p = {};
    p.x = (const __half*)x->ptr;
    p.out = (__half*)const_cast<void*>(out->ptr);
    p.xL = x->stride[1], p.xH = x->stride[2], p.xB = x->stride[3];
    p.oL = out->stride[1], p.oH = out->stride[2], p.oB = out->stride[3];
    p.weight = weight, p.weight_ld = weight_ld, p.weight_f32 = weight_dtype == B200_F32;
    p.split = (int)(split < 0 && weight_ld == 0 ? H : split);      // one column: loaded once a lane
    p.freq = (const unsigned long long*)freq;
    p.at = {positions, lens, news, pos_l, pos_b, (int)L};
    p.gain = gain, p.eps = eps;
    p.E = (int)E, p.rot = (int)rot, p.L = (int)L, p.H = (int)H;
    p.interleaved = interleaved;
    const auto whole = [&](const b200_strided4* a) {
        return ((uintptr_t)a->ptr % 16 | (uint64_t)a->stride[1] % 8 | (uint64_t)a->stride[2] % 8 | (uint64_t)a->stride[3] % 8) == 0;
    };
    const bool vec = E <= 512 && rot % 16 == 0 && E % 16 == 0 && whole(x) && whole(out) &&
                     (weight == nullptr || ((uintptr_t)weight % 16 == 0 && weight_ld % 8 == 0));
    int G = 1;
    while (vec && G * 16 < E) G *= 2;
    // Heads of a warp: all of a token's, halved while there are fewer than 16 warps an SM and each still has a head for every group.  Each warp
    // computes its token's turns: with up to 128 warps an SM 2 x 8192 tokens take 56.5 us for 52, 7 x 611 17.7 for 11.3.
    const int64_t tokens = L * B, sms = ctx->prop.multiProcessorCount, least = vec ? 32 / G : 1;
    int64_t heads = H;
    while (heads > least && tokens * cdiv(H, heads) < 16 * sms) heads = cdiv(heads, 2 * least) * least;
    p.heads = (int)heads;
    p.chunks = (uint32_t)cdiv(H, heads);
    const int64_t units = tokens * p.chunks;
    B200_REQUIRE(tokens < (1ll << 31) && units < (1ll << 32) - NR_WARPS, B200_DECLINE_EXTENT, "norm_rotary: %lld tokens of %lld heads",
                 (long long)tokens, (long long)H);
    p.units = (uint32_t)units;
    const dim3 grid((unsigned)cdiv(units, NR_WARPS)), block(32 * NR_WARPS);
    auto run = [&](auto kern) { return launch_dep(kern, grid, block, 0, ctx->stream, 1, p); };
    cudaError_t e;
    if (!vec) e = run(norm_rotary_any_kernel);
    else if (G == 1) e = run(norm_rotary_kernel<1, 2>);
    else if (G == 2) e = run(norm_rotary_kernel<2, 2>);
    else if (G == 4) e = run(norm_rotary_kernel<4, 2>);
    else if (G == 8) e = run(norm_rotary_kernel<8, 2>);
    else if (G == 16) e = run(norm_rotary_kernel<16, 2>);
    else e = run(norm_rotary_kernel<32, 2>);
    B200_CUDA(e);
    ctx->launches++;
    return B200_OK;
}

} // extern "C"
