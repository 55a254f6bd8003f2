// Attention over the paged 8-bit cache (cache8.cuh) for few query rows a key head: a decoder's step.
//     out = softmax(scale Q K^T, keys below the sequence's length and, when causal, up to the query's own position) V
//
// Bandwidth-bound: the cache is read once, E + 4 / T bytes a key, head and side, against 4 E flops a query head and key.  The
// query rows of a key head (the heads that share it, times the new tokens) are stacked, 16 to a tile, so the cache is read
// once for all of them; the products are warp-level m16n8k16 tiles whose 8-bit operands become fp16 in registers, exactly.
// A page's scales never touch the operands: the key scale multiplies the fp32 scores of its page, the value scale goes
// onto P, relative to the largest one so far, whose change is one more factor of the running rescale.  P is rounded to fp16
// times 2^12, so that weights down to 2^-26 of the row's largest keep all their bits.
//
// The work is one list of key tiles over all (sequence, key head, row tile), computed from the lengths on the device and dealt
// out in equal shares, so ragged lengths and few sequences fill the GPU alike.  A share's first and last pieces may be parts
// of a list entry; their rows meet in the workspace and the last block to arrive joins them, in block order.
#include <cuda_fp16.h>

#include "cache8.cuh"

namespace b200 {

constexpr int CF_THREADS = 128;
constexpr int CF_WARPS = 4;
constexpr int CF_TILE = 64;               // keys of a tile, 16 a warp
constexpr int CF_STAGES = 4;
constexpr int CF_SHARE = 2;               // tiles of a share at least
constexpr int CF_SCALES = 2 * CF_TILE / 16;   // scales of a tile: key and value scale of each 16 keys

struct CacheAttnParams {
    CacheView c;
    const __half* q;
    void* out;
    int64_t qL, qH, qB, oL, oH, oB;
    const int32_t *lens, *news;
    int L, B, G;                          // rows at most, sequences, query heads a key head
    int causal, out_f32, whole;           // whole: rows of q start on 16-byte boundaries
    float scale_log2;
    float* part;                          // [block][first or last][16 rows][EP + 4]
    int* arrived;
};

template <int EP> struct CfCfg {
    static constexpr int SIDE = CF_TILE * EP;                 // bytes of a tile's keys, or values
    static constexpr int STAGE = 2 * SIDE;
    static constexpr int RING = CF_STAGES * STAGE;
    static constexpr int ROW = EP + 4;                        // floats: the row, its reference point, its sum
    static constexpr int SMEM = RING + CF_STAGES * CF_SCALES * 4;
    static_assert(CF_WARPS * 16 * ROW * 4 <= RING, "the warps' rows fit over the ring");
};

// Where 16-byte chunk c of row r of a tile lies, so that the eight lanes of a shared-memory phase meet all banks both when they
// read rows (keys: two rows' four chunks) and when they read columns (values: rows 2 t + i).
template <int EP> __device__ __forceinline__ int cf_place(int r, int c) {
    if constexpr (EP == 128) return r * 128 + ((c ^ ((r & 1) << 2) ^ (((r >> 1) & 3) << 1)) << 4);
    else return (r >> 1) * 128 + ((((r ^ r >> 2) & 1) << 2 | (c ^ (r & 2))) << 4);
}
// The row of a 16-key group that a key tile's column g (tile 0 or 1) stands for.  At EP = 64 a lane's four values lie in rows t,
// t + 4, t + 8, t + 12, at EP = 128 in rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9: both free of bank conflicts under cf_place.
template <int EP> __device__ __forceinline__ int cf_key(int tile, int g) {
    return EP == 128 ? tile * 8 + g : tile * 8 + (g >> 1) + (g & 1) * 4;
}

__device__ __forceinline__ void cf_copy16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cf_copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint32_t cf_pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Four tokens' words (four elements each) as the value operands of those elements: pair i of tokens 0, 1 and of tokens 2, 3.
template <bool FP8> __device__ __forceinline__ void cf_values(uint32_t a, uint32_t b, uint32_t (&r)[4]) {
    const uint32_t x = __byte_perm(a, b, 0x5140), y = __byte_perm(a, b, 0x7362);   // (a0 b0 a1 b1), (a2 b2 a3 b3)
    cache_halves<FP8>(x, r[0], r[1]);
    cache_halves<FP8>(y, r[2], r[3]);
    if constexpr (FP8) {   // the code of a NaN in a place that this row may not see must not reach it: it reads as 448
        const __half2 most = __half2half2(__ushort_as_half(0x5f00));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 v = __hmin2(*reinterpret_cast<__half2*>(&r[i]), most);
            r[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
}

template <int EP, bool FP8>
__global__ void __launch_bounds__(CF_THREADS, EP == 64 ? 4 : 3)
cache_attention_kernel(const CacheAttnParams p) {
    using Cfg = CfCfg<EP>;
    constexpr int CH = EP / 16, W = EP / 8, ROW = Cfg::ROW, HH = EP / 64;
    extern __shared__ __align__(128) uint8_t cf_smem[];
    float* scales = reinterpret_cast<float*>(cf_smem + Cfg::RING);
    __shared__ long long start_s;
    __shared__ int where_s, last_s;
    __shared__ long long sums_s[CF_WARPS];
    const CacheView& c = p.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    grid_dep_wait();
    grid_dep_launch();

    // ---- this block's share of the list
    auto entry = [&](int b, int& n, int& m, int& tiles) -> long long {   // tiles of sequence b, over its heads and row tiles
        n = c.tokens(b, p.lens);
        m = c.fresh(b, p.news, p.L);
        tiles = n > 0 ? (n + CF_TILE - 1) / CF_TILE : 1;
        return (long long)tiles * c.H * ((m * p.G + 15) / 16);
    };
    auto before = [&](long long v, long long& all) -> long long {        // sum over the threads before this one, and over all
        long long x = v;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const long long y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        if (lane == 31) sums_s[warp] = x;
        __syncthreads();
        long long add = 0;
        all = 0;
#pragma unroll
        for (int i = 0; i < CF_WARPS; ++i) {
            if (i < warp) add += sums_s[i];
            all += sums_s[i];
        }
        __syncthreads();
        return x - v + add;
    };
    long long total = 0;
    for (int b0 = 0; b0 < p.B; b0 += CF_THREADS) {
        int n, m, tiles;
        long long all;
        before(b0 + tid < p.B ? entry(b0 + tid, n, m, tiles) : 0, all);
        total += all;
    }
    long long share = (total + gridDim.x - 1) / gridDim.x;
    if (share < CF_SHARE) share = CF_SHARE;
    const long long from = blockIdx.x * share, to = from + share < total ? from + share : total;
    if (from >= to) return;
    {
        long long base = 0;
        for (int b0 = 0; b0 < p.B; b0 += CF_THREADS) {
            int n, m, tiles;
            long long all;
            const long long mine = b0 + tid < p.B ? entry(b0 + tid, n, m, tiles) : 0, at = base + before(mine, all);
            if (at <= from && from < at + mine) {
                where_s = b0 + tid;
                start_s = at;
            }
            base += all;
            if (base > from) break;
        }
        __syncthreads();
    }
    int b = where_s;
    long long bstart = start_s;

    // ---- its pieces
    for (long long at = from; at < to;) {
        int n, m, tiles;
        long long size = entry(b, n, m, tiles);
        while (at >= bstart + size) {          // the next sequence with work
            bstart += size;
            size = entry(++b, n, m, tiles);
        }
        const int rts = (m * p.G + 15) / 16;
        const long long off = at - bstart;
        const int piece = (int)(off / tiles), j0 = (int)(off - (long long)piece * tiles);
        const int h = piece / rts, rt = piece - h * rts;
        const long long pstart = bstart + (long long)piece * tiles;
        const int j1 = to - pstart < tiles ? (int)(to - pstart) : tiles;

        // rows g and g + 8 of the tile: new token l, query head of the group
        const int rows = m * p.G - rt * 16 < 16 ? m * p.G - rt * 16 : 16;
        int last0 = -1, last1 = -1;           // the last key each may see
        const __half *q0 = nullptr, *q1 = nullptr;
        {
            const int r0 = rt * 16 + g, r1 = r0 + 8;
            if (g < rows) {
                const int l = r0 / p.G;
                q0 = p.q + l * p.qL + (h * p.G + r0 - l * p.G) * p.qH + b * p.qB;
                last0 = p.causal ? n - m + l : n - 1;
            }
            if (g + 8 < rows) {
                const int l = r1 / p.G;
                q1 = p.q + l * p.qL + (h * p.G + r1 - l * p.G) * p.qH + b * p.qB;
                last1 = p.causal ? n - m + l : n - 1;
            }
        }
        auto fetch = [&](int j) {   // tile j0 + j into its stage; a commit group even when there is none
            if (j0 + j < j1) {
                const int st = j % CF_STAGES, key0 = (j0 + j) * CF_TILE;
                const uint32_t ring = smem_u32(cf_smem) + st * Cfg::STAGE;
#pragma unroll
                for (int i = 0; i < CF_TILE * CH / CF_THREADS; ++i) {
                    const int idx = tid + i * CF_THREADS, row = idx / CH, ch = idx % CH, key = key0 + row;
                    const int64_t page = key < n ? c.page(b, key >> c.logT) : -1;
                    const bool live = page >= 0 && ch * 16 < c.E;
                    const int in = key & (c.T - 1);
                    const uint8_t* k = live ? c.k + page * c.kP + h * c.kH + in * c.kT + ch * 16 : c.k;
                    const uint8_t* v = live ? c.v + page * c.vP + h * c.vH + in * c.vT + ch * 16 : c.v;
                    const uint32_t dst = ring + cf_place<EP>(row, ch);
                    cf_copy16(dst, k, live);
                    cf_copy16(dst + Cfg::SIDE, v, live);
                }
                if (tid < CF_SCALES) {   // a group without a page gets a key scale below any magnitude
                    const int key = key0 + (tid >> 1) * 16, side = tid & 1;
                    const int64_t page = key < n ? c.page(b, key >> c.logT) : -1;
                    float* dst = scales + st * CF_SCALES + tid;
                    if (page >= 0) cf_copy4(smem_u32(dst), (side ? c.vmax : c.kmax) + page * c.H + h);
                    else *dst = side ? 0.f : -1.f;
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int j = 0; j < CF_STAGES - 1; ++j) fetch(j);

        // Q: lane (g, t) holds, for keys' elements 64 hh + 16 t + 4 s + (0 .. 3) of step (hh, s), rows g and g + 8
        uint32_t qa[HH * 4][4];
#pragma unroll
        for (int hh = 0; hh < HH; ++hh)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const __half* q = r ? q1 : q0;
                const int e = hh * 64 + t * 16;
                uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (q != nullptr && e < c.E) {
                    if (p.whole) {
                        const uint4 a = __ldg(reinterpret_cast<const uint4*>(q + e)), d = __ldg(reinterpret_cast<const uint4*>(q + e + 8));
                        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = d.x, w[5] = d.y, w[6] = d.z, w[7] = d.w;
                    } else {
                        const unsigned short* u = reinterpret_cast<const unsigned short*>(q + e);
#pragma unroll
                        for (int i = 0; i < 8; ++i) w[i] = u[2 * i] | (uint32_t)u[2 * i + 1] << 16;
                    }
                }
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    qa[hh * 4 + s][r] = w[2 * s];
                    qa[hh * 4 + s][2 + r] = w[2 * s + 1];
                }
            }
        float o[W][4];
#pragma unroll
        for (int i = 0; i < W; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, vref = 0.f;   // vref: the value scale P is relative to

        for (int j = 0; j0 + j < j1; ++j) {
            asm volatile("cp.async.wait_group %0;" ::"n"(CF_STAGES - 2) : "memory");
            __syncthreads();   // tile j has landed for everyone, and tile j - 1 has been read by everyone
            fetch(j + CF_STAGES - 1);
            const int st = j % CF_STAGES, key0 = (j0 + j) * CF_TILE + warp * 16;
            const uint8_t* K = cf_smem + st * Cfg::STAGE;
            const uint8_t* V = K + Cfg::SIDE;
            const float ks = scales[st * CF_SCALES + 2 * warp], vs = scales[st * CF_SCALES + 2 * warp + 1];
            if (key0 >= n || ks < 0.f) continue;   // nothing of this warp's group (uniform over the warp)
            float s[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
                for (int hh = 0; hh < HH; ++hh) {
                    const uint4 w4 = *reinterpret_cast<const uint4*>(K + cf_place<EP>(warp * 16 + cf_key<EP>(i, g), hh * 4 + t));
                    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t b0, b1;
                        cache_halves<FP8>(w[k], b0, b1);
                        mma_16816(s[i], qa[hh * 4 + k], b0, b1);
                    }
                }
            }
            const float ksl = ks * p.scale_log2;
            float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int key = key0 + cf_key<EP>(i, 2 * t + (k & 1));
                    s[i][k] = key <= (k < 2 ? last0 : last1) ? s[i][k] * ksl : -INFINITY;
                    if (k < 2) x0 = fmaxf(x0, s[i][k]);
                    else x1 = fmaxf(x1, s[i][k]);
                }
#pragma unroll
            for (int d = 1; d < 4; d *= 2) {   // a quad of lanes shares a row
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
            }
            x0 = fmaxf(m0, x0);
            x1 = fmaxf(m1, x1);
            float vnew = vref;
            if (vs < INFINITY && vs > vref) vnew = vs;            // one that is not finite is nobody's reference
            if (__any_sync(0xffffffffu, x0 != m0 || x1 != m1 || vnew != vref)) {
                // a row that has seen nothing but hidden keys keeps the reference point -inf and contributes zeros
                const float a0 = m0 == x0 ? 1.f : exp2f(m0 - x0), a1 = m1 == x1 ? 1.f : exp2f(m1 - x1);
                const float f = vnew == vref ? 1.f : vref / vnew;
                l0 *= a0;
                l1 *= a1;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    o[i][0] *= a0 * f;
                    o[i][1] *= a0 * f;
                    o[i][2] *= a1 * f;
                    o[i][3] *= a1 * f;
                }
                m0 = x0, m1 = x1, vref = vnew;
            }
            const float n0 = m0 == -INFINITY ? 0.f : m0, n1 = m1 == -INFINITY ? 0.f : m1;
            const float f = (vs == vref ? 1.f : vs / vref) * 4096.f;   // both 0 while there are only pages of zeros
            uint32_t pa[4];
            float e[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    e[i][k] = exp2f(s[i][k] - (k < 2 ? n0 : n1));
                    if (k < 2) l0 += e[i][k];
                    else l1 += e[i][k];
                    e[i][k] = s[i][k] == -INFINITY ? 0.f : e[i][k] * f;
                }
            pa[0] = cf_pack(e[0][0], e[0][1]);
            pa[1] = cf_pack(e[0][2], e[0][3]);
            pa[2] = cf_pack(e[1][0], e[1][1]);
            pa[3] = cf_pack(e[1][2], e[1][3]);
            // V: lane (g, t) holds four tokens' elements W g ... W g + W - 1, in the order of P's columns
            const int row0 = warp * 16;
            uint32_t w[4][W / 4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t* at = V + cf_place<EP>(row0 + cf_key<EP>(i >> 1, 2 * t + (i & 1)), g * W >> 4) + (g * W & 15);
                if constexpr (W == 16) {
                    const uint4 v = *reinterpret_cast<const uint4*>(at);
                    w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
                } else {
                    const uint2 v = *reinterpret_cast<const uint2*>(at);
                    w[i][0] = v.x, w[i][1] = v.y;
                }
            }
#pragma unroll
            for (int u = 0; u < W / 4; ++u) {
                uint32_t b0[4], b1[4];
                cf_values<FP8>(w[0][u], w[1][u], b0);
                cf_values<FP8>(w[2][u], w[3][u], b1);
#pragma unroll
                for (int i = 0; i < 4; ++i) mma_16816(o[u * 4 + i], pa, b0[i], b1[i]);
            }
        }
#pragma unroll
        for (int d = 1; d < 4; d *= 2) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, d);
            l1 += __shfl_xor_sync(0xffffffffu, l1, d);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();   // the ring is free
        // this warp's rows: [row][EP values, reference point, sum]
        float* mine = reinterpret_cast<float*>(cf_smem) + warp * 16 * ROW;
        const float back = vref * (1.f / 4096.f) / cache_top<FP8>();
#pragma unroll
        for (int i = 0; i < W; i += 4)
#pragma unroll
            for (int col = 0; col < 2; ++col)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    *reinterpret_cast<float4*>(mine + (g + 8 * r) * ROW + W * (2 * t + col) + i) =
                        make_float4(o[i][2 * r + col] * back, o[i + 1][2 * r + col] * back, o[i + 2][2 * r + col] * back, o[i + 3][2 * r + col] * back);
        if (t == 0) {
            *reinterpret_cast<float2*>(mine + g * ROW + EP) = make_float2(m0, l0);
            *reinterpret_cast<float2*>(mine + (g + 8) * ROW + EP) = make_float2(m1, l1);
        }
        __syncthreads();
        const bool whole = j0 == 0 && j1 == tiles;
        const long long first = pstart / share, final = (pstart + tiles - 1) / share;   // blocks that hold parts of this piece
        float* part = p.part + ((int64_t)blockIdx.x * 2 + (j0 == 0)) * 16 * ROW;
        auto store = [&](int row, int e4, float4 v) {
            const int r = rt * 16 + row, l = r / p.G;
            const int64_t at = l * p.oL + (h * p.G + r - l * p.G) * p.oH + b * p.oB + e4;
            if (e4 >= c.E) return;
            if (p.out_f32) {
                float* d = (float*)p.out + at;
                d[0] = v.x, d[1] = v.y, d[2] = v.z, d[3] = v.w;
            } else {
                __half* d = (__half*)p.out + at;
                d[0] = __float2half_rn(v.x), d[1] = __float2half_rn(v.y), d[2] = __float2half_rn(v.z), d[3] = __float2half_rn(v.w);
            }
        };
        for (int i = tid; i < rows * (EP / 4); i += CF_THREADS) {   // the warps of a row
            const int row = i / (EP / 4), e4 = i % (EP / 4) * 4;
            const float* src = reinterpret_cast<const float*>(cf_smem) + row * ROW;
            float M = -INFINITY, l = 0.f;
#pragma unroll
            for (int w = 0; w < CF_WARPS; ++w) M = fmaxf(M, src[w * 16 * ROW + EP]);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < CF_WARPS; ++w) {
                const float mw = src[w * 16 * ROW + EP], f = mw == M ? 1.f : exp2f(mw - M);   // 1: both may be -inf, with zeros or a NaN
                const float4 x = *reinterpret_cast<const float4*>(src + w * 16 * ROW + e4);
                v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
                l = fmaf(src[w * 16 * ROW + EP + 1], f, l);
            }
            if (whole) {
                const float inv = l == 0.f ? 1.f : 1.f / l;
                store(row, e4, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
            } else {
                __stcg(reinterpret_cast<float4*>(part + row * ROW + e4), v);
                if (e4 == 0) __stcg(reinterpret_cast<float2*>(part + row * ROW + EP), make_float2(M, l));
            }
        }
        if (!whole) {   // whoever is last joins the parts, in block order
            __threadfence();
            __syncthreads();
            if (tid == 0) last_s = atomicAdd(p.arrived + first, 1) == (int)(final - first);
            __syncthreads();
            if (last_s) {
                __threadfence();
                for (int i = tid; i < rows * (EP / 4); i += CF_THREADS) {
                    const int row = i / (EP / 4), e4 = i % (EP / 4) * 4;
                    float M = -INFINITY, l = 0.f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (long long k = first; k <= final; ++k) {
                        const float* src = p.part + (k * 2 + (k == first)) * 16 * ROW + row * ROW;
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + EP));
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(src + e4));
                        const float top = fmaxf(M, ml.x);
                        const float a = M == top ? 1.f : exp2f(M - top), f = ml.x == top ? 1.f : exp2f(ml.x - top);
                        v.x = v.x * a + x.x * f, v.y = v.y * a + x.y * f, v.z = v.z * a + x.z * f, v.w = v.w * a + x.w * f;
                        l = l * a + ml.y * f;
                        M = top;
                    }
                    const float inv = l == 0.f ? 1.f : 1.f / l;
                    store(row, e4, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                }
                if (tid == 0) p.arrived[first] = 0;
            }
        }
        __syncthreads();   // the ring may be filled again
        at = pstart + j1;
    }
}

template <int EP, bool FP8>
static int cf_launch(b200_ctx* ctx, CacheAttnParams& p) {
    using Cfg = CfCfg<EP>;
    auto kern = cache_attention_kernel<EP, FP8>;
    B200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    // One resident wave at most, and no more blocks than there can be shares.
    int64_t grid = (int64_t)ctx->prop.multiProcessorCount * (EP == 64 ? 4 : 3);
    if (grid > GEMV_COUNTER_COUNT) grid = GEMV_COUNTER_COUNT;
    const int64_t tiles = cdiv((int64_t)p.c.width * p.c.T, CF_TILE), rts = cdiv((int64_t)p.L * p.G, 16);
    const double most = (double)tiles * rts * p.c.H * p.B / CF_SHARE;
    if (most + 1 < (double)grid) grid = (int64_t)most + 1;
    void* ws = nullptr;
    int rc = ws_scratch(ctx, (size_t)grid * 2 * 16 * Cfg::ROW * sizeof(float), &ws);
    if (rc) return rc;
    p.part = static_cast<float*>(ws);
    p.arrived = ctx->sk_flags + SK_FLAG_COUNT;
    B200_CUDA(launch_dep(kern, dim3((unsigned)grid), dim3(CF_THREADS), Cfg::SMEM, ctx->stream, 1, p));
    ctx->launches++;
    return B200_OK;
}

} // namespace b200

using namespace b200;

extern "C" {

int b200_cache_attention(b200_ctx* ctx, const b200_cache8* cache, int64_t L, int64_t Hq, int64_t B, const b200_strided4* q,
                         const b200_strided4* out, int out_dtype, float scale, int causal, const int32_t* lens, const int32_t* news) {
    CacheAttnParams p = {};
    int rc = cache_view(ctx, cache, "cache_attention", &p.c);
    if (rc) return rc;
    B200_REQUIRE(q && out, B200_EINVAL, "cache_attention: null argument");
    B200_REQUIRE(L >= 0 && B >= 0 && Hq >= 0, B200_EINVAL, "cache_attention: L=%lld B=%lld H=%lld", (long long)L, (long long)B, (long long)Hq);
    B200_REQUIRE(Hq % p.c.H == 0, B200_DECLINE_EXTENT, "cache_attention: %lld query heads over %d key heads", (long long)Hq, p.c.H);
    B200_REQUIRE(Hq < 65536 && L < (1ll << 24) && B < (1ll << 24) && L * (Hq / p.c.H) < (1ll << 30), B200_DECLINE_EXTENT,
                 "cache_attention: L=%lld B=%lld H=%lld", (long long)L, (long long)B, (long long)Hq);
    B200_REQUIRE(out_dtype == B200_F16 || out_dtype == B200_F32, B200_DECLINE_ELTYPE, "cache_attention: out dtype %d", out_dtype);
    if (L == 0 || B == 0 || Hq == 0) return B200_OK;
    B200_REQUIRE(q->ptr && out->ptr && lens, B200_EINVAL, "cache_attention: null array");
    B200_REQUIRE(q->stride[0] == 1 && out->stride[0] == 1, B200_DECLINE_ALIGN, "cache_attention: E is not contiguous");
    p.q = (const __half*)q->ptr;
    p.qL = q->stride[1], p.qH = q->stride[2], p.qB = q->stride[3];
    p.out = const_cast<void*>(out->ptr);
    p.oL = out->stride[1], p.oH = out->stride[2], p.oB = out->stride[3];
    p.lens = lens, p.news = news;
    p.L = (int)L, p.B = (int)B, p.G = (int)(Hq / p.c.H);
    p.causal = causal, p.out_f32 = out_dtype == B200_F32;
    p.whole = ((uintptr_t)q->ptr % 16 | (uint64_t)q->stride[1] % 8 | (uint64_t)q->stride[2] % 8 | (uint64_t)q->stride[3] % 8) == 0;
    const bool fp8 = cache->kind == B200_E4M3;
    p.scale_log2 = (float)((double)scale * 1.4426950408889634 / (fp8 ? 448.0 : 127.0));
    B200_CUDA(cudaSetDevice(ctx->device));
    if (p.c.E <= 64) return fp8 ? cf_launch<64, true>(ctx, p) : cf_launch<64, false>(ctx, p);
    return fp8 ? cf_launch<128, true>(ctx, p) : cf_launch<128, false>(ctx, p);
}

} // extern "C"
