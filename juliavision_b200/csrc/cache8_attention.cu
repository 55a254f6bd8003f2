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
// Each warp streams keys of its own, 32 at a time, through a ring that its first lane fills with TMA: nothing but the end of a
// piece of work brings a block's warps together, and what a copy costs is one lane's few instructions (64-key tiles shared by
// the block and copied 16 bytes a thread spent a third of the instructions on addresses: 32 x 8192 tokens 128 us).
//
// The work is one list of key tiles over all (sequence, key head, row tile), computed from the lengths on the device and dealt
// out in equal shares, so ragged lengths and few sequences fill the GPU alike.  A share's first and last pieces may be parts
// of a list entry; their rows meet in the workspace and the last block to arrive joins them, in block order.
#include <cuda_fp16.h>

#include "cache8.cuh"

namespace b200 {

constexpr int CF_THREADS = 128;
constexpr int CF_WARPS = 4;
constexpr int CF_KEYS = 32;                      // keys of a warp's stage
constexpr int CF_TILE = CF_WARPS * CF_KEYS;      // keys of a tile
constexpr int CF_SHARE = 1;                      // tiles of a share at least

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
    static constexpr int STAGES = EP == 128 ? 2 : 3;          // of each warp's own ring
    static constexpr int SIDE = CF_KEYS * EP;                 // bytes of a stage's keys, or values
    static constexpr int STAGE = 2 * SIDE;
    static constexpr int RING = CF_WARPS * STAGES * STAGE;
    static constexpr int ROW = EP + 4;                        // floats: the row, its reference point, its sum
    static constexpr int CTAS = EP == 128 ? 3 : 4;            // per SM
    static constexpr int SMEM = RING + 1024;                  // the swizzle wants the ring on a 1024-byte boundary
    static_assert(CF_WARPS * 16 * ROW * 4 <= RING, "the warps' rows fit over the ring");
};

// Byte of 16-byte chunk c of row r of a stage's side, as the tensor map's swizzle lays it: 128-byte rows with the chunk turned
// by r % 8, or two 64-byte rows a line with the chunk turned by r / 2 % 4.
template <int EP> __device__ __forceinline__ int cf_place(int r, int c) {
    if constexpr (EP == 128) return r * 128 + ((c ^ (r & 7)) << 4);
    else return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}
// The row of a 16-key group that column g of its key tile (0 or 1) stands for, and the chunk of a row that column g of the value
// tiles stands for; both free, and chosen so that the eight (or sixteen) lanes of a shared-memory phase meet all banks: keys read
// the same four chunks of two rows, values one or two chunks of four rows.
template <int EP> __device__ __forceinline__ int cf_key(int tile, int g) {
    if constexpr (EP == 128) return tile * 8 + (g >> 1) + (g & 1) * 4;   // two rows that differ in bit 2
    else return tile * 8 + (g ^ ((g >> 1) & 1));                         // rows 0 1 3 2 4 5 7 6: an odd one to every even one
}
__device__ __forceinline__ int cf_chunk(int g) { return (g >> 1) | (g & 1) << 2; }   // EP = 128

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

__device__ __forceinline__ float cf_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int EP, bool FP8>
__global__ void __launch_bounds__(CF_THREADS, CfCfg<EP>::CTAS)
cache_attention_kernel(const __grid_constant__ CUtensorMap tmapK, const __grid_constant__ CUtensorMap tmapV, const CacheAttnParams p) {
    using Cfg = CfCfg<EP>;
    constexpr int W = EP / 8, ROW = Cfg::ROW, HH = EP / 64, STAGES = Cfg::STAGES;
    extern __shared__ uint8_t cf_raw[];
    __shared__ __align__(8) uint64_t full_s[CF_WARPS][STAGES];
    __shared__ __align__(16) float scales_s[CF_WARPS][STAGES][4];   // key and value scale of each 16 keys
    __shared__ long long start_s, sums_s[CF_WARPS];
    __shared__ int where_s, last_s, abort_s;
    uint8_t* cf_smem = cf_raw + ((1024 - (smem_u32(cf_raw) & 1023)) & 1023);
    const CacheView& c = p.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    if (lane == 0) {
        for (int i = 0; i < STAGES; ++i) mbar_init(&full_s[warp][i], 1);
        fence_barrier_init();
    }
    if (tid == 0) {
        abort_s = 0;
        prefetch_tmap(&tmapK);
        prefetch_tmap(&tmapV);
    }
    __syncthreads();
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
    uint32_t fill = 0, use = 0;   // stages this warp has asked for, and has waited for
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
        // This warp's keys of tile j: 32 j' on, j' = 4 (j0 + j) + warp; its page or pages, looked up a tile ahead of the copies.
        int64_t page0 = -1, page1 = -1;
        auto look = [&](int j) {
            const int key = (j0 + j) * CF_TILE + warp * CF_KEYS;
            page0 = page1 = -1;
            if (j0 + j < j1 && key < n) {
                page0 = c.page(b, key >> c.logT);
                page1 = key + 16 >= n ? -1 : c.T == 16 ? c.page(b, (key >> 4) + 1) : page0;
            }
        };
        auto fetch = [&](int j) {   // a commit group even when there is none
            const int key = (j0 + j) * CF_TILE + warp * CF_KEYS;
            if (j0 + j < j1 && key < n) {
                const int st = fill % STAGES;
                if (lane < 4) {   // a group without a page gets a key scale below any magnitude
                    const int64_t page = lane < 2 ? page0 : page1;
                    float* dst = &scales_s[warp][st][lane];
                    if (page >= 0) cf_copy4(smem_u32(dst), ((lane & 1) ? c.vmax : c.kmax) + page * c.H + h);
                    else *dst = (lane & 1) ? 0.f : -1.f;
                }
                if (lane == 0) {
                    uint8_t* dst = cf_smem + (warp * STAGES + st) * Cfg::STAGE;
                    const int in = key & (c.T - 1);
                    if (c.T == 16) {
                        mbar_arrive_expect_tx(&full_s[warp][st], (uint32_t)((page0 >= 0) + (page1 >= 0)) * Cfg::SIDE);
                        if (page0 >= 0) {
                            tma_load_4d(dst, &tmapK, &full_s[warp][st], 0, 0, h, (int)page0);
                            tma_load_4d(dst + Cfg::SIDE, &tmapV, &full_s[warp][st], 0, 0, h, (int)page0);
                        }
                        if (page1 >= 0) {
                            tma_load_4d(dst + Cfg::SIDE / 2, &tmapK, &full_s[warp][st], 0, 0, h, (int)page1);
                            tma_load_4d(dst + Cfg::SIDE + Cfg::SIDE / 2, &tmapV, &full_s[warp][st], 0, 0, h, (int)page1);
                        }
                    } else {
                        mbar_arrive_expect_tx(&full_s[warp][st], page0 >= 0 ? Cfg::STAGE : 0);
                        if (page0 >= 0) {
                            tma_load_4d(dst, &tmapK, &full_s[warp][st], 0, in, h, (int)page0);
                            tma_load_4d(dst + Cfg::SIDE, &tmapV, &full_s[warp][st], 0, in, h, (int)page0);
                        }
                    }
                }
                ++fill;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int j = 0; j < STAGES; ++j) {
            look(j);
            fetch(j);
        }

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
        float m0 = -INFINITY, m1 = -INFINITY, vref = 0.f;   // vref: the value scale P is relative to
        uint64_t l0p = 0, l1p = 0;                          // sums of rows g and g + 8, in pairs
        const int all_see = p.causal ? n - m + rt * 16 / p.G : n - 1;   // the last key that every row may see

        for (int j = 0; j0 + j < j1; ++j) {
            const int key0 = (j0 + j) * CF_TILE + warp * CF_KEYS;
            if (key0 >= n) break;   // uniform over the warp, and so is every later tile
            look(j + STAGES);
            const int st = use % STAGES;
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
            if (!mbar_wait(&full_s[warp][st], (use / STAGES) & 1, c.d_status, KST_WAIT_FULL, &abort_s)) break;
            __syncwarp();
            ++use;
            const uint8_t* K = cf_smem + (warp * STAGES + st) * Cfg::STAGE;
            const uint8_t* V = K + Cfg::SIDE;
            const float4 sc = *reinterpret_cast<const float4*>(scales_s[warp][st]);   // key, value scale of group 0, of group 1
            float s[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
                for (int hh = 0; hh < HH; ++hh) {
                    const uint4 w4 = *reinterpret_cast<const uint4*>(K + cf_place<EP>((i >> 1) * 16 + cf_key<EP>(i & 1, g), hh * 4 + t));
                    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t b0, b1;
                        cache_halves<FP8>(w[k], b0, b1);
                        mma_16816(s[i], qa[hh * 4 + k], b0, b1);
                    }
                }
            }
            uint64_t s0[4], s1[4];   // scaled, in pairs, of rows g and g + 8
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float ksl = (i < 2 ? sc.x : sc.z) * p.scale_log2;
                s0[i] = mul2(pack2(s[i][0], s[i][1]), pack2(ksl, ksl));
                s1[i] = mul2(pack2(s[i][2], s[i][3]), pack2(ksl, ksl));
                unpack2(s0[i], s[i][0], s[i][1]);
                unpack2(s1[i], s[i][2], s[i][3]);
            }
            if (key0 + CF_KEYS - 1 > all_see || sc.x < 0.f || sc.z < 0.f) {   // someone does not see all of these
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool hidden = (i < 2 ? sc.x : sc.z) < 0.f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int key = key0 + (i >> 1) * 16 + cf_key<EP>(i & 1, 2 * t + (k & 1));
                        if (hidden || key > (k < 2 ? last0 : last1)) s[i][k] = -INFINITY;
                    }
                    s0[i] = pack2(s[i][0], s[i][1]);
                    s1[i] = pack2(s[i][2], s[i][3]);
                }
            }
            float x0 = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])), fmaxf(fmaxf(s[2][0], s[2][1]), fmaxf(s[3][0], s[3][1])));
            float x1 = fmaxf(fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3])), fmaxf(fmaxf(s[2][2], s[2][3]), fmaxf(s[3][2], s[3][3])));
#pragma unroll
            for (int d = 1; d < 4; d *= 2) {   // a quad of lanes shares a row
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
            }
            x0 = fmaxf(m0, x0);
            x1 = fmaxf(m1, x1);
            float vnew = vref;                                     // a scale that is not finite is nobody's reference
            if (sc.y < INFINITY && sc.y > vnew) vnew = sc.y;
            if (sc.w < INFINITY && sc.w > vnew) vnew = sc.w;
            if (__any_sync(0xffffffffu, x0 != m0 || x1 != m1 || vnew != vref)) {
                // a row that has seen nothing but hidden keys keeps the reference point -inf and contributes zeros
                const float a0 = m0 == x0 ? 1.f : cf_ex2(m0 - x0), a1 = m1 == x1 ? 1.f : cf_ex2(m1 - x1);
                const float f = vnew == vref ? 1.f : vref / vnew;
                l0p = mul2(l0p, pack2(a0, a0));
                l1p = mul2(l1p, pack2(a1, a1));
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    o[i][0] *= a0 * f;
                    o[i][1] *= a0 * f;
                    o[i][2] *= a1 * f;
                    o[i][3] *= a1 * f;
                }
                m0 = x0, m1 = x1, vref = vnew;
            }
            const float n0 = m0 == -INFINITY ? 0.f : -m0, n1 = m1 == -INFINITY ? 0.f : -m1;
            uint32_t pa[2][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float vs = i < 2 ? sc.y : sc.w, f = (vs == vref ? 1.f : vs / vref) * 4096.f;   // both 0 while there are only pages of zeros
                float e0, e1, e2, e3;
                unpack2(add2(s0[i], pack2(n0, n0)), e0, e1);
                unpack2(add2(s1[i], pack2(n1, n1)), e2, e3);
                e0 = cf_ex2(e0), e1 = cf_ex2(e1), e2 = cf_ex2(e2), e3 = cf_ex2(e3);
                l0p = add2(l0p, pack2(e0, e1));
                l1p = add2(l1p, pack2(e2, e3));
                unpack2(mul2(pack2(e0, e1), pack2(f, f)), e0, e1);
                unpack2(mul2(pack2(e2, e3), pack2(f, f)), e2, e3);
                if (!(vs < INFINITY)) {   // 0 times it is no number: a hidden key has no part
                    if (s[i][0] == -INFINITY) e0 = 0.f;
                    if (s[i][1] == -INFINITY) e1 = 0.f;
                    if (s[i][2] == -INFINITY) e2 = 0.f;
                    if (s[i][3] == -INFINITY) e3 = 0.f;
                }
                pa[i >> 1][(i & 1) * 2] = cf_pack(e0, e1);
                pa[i >> 1][(i & 1) * 2 + 1] = cf_pack(e2, e3);
            }
            // V: lane (g, t) holds four tokens' W elements of column g, in the order of P's columns
#pragma unroll
            for (int grp = 0; grp < 2; ++grp) {
                uint32_t w[4][W / 4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = grp * 16 + cf_key<EP>(i >> 1, 2 * t + (i & 1));
                    if constexpr (W == 16) {
                        const uint4 v = *reinterpret_cast<const uint4*>(V + cf_place<EP>(row, cf_chunk(g)));
                        w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(V + cf_place<EP>(row, g >> 1) + (g & 1) * 8);
                        w[i][0] = v.x, w[i][1] = v.y;
                    }
                }
#pragma unroll
                for (int u = 0; u < W / 4; ++u) {
                    uint32_t b0[4], b1[4];
                    cf_values<FP8>(w[0][u], w[1][u], b0);
                    cf_values<FP8>(w[2][u], w[3][u], b1);
#pragma unroll
                    for (int i = 0; i < 4; ++i) mma_16816(o[u * 4 + i], pa[grp], b0[i], b1[i]);
                }
            }
            __syncwarp();   // the stage has been read
            fetch(j + STAGES);
        }
        float l0, l1, l0b, l1b;
        unpack2(l0p, l0, l0b);
        unpack2(l1p, l1, l1b);
        l0 += l0b;
        l1 += l1b;
#pragma unroll
        for (int d = 1; d < 4; d *= 2) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, d);
            l1 += __shfl_xor_sync(0xffffffffu, l1, d);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();   // the ring is free: every copy that was asked for has been waited for
        // this warp's rows: [row][EP values, reference point, sum]
        float* mine = reinterpret_cast<float*>(cf_smem) + warp * 16 * ROW;
        const float back = vref * (1.f / 4096.f) / cache_top<FP8>();
#pragma unroll
        for (int i = 0; i < W; i += 4)
#pragma unroll
            for (int col = 0; col < 2; ++col)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    *reinterpret_cast<float4*>(mine + (g + 8 * r) * ROW + (EP == 128 ? 64 * col + 16 * t : 16 * t + 8 * col) + i) =
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
                const float mw = src[w * 16 * ROW + EP], f = mw == M ? 1.f : cf_ex2(mw - M);   // 1: both may be -inf, with zeros or a NaN
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
                        const float a = M == top ? 1.f : cf_ex2(M - top), f = ml.x == top ? 1.f : cf_ex2(ml.x - top);
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
        fence_proxy_async_smem();
        __syncthreads();   // the ring may be filled again
        at = pstart + j1;
    }
}

// A tensor map over one side of the cache, boxes of `rows` tokens of a page and head.
static int cf_map(b200_ctx* ctx, CUtensorMap* m, const void* base, const CacheView& c, int64_t sT, int64_t sH, int64_t sP, int EP, int rows) {
    const uint64_t dims[4] = {(uint64_t)c.E, (uint64_t)c.T, (uint64_t)c.H, (uint64_t)c.P};
    const uint64_t strides[3] = {(uint64_t)sT, (uint64_t)sH, (uint64_t)sP};
    const uint32_t box[4] = {(uint32_t)EP, (uint32_t)rows, 1, 1};
    return make_tmap(ctx, m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, base, dims, strides, box, EP == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

template <int EP, bool FP8>
static int cf_launch(b200_ctx* ctx, CacheAttnParams& p) {
    using Cfg = CfCfg<EP>;
    auto kern = cache_attention_kernel<EP, FP8>;
    CUtensorMap mk, mv;
    const int rows = p.c.T < CF_KEYS ? p.c.T : CF_KEYS;
    int rc = cf_map(ctx, &mk, p.c.k, p.c, p.c.kT, p.c.kH, p.c.kP, EP, rows);
    if (!rc) rc = cf_map(ctx, &mv, p.c.v, p.c, p.c.vT, p.c.vH, p.c.vP, EP, rows);
    if (rc) return rc;
    B200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    // One resident wave at most, and no more blocks than there can be shares.
    int64_t grid = (int64_t)ctx->prop.multiProcessorCount * Cfg::CTAS;
    if (grid > GEMV_COUNTER_COUNT) grid = GEMV_COUNTER_COUNT;
    const int64_t tiles = cdiv((int64_t)p.c.width * p.c.T, CF_TILE), rts = cdiv((int64_t)p.L * p.G, 16);
    const double most = (double)tiles * rts * p.c.H * p.B / CF_SHARE;
    if (most + 1 < (double)grid) grid = (int64_t)most + 1;
    void* ws = nullptr;
    rc = ws_scratch(ctx, (size_t)grid * 2 * 16 * Cfg::ROW * sizeof(float), &ws);
    if (rc) return rc;
    p.part = static_cast<float*>(ws);
    p.arrived = ctx->sk_flags + SK_FLAG_COUNT;
    B200_CUDA(launch_dep(kern, dim3((unsigned)grid), dim3(CF_THREADS), Cfg::SMEM, ctx->stream, 1, mk, mv, p));
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
