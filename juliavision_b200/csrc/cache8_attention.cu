// Attention over the paged 8-bit cache (cache8.cuh) for few query rows a key head: a decoder's step.
//     out = softmax(scale Q K^T, keys below the sequence's length and, when causal, up to the query's own position) V
//
// Bandwidth-bound: the cache is read once, E + 4 / T bytes a key, head and side, against 4 E flops a query head and key.  The
// query rows of a key head (the heads that share it, times the new tokens) are stacked, 8 or 16 to a tile, so the cache is read
// once for all of them.  What the SMs are short of is instructions, most of them spent on making 8-bit operands into fp16
// (exactly); so both products are taken transposed, S^T = K Q^T and O^T = V^T P^T, as warp-level m16n8k16 tiles whose 16 rows
// are keys, then elements, and whose 8 columns are query rows: every converted register pair serves a full tile, where tiles
// of 16 query rows would be half empty for a group of four or eight heads.  P^T reaches its operand layout by movmatrix.
//
// A page's scales never touch the operands: the key scale multiplies the fp32 scores of its page, the value scale goes onto P, its
// power of two as a summand of the exponents, the rest as a factor.  A row's reference point is its largest exponent with that
// summand: P has its bits where weight times scale is largest, whatever pages hold that the row does not see or gives no weight.  The
// rescale waits until an exponent is 7 past the reference point; P goes in times 2^7, so that it stays below 2^15, as two fp16
// halves (the rounded weight and what that lost): 22 bits of weight for half as many more products, which hide behind the conversions (an error of
// 2.1e-4 of the result's scale against 2.9e-4 with the upper half alone; 32 x 8192 tokens 65 us with both and 64 with one).
//
// The work is one list of 64-key tiles over all (sequence, key head, row tile): pieces.  It is computed from the lengths on the
// device and dealt out to the warps in equal contiguous shares, so ragged lengths and few sequences fill the GPU alike.  A warp
// streams its tiles by TMA and meets nobody before its block's end: it asks for the next piece's first tile before it writes the
// results of the last.  (Blocks that walked the list together lost 8 us at every change of piece, the slowest warp's tile and
// the trips to memory that nothing hid.)  A piece that one warp holds whole is stored at once.  Of the others, what ends inside a
// warp's share waits in the workspace; the last pieces of a block's warps are joined in shared memory at its end, and a second
// launch joins what then still lies in several places, in the order of the list: the result does not depend on timing.
//
// 32 sequences of 1000 to 8192 tokens, 32 heads on 8, E = 128: 310 MB in 68 us a call (4.6 TB/s; some 5 us of it before the first tile
// and in the join, 2 at the uneven ends of the shares, the rest waits for stages that are asked for only once they are read); 131071 tokens of one in 54 us (5.0 TB/s).
#include <cuda_fp16.h>

#include "cache8.cuh"
#include "shares.cuh"

namespace b200 {

constexpr int CF_THREADS = 128;
constexpr int CF_WARPS = 4;
constexpr int CF_JOIN_THREADS = 512;    // of a block that joins what began in a block's shares
constexpr int CF_KEYS = 64;                      // keys a warp takes at a time: a tile of the list
constexpr int CF_GROUPS = CF_KEYS / 16;          // of one page each

struct CfJoin {               // a piece that lies in several places: sequence, key head, row tile, rows (0: there is none), where
    int b, h, rt, rows;
    PieceParts parts;
};
struct CacheAttnParams {
    CacheView c;
    const __half* q;
    void* out;
    int64_t qL, qH, qB, oL, oH, oB;
    const int32_t *lens, *news;
    int L, B, G;                          // rows at most, sequences, query heads a key head
    int causal, out_f32, whole, out_whole;   // rows of q start on 16-byte boundaries, fours of out on their own size
    float scale_log2;
    float* part;                          // [warp][ended inside its share, or its last][row][EP + 4]
    CfJoin* joins;                        // [warp]
};

template <int EP, int NT> struct CfCfg {
    static constexpr int SIDE = CF_KEYS * EP;                 // bytes of a warp's keys, or values
    static constexpr int STAGE = 2 * SIDE;
    static constexpr int RING = CF_WARPS * STAGE;
    static constexpr int RT = 8 * NT;                         // query rows of a tile
    static constexpr int ROW = EP + 4;                        // floats: the row, its reference point, its sum
    // Per SM.  A third block of 128-wide rows adds parts to join and nothing to the rate (131071 tokens 57.7 -> 53.1 us with two).
    static constexpr int CTAS = NT == 1 && EP == 64 ? 4 : 2;
    static constexpr int SMEM = RING + 1024;                  // the swizzle wants the ring on a 1024-byte boundary
    static_assert(CF_WARPS * RT * ROW * 4 <= RING, "the warps' rows fit over the ring");
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

__device__ __forceinline__ float cf_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Four results of a row of a piece.
__device__ __forceinline__ void cf_store(const CacheAttnParams& p, int rows, int b, int h, int rt, int row, int e4, float4 v) {
    const int r = rt * rows + row, l = r / p.G;
    const int64_t at = l * p.oL + (h * p.G + r - l * p.G) * p.oH + b * p.oB + e4;
    if (e4 >= p.c.E) return;
    if (p.out_f32) {
        float* d = (float*)p.out + at;
        if (p.out_whole) *reinterpret_cast<float4*>(d) = v;
        else d[0] = v.x, d[1] = v.y, d[2] = v.z, d[3] = v.w;
    } else {
        __half* d = (__half*)p.out + at;
        if (p.out_whole) *reinterpret_cast<uint2*>(d) = make_uint2(cf_pack(v.x, v.y), cf_pack(v.z, v.w));
        else d[0] = __float2half_rn(v.x), d[1] = __float2half_rn(v.y), d[2] = __float2half_rn(v.z), d[3] = __float2half_rn(v.w);
    }
}
// the transpose of an 8 x 8 matrix of fp16, two neighbours of a row a lane
__device__ __forceinline__ uint32_t cf_transpose(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

struct CfPiece {
    long long start;          // its first tile in the list
    int b, n, m, tiles;       // sequence, its length and new tokens; tiles of a piece of it
    int h, rt, rows;          // key head, row tile, rows that count
    int j0, j1;               // the tiles of it that this warp has
};

template <int EP, bool FP8, int NT>
__global__ void __launch_bounds__(CF_THREADS, CfCfg<EP, NT>::CTAS)
cache_attention_kernel(const __grid_constant__ CUtensorMap tmapK, const __grid_constant__ CUtensorMap tmapV, const CacheAttnParams p) {
    using Cfg = CfCfg<EP, NT>;
    constexpr int W = EP / 8, ROW = Cfg::ROW, HH = EP / 64, NG = CF_GROUPS, RT = Cfg::RT;
    extern __shared__ uint8_t cf_raw[];
    __shared__ __align__(8) uint64_t full_s[CF_WARPS][2];              // keys have landed, values have landed
    __shared__ __align__(16) float scales_s[CF_WARPS][2][2][NG];       // of the tile at hand and the next: key and value scales of each 16 keys
    __shared__ long long start_s[CF_WARPS], sums_s[CF_WARPS];
    __shared__ int where_s[CF_WARPS], abort_s;
    __shared__ CfPiece given_s[2 * CF_WARPS];                          // parts of pieces this block's warps have: ended, last
    __shared__ PieceParts parts_s[2 * CF_WARPS];
    __shared__ int has_s[2 * CF_WARPS];                                // there is one
    if (threadIdx.x < 2 * CF_WARPS) has_s[threadIdx.x] = 0;
    uint8_t* cf_smem = cf_raw + ((1024 - (smem_u32(cf_raw) & 1023)) & 1023);
    const CacheView& c = p.c;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, t = lane & 3;
    if (lane == 0) {
        for (int i = 0; i < 2; ++i) mbar_init(&full_s[warp][i], 1);
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
        tiles = n > 0 ? (n + CF_KEYS - 1) / CF_KEYS : 1;
        return (long long)tiles * (c.H * ((m * p.G + RT - 1) / RT));
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
    long long total = 0, bstart = 0, from = 0, to = 0;
    int b = 0;
    const int me = blockIdx.x * CF_WARPS + warp;
    auto deal = [&]() {
        const Shares s(total, gridDim.x * CF_WARPS);
        if (me < s.warps) {
            from = s.begin(me);
            to = s.begin(me + 1);
        }
        from = __shfl_sync(0xffffffffu, from, 0), to = __shfl_sync(0xffffffffu, to, 0);   // the same for all lanes, which the compiler sees
    };
    if (p.B <= 32) {              // every warp for itself
        int n, m, tiles;
        const long long mine = lane < p.B ? entry(lane, n, m, tiles) : 0;
        long long x = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const long long y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        total = __shfl_sync(0xffffffffu, x, 31);
        deal();
        b = __ffs(__ballot_sync(0xffffffffu, from < x)) - 1;    // the first sequence that ends behind `from`
        bstart = __shfl_sync(0xffffffffu, x - mine, b < 0 ? 0 : b);
    } else {
        for (int b0 = 0; b0 < p.B; b0 += CF_THREADS) {
            int n, m, tiles;
            long long all;
            before(b0 + tid < p.B ? entry(b0 + tid, n, m, tiles) : 0, all);
            total += all;
        }
        deal();
        long long base = 0;
        for (int b0 = 0; b0 < p.B; b0 += CF_THREADS) {
            int n, m, tiles;
            long long all;
            const long long mine = b0 + tid < p.B ? entry(b0 + tid, n, m, tiles) : 0, at = base + before(mine, all);
#pragma unroll
            for (int w = 0; w < CF_WARPS; ++w) {
                const int who = blockIdx.x * CF_WARPS + w;
                const Shares s(total, gridDim.x * CF_WARPS);
                if (who >= s.warps) break;
                const long long f = s.begin(who);
                if (at <= f && f < at + mine) {
                    where_s[w] = b0 + tid;
                    start_s[w] = at;
                }
            }
            base += all;
        }
        __syncthreads();
        b = where_s[warp];
        bstart = start_s[warp];
    }

    // ---- its pieces
    uint32_t phase = 0;           // of this warp's two barriers
    const int rows_box = c.T < CF_KEYS ? c.T : CF_KEYS, boxes = CF_KEYS / rows_box;   // tokens that one copy brings, copies a side
    uint8_t* const K = cf_smem + warp * Cfg::STAGE;
    uint8_t* const V = K + Cfg::SIDE;
    auto locate = [&](CfPiece& pc, long long at) {
        int n, m, tiles;
        long long size = entry(b, n, m, tiles);
        while (at >= bstart + size) {          // the next sequence with work
            bstart += size;
            size = entry(++b, n, m, tiles);
        }
        const int rts = (m * p.G + RT - 1) / RT;
        const long long off = at - bstart;
        const int piece = (int)floor_div(off, tiles);
        pc.b = b, pc.n = n, pc.m = m, pc.tiles = tiles;
        pc.h = piece / rts, pc.rt = piece - pc.h * rts;
        pc.rows = m * p.G - pc.rt * RT < RT ? m * p.G - pc.rt * RT : RT;
        pc.start = bstart + (long long)piece * tiles;
        pc.j0 = (int)(at - pc.start);
        pc.j1 = to - pc.start < tiles ? (int)(to - pc.start) : tiles;
    };
    // The tile to be asked for next, of this piece or the one behind it.  Lane i looks up box i of it (the tokens of one page) a tile
    // ahead of its copies; keys and values have one stage each, refilled as soon as they are read: the other half of the work hides
    // the way.
    int tb = 0, tn = 0, th = 0, tj = -1, page = -1, slot = 1;
    auto look = [&](const CfPiece& q, int j) {
        tb = q.b, tn = q.n, th = q.h, tj = j;
        const int key = j * CF_KEYS + lane * rows_box;
        page = lane < boxes && key < tn ? (int)c.page(tb, key >> c.logT) : -1;
    };
    auto copy = [&](int side) {
        uint64_t* bar = &full_s[warp][side];
        const uint32_t live = __ballot_sync(0xffffffffu, page >= 0);
        if (lane == 0) mbar_arrive_expect_tx(bar, __popc(live) * rows_box * EP);
        __syncwarp();
        if (page >= 0)
            tma_load_4d((side ? V : K) + lane * rows_box * EP, side ? &tmapV : &tmapK, bar, 0, tj * CF_KEYS & (c.T - 1), th, page);
    };
    auto scales = [&]() {   // into the other slot; a group without a page gets a key scale below any magnitude
        slot ^= 1;
        const int grp = lane & (NG - 1), side = lane / NG & 1;
        const int pg = __shfl_sync(0xffffffffu, page, grp * 16 / rows_box);
        float* dst = &scales_s[warp][slot][side][grp];
        if (lane < 2 * NG) {
            if (pg >= 0) cf_copy4(smem_u32(dst), (side ? c.vmax : c.kmax) + (int64_t)pg * c.H + th);
            else *dst = side ? 0.f : -1.f;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // Query row r of a piece: new token l, query head of the group.  As the products' second operand lane (g, t) holds row
    // 8 i + g, elements 64 hh + 16 t + 4 s + (0 .. 3) in step (hh, s), the order in which it reads the keys.
    uint32_t qb[NT][HH * 4][2];
    auto queries = [&](const CfPiece& x) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int r = x.rt * RT + i * 8 + g, l = r / p.G;
            const __half* q = p.q + l * p.qL + (x.h * p.G + r - l * p.G) * p.qH + x.b * p.qB;
#pragma unroll
            for (int hh = 0; hh < HH; ++hh) {
                const int e = hh * 64 + t * 16;
                uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (i * 8 + g < x.rows && e < c.E) {
                    if (p.whole) {
                        const uint4 a = __ldg(reinterpret_cast<const uint4*>(q + e)), d = __ldg(reinterpret_cast<const uint4*>(q + e + 8));
                        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = d.x, w[5] = d.y, w[6] = d.z, w[7] = d.w;
                    } else {
                        const unsigned short* u = reinterpret_cast<const unsigned short*>(q + e);
#pragma unroll
                        for (int k = 0; k < 8; ++k) w[k] = u[2 * k] | (uint32_t)u[2 * k + 1] << 16;
                    }
                }
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    qb[i][hh * 4 + s][0] = w[2 * s];
                    qb[i][hh * 4 + s][1] = w[2 * s + 1];
                }
            }
        }
    };
    auto store = [&](const CfPiece& q, int row, int e4, float4 v) { cf_store(p, RT, q.b, q.h, q.rt, row, e4, v); };
    float o[NT][W / 2][4], mref[NT][2];                             // mref: rows' reference points
    uint64_t lsum[NT];
    const int e0 = W * (EP == 128 ? cf_chunk(g) : g);               // this lane's W elements of its rows
    // This warp's rows of piece q: `put` gets (row, element, four values times f(row's sum)) and `ends` (row, reference point, sum).
    auto results = [&](const CfPiece& q, auto factor, auto put, auto ends) {
        const float back = 1.f / cache_top<FP8>();
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            float l[2];
            unpack2(lsum[i], l[0], l[1]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int row = i * 8 + 2 * t + k;
#pragma unroll
                for (int d = 4; d < 32; d *= 2) l[k] += __shfl_xor_sync(0xffffffffu, l[k], d);
                if (row < q.rows) {
                    const float f = back * factor(l[k]);
#pragma unroll
                    for (int u = 0; u < W / 2; u += 2)
                        put(row, e0 + 2 * u, make_float4(o[i][u][k] * f, o[i][u][2 + k] * f, o[i][u + 1][k] * f, o[i][u + 1][2 + k] * f));
                    if (g == 0) ends(row, mref[i][k], l[k]);
                }
            }
        }
    };
    const auto one = [](float) { return 1.f; };
    auto keep = [&](float* to_p, const CfPiece& q) {   // as rows of [EP values, reference point, sum]
        results(q, one, [&](int row, int e4, float4 v) { *reinterpret_cast<float4*>(to_p + row * ROW + e4) = v; },
                [&](int row, float mr, float l) { *reinterpret_cast<float2*>(to_p + row * ROW + EP) = make_float2(mr, l); });
    };

    CfPiece pc, nx;
    bool ok = true;               // no wait has run out
    if (from < to) {
        locate(pc, from);
        look(pc, pc.j0);
        copy(0);
        copy(1);
        scales();
        queries(pc);
    }
    for (long long at = from; ok && at < to;) {
        const int n = pc.n, m = pc.m, rt = pc.rt;
        at = pc.start + pc.j1;
        // As results lane (g, t) holds rows 8 i + 2 t and 8 i + 2 t + 1.
        int last[NT][2];                                     // the last key each may see
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) last[i][k] = p.causal ? n - m + (rt * RT + i * 8 + 2 * t + k) / p.G : n - 1;
        const int all_see = p.causal ? n - m + rt * RT / p.G : n - 1;   // that every row may see
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int u = 0; u < W / 2; ++u) o[i][u][0] = o[i][u][1] = o[i][u][2] = o[i][u][3] = 0.f;
            mref[i][0] = mref[i][1] = -INFINITY;
            lsum[i] = 0;
        }

        for (int j = pc.j0; j < pc.j1; ++j) {
            const int key0 = j * CF_KEYS;
            const bool last_one = j + 1 == pc.j1, more = !last_one || at < to;
            if (!last_one) {
                look(pc, j + 1);
            } else if (more) {   // the next piece's first tile
                locate(nx, at);
                look(nx, nx.j0);
            }
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&full_s[warp][0], phase, c.d_status, KST_WAIT_FULL, &abort_s)))) break;
            float s[NT][NG][4];     // rows g and g + 8 of a group's keys, query rows 2 t and 2 t + 1
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
#pragma unroll
                for (int i = 0; i < NT; ++i) s[i][grp][0] = s[i][grp][1] = s[i][grp][2] = s[i][grp][3] = 0.f;
#pragma unroll
                for (int hh = 0; hh < HH; ++hh) {
                    const uint4 lo = *reinterpret_cast<const uint4*>(K + cf_place<EP>(grp * 16 + cf_key<EP>(0, g), hh * 4 + t));
                    const uint4 hi = *reinterpret_cast<const uint4*>(K + cf_place<EP>(grp * 16 + cf_key<EP>(1, g), hh * 4 + t));
                    const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t a[4];
                        cache_halves<FP8>(wl[k], a[0], a[2]);
                        cache_halves<FP8>(wh[k], a[1], a[3]);
#pragma unroll
                        for (int i = 0; i < NT; ++i) mma_16816_free(s[i][grp], a[0], a[1], a[2], a[3], qb[i][hh * 4 + k][0], qb[i][hh * 4 + k][1]);
                    }
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();            // the keys have been read, and this tile's scales are there for every lane
            float ks[NG], vs[NG];
            *reinterpret_cast<float4*>(ks) = *reinterpret_cast<const float4*>(scales_s[warp][slot][0]);
            *reinterpret_cast<float4*>(vs) = *reinterpret_cast<const float4*>(scales_s[warp][slot][1]);
            if (more) {
                copy(0);
                scales();
                if (last_one) queries(nx);
            }
            // A value scale as 2^vk times vm, exactly, and 2^-vk, which takes a weight back for the row's sum.  2^-80 stands for less and for
            // 0, whose weights count but whose vm is 0: fp32 holds them beside fp16's largest down to 2^-30 of the row's largest weight.
            float vk[NG], vm[NG], vb[NG];
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
                const int e = min(max((__float_as_int(vs[grp]) >> 23) - 127, -80), 126);
                vk[grp] = (float)e;
                vb[grp] = __int_as_float((127 - e) << 23);
                vm[grp] = vs[grp] * vb[grp];
            }
            const bool plain = key0 + CF_KEYS - 1 <= all_see && fminf(fminf(ks[0], ks[1]), fminf(ks[2], ks[3])) >= 0.f;   // every row sees all of these
            const bool odd = !(vs[0] + vs[1] + vs[2] + vs[3] < INFINITY);
            bool grown = false;
            float top[NT][2];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                top[i][0] = top[i][1] = -INFINITY;
#pragma unroll
                for (int grp = 0; grp < NG; ++grp) {
                    const float ksl = ks[grp] * p.scale_log2;
                    float* x = s[i][grp];
                    unpack2(fma2(pack2(x[0], x[1]), pack2(ksl, ksl), pack2(vk[grp], vk[grp])), x[0], x[1]);
                    unpack2(fma2(pack2(x[2], x[3]), pack2(ksl, ksl), pack2(vk[grp], vk[grp])), x[2], x[3]);
                    if (!plain) {
                        const int k0 = key0 + grp * 16 + cf_key<EP>(0, g), k1 = key0 + grp * 16 + cf_key<EP>(1, g);
                        const bool hidden = ks[grp] < 0.f;
                        if (hidden || k0 > last[i][0]) x[0] = -INFINITY;
                        if (hidden || k0 > last[i][1]) x[1] = -INFINITY;
                        if (hidden || k1 > last[i][0]) x[2] = -INFINITY;
                        if (hidden || k1 > last[i][1]) x[3] = -INFINITY;
                    }
                    top[i][0] = cf_max3(top[i][0], x[0], x[2]);
                    top[i][1] = cf_max3(top[i][1], x[1], x[3]);
                }
                grown = grown || top[i][0] > mref[i][0] + 7.f || top[i][1] > mref[i][1] + 7.f;
            }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float x = top[i][k];
#pragma unroll
                        for (int d = 4; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));   // the lanes of a row
                        x = fmaxf(x, mref[i][k]);
                        // a row that has seen nothing but hidden keys keeps the reference point -inf and contributes zeros
                        const float a = mref[i][k] == x ? 1.f : cf_ex2(mref[i][k] - x);
                        mref[i][k] = x;
                        float l0, l1;
                        unpack2(lsum[i], l0, l1);
                        if (k == 0) l0 *= a;
                        else l1 *= a;
                        lsum[i] = pack2(l0, l1);
#pragma unroll
                        for (int u = 0; u < W / 2; ++u) {
                            o[i][u][k] *= a;
                            o[i][u][2 + k] *= a;
                        }
                    }
            }
            uint32_t pb[NT][NG][2], pl[NT][NG][2];   // the weights' upper and lower halves
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const uint64_t nm = pack2(mref[i][0] == -INFINITY ? 0.f : 7.f - mref[i][0], mref[i][1] == -INFINITY ? 0.f : 7.f - mref[i][1]);
#pragma unroll
                for (int grp = 0; grp < NG; ++grp) {
                    const uint64_t f = pack2(vm[grp], vm[grp]), b2 = pack2(vb[grp], vb[grp]);
                    const float* x = s[i][grp];
                    float e[4];
                    unpack2(add2(pack2(x[0], x[1]), nm), e[0], e[1]);
                    unpack2(add2(pack2(x[2], x[3]), nm), e[2], e[3]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) e[k] = cf_ex2(e[k]);
                    lsum[i] = fma2(add2(pack2(e[0], e[1]), pack2(e[2], e[3])), b2, lsum[i]);
                    unpack2(mul2(pack2(e[0], e[1]), f), e[0], e[1]);
                    unpack2(mul2(pack2(e[2], e[3]), f), e[2], e[3]);
                    if (odd) {   // 0 times what is not finite is no number: a hidden key has no part
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (x[k] == -INFINITY) e[k] = 0.f;
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t hi = cf_pack(e[2 * k], e[2 * k + 1]);
                        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                        float r0, r1;
                        unpack2(add2(pack2(e[2 * k], e[2 * k + 1]), pack2(-back.x, -back.y)), r0, r1);
                        pb[i][grp][k] = cf_transpose(hi);
                        pl[i][grp][k] = cf_transpose(cf_pack(r0, r1));
                    }
                }
            }
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&full_s[warp][1], phase, c.d_status, KST_WAIT_FULL, &abort_s)))) break;
            phase ^= 1;
            // V: lane (g, t) holds four tokens' W elements of its chunk, in the order of P's rows; elements 2 u and 2 u + 1 of the chunks are
            // rows g and g + 8 of tile u
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
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
                    for (int i = 0; i < NT; ++i) {
                        mma_16816_free(o[i][2 * u], b0[0], b0[1], b1[0], b1[1], pb[i][grp][0], pb[i][grp][1]);
                        mma_16816_free(o[i][2 * u + 1], b0[2], b0[3], b1[2], b1[3], pb[i][grp][0], pb[i][grp][1]);
                        mma_16816_free(o[i][2 * u], b0[0], b0[1], b1[0], b1[1], pl[i][grp][0], pl[i][grp][1]);
                        mma_16816_free(o[i][2 * u + 1], b0[2], b0[3], b1[2], b1[3], pl[i][grp][0], pl[i][grp][1]);
                    }
                }
            }
            __syncwarp();   // the values have been read
            if (more) copy(1);
        }
        if (!ok) break;
        // the next piece's first tile is on its way while this one's results leave
        const CfPiece done = pc;
        const bool mine = done.j0 == 0 && done.j1 == done.tiles;
        if (at < to) pc = nx;
        if (mine)
            results(done, [](float l) { return l == 0.f ? 1.f : 1.f / l; }, [&](int row, int e4, float4 v) { store(done, row, e4, v); },
                    [](int, float, float) {});
        else if (at < to) keep(p.part + (int64_t)(2 * me) * RT * ROW, done);
        if (!mine && lane == 0) {
            const int i = 2 * warp + (at == to);
            given_s[i] = done;
            has_s[i] = 1;
        }
        __syncwarp();
    }

    // ---- the block's parts of pieces
    if (!ok)                      // copies may still land
        for (int i = 0; i < 4; ++i) __nanosleep(1000000);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();   // the ring is free: every copy that was asked for has been waited for
    float* rows_s = reinterpret_cast<float*>(cf_smem);
    if (has_s[2 * warp + 1]) keep(rows_s + warp * RT * ROW, pc);
    if (tid < 2 * CF_WARPS && has_s[tid])
        parts_s[tid] = PieceParts::of<CF_WARPS>(Shares(total, gridDim.x * CF_WARPS), given_s[tid].start, given_s[tid].start + given_s[tid].tiles);
    __syncthreads();
    auto same = [&](int w) {   // warps w and w + 1 have the same last piece
        return w + 1 < CF_WARPS && has_s[2 * w + 1] && has_s[2 * w + 3] && given_s[2 * w + 1].start == given_s[2 * w + 3].start;
    };
    for (int w = 0, end; w < CF_WARPS; w = end) {
        end = w + 1;
        while (same(end - 1)) ++end;
        if (!has_s[2 * w + 1]) continue;
        const CfPiece& q = given_s[2 * w + 1];
        const bool all = parts_s[2 * w + 1].count == 1;
        float* part = p.part + (int64_t)(2 * (blockIdx.x * CF_WARPS + w) + 1) * RT * ROW;
        for (int i = tid; i < q.rows * (EP / 4); i += CF_THREADS) {
            const int row = i / (EP / 4), e4 = i % (EP / 4) * 4;
            const float* src = rows_s + row * ROW;
            float M = -INFINITY, l = 0.f;
            for (int k = w; k < end; ++k) M = fmaxf(M, src[k * RT * ROW + EP]);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k = w; k < end; ++k) {
                const float mw = src[k * RT * ROW + EP], f = mw == M ? 1.f : cf_ex2(mw - M);   // 1: both may be -inf, with zeros or a NaN
                const float4 x = *reinterpret_cast<const float4*>(src + k * RT * ROW + e4);
                v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
                l = fmaf(src[k * RT * ROW + EP + 1], f, l);
            }
            if (all) {
                const float inv = l == 0.f ? 1.f : 1.f / l;
                store(q, row, e4, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
            } else {
                *reinterpret_cast<float4*>(part + row * ROW + e4) = v;
                if (e4 == 0) *reinterpret_cast<float2*>(part + row * ROW + EP) = make_float2(M, l);
            }
        }
    }
    if (lane == 0) {      // the warp in whose share a piece begins says where its parts are
        const CfPiece& q = given_s[2 * warp + 1];
        CfJoin d = {};
        if (has_s[2 * warp + 1] && q.j0 == 0 && parts_s[2 * warp + 1].count > 1)
            d = {q.b, q.h, q.rt, q.rows, parts_s[2 * warp + 1]};
        p.joins[me] = d;
    }
}

// One block for each of the launch before: joins the parts of the pieces that began in its warps' shares, in the order of the list,
// several parts at a time where there are more threads than fours of results.
template <int EP, int NT>
__global__ void __launch_bounds__(CF_JOIN_THREADS)
cache_attention_join_kernel(const CacheAttnParams p) {
    constexpr int ROW = CfCfg<EP, NT>::ROW, RT = CfCfg<EP, NT>::RT, AT_ONCE = 8;   // parts in flight: each is a trip to L2
    __shared__ float4 rows_s[CF_JOIN_THREADS];
    __shared__ float2 ml_s[CF_JOIN_THREADS];
    grid_dep_wait();
    grid_dep_launch();
    __shared__ CfJoin joins_s[CF_WARPS];
    if (threadIdx.x < CF_WARPS) joins_s[threadIdx.x] = p.joins[blockIdx.x * CF_WARPS + threadIdx.x];
    __syncthreads();
    const int tid = threadIdx.x;
    for (int w = 0; w < CF_WARPS; ++w) {
        const CfJoin& d = joins_s[w];
        const int items = d.rows * (EP / 4);
        if (items == 0) continue;
        const int groups = items < CF_JOIN_THREADS ? CF_JOIN_THREADS / items : 1, grp = items < CF_JOIN_THREADS ? tid / items : 0;
        const int i = tid - grp * items;      // 16 rows of 128 elements have as many fours as there are threads
        static_assert(RT * EP / 4 <= CF_JOIN_THREADS, "a thread for each four of a piece's results");
        const int row = i / (EP / 4), e4 = i % (EP / 4) * 4;
        float M = -INFINITY, l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (grp < groups)
            for (int k0 = grp; k0 < d.parts.count; k0 += groups * AT_ONCE) {
                float2 ml[AT_ONCE];
                float4 x[AT_ONCE];
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u) {
                    const int k = k0 + u * groups;
                    ml[u] = make_float2(-INFINITY, 0.f);
                    x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (k < d.parts.count) {
                        const float* src = p.part + d.parts.place<CF_WARPS>(k) * RT * ROW + row * ROW;
                        ml[u] = *reinterpret_cast<const float2*>(src + EP);
                        x[u] = *reinterpret_cast<const float4*>(src + e4);
                    }
                }
                float top = M;
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u) top = fmaxf(top, ml[u].x);
                const float a = M == top ? 1.f : cf_ex2(M - top);      // 1: both may be -inf, with zeros or a NaN
                v.x *= a, v.y *= a, v.z *= a, v.w *= a, l *= a;
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u) {
                    const float f = ml[u].x == top ? 1.f : cf_ex2(ml[u].x - top);
                    v.x = fmaf(x[u].x, f, v.x), v.y = fmaf(x[u].y, f, v.y), v.z = fmaf(x[u].z, f, v.z), v.w = fmaf(x[u].w, f, v.w);
                    l = fmaf(ml[u].y, f, l);
                }
                M = top;
            }
        rows_s[tid] = v;
        ml_s[tid] = make_float2(M, l);
        __syncthreads();
        if (grp == 0) {
            for (int k = 1; k < groups; ++k) M = fmaxf(M, ml_s[k * items + i].x);
            float f = ml_s[i].x == M ? 1.f : cf_ex2(ml_s[i].x - M);
            v.x *= f, v.y *= f, v.z *= f, v.w *= f, l *= f;
            for (int k = 1; k < groups; ++k) {
                const float2 ml = ml_s[k * items + i];
                const float4 x = rows_s[k * items + i];
                f = ml.x == M ? 1.f : cf_ex2(ml.x - M);
                v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
                l = fmaf(ml.y, f, l);
            }
            const float inv = l == 0.f ? 1.f : 1.f / l;
            cf_store(p, RT, d.b, d.h, d.rt, row, e4, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        }
        __syncthreads();
    }
}

// A tensor map over one side of the cache, boxes of `rows` tokens of a page and head.
static int cf_map(b200_ctx* ctx, CUtensorMap* m, const void* base, const CacheView& c, int64_t sT, int64_t sH, int64_t sP, int EP, int rows) {
    const uint64_t dims[4] = {(uint64_t)c.E, (uint64_t)c.T, (uint64_t)c.H, (uint64_t)c.P};
    const uint64_t strides[3] = {(uint64_t)sT, (uint64_t)sH, (uint64_t)sP};
    const uint32_t box[4] = {(uint32_t)EP, (uint32_t)rows, 1, 1};
    return make_tmap(ctx, m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, base, dims, strides, box, EP == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

template <int EP, bool FP8, int NT>
static int cf_launch(b200_ctx* ctx, CacheAttnParams& p) {
    using Cfg = CfCfg<EP, NT>;
    auto kern = cache_attention_kernel<EP, FP8, NT>;
    CUtensorMap mk, mv;
    const int rows = p.c.T < CF_KEYS ? p.c.T : CF_KEYS;
    int rc = cf_map(ctx, &mk, p.c.k, p.c, p.c.kT, p.c.kH, p.c.kP, EP, rows);
    if (!rc) rc = cf_map(ctx, &mv, p.c.v, p.c, p.c.vT, p.c.vH, p.c.vP, EP, rows);
    if (rc) return rc;
    static std::atomic<uint64_t> asked{0};
    B200_CUDA(allow_smem(ctx, kern, Cfg::SMEM, asked));
    // One resident wave at most, and no more blocks than there can be shares.
    int64_t grid = (int64_t)ctx->prop.multiProcessorCount * Cfg::CTAS;
    const int64_t tiles = cdiv((int64_t)p.c.width * p.c.T, CF_KEYS), rts = cdiv((int64_t)p.L * p.G, Cfg::RT);
    const double most = (double)tiles * rts * p.c.H * p.B / CF_WARPS;
    if (most + 1 < (double)grid) grid = (int64_t)most + 1;
    void* ws = nullptr;
    const size_t floats = (size_t)grid * CF_WARPS * 2 * Cfg::RT * Cfg::ROW;
    rc = ws_scratch(ctx, floats * sizeof(float) + (size_t)grid * CF_WARPS * sizeof(CfJoin), &ws);
    if (rc) return rc;
    p.part = static_cast<float*>(ws);
    p.joins = reinterpret_cast<CfJoin*>(p.part + floats);
    B200_CUDA(launch_dep(kern, dim3((unsigned)grid), dim3(CF_THREADS), Cfg::SMEM, ctx->stream, 1, mk, mv, p));
    B200_CUDA(launch_dep(cache_attention_join_kernel<EP, NT>, dim3((unsigned)grid), dim3(CF_JOIN_THREADS), 0, ctx->stream, 1, p));
    ctx->launches += 2;
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
    const int64_t four = p.out_f32 ? 16 : 8, size = four / 4;
    p.out_whole = ((uintptr_t)out->ptr | (uint64_t)(out->stride[1] * size) | (uint64_t)(out->stride[2] * size) | (uint64_t)(out->stride[3] * size)) % four == 0;
    const bool fp8 = cache->kind == B200_E4M3;
    p.scale_log2 = (float)((double)scale * 1.4426950408889634 / (fp8 ? 448.0 : 127.0));
    B200_CUDA(cudaSetDevice(ctx->device));
    // Each tile of 16 rows converts the cache again; tiles of 128 rows convert it once.  By few rows and by many, us, E = 128, 32 query heads on 8 but
    // where noted: 32 rows (two tiles) 4 x 4096 tokens 29 and 36, 16 x 8192 120 and 152, 1 x 60000 63 and 87, 32 x 500 of 8 on 2 15.9 and 17.4; 48
    // rows 36 and 36, 171 and 152, 87 and 87, 23 and 17.5.  E = 64: 48 rows 26 and 31, 121 and 133, 61 and 77, 19 and 14; 64 rows 32 and 31, 155
    // and 133, 75 and 77, 20 and 14.  Short caches of few items gain from few rows for longer (1 x 1500 of 16 on 4, E = 128: 48 rows 14 and 21),
    // but lengths are not known here.
    if ((int64_t)p.L * p.G > (p.c.E > 64 ? 32 : 48)) return cache_prompt_run(ctx, p.c, L, B, p.G, q, out, out_dtype, scale, fp8, causal, lens, news);
    if (p.L * p.G <= 8) {
        if (p.c.E <= 64) return fp8 ? cf_launch<64, true, 1>(ctx, p) : cf_launch<64, false, 1>(ctx, p);
        return fp8 ? cf_launch<128, true, 1>(ctx, p) : cf_launch<128, false, 1>(ctx, p);
    }
    if (p.c.E <= 64) return fp8 ? cf_launch<64, true, 2>(ctx, p) : cf_launch<64, false, 2>(ctx, p);
    return fp8 ? cf_launch<128, true, 2>(ctx, p) : cf_launch<128, false, 2>(ctx, p);
}

} // extern "C"
