// Attention over the paged 8-bit cache (cache8.cuh) for many query rows a key head: a piece of a prompt, the formula of
// cache8_attention.cu.
//
// Tensor-bound in the limit: 4 E flops a row and visible key; 2048 new tokens of 10240, 16 heads on 4, E = 128: 229 us a call
// between others, 208 back to back (0.68 and 0.74 PFLOP/s).
// What it waits for is the chain of one tile (scores into registers, maximum, exponentials, P V, the next Q K', some 4600 clocks a block
// of 128 keys for two tiles whose products take two thirds of that), which the other tile's covers in part.
//
// The query rows of a key head (the heads that share it, times the new tokens) are stacked; a block takes two tiles of 128 of them
// and walks their keys in blocks of 128: S = Q K^T and O += P V on tcgen05 with S, P (two fp16 halves, 21 bits and more of a
// weight, as for few rows) and O in tensor memory.  The 8-bit operands become fp16 on the way to shared memory, exactly, once for 256 rows: four warps
// read them from the pages into registers a side ahead and write them in the 128-byte swizzle.  No operand carries a scale: a
// page's key scale (and the softmax's own) is the factor of its columns' exponents, its value scale a summand of them; the row sum
// takes that back a group of 16 keys at a time.  A row's reference point is its largest exponent with that summand (cache8_attention.cu).
//
//   warps 0-3  softmax of tile 0, warps 4-7 of tile 1: one thread a row, the row's 128 scores in registers
//   warps 8-11 fetch and convert: K(j), V(j), K(j+1), ...
//   warps 12, 13  issue one tile's products each:  Q K(j)',  P(j) V(j), Q K(j+1)', ...; P's halves lie over the halves of S
//   warp 14    looks up pages and scales and lays out each block's constants, two blocks ahead
//   warp 15    walks the block's share of the items' keys (CpWalk), an item's part at a time, and tells the others
#include <cuda_fp16.h>

#include "cache8.cuh"
#include "shares.cuh"

namespace b200 {

constexpr int CP_THREADS = 512;
constexpr int CP_ROWS = 128, CP_KEYS = 128;     // of a tile
constexpr int CP_ATOM = 128 * 128;              // 128 rows x 64 fp16
constexpr int CP_LEAST = 2;                     // blocks of keys of a share
constexpr int CP_START = 3;                     // blocks of keys that an item's start and end take as long as
constexpr int CP_SCALES = 4;                    // blocks of constants in flight
constexpr int CP_SOFTMAX_REGS = 176, CP_CONVERT_REGS = 104, CP_OTHER_REGS = 56;
static_assert(2 * 128 * CP_SOFTMAX_REGS + 128 * CP_CONVERT_REGS + 128 * CP_OTHER_REGS <= CP_THREADS * 128, "what the launch holds");

struct __align__(16) CpScales {              // of one block of keys, a group of 16 keys an entry
    float2 score[8];           // score to exponent: a factor, finite and above 0, so that a hidden score of -inf stays that; log2 of the value scale
    float back[8];             // an exponential of the group back to a weight
    int hidden, odd;           // bit g: the group has no page; one of its scales is not finite
};

struct CachePromptParams {
    CacheView c;
    const __half* q;
    void* out;
    int64_t qL, qH, qB, oL, oH, oB;
    const int32_t *lens, *news;
    int L, B, G;
    int causal, out_f32, whole, out_whole;
    float scale_log2;         // without its sign, which goes onto Q
    int negate;
    int items, shared;        // row pairs x heads x sequences; whether the blocks have equal shares of their keys, or an item each
    float* part;              // [2 grid][EP / 4][256 rows][4]: a block's share that begins inside an item, and the one that ends inside one
    float* part_ml;           // [2 grid][256][2]: reference point, sum
    int4* joins;              // [grid]: the item of a block's first share and its first and last block, if it is the second of them
};

__device__ __forceinline__ float cp_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float cp_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void cp_tmem_st16(uint32_t taddr, const uint32_t* r) {
    uint32_t v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = r[i];
    tmem_st16(taddr, v);
}
// Two weights as two halves each: what fp16 holds of them, cut off, and what is left, rounded; off by 2^-21 of themselves, or, below
// 2^-14, by a step of 2^-24.  (One half alone: 163 us for 208 at 2048 tokens over 10240, and 2.9e-4 of the result for 2.1e-4.  The upper
// ones rounded to nearest and converted back 217; the lower ones made after the exponentials' turn has passed, beside the upper ones'
// product, 216.)
__device__ __forceinline__ void cp_halves(float a, float b, uint32_t& upper, uint32_t& lower) {
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(upper) : "f"(b), "f"(a));
    const float ma = __uint_as_float((__float_as_uint(a) & 0xffffe000u) ^ 0x80000000u), mb = __uint_as_float((__float_as_uint(b) & 0xffffe000u) ^ 0x80000000u);
    float ra, rb;
    unpack2(add2(pack2(a, b), pack2(ma, mb)), ra, rb);
    const __half2 l = __floats2half2_rn(ra, rb);
    lower = *reinterpret_cast<const uint32_t*>(&l);
}
// 16 bytes to shared memory on their own, zeros where there are none to read
__device__ __forceinline__ void cp_async16(uint32_t to, const void* from, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void cp_load8(uint32_t (&v)[4], const __half* at, bool whole) {
    if (whole) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(at));
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
        const unsigned short* u = reinterpret_cast<const unsigned short*>(at);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = u[2 * k] | (uint32_t)u[2 * k + 1] << 16;
    }
}
// eight results of a row, 16 bytes at a time where rows allow it
__device__ __forceinline__ void cp_store8(const CachePromptParams& p, int64_t at, const float (&v)[8]) {
    if (p.out_f32) {
        float* d = (float*)p.out + at;
        if (p.out_whole) {
            reinterpret_cast<float4*>(d)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(d)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = v[i];
        }
    } else {
        __half* d = (__half*)p.out + at;
        if (p.out_whole) {
            uint4 w;
            __half2* h = reinterpret_cast<__half2*>(&w);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            *reinterpret_cast<uint4*>(d) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = __float2half_rn(v[i]);
        }
    }
}

// What the rows of an item see: item -> (row pair, head, sequence), later rows, whose keys are more, first.
struct CpItem {
    int b, h, r0, rows, n, m, blocks;   // first row, rows of the sequence (all of its heads), length, new tokens, blocks of keys
    // Its length in the list that is shared out: `start` for its start and end, then its blocks.  An item without keys has rows of zeros
    // to write.
    __device__ __forceinline__ int weight(int start) const { return r0 >= rows ? 0 : start + (blocks > 0 ? blocks : 1); }
    __device__ __forceinline__ int block(int j, int start) const { return j <= start ? 0 : j - start < blocks ? j - start : blocks; }
};
__device__ __forceinline__ CpItem cp_item(const CachePromptParams& p, int item) {
    CpItem it;
    const int pairs = (p.L * p.G + 2 * CP_ROWS - 1) / (2 * CP_ROWS), hb = p.c.H * p.B;
    const int rp = pairs - 1 - item / hb, rest = item % hb;
    it.h = rest % p.c.H;
    it.b = rest / p.c.H;
    it.r0 = rp * 2 * CP_ROWS;
    it.n = p.c.tokens(it.b, p.lens);
    it.m = p.c.fresh(it.b, p.news, p.L);
    it.rows = it.m * p.G;
    const int top = it.r0 + 2 * CP_ROWS < it.rows ? it.r0 + 2 * CP_ROWS : it.rows;
    int seen = p.causal && top > 0 ? it.n - it.m + (top - 1) / p.G + 1 : it.n;   // keys that some row sees
    if (seen < 0) seen = 0;
    it.blocks = (seen + CP_KEYS - 1) / CP_KEYS;
    return it;
}

// A block's share of the list of all items' blocks of keys, an item's part at a time.
struct CpWalk {
    long long left;     // blocks of the share from here on
    int item, j;        // where the next part begins
    int start;          // CpItem::weight

    __device__ __forceinline__ bool next(const CachePromptParams& p, CpItem& it, int& at, int& j0, int& nblk) {
        while (left > 0 && item < p.items) {
            it = cp_item(p, item);
            const int w = it.weight(start);
            if (w == 0) {                     // nor has any other head of these rows
                item += p.c.H - item % p.c.H;
                j = 0;
                continue;
            }
            const int from = j, take = w - j < left ? w - j : (int)left;
            at = item, j0 = it.block(j, start), nblk = it.block(j + take, start) - j0;
            left -= take;
            j += take;
            if (j == w) ++item, j = 0;
            if (nblk > 0 || (it.blocks == 0 && from == 0)) return true;
        }
        return false;
    }
};

constexpr int CP_PARTS = 2;    // on their way from the warp that walks to the others
struct CpPart {
    CpItem it;
    int item, j0, nblk, more;
};

template <int EP> struct CpCfg {
    static constexpr int ATOMS = EP / 64;
    static constexpr int SIDE = ATOMS * CP_ATOM;                 // an operand tile
    static constexpr int STAGES = 2;
    static constexpr int S_Q = 0, S_K = 2 * SIDE, S_V = S_K + STAGES * SIDE, S_C = S_V + STAGES * SIDE;
    static constexpr int S_BARS = S_C + (CP_SCALES * (int)sizeof(CpScales) + 15) / 16 * 16;
    static constexpr int BARRIERS = 2 + 4 * STAGES + 2 * 5 + 2 * CP_SCALES + 2 * CP_PARTS;
    static constexpr int S_WALK = S_BARS + (BARRIERS + 1) * 8;   // where the share begins; what finding it adds up
    static constexpr int S_PART = S_WALK + (int)sizeof(CpWalk) + 48 * 8;
    static constexpr int SMEM = S_PART + CP_PARTS * (int)sizeof(CpPart);
    static constexpr int O_COL = 2 * CP_KEYS;
};

template <int EP, bool FP8>
__global__ void __launch_bounds__(CP_THREADS, 1)
cache_prompt_kernel(const CachePromptParams p) {
    using Cfg = CpCfg<EP>;
    constexpr int STAGES = Cfg::STAGES, ATOMS = Cfg::ATOMS;
    extern __shared__ __align__(1024) uint8_t smem[];
    const CacheView& c = p.c;
    if ((smem_u32(smem) & 1023u) != 0) {   // uniform across the grid
        if (threadIdx.x == 0) atomicCAS(c.d_status, 0, KST_SMEM_LAYOUT);
        return;
    }
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::S_BARS);
    uint64_t* q_full = bars;                       // [2] four softmax warps
    uint64_t* k_full = q_full + 2;                 // [STAGES] four converting warps
    uint64_t* k_empty = k_full + STAGES;           // one arrival a tile
    uint64_t* v_full = k_empty + STAGES;
    uint64_t* v_empty = v_full + STAGES;
    uint64_t* s_full = v_empty + STAGES;           // [2] a tile's scores are there
    uint64_t* p_half = s_full + 2;                 // [2] half of its P
    uint64_t* p_full = p_half + 2;                 // [2] all of it
    uint64_t* pv_done = p_full + 2;                // [2] its last product
    uint64_t* exp_turn = pv_done + 2;              // [2] whose turn it is to run its exponentials
    uint64_t* c_full = exp_turn + 2;                 // [CP_SCALES] a block's constants
    uint64_t* c_empty = c_full + CP_SCALES;        // four softmax warps a tile
    uint64_t* a_full = c_empty + CP_SCALES;        // [CP_PARTS] a part of an item
    uint64_t* a_empty = a_full + CP_PARTS;         // every other warp
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(a_empty + CP_PARTS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    CpScales* consts = reinterpret_cast<CpScales*>(smem + Cfg::S_C);
    static_assert(Cfg::BARRIERS == 2 + 4 * STAGES + 10 + 2 * CP_SCALES + 2 * CP_PARTS, "barriers counted by the layout");

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(&q_full[t], 4);
            mbar_init(&s_full[t], 1);
            mbar_init(&p_half[t], 4);
            mbar_init(&p_full[t], 4);
            mbar_init(&pv_done[t], 1);
            mbar_init(&exp_turn[t], 4);
        }
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&k_full[s], 4);
            mbar_init(&k_empty[s], 2);
            mbar_init(&v_full[s], 4);
            mbar_init(&v_empty[s], 2);
        }
        for (int s = 0; s < CP_SCALES; ++s) {
            mbar_init(&c_full[s], 1);
            mbar_init(&c_empty[s], 8);
        }
        for (int s = 0; s < CP_PARTS; ++s) {
            mbar_init(&a_full[s], 1);
            mbar_init(&a_empty[s], CP_THREADS / 32 - 1);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    grid_dep_wait();          // the lengths may come from the launch before
    grid_dep_launch();
    CpWalk* walk = reinterpret_cast<CpWalk*>(smem + Cfg::S_WALK);
    if (!p.shared) {
        const int w = cp_item(p, blockIdx.x).weight(0);
        if (w == 0) return;                        // uniform: before any barrier or tensor memory exists
        if (threadIdx.x == 0) *walk = {w, (int)blockIdx.x, 0, 0};
    } else {
        // Weights are the same for all heads: an entry has the H items of a row pair of a sequence.  A thread sums a run of
        // them; the sums before it tell which thread's run the share of this block begins in.
        long long* sums = reinterpret_cast<long long*>(smem + Cfg::S_WALK + sizeof(CpWalk));
        const int entries = p.items / c.H, run = (entries + CP_THREADS - 1) / CP_THREADS, e0 = threadIdx.x * run;
        long long mine = 0, some = 0;              // blocks of keys, items
        int longest = 0;
        for (int e = e0; e < e0 + run && e < entries; ++e) {
            const int w = cp_item(p, e * c.H).weight(0);
            mine += (long long)w * c.H;
            some += w > 0 ? c.H : 0;
            longest = w > longest ? w : longest;
        }
        long long upto = mine, items = some;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const long long x = __shfl_up_sync(0xffffffffu, upto, d), z = __shfl_up_sync(0xffffffffu, items, d);
            if (lane >= d) upto += x, items += z;
            const int y = __shfl_xor_sync(0xffffffffu, longest, d);
            longest = y > longest ? y : longest;
        }
        if (lane == 31) sums[warp] = upto, sums[16 + warp] = items, sums[32 + warp] = longest;
        __syncthreads();
        long long total = 0, pieces = 0;
        for (int i = 0; i < CP_THREADS / 32; ++i) {
            if (i == warp) upto += total, items += pieces;
            total += sums[i], pieces += sums[16 + i];
            if (sums[32 + i] > longest) longest = (int)sums[32 + i];
        }
        // as many shares as blocks, but of CP_LEAST blocks of keys at least where there are no more items than that makes
        const long long want = pieces > total / CP_LEAST ? pieces : total / CP_LEAST;
        long long many = want < gridDim.x ? want : gridDim.x;
        // Lengths far apart: what the start and end of an item take counts too, or a share of many short ones is the last to end (74
        // items of 4 to 39 blocks 56 us without and 51 with; 128 of 64 to 80 213 and 212, 32 of 32 36.0 and 38.8).
        const int start = 4 * total < 3 * pieces * longest && total >= 4 * many ? CP_START : 0;
        total += start * pieces, upto += start * items, mine += start * some, longest += start;
        // Items of one length: whole shares an item, where the blocks that this leaves out would save the others less than the four
        // blocks of keys that a second part's start and end cost (32 items of 32 blocks: 39.5 us with 148 shares, 36.1 with 128; 64 of 64 86.8 and 90.4).
        const long long even = pieces > 0 && pieces <= many ? many - many % pieces : many;
        if (pieces * longest == total && total * (many - even) <= 4 * many * even) many = even;
        const Shares shares(total, (int)many);
        if ((int)blockIdx.x >= shares.warps) {     // uniform
            if (threadIdx.x == 0) p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
            return;
        }
        const long long begin = shares.begin(blockIdx.x), end = shares.begin(blockIdx.x + 1);
        __syncthreads();        // the sums are read
        if (begin >= upto - mine && begin < upto) {
            long long at = upto - mine;
            for (int e = e0; e < e0 + run && e < entries; ++e) {
                const int w = cp_item(p, e * c.H).weight(start);
                if (begin < at + (long long)w * c.H) {
                    const int h = (int)floor_div(begin - at, w);
                    at += (long long)h * w;
                    *walk = {end - begin, e * c.H + h, (int)(begin - at), start};
                    sums[0] = at + start, sums[1] = at + w - 1, sums[2] = total;   // its first block, its last
                    sums[3] = shares.warps;
                    break;
                }
                at += (long long)w * c.H;
            }
        }
    }

    if (warp == 15) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    CpPart* part = reinterpret_cast<CpPart*>(smem + Cfg::S_PART);
    // A warp leaves a wait that runs out as one: lanes that went on alone would wait for the others in the next vote, for good.
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, c.d_status, code, abort_flag));
    };
    // The next part of the block's share; barriers go on over all of them.
    CpItem it;
    int item = 0, j_begin = 0, nblk = 0, parts_seen = 0;
    auto next = [&]() -> bool {
        const int s = parts_seen % CP_PARTS;
        if (!wait(&a_full[s], (uint32_t)((parts_seen / CP_PARTS) & 1), KST_WAIT_FULL)) return false;
        CpPart x = part[s];
        // the same for all lanes, which the compiler sees: what depends on them stays in the warp's own registers
        for (int* v : {&x.it.b, &x.it.h, &x.it.r0, &x.it.rows, &x.it.n, &x.it.m, &x.it.blocks, &x.item, &x.j0, &x.nblk, &x.more})
            *v = __shfl_sync(0xffffffffu, *v, 0);
        if (lane == 0) mbar_arrive(&a_empty[s]);
        ++parts_seen;
        it = x.it, item = x.item, j_begin = x.j0, nblk = x.nblk;
        return x.more != 0;
    };

    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CP_OTHER_REGS));
        if (warp == 14) {
            // -------------------------------------------------- pages and scales of the blocks
            int done = 0;
            bool ok = true;
            while (ok && next()) {
                auto page = [&](int j) {
                    const int key = (j_begin + j) * CP_KEYS + (lane & 7) * 16;
                    return j < nblk && key < it.n ? (int)c.page(it.b, key >> c.logT) : -1;
                };
                int pg = page(0), pg1 = page(1);
                float k0 = 0.f, v0 = 0.f;
                auto load = [&](int q, float& k, float& v) {
                    k = q >= 0 ? __ldg(c.kmax + (int64_t)q * c.H + it.h) : 0.f;
                    v = q >= 0 ? __ldg(c.vmax + (int64_t)q * c.H + it.h) : 0.f;
                };
                load(pg, k0, v0);
                for (int j = 0; j < nblk; ++j) {
                    const int pg2 = page(j + 2);
                    float k1, v1;
                    load(pg1, k1, v1);
                    const int s = done % CP_SCALES;
                    if (!wait(&c_empty[s], (uint32_t)((done / CP_SCALES) & 1) ^ 1, KST_WAIT_EMPTY)) { ok = false; break; }
                    ++done;
                    const float f = fmaxf(v0, 0x1p-80f);      // of a page of zeros, whose weights count: as for few rows
                    const float kf = k0 * p.scale_log2;
                    const bool strange = !(kf < INFINITY) || !(v0 < INFINITY);
                    const unsigned hidden = __ballot_sync(0xffffffffu, pg < 0) & 255u, odd = __ballot_sync(0xffffffffu, strange) & 255u;
                    if (lane < 8) {
                        // a page of zeros: its scores are zeros whatever the factor
                        consts[s].score[lane] = make_float2(strange ? 1.f : fmaxf(kf, 0x1p-100f), strange ? 0.f : log2f(f));
                        consts[s].back[lane] = strange ? 1.f : 1.f / f;
                    }
                    if (lane == 0) {
                        consts[s].hidden = (int)hidden;
                        consts[s].odd = (int)odd;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&c_full[s]);
                    pg = pg1, pg1 = pg2, k0 = k1, v0 = v1;
                }
            }
        } else if (warp == 15) {
            // -------------------------------------------------- parts of items
            CpWalk mine = *walk;
            const int first = mine.j > mine.start ? mine.item : -1;      // its share begins inside this item's blocks
            int s = 0;
            CpPart x;
            do {
                x.more = mine.next(p, x.it, x.item, x.j0, x.nblk);
                if (!wait(&a_empty[s % CP_PARTS], (uint32_t)((s / CP_PARTS) & 1) ^ 1, KST_WAIT_EMPTY)) break;
                if (lane == 0) {
                    part[s % CP_PARTS] = x;
                    mbar_arrive(&a_full[s % CP_PARTS]);
                }
                __syncwarp();
                ++s;
            } while (x.more);
            if (p.shared && lane == 0) {     // who joins the item that the share begins inside
                const long long* at = reinterpret_cast<const long long*>(smem + Cfg::S_WALK + sizeof(CpWalk));
                const Shares shares(at[2], (int)at[3]);
                const int w0 = shares.holder(at[0]), w1 = shares.holder(at[1]);
                p.joins[blockIdx.x] = make_int4(w0 + 1 == (int)blockIdx.x ? first : -1, w0, w1, 0);
            }
        } else if (warp < 14) {
            // -------------------------------------------------- issuers: the whole warp waits, one thread issues
            const int t = warp - 12;
            constexpr uint32_t idesc_s = make_idesc_f16(CP_ROWS, CP_KEYS, 0, 0);
            constexpr uint32_t idesc_o = make_idesc_f16(CP_ROWS, EP, 0, 1);
            constexpr uint64_t kdesc0 = make_smem_desc(16, 1024);
            constexpr uint64_t vdesc0 = make_smem_desc(CP_ATOM, 1024);
            const uint32_t q_addr = smem_u32(smem + Cfg::S_Q + t * Cfg::SIDE);
            const uint32_t s_tmem = tmem_base + t * CP_KEYS, o_tmem = tmem_base + Cfg::O_COL + t * EP;
            int done = 0, busy = 0, parts = 0;      // blocks of the share, of this tile, parts of this tile, before this part
            auto issue_qk = [&](int j) -> bool {
                const int i = done + j, sk = i % STAGES;
                if (!wait(&k_full[sk], (uint32_t)((i / STAGES) & 1), KST_WAIT_FULL)) return false;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t k_addr = smem_u32(smem + Cfg::S_K + sk * Cfg::SIDE);
#pragma unroll
                    for (int k = 0; k < EP / 16; ++k) {
                        if (k * 16 >= c.E) break;
                        const uint32_t in = (uint32_t)(k >> 2) * CP_ATOM + (uint32_t)(k & 3) * 32;
                        umma_ss(s_tmem, smem_desc_at(kdesc0, q_addr + in), smem_desc_at(kdesc0, k_addr + in), idesc_s, k != 0);
                    }
                    umma_commit(&s_full[t]);
                    umma_commit(&k_empty[sk]);
                }
                __syncwarp();
                return true;
            };
            auto issue_pv = [&](int j, int sv, int k0, int k1) {
                const uint32_t v_addr = smem_u32(smem + Cfg::S_V + sv * Cfg::SIDE);
#pragma unroll
                for (int k = k0; k < k1; ++k) {
                    const uint64_t vdesc = smem_desc_at(vdesc0, v_addr + k * 2048);
                    umma_ts(o_tmem, s_tmem + k * 8, vdesc, idesc_o, (j | k) != 0);
                    umma_ts(o_tmem, s_tmem + CP_KEYS / 2 + k * 8, vdesc, idesc_o, 1);
                }
            };
            bool ok = true;
            while (ok && next()) {
                if (it.r0 + t * CP_ROWS >= it.rows) {      // no rows: what the other tile reads is released from here too
                    for (int j = 0; ok && j < nblk; ++j) {
                        const int i = done + j, s = i % STAGES;
                        const uint32_t ph = (uint32_t)((i / STAGES) & 1);
                        ok = wait(&k_full[s], ph, KST_WAIT_FULL);
                        if (ok && elect_one()) mbar_arrive(&k_empty[s]);
                        ok = ok && wait(&v_full[s], ph, KST_WAIT_FULL);
                        if (ok && elect_one()) mbar_arrive(&v_empty[s]);
                        __syncwarp();
                    }
                    done += nblk;
                    continue;
                }
                if (nblk == 0) continue;
                ok = wait(&q_full[t], (uint32_t)(parts & 1), KST_WAIT_FULL) && issue_qk(0);
                for (int j = 0; ok && j < nblk; ++j) {
                    const int i = done + j, sv = i % STAGES;
                    const uint32_t ph = (uint32_t)((busy + j) & 1);
                    ok = wait(&v_full[sv], (uint32_t)((i / STAGES) & 1), KST_WAIT_FULL) && wait(&p_half[t], ph, KST_WAIT_SOFTMAX);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) issue_pv(j, sv, 0, 4);
                    __syncwarp();
                    ok = wait(&p_full[t], ph, KST_WAIT_SOFTMAX);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        issue_pv(j, sv, 4, 8);
                        umma_commit(&pv_done[t]);
                        umma_commit(&v_empty[sv]);
                    }
                    __syncwarp();
                    if (j + 1 < nblk) ok = issue_qk(j + 1);   // over P(j): after the product that reads it, in issue order
                }
                done += nblk, busy += nblk, ++parts;
            }
        }
    } else if (warp >= 8) {
        // ------------------------------------------------------ 8 bits to fp16, in the swizzle
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CP_CONVERT_REGS));
        // Lane (sub, ch) of a warp has keys 32 w + 8 i + sub of a block and elements 64 a + 16 ch on: the eight lanes that a store to
        // shared memory serves at a time hold four chunks of two neighbouring rows, which the swizzle puts into all banks.
        const int w = warp - 8, ch = lane & 3, sub = lane >> 2;
        constexpr int NV = 4 * ATOMS;           // vectors a lane holds of a side
        int page0 = -1, page1 = -1;             // of the warp's first and second 16 keys
        auto look = [&](int j) {
            const int key = (j_begin + j) * CP_KEYS + w * 32;
            page0 = page1 = -1;
            if (j < nblk && key < it.n) {
                page0 = (int)c.page(it.b, key >> c.logT);
                page1 = c.T > 16 ? page0 : key + 16 < it.n ? (int)c.page(it.b, (key >> 4) + 1) : -1;
            }
        };
        // Sides in turn: K(0), V(0), K(1), ...  One copy of the code serves both: the loops of all warps together do not fit the nearer
        // instruction caches, and this one's length is everyone's wait (2048 tokens over 10240, with one half a weight, 177 us with a copy each, 163 with one).
        // What it costs is a side less on its way from memory, which a cache that is read once misses: 64 tokens over 100000 122 us
        // and 127.  Asking L2 for later rows gave some of that back, and its code took as much from the others.
        uint4 cur[NV], nxt[NV];
        auto fetch = [&](uint4 (&to)[NV], int j, int side) {   // zeros where there is no key: what P = 0 multiplies is a number
            const int key0 = (j_begin + j) * CP_KEYS + w * 32, in = (key0 & (c.T - 1)) + sub;
            const uint8_t* base = (side ? c.v : c.k) + it.h * (side ? c.vH : c.kH) + ch * 16;
            const int64_t sT = side ? c.vT : c.kT, sP = side ? c.vP : c.kP;
            const uint8_t* at0 = base + page0 * sP + in * sT;
            const uint8_t* at1 = base + page1 * sP + (c.T > 16 ? in + 16 : sub) * sT;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int a = i % ATOMS, r = i / ATOMS;
                const bool on = (r < 2 ? page0 : page1) >= 0 && key0 + 8 * r + sub < it.n && a * 64 + ch * 16 < c.E;
                to[i] = make_uint4(0, 0, 0, 0);
                if (on) to[i] = __ldg(reinterpret_cast<const uint4*>((r < 2 ? at0 : at1) + (r & 1) * 8 * sT + a * 64));
            }
        };
        // A value that is the code of a NaN reads as 448: a row that may not see it must not meet it.  The lesser of a number and a NaN is
        // the number, so for keys the bound is a NaN and all stays as it is.
        auto write = [&](uint32_t tile, __half2 most) {
            const uint32_t even = tile + (w * 32 + sub) * 128 + (((2 * ch) ^ sub) << 4);   // a row's place modulo 8 is sub
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const uint32_t v[4] = {cur[i].x, cur[i].y, cur[i].z, cur[i].w};
                uint32_t h[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    cache_halves<FP8>(v[k], h[2 * k], h[2 * k + 1]);
                    if (FP8) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const __half2 x = __hmin2(*reinterpret_cast<__half2*>(&h[2 * k + u]), most);
                            h[2 * k + u] = *reinterpret_cast<const uint32_t*>(&x);
                        }
                    }
                }
                const uint32_t at = even + (uint32_t)((i % ATOMS) * CP_ATOM + (i / ATOMS) * 1024);
                st_shared_v4(at, h);
                st_shared_v4(at ^ 16u, h + 4);   // the chunk's neighbour
            }
            fence_proxy_async_smem();
            __syncwarp();
        };
        int done = 0;
        bool ok = true;
        while (ok && next()) {
            look(0);
            fetch(cur, 0, 0);
#pragma unroll 1
            for (int j = 0; ok && j < nblk; ++j) {
                const int s = (done + j) % STAGES;
                const uint32_t ph = (uint32_t)(((done + j) / STAGES) & 1) ^ 1;
#pragma unroll 1
                for (int side = 0; side < 2; ++side) {
                    fetch(nxt, j + side, side ^ 1);
                    if (side == 0) look(j + 1);      // what is fetched next is of the next block
                    uint64_t *empty = side ? v_empty : k_empty, *full = side ? v_full : k_full;
                    if (!wait(&empty[s], ph, KST_WAIT_EMPTY)) { ok = false; break; }
                    write(smem_u32(smem + Cfg::S_K + (side * STAGES + s) * Cfg::SIDE), __half2half2(__ushort_as_half(side ? 0x5f00 : 0x7fff)));
                    if (lane == 0) mbar_arrive(&full[s]);
#pragma unroll
                    for (int u = 0; u < NV; ++u) cur[u] = nxt[u];
                }
            }
            done += nblk;
        }
    } else {
        // ------------------------------------------------------ softmax and results
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(CP_SOFTMAX_REGS));
        const int t = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lane_base = uint32_t(quad * 32) << 16;
        const uint32_t s_tmem = tmem_base + lane_base + t * CP_KEYS, o_tmem = tmem_base + lane_base + Cfg::O_COL + t * EP;
        int done = 0, busy = 0, turns = 0;          // blocks of the share, of this tile, of both tiles, before this one
        bool ok = true;
        while (ok && next()) {
            if (it.r0 + t * CP_ROWS >= it.rows) {
                for (int j = 0; ok && j < nblk; ++j, ++done) {
                    const int cs = done % CP_SCALES;
                    ok = wait(&c_full[cs], (uint32_t)((done / CP_SCALES) & 1), KST_WAIT_FULL);
                    if (ok && lane == 0) mbar_arrive(&c_empty[cs]);
                }
                continue;
            }
            const int r = it.r0 + t * CP_ROWS + row, l = r / p.G, hq = it.h * p.G + r - l * p.G;   // new token, query head
            const bool live = r < it.rows;
            if (nblk > 0) {
                // a row's chunks are read by neighbouring lanes, whole lines; all of them are on their way at once
                constexpr int CH = EP / 8, STEP = 32 / CH;
                const int ch = lane % CH;
                const uint32_t dst = smem_u32(smem + Cfg::S_Q + t * Cfg::SIDE) + (uint32_t)(ch >> 3) * CP_ATOM;
                int to = quad * 32 + lane / CH, lq = (it.r0 + t * CP_ROWS + to) / p.G, g = it.r0 + t * CP_ROWS + to - lq * p.G;
                const __half* q = p.q + it.h * p.G * p.qH + it.b * p.qB + ch * 8;
#pragma unroll 1
                for (int i = 0; i < CH; ++i, to += STEP) {
                    const bool on = it.r0 + t * CP_ROWS + to < it.rows && ch * 8 < c.E;
                    const __half* at = on ? q + lq * p.qL + g * p.qH : p.q;
                    const uint32_t to_smem = dst + to * 128 + (((ch & 7) ^ (to & 7)) << 4);
                    if (p.whole && !p.negate) {
                        cp_async16(to_smem, at, on);
                    } else {
                        uint32_t v[4] = {0, 0, 0, 0};
                        if (on) cp_load8(v, at, p.whole);
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[k] ^= p.negate ? 0x80008000u : 0u;
                        st_shared_v4(to_smem, v);
                    }
                    for (g += STEP; g >= p.G; g -= p.G) ++lq;
                }
                cp_async_wait();
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[t]);
            }
            const int last = p.causal ? it.n - it.m + l : it.n - 1;                       // the last key this row sees
            const int all_see = p.causal ? it.n - it.m + (it.r0 + t * CP_ROWS) / p.G : it.n - 1;   // that every row of the tile sees
            float m_run = -INFINITY, l_run = 0.f;
            const bool pingpong = it.r0 + CP_ROWS < it.rows;
            for (int j = 0; ok && j < nblk; ++j, ++done, ++busy) {
                const int cs = done % CP_SCALES, key0 = (j_begin + j) * CP_KEYS;
                const CpScales& k = consts[cs];
                ok = __all_sync(0xffffffffu, mbar_wait(&c_full[cs], (uint32_t)((done / CP_SCALES) & 1), c.d_status, KST_WAIT_FULL, abort_flag) &&
                                             mbar_wait(&s_full[t], (uint32_t)(busy & 1), c.d_status, KST_WAIT_TMEM_FULL, abort_flag));
                if (!ok) break;
                tc_fence_after();
                uint32_t x[4][32];
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld32(s_tmem + i * 32, x[i]);
                const int hidden = k.hidden;
                const bool masked = key0 + CP_KEYS - 1 > all_see || hidden != 0;
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int u = 0; u < 32; ++u) asm volatile("" : "+r"(x[i][u]));   // in registers from here on
                if (masked) {
                    const int seen = last - key0;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int u = 0; u < 32; ++u)
                            if (i * 32 + u > seen || (hidden >> (i * 2 + u / 16) & 1)) x[i][u] = 0xff800000u;
                }
                if (k.odd != 0) {     // whoever sees one of the group's keys sees no number
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int u = 0; u < 32; ++u)
                            if ((k.odd >> (i * 2 + u / 16) & 1) && x[i][u] != 0xff800000u) x[i][u] = 0x7fffffffu;
                }
                float top = -INFINITY;
#pragma unroll
                for (int gq = 0; gq < 8; ++gq) {
                    const uint32_t* y = &x[gq >> 1][(gq & 1) * 16];
                    float a = __uint_as_float(y[0]), b2 = __uint_as_float(y[1]);
#pragma unroll
                    for (int u = 2; u < 16; u += 4) {
                        a = cp_max3(a, __uint_as_float(y[u]), __uint_as_float(y[u + 1]));
                        if (u + 2 < 16) b2 = cp_max3(b2, __uint_as_float(y[u + 2]), __uint_as_float(y[u + 3]));
                    }
                    top = fmaxf(top, fmaf(fmaxf(a, b2), k.score[gq].x, k.score[gq].y));
                }
                // the reference point follows lazily: only when the maximum has grown by more than 2^8; P goes in times 2^7
                const float m_new = top > m_run + 8.f ? top : m_run, m_sub = m_new == -INFINITY ? 0.f : m_new - 7.f;
                if (__any_sync(0xffffffffu, m_new != m_run)) {
                    const float alpha = m_run == m_new ? 1.f : cp_ex2(m_run - m_new);
                    l_run *= alpha;
                    if (j > 0) {          // these scores were issued after the last P V: it is done
#pragma unroll 1
                        for (int i = 0; i < EP / 16; ++i) {
                            uint32_t o16[16];
                            tmem_ld16(o_tmem + i * 16, o16);
                            tmem_wait_ld();
#pragma unroll
                            for (int u = 0; u < 16; ++u) o16[u] = __float_as_uint(__uint_as_float(o16[u]) * alpha);
                            tmem_st16(o_tmem + i * 16, o16);
                        }
                        tmem_wait_st();
                    }
                    m_run = m_new;
                }
                if (pingpong && (t == 1 || turns > 0) &&
                    !wait(&exp_turn[t], (uint32_t)((t == 1 ? turns : turns - 1) & 1), KST_WAIT_SOFTMAX)) { ok = false; break; }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t pk[16], pl[16];
#pragma unroll
                    for (int g2 = 0; g2 < 2; ++g2) {
                        const float kf = k.score[2 * i + g2].x, add = k.score[2 * i + g2].y - m_sub;
                        const uint64_t k2 = pack2(kf, kf), a2 = pack2(add, add);
                        uint64_t sum = pack2(0.f, 0.f);
#pragma unroll
                        for (int u = 0; u < 8; ++u) {
                            const uint32_t u0 = x[i][g2 * 16 + 2 * u], u1 = x[i][g2 * 16 + 2 * u + 1];
                            float e0, e1;
                            unpack2(fma2(pack2(__uint_as_float(u0), __uint_as_float(u1)), k2, a2), e0, e1);
                            e0 = cp_ex2(e0), e1 = cp_ex2(e1);
                            sum = add2(sum, pack2(e0, e1));
                            cp_halves(e0, e1, pk[g2 * 8 + u], pl[g2 * 8 + u]);
                        }
                        float s0, s1;
                        unpack2(sum, s0, s1);
                        l_run = fmaf(s0 + s1, k.back[2 * i + g2], l_run);
                    }
                    cp_tmem_st16(s_tmem + i * 16, pk);
                    cp_tmem_st16(s_tmem + CP_KEYS / 2 + i * 16, pl);
                    if (i == 1) {
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_half[t]);
                    }
                }
                if (pingpong) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&exp_turn[1 - t]);
                    ++turns;
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&p_full[t]);
                    mbar_arrive(&c_empty[cs]);
                }
            }
            if (ok && nblk > 0) ok = wait(&pv_done[t], (uint32_t)((busy - 1) & 1), KST_WAIT_SOFTMAX);
            __syncwarp();
            if (ok) {
                tc_fence_after();
                const float back = 1.f / cache_top<FP8>();
                const bool whole = j_begin == 0 && nblk == it.blocks;
                const float f = !whole ? back : back / (l_run == 0.f ? 1.f : l_run);
                const int64_t at = l * p.oL + hq * p.oH + it.b * p.oB;
                const int64_t place = (int64_t)blockIdx.x * 2 + (j_begin == 0 ? 1 : 0);
                const int prow = t * CP_ROWS + row;
#pragma unroll 1
                for (int i = 0; i < EP / 16; ++i) {
                    uint32_t o16[16];
                    __syncwarp();
                    if (nblk > 0) {
                        tmem_ld16(o_tmem + i * 16, o16);
                        tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int u = 0; u < 16; ++u) o16[u] = 0;
                    }
                    if (!live || i * 16 >= c.E) continue;
                    float v[2][8];
#pragma unroll
                    for (int u = 0; u < 16; ++u) v[u >> 3][u & 7] = __uint_as_float(o16[u]) * f;
                    if (!whole) {
                        float4* d = reinterpret_cast<float4*>(p.part + place * (2 * CP_ROWS * EP)) + i * 4 * (2 * CP_ROWS) + prow;
#pragma unroll
                        for (int u = 0; u < 4; ++u) d[u * 2 * CP_ROWS] = make_float4(v[u >> 1][(u & 1) * 4], v[u >> 1][(u & 1) * 4 + 1], v[u >> 1][(u & 1) * 4 + 2], v[u >> 1][(u & 1) * 4 + 3]);
                    } else {
                        cp_store8(p, at + i * 16, v[0]);
                        cp_store8(p, at + i * 16 + 8, v[1]);
                    }
                }
                if (live && !whole) *reinterpret_cast<float2*>(p.part_ml + (place * 2 * CP_ROWS + prow) * 2) = make_float2(m_run, l_run);
            }
        }
    }
    if (*abort_flag) {
        for (int i = 0; i < 4; ++i) __nanosleep(1000000);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 15) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// The items that several blocks have parts of, sixteen elements of a row a thread: the second block of an item stands for it.
template <int EP>
__global__ void __launch_bounds__(256)
cache_prompt_join_kernel(const CachePromptParams p) {
    grid_dep_wait();
    grid_dep_launch();
    const int4 at = p.joins[blockIdx.x / (EP / 16)];
    if (at.x < 0) return;
    const int row = threadIdx.x, e = (int)(blockIdx.x % (EP / 16)) * 16;
    const CpItem it = cp_item(p, at.x);
    const int r = it.r0 + row;
    if (r >= it.rows || e >= p.c.E) return;
    const int l = r / p.G, hq = it.h * p.G + r - l * p.G;
    auto place = [&](int w) { return (int64_t)w * 2 + (w == at.y ? 1 : 0); };
    auto stat = [&](int w) { return *reinterpret_cast<const float2*>(p.part_ml + (place(w) * 2 * CP_ROWS + row) * 2); };
    float M = -INFINITY, sum = 0.f, v[2][8] = {};
    for (int w = at.y; w <= at.z; ++w) M = fmaxf(M, stat(w).x);
    for (int w = at.y; w <= at.z; ++w) {
        const float2 ml = stat(w);
        const float f = ml.x == M ? 1.f : exp2f(ml.x - M);
        const float4* x = reinterpret_cast<const float4*>(p.part + place(w) * (2 * CP_ROWS * EP)) + e / 4 * (2 * CP_ROWS) + row;
        sum = fmaf(ml.y, f, sum);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float4 a = x[u * 2 * CP_ROWS];
            float* d = &v[u >> 1][(u & 1) * 4];
            d[0] = fmaf(a.x, f, d[0]), d[1] = fmaf(a.y, f, d[1]), d[2] = fmaf(a.z, f, d[2]), d[3] = fmaf(a.w, f, d[3]);
        }
    }
    const float inv = sum == 0.f ? 1.f : 1.f / sum;
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k >> 3][k & 7] *= inv;
    const int64_t to = l * p.oL + hq * p.oH + it.b * p.oB + e;
    cp_store8(p, to, v[0]);
    cp_store8(p, to + 8, v[1]);
}

template <int EP, bool FP8>
static int cp_launch(b200_ctx* ctx, CachePromptParams& p) {
    using Cfg = CpCfg<EP>;
    auto kern = cache_prompt_kernel<EP, FP8>;
    static std::atomic<uint64_t> asked{0};
    B200_CUDA(allow_smem(ctx, kern, Cfg::SMEM, asked));
    const int64_t sms = ctx->prop.multiProcessorCount;
    const int64_t items = cdiv((int64_t)p.L * p.G, 2 * CP_ROWS) * p.c.H * p.B;
    B200_REQUIRE(items < (1ll << 24), B200_DECLINE_EXTENT, "cache_attention: %lld row tiles", (long long)items);
    p.items = (int)items;
    // Equal shares keep every SM busy to the end.  They cost a look for the share's place and a second launch that joins, together
    // about what four blocks of keys do, and a further start and end for most items, about six (of 2 us at E = 128).  An item a launch
    // block / shares, us: 128 items of 64 to 80 blocks 225 / 214 (E = 128), 191 / 163 (E = 64); 74 of 4 to 39 91 / 51; 8 of 782 1989 / 151;
    // 32 of 2 to 8 31 / 25; 140 of 50 123 / 128; 256 of 28 to 32 182 / 203; 48 of 1 to 5 20 / 25; 1680 of 1 to 6 199 / 251.  Lengths are not
    // known here: sequences much shorter than their table get shares as if they filled it, and lose what the last four do.
    const int64_t blocks = cdiv((int64_t)p.c.width * p.c.T, CP_KEYS);
    p.shared = items <= 8 * sms && items * (blocks + 6) + 4 * sms < cdiv(items, sms) * blocks * sms;
    const int64_t grid = p.shared ? sms : items;
    if (p.shared) {
        void* ws = nullptr;
        const size_t rows = (size_t)grid * 4 * CP_ROWS;
        int rc = ws_scratch(ctx, rows * (EP + 2) * sizeof(float) + grid * sizeof(int4), &ws);
        if (rc) return rc;
        p.part = static_cast<float*>(ws);
        p.part_ml = p.part + rows * EP;
        p.joins = reinterpret_cast<int4*>(p.part_ml + rows * 2);
    }
    B200_CUDA(launch_dep(kern, dim3((unsigned)grid), dim3(CP_THREADS), Cfg::SMEM, ctx->stream, 1, p));
    ctx->launches++;
    if (p.shared) {
        B200_CUDA(launch_dep(cache_prompt_join_kernel<EP>, dim3((unsigned)(grid * (EP / 16))), dim3(256), 0, ctx->stream, 1, p));
        ctx->launches++;
    }
    return B200_OK;
}

int cache_prompt_run(b200_ctx* ctx, const CacheView& c, int64_t L, int64_t B, int64_t G, const b200_strided4* q, const b200_strided4* out,
                     int out_dtype, float scale, bool fp8, int causal, const int32_t* lens, const int32_t* news) {
    CachePromptParams p = {};
    p.c = c;
    p.q = (const __half*)q->ptr;
    p.qL = q->stride[1], p.qH = q->stride[2], p.qB = q->stride[3];
    p.out = const_cast<void*>(out->ptr);
    p.oL = out->stride[1], p.oH = out->stride[2], p.oB = out->stride[3];
    p.lens = lens, p.news = news;
    p.L = (int)L, p.B = (int)B, p.G = (int)G;
    p.causal = causal, p.out_f32 = out_dtype == B200_F32;
    p.whole = ((uintptr_t)q->ptr % 16 | (uint64_t)q->stride[1] % 8 | (uint64_t)q->stride[2] % 8 | (uint64_t)q->stride[3] % 8) == 0;
    const int64_t size = p.out_f32 ? 4 : 2;
    p.out_whole = ((uintptr_t)out->ptr | (uint64_t)(out->stride[1] * size) | (uint64_t)(out->stride[2] * size) | (uint64_t)(out->stride[3] * size)) % 16 == 0;
    p.negate = scale < 0.f;
    p.scale_log2 = (float)(fabs((double)scale) * 1.4426950408889634 / (fp8 ? 448.0 : 127.0));
    if (c.E <= 64) return fp8 ? cp_launch<64, true>(ctx, p) : cp_launch<64, false>(ctx, p);
    return fp8 ? cp_launch<128, true>(ctx, p) : cp_launch<128, false>(ctx, p);
}

} // namespace b200
