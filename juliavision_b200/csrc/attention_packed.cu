// Attention of packed sequences: sequence b has the query rows starts[b] .. starts[b+1] - 1 of q and the keys kstarts[b] ..
// kstarts[b+1] - 1, query head i reads key head i / (Hq / H), and the last query row stands at the last key:
//     out = softmax(scale Q K' + mask) V, row i of n seeing, when causal, the keys up to i + keys - n, else all of its sequence's.
//
// 4 E flops a row and visible key on tcgen05, and as many clocks of the exponential unit as of the products at E = 128, twice as many at 64.
// What bounds it at E = 128 is the chain of a block of keys, which two tiles have between them to hide: 2900 clocks for two tiles and 128 keys, where
// the products are 2048. A tile's softmax is 1300 for exponentials and sums, 240 to 430 for the maximum and 75 for the load of S, and its
// product goes out only then; at E = 64 it is the exponentials (2600 clocks, 2048 of them the unit's).  From one part of the work to the next a
// block takes 1500 to 2500 clocks more.  Once the power limit holds, fewer clocks alone gain little (below, and at the exponentials).  32 query
// heads on 8 key heads of 128, causal: 16384 rows 1980 us (1.11 PFLOP/s), 37 sequences of up to 2000 570 us (0.77); 20 heads
// of 64: 16 sequences of up to 1500 162 us, one of 77 rows 7.2; 20 of 80 on 4, 3 sequences of 500 rows behind 30000 keys: 262.
//
// Query heads that share a key head are stacked with the tokens: a tile's 128 rows are T tokens of G heads, G being the largest power of two up to 128
// that divides the number that share, so that keys and values are read once for G heads and a tile's rows lie close together under the causal
// mask; of 3, 5 or 7 heads each reads them for itself.  A block takes two tiles and walks their keys in blocks of 128: S = Q K' and O += P V with
// S, P (fp16) and O in tensor memory, Q, K and V by TMA through the caller's strides.
//
//   warps 0-3  softmax of tile 0, warps 4-7 of tile 1: one thread a row, its 128 scores in registers
//   warp 8     finds the block's next part of the work (below), tells the others, and asks for Q, K and V
//   warps 9, 10  issue one tile's products each:  Q K(0)', P(0) V(0), Q K(1)', ...
//   warp 11    hands V on to them; where a row does not see a key of the block, it first takes out of the tile what is not finite
//   warps 12-15  take both tiles' results out while the softmax is at the next part
//
// Lengths are on the device, so the work is listed there: the row pairs of all sequences, longest first (packed_plan_kernel).  Blocks take the
// list's units in order as they become free.  Where some pairs are a large part of what an SM has to do, such pairs' blocks of keys are dealt out
// first, the same number in a row to each SM, which cuts pairs along their keys; a second launch joins what was cut.  Calls whose pairs all
// run at once, over few keys, take them as they come and need neither.
#include <cuda_fp16.h>

#include "internal.h"
#include "ptx.cuh"

namespace b200 {

constexpr int PK_THREADS = 512;
constexpr int PK_ROWS = 128, PK_KEYS = 128;      // of a tile
constexpr int PK_ATOM = 128 * 128;               // 128 rows x 64 fp16
constexpr int PK_PARTS = 3;                      // parts of the work on their way from warp 8 to the others
constexpr int PK_SOFTMAX_REGS = 184, PK_OTHER_REGS = 56, PK_OUT_REGS = 88;
static_assert(256 * PK_SOFTMAX_REGS + 128 * PK_OTHER_REGS + 128 * PK_OUT_REGS <= PK_THREADS * 128, "what the launch holds");
constexpr int PK_IDLE = 10;                      // blocks of keys an SM may stand idle before pairs are cut
constexpr int PK_BUCKETS = 1024;                 // lengths that the list tells apart

// mbar_wait in as few instructions as it takes: what the roles of a block run through, all together, has to fit the nearer instruction caches.  A
// try sleeps for 1.5 us at most, so that the tries end after some three seconds; why is left in shared memory, for the block's end.
constexpr uint32_t PK_TRIES = 1u << 21;
__device__ __forceinline__ bool pk_wait(uint64_t* bar, uint32_t parity, int code, volatile int* why) {
#pragma unroll 1
    for (uint32_t n = PK_TRIES; n != 0; --n)
        if (mbar_try_wait(bar, parity)) return true;
    *why = code;
    return false;
}

struct __align__(16) PackedEntry {
    int q0, n, k0, m;                  // the sequence: first row, rows, first key, keys
    int pair, blocks, pad[2];
};
struct __align__(16) PackedCut {
    int slot, parts, head, token;      // first slot (the others are the next even ones), parts; unit of the row pair; first token of tile 0
    int q0, n, pad[2];
};

struct PackedParams {
    const __half* v;                   // for what is not finite
    int64_t vN, vH;
    void* out;
    int64_t oN, oH;
    const int32_t *starts, *kstarts;
    int N, Nk, B, H, Hq, E;
    int G, T, groups, share;           // heads and tokens of a tile, G T = 128; tiles' worth of heads of a key head; heads that share a key head
    int log_g;
    int causal, out_f32, out_whole;
    float scale_log2;
    int heads;                         // H * groups: units of a row pair
    int most;                          // row pairs that the list has room for: what sequences in order can have
    int planned;
    // The list (null without one): row pairs with their sequence's place and size, pair and blocks of keys, the long ones first; how many blocks the
    // long ones before have, of all heads; counters; what is cut, a head at a time, as the launch that joins it wants it.
    PackedEntry* entry;
    int* before;
    int4* counts;                      // units, long entries, cut heads, units taken beyond the first of each block;
                                       // blocks dealt to an SM, the first of them, the long ones' blocks, units before what is dealt
    int* first;                        // [B] first pair of a sequence, where they are too many for shared memory
    PackedCut* cut;
    float *part, *part_ml;             // [2 an SM][E / 4][256 rows][4] and [2 an SM][256][2]: reference point, sum
    int sms;
    int* d_status;
};

__device__ __forceinline__ float pk_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pk_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void pk_tmem_st16(uint32_t taddr, const uint32_t* r) {
    uint32_t v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = r[i];
    tmem_st16(taddr, v);
}

// Where a sequence lies.  Whatever starts and kstarts hold, it is inside the arrays.
struct PackedSeq {
    int q0, n, k0, m;      // first row, rows, first key, keys
    __device__ __forceinline__ void range(const PackedParams& p, const int32_t* s, int b, int most, int& at, int& count) const {
        int lo = s[b], hi = s[b + 1];
        if (lo < 0 || hi < lo || hi > most) {
            atomicCAS(p.d_status, 0, KST_PACKED_STARTS);
            lo = lo < 0 ? 0 : lo > most ? most : lo;
            hi = hi < lo ? lo : hi > most ? most : hi;
        }
        at = lo, count = hi - lo;
    }
    __device__ __forceinline__ void of(const PackedParams& p, int b) {
        range(p, p.starts, b, p.N, q0, n);
        range(p, p.kstarts, b, p.Nk, k0, m);
    }
    __device__ __forceinline__ int pairs(const PackedParams& p) const { return (n + 2 * p.T - 1) / (2 * p.T); }
    __device__ __forceinline__ int blocks(const PackedParams& p, int pair) const {   // of keys that some row of the pair sees
        const int top = (pair + 1) * 2 * p.T < n ? (pair + 1) * 2 * p.T : n;
        const int seen = p.causal ? m - n + top : m;
        return seen <= 0 ? 0 : (seen + PK_KEYS - 1) / PK_KEYS;
    }
};

// ------------------------------------------------------------------------------------------ the list of the work
// One block, which the launch behind it waits for: sequences in shared memory, few barriers, no lane waits for another's atomic (10 to 31 us with
// sequences in global memory and sums by atomics, 6 to 8 so).
constexpr int PL_THREADS = 1024, PL_SEQS = 1024;    // sequences kept in shared memory

__device__ __forceinline__ int pl_scan(int x, int* sums, int& total) {   // exclusive; sums: 32 of its own
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int upto = x;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += y;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    const int mine = sums[lane];
    int all = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, all, d);
        if (lane >= d) all += y;
    }
    total = __shfl_sync(0xffffffffu, all, 31);
    return __shfl_sync(0xffffffffu, all - mine, warp) + upto - x;
}
// One more in bucket b for each lane that is `on`; the lane's place in it.
__device__ __forceinline__ int pl_count(int* bucket, int b, bool on) {
    const unsigned same = __match_any_sync(0xffffffffu, on ? b : -1);
    const int lane = threadIdx.x & 31, leader = __ffs(same) - 1;
    int at = 0;
    if (on && lane == leader) at = atomicAdd(&bucket[b], __popc(same));
    return __shfl_sync(0xffffffffu, at, leader) + __popc(same & ((1u << lane) - 1));
}

__global__ void __launch_bounds__(PL_THREADS)
packed_plan_kernel(const PackedParams p) {
    __shared__ int sums[32], bucket[PK_BUCKETS], first_here[PL_SEQS];
    __shared__ int4 seqs[PL_SEQS];
    static_assert(PK_BUCKETS == PL_THREADS, "a bucket a thread");
    const int tid = threadIdx.x;
    grid_dep_wait();
    grid_dep_launch();
    const bool here = p.B <= PL_SEQS;
    int* first = here ? first_here : p.first;
    int entries = 0;
    for (int base = 0; base < p.B; base += PL_THREADS) {
        PackedSeq s = {0, 0, 0, 0};
        if (base + tid < p.B) s.of(p, base + tid);
        int total;
        const int at = pl_scan(s.pairs(p), sums, total);
        if (base + tid < p.B) {
            first[base + tid] = entries + at;
            if (here) seqs[tid] = make_int4(s.q0, s.n, s.k0, s.m);
        }
        entries = entries + total < p.most ? entries + total : p.most;      // sequences that overlap, which has been reported
    }
    bucket[tid] = 0;
    __syncthreads();
    auto entry = [&](int e, PackedSeq& s, int& pair, int& blocks) {
        int lo = 0, hi = p.B;          // the last sequence whose first pair is at or before e
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (first[mid] <= e) lo = mid;
            else hi = mid;
        }
        if (here) {
            const int4 x = seqs[lo];
            s = {x.x, x.y, x.z, x.w};
        } else {
            s.of(p, lo);
        }
        pair = e - first[lo];
        blocks = s.blocks(p, pair);
    };
    // Blocks of keys of all pairs and heads; what an SM's share of them is.  The first 1024 pairs stay in registers.
    PackedSeq s0 = {0, 0, 0, 0};
    int pair0 = 0, blocks0 = 0;
    long long mine = 0;
    int longest = 0;
    for (int e = tid; e < entries; e += PL_THREADS) {
        PackedSeq s;
        int pair, n;
        entry(e, s, pair, n);
        if (e == tid) s0 = s, pair0 = pair, blocks0 = n;
        mine += n > 0 ? n : 1;
        longest = n > longest ? n : longest;
    }
#pragma unroll
    for (int d = 1; d < 32; d *= 2) mine += __shfl_xor_sync(0xffffffffu, mine, d);
    longest = __reduce_max_sync(0xffffffffu, longest);
    __shared__ long long total_of[32];
    __shared__ int longest_of[32];
    if ((tid & 31) == 0) total_of[tid >> 5] = mine, longest_of[tid >> 5] = longest;
    __syncthreads();
    long long all = total_of[tid & 31];
    longest = __reduce_max_sync(0xffffffffu, longest_of[tid & 31]);
#pragma unroll
    for (int d = 1; d < 32; d *= 2) all += __shfl_xor_sync(0xffffffffu, all, d);
    all *= p.heads;
    // Long: more than an SM's share, or a quarter of it where all pairs are alike, whose last round leaves SMs idle (where they differ, longest first
    // evens that out: 320 of 16 to 32 blocks, E = 128, 148 us; with the longer ones dealt out, which then share fewer of their keys in the L2 cache,
    // 170).  They stand first, in the sequences' order, for some of them are cut, and which ones must not hang on the order of atomics.  The
    // others follow, longest first; pairs of a bucket come in any order, which changes no result.
    const bool alike = (long long)entries * p.heads * longest * 4 <= all * 5;
    const long long least = alike ? all / 4 / p.sms : all / p.sms;
    const bool longs = longest > least + (alike ? 0 : PK_IDLE) && all < 0x7fffffff - p.sms;
    auto bucket_of = [&](int blocks) { return blocks < PK_BUCKETS ? PK_BUCKETS - 1 - blocks : 0; };
    auto set_down = [&](int at, const PackedSeq& s, int pair, int n) {
        int4* to = reinterpret_cast<int4*>(p.entry + at);
        to[0] = make_int4(s.q0, s.n, s.k0, s.m);
        to[1] = make_int4(pair, n, 0, 0);
    };
    const int rounds = (entries + PL_THREADS - 1) / PL_THREADS;
    int many_long = 0, blocks_long = 0;
    for (int r = 0; r < rounds; ++r) {
        const int e = r * PL_THREADS + tid;
        PackedSeq s = s0;
        int pair = pair0, n = blocks0;
        if (r > 0 && e < entries) entry(e, s, pair, n);
        const bool is = longs && e < entries && n > least;
        pl_count(bucket, bucket_of(n), e < entries && !is);
        if (longs) {
            int total;
            int at = many_long + pl_scan(is, sums, total);
            many_long += total;
            if (is) set_down(at, s, pair, n);
            const int before = blocks_long + pl_scan(is ? n * p.heads : 0, sums, total);
            blocks_long += total;
            if (is) p.before[at] = before;
        }
    }
    __syncthreads();
    {
        int total;
        const int n = bucket[tid], at = pl_scan(n, sums, total);
        bucket[tid] = at;
    }
    __syncthreads();
    for (int r = 0; r < rounds; ++r) {
        const int e = r * PL_THREADS + tid;
        PackedSeq s = s0;
        int pair = pair0, n = blocks0;
        if (r > 0 && e < entries) entry(e, s, pair, n);
        const bool is = longs && e < entries && n > least;
        const int at = pl_count(bucket, bucket_of(n), e < entries && !is);
        if (e < entries && !is) set_down(many_long + at, s, pair, n);
    }
    // Which long ones are dealt out: all of them, or, where they are alike, those that are left when each SM has had as many whole ones as go
    // round; and none where the SMs that would stand idle then lose less than ten blocks of keys (20 heads of 64, 4096 rows, 27 blocks: 127 us
    // for 146 whole; 100 rows over 3000 keys, 15 blocks: 23 for 32; 16 heads of 128, 4096 rows, 9 blocks: 158 for 149).
    int whole = many_long * p.heads, each = 0, many = 0, from = blocks_long;
    if (many_long > 0) {
        const int items = whole, left = items % p.sms;
        if (!alike) whole = 0;
        else if (left > 0 && longest - (long long)longest * left / p.sms > PK_IDLE) whole = items - left;
        __syncthreads();
        if (whole < items) {
            const int e = whole / p.heads;
            from = p.before[e] + (whole - e * p.heads) * p.entry[e].blocks;
            each = (blocks_long - from + p.sms - 1) / p.sms;
        }
        // SM c's first block of keys is from + c * each; where that is inside a pair, the pair is cut, and the first such SM lists it.
        for (int base = 0; each > 0 && base < p.sms; base += PL_THREADS) {
            const int c = base + tid;
            PackedCut x = {};
            if (c > 0 && c < p.sms && from + (long long)c * each < blocks_long) {
                const int at = from + c * each;
                int lo = 0, hi = many_long;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) / 2;
                    if (p.before[mid] <= at) lo = mid;
                    else hi = mid;
                }
                const PackedEntry y = p.entry[lo];
                const int rel = at - p.before[lo], size = y.blocks, head = rel / size, start = at - (rel - head * size);
                if (start < at && start >= at - each) {
                    x.parts = (start - from + size - 1) / each - (c - 1) + 1;
                    x.slot = 2 * (c - 1) + (start > at - each), x.head = head, x.token = y.pair * 2 * p.T, x.q0 = y.q0, x.n = y.n;
                }
            }
            int total;
            const int at = pl_scan(x.parts > 0, sums, total);
            if (x.parts > 0) {
                int4* to = reinterpret_cast<int4*>(p.cut + many + at);
                to[0] = make_int4(x.slot, x.parts, x.head, x.token);
                to[1] = make_int4(x.q0, x.n, 0, 0);
            }
            many += total;
        }
    }
    if (tid == 0) {
        p.counts[0] = make_int4(entries * p.heads, many_long, many, 0);
        p.counts[1] = make_int4(each, from, blocks_long, whole);
    }
}

// A block's work: some of the key blocks of two tiles.
struct PackedPart {
    int q0, n, k0, m;            // the sequence
    int h, g0, token;            // key head, first of its query heads, first token of tile 0
    int j0, nblk, slot, more;    // key blocks; slot < 0: the whole of the item
};

// A unit of the work: a row pair, or a part of its keys, for one group of heads of a key head.
struct PackedUnit {
    PackedSeq s;
    int pair, blocks, head, j0, slot;
    int next;                    // of the blocks dealt out, the first behind this unit; -1 before, PK_DEALT behind them
};
__device__ __forceinline__ void pk_part(const PackedParams& p, PackedPart& x, const PackedUnit& u) {
    x.q0 = u.s.q0, x.n = u.s.n, x.k0 = u.s.k0, x.m = u.s.m;
    x.h = u.head / p.groups, x.g0 = (u.head - x.h * p.groups) * p.G;
    x.token = u.pair * 2 * p.T;
    x.j0 = u.j0, x.nblk = u.blocks, x.slot = u.slot;
}

// The next of what is dealt out to this block, and then unit `unit` of the list; found by a whole warp.
constexpr int PK_DEALT = -2;     // PackedUnit::next behind what was dealt out
__device__ __forceinline__ bool pk_listed(const PackedParams& p, int unit, PackedUnit& x) {
    const int lane = threadIdx.x & 31;
    // where nothing is dealt out it is its pair's `heads` units on; asked for along with the counters
    int e = unit / p.heads, rel = unit - e * p.heads;
    PackedEntry it = p.entry[e < p.most ? e : p.most - 1];
    const int4 counts = p.counts[0], dealt = p.counts[1];
    x.j0 = 0, x.slot = -1;
    if (dealt.x > 0 && x.next != PK_DEALT) {
        const long long mine = dealt.y + (long long)blockIdx.x * dealt.x;
        const int start = mine < dealt.z ? (int)mine : dealt.z, end = dealt.z - start < dealt.x ? dealt.z : start + dealt.x;
        const int at = x.next < 0 ? start : x.next;
        if (at < end) {
            int lo = 0, hi = counts.y;          // the last entry that begins at or before this block of keys
#pragma unroll 1
            while (hi - lo > 1) {
                const int step = (hi - lo + 31) / 32, to = lo + lane * step;
                const bool before = to < hi && p.before[to] <= at;
                const int k = 31 - __clz(__ballot_sync(0xffffffffu, before));
                lo += k * step;
                hi = lo + step < hi ? lo + step : hi;
            }
            it = p.entry[lo];
            const int into = at - p.before[lo], size = it.blocks;
            x.head = into / size;
            x.j0 = into - x.head * size;
            const int here = size - x.j0 < end - at ? size - x.j0 : end - at;
            x.blocks = here;
            x.next = at + here;
            if (here < size) x.slot = 2 * blockIdx.x + (at > start);      // at most the first and the last of a block
            x.s = {it.q0, it.n, it.k0, it.m};
            x.pair = it.pair;
            return true;
        }
    }
    x.next = PK_DEALT;
    if (dealt.x > 0 && unit >= dealt.w) {       // behind what was dealt out
        const int skipped = unit + counts.y * p.heads - dealt.w;
        e = skipped / p.heads, rel = skipped - e * p.heads;
        if (skipped < counts.x) it = p.entry[e];
        unit = skipped;
    }
    if (unit >= counts.x) return false;
    x.blocks = it.blocks;
    x.s = {it.q0, it.n, it.k0, it.m};
    x.pair = it.pair, x.head = rel;
    return true;
}
// Without a list: the row pairs of all sequences in their order.
__device__ __forceinline__ bool pk_direct(const PackedParams& p, int unit, PackedUnit& x) {
    const int lane = threadIdx.x & 31, pair = unit / p.heads;
    int before = 0;
#pragma unroll 1
    for (int base = 0; base < p.B; base += 32) {
        PackedSeq s = {0, 0, 0, 0};
        if (base + lane < p.B) s.of(p, base + lane);
        const int n = s.pairs(p);
        int upto = n;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int y = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += y;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + upto > pair);
        if (past) {
            const int k = __ffs(past) - 1;
            x.pair = pair - before - __shfl_sync(0xffffffffu, upto - n, k);
            for (int* v : {&s.q0, &s.n, &s.k0, &s.m}) *v = __shfl_sync(0xffffffffu, *v, k);
            x.s = s;
            x.blocks = s.blocks(p, x.pair), x.head = unit - pair * p.heads;
            x.j0 = 0, x.slot = -1;
            return true;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

template <int EP, bool TWO> struct PkCfg {                       // TWO: fp32 results, weights as two fp16 numbers
    static constexpr int ATOMS = EP / 64;
    static constexpr int SIDE = ATOMS * PK_ATOM;                 // an operand tile
    // P beside S in tensor memory where there is room for it, so that the next scores come while P V reads; else over S, whose 128 columns two
    // halves of P fill.
    static constexpr bool SMALL = EP == 64, OWN_P = SMALL && !TWO;
    static constexpr int STAGES = SMALL ? 8 : 4;                 // K(0), V(0), K(1), ...
    static_assert(STAGES % 2 == 0, "V has stages of its own, every fill of which warp 11 waits for");
    // Quarters of P that P V starts with, where P lies over S: three, 2922 clocks for two tiles and a block of keys; with two 3062.
    static constexpr int FIRST = 3;
    static constexpr int S_Q = 0, S_KV = 2 * SIDE, S_OUT = S_KV + STAGES * SIDE;   // operands; 128 bytes of a tile's rows on their way out, twice
    static constexpr int S_STAT = S_OUT + 2 * PK_ATOM;           // a row's reference point and sum
    static constexpr int S_BARS = S_STAT + 2 * PK_ROWS * 8;
    static constexpr int BARRIERS = 2 * 2 + 3 * STAGES + 2 * 8 + 2 * PK_PARTS;
    static constexpr int S_PART = S_BARS + (BARRIERS + 1) * 8;
    static constexpr int SMEM = S_PART + PK_PARTS * ((int)sizeof(PackedPart) + 4);
    static constexpr int O_COL = 2 * PK_KEYS, P_COL = O_COL + 2 * EP;
    static_assert(SMEM <= 232448, "shared memory over budget");
};

__device__ __forceinline__ void pk_store8(const PackedParams& p, int64_t at, int count, const float (&v)[8]) {   // eight results of a row, or fewer
    if (p.out_whole && count >= 8) {
        if (p.out_f32) {
            float4* d = reinterpret_cast<float4*>((float*)p.out + at);
            d[0] = make_float4(v[0], v[1], v[2], v[3]);
            d[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint4 w;
            __half2* h = reinterpret_cast<__half2*>(&w);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            *reinterpret_cast<uint4*>((__half*)p.out + at) = w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < count) {
            if (p.out_f32) ((float*)p.out)[at + i] = v[i];
            else ((__half*)p.out)[at + i] = __float2half_rn(v[i]);
        }
}

template <int EP, bool TWO>
__global__ void __launch_bounds__(PK_THREADS, 1)
attention_packed_kernel(const __grid_constant__ CUtensorMap tmapQ, const __grid_constant__ CUtensorMap tmapK,
                        const __grid_constant__ CUtensorMap tmapV, const __grid_constant__ CUtensorMap tmapO, const PackedParams p) {
    using Cfg = PkCfg<EP, TWO>;
    constexpr int STAGES = Cfg::STAGES, ATOMS = Cfg::ATOMS;
    constexpr bool OWN_P = Cfg::OWN_P, HALVES = !OWN_P;
    extern __shared__ __align__(1024) uint8_t smem[];
    if ((smem_u32(smem) & 1023u) != 0) {   // uniform across the grid
        if (threadIdx.x == 0) atomicCAS(p.d_status, 0, KST_SMEM_LAYOUT);
        return;
    }
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::S_BARS);
    uint64_t* q_full = bars;                       // [2]
    uint64_t* q_empty = q_full + 2;                // [2] a part's last Q K' is done
    uint64_t* full = q_empty + 2;                  // [STAGES] K or V has landed
    uint64_t* ready = full + STAGES;               // [STAGES, in the order of the blocks] V may be multiplied
    uint64_t* empty = ready + STAGES;              // [STAGES] one arrival a tile
    uint64_t* s_full = empty + STAGES;             // [2] a tile's scores are there
    uint64_t* s_empty = s_full + 2;                // [2] and in registers
    uint64_t* p_half = s_empty + 2;                // [2] the first FIRST quarters of its P
    uint64_t* p_full = p_half + 2;                 // [2] all of it
    uint64_t* pv_done = p_full + 2;                // [2] its last product
    uint64_t* exp_turn = pv_done + 2;              // [2] whose turn it is to run its exponentials
    uint64_t* o_full = exp_turn + 2;               // [2] a part's row sums are there, and the last of its P
    uint64_t* o_empty = o_full + 2;                // [2] they and O have been read
    uint64_t* a_full = o_empty + 2;                // [PK_PARTS] a part of the work
    uint64_t* a_empty = a_full + PK_PARTS;         // every other warp
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(a_empty + PK_PARTS);
    volatile int* why = reinterpret_cast<volatile int*>(tmem_slot + 1);       // 0, or the code of a wait that ran out
    PackedPart* part = reinterpret_cast<PackedPart*>(smem + Cfg::S_PART);
    int* odd = reinterpret_cast<int*>(part + PK_PARTS);   // [PK_PARTS] the first key block of a part from which something was taken out
    static_assert(Cfg::BARRIERS == 4 + 3 * STAGES + 16 + 2 * PK_PARTS, "barriers counted by the layout");

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
#pragma unroll 1
        for (int t = 0; t < 2; ++t) {
            mbar_init(&q_full[t], 1);
            mbar_init(&q_empty[t], 1);
            mbar_init(&s_full[t], 1);
            mbar_init(&s_empty[t], 4);
            mbar_init(&p_half[t], 4);
            mbar_init(&p_full[t], 4);
            mbar_init(&pv_done[t], 1);
            mbar_init(&exp_turn[t], 4);
            mbar_init(&o_full[t], 4);
            mbar_init(&o_empty[t], 4);
        }
#pragma unroll 1
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&ready[s], 1);
            mbar_init(&empty[s], 2);
        }
#pragma unroll 1
        for (int s = 0; s < PK_PARTS; ++s) {
            mbar_init(&a_full[s], 1);
            mbar_init(&a_empty[s], PK_THREADS / 32 - 1);
        }
        *why = 0;
        fence_barrier_init();
        prefetch_tmap(&tmapQ);
        prefetch_tmap(&tmapK);
        prefetch_tmap(&tmapV);
    }
    if (warp == 8) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    grid_dep_wait();
    grid_dep_launch();

    // A warp leaves a wait that runs out as one: lanes that went on alone would wait for the others in the next vote, for good.
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
        return __all_sync(0xffffffffu, pk_wait(bar, parity, code, why));
    };
    PackedPart it;
    int parts_seen = 0;
    auto take = [&]() -> int {        // the next part: its place in the ring, or -1
        const int s = parts_seen % PK_PARTS;
        if (!wait(&a_full[s], (uint32_t)((parts_seen / PK_PARTS) & 1), KST_WAIT_FULL)) return -1;
        it = part[s];
        // the same for all lanes, which the compiler sees: what depends on them stays in the warp's own registers
        for (int* v : {&it.q0, &it.n, &it.k0, &it.m, &it.h, &it.g0, &it.token, &it.j0, &it.nblk, &it.slot, &it.more})
            *v = __shfl_sync(0xffffffffu, *v, 0);
        return it.more ? s : -1;
    };
    auto done_with = [&](int s) {     // nobody of this warp reads the part's place any more
        __syncwarp();
        if (lane == 0) mbar_arrive(&a_empty[s]);
        ++parts_seen;
    };
    // The last key that every row of both tiles sees; blocks that end behind it are masked.
    auto all_see = [&](int token) { return p.causal && it.m - it.n + token < it.m - 1 ? it.m - it.n + token : it.m - 1; };
    // The last key whose value is multiplied whatever it holds.  A weight's lower half may be 0 or below, which makes a NaN of an infinity: none then.
    auto as_it_is = [&]() { return TWO ? -1 : all_see(it.token); };

    float2* stats = reinterpret_cast<float2*>(smem + Cfg::S_STAT);
    // A row of a tile: its token in the tile, its head.  Which rows are any sequence's, and the last key that each sees.
    auto live_row = [&](int t, int l0) { return l0 < it.n - it.token - t * p.T; };
    auto last_key = [&](int t, int l0) { return p.causal ? min(it.m - it.n + it.token + t * p.T + l0, it.m - 1) : it.m - 1; };

    if (warp >= 12) {
        // ------------------------------------------------------ results
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PK_OUT_REGS));
        const int quad = warp & 3, row = quad * 32 + lane, l0 = row >> p.log_g, g = row & (p.G - 1);
        int busy0 = 0, busy1 = 0, parts0 = 0, parts1 = 0;        // blocks and parts of a tile before this one
        constexpr int BAR = 1;                  // the four warps' own barrier
        const uint32_t out = smem_u32(smem + Cfg::S_OUT), swz = (uint32_t)(row & 7) << 4;
        // They leave together, wherever a wait runs out: one alone would leave the others at their barrier for good.
        // what the loops ask for each time round, out of the constant bank
        int E = p.E;
        asm volatile("" : "+r"(E));
        bool ok = true;
#pragma unroll 1
        for (;;) {
            const int s = take();
            if (named_bar_or(BAR, 128, s < 0)) break;
#pragma unroll 1
            for (int t = 0; t < 2; ++t) {
                if (it.token + t * p.T >= it.n) continue;
                const uint32_t o_tmem = tmem_base + (uint32_t(quad * 32) << 16) + Cfg::O_COL + t * EP;
                const bool live = live_row(t, l0);
                const int row0 = it.q0 + it.token + t * p.T, head0 = it.h * p.share + it.g0;
                // Whole tiles of fp16 go out through shared memory and a tensor map, others a row a lane.  A store for every 16 bytes of all tiles cost the
                // SM 6000 clocks an item in instructions and waits for them, two blocks of keys; a bulk copy for every row more.
                const bool whole = p.out_whole && it.token + (t + 1) * p.T <= it.n;
                const int64_t at = (int64_t)(row0 + l0) * p.oN + (int64_t)(head0 + g) * p.oH;
                const int turn = t ? parts1++ : parts0++, blocks = t ? (busy1 += it.nblk) : (busy0 += it.nblk);
                ok = wait(&o_full[t], (uint32_t)(turn & 1), KST_WAIT_SOFTMAX);
                if (ok && it.nblk > 0) ok = wait(&pv_done[t], (uint32_t)((blocks - 1) & 1), KST_WAIT_SOFTMAX);
                if (named_bar_or(BAR, 128, !ok)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const int nblk = it.nblk, slot = it.slot;
                const float2 stat = stats[t * PK_ROWS + row];
                const float f = it.slot >= 0 || stat.y == 0.f ? 1.f : 1.f / stat.y;
                const int bad = *reinterpret_cast<volatile int*>(&odd[s]);      // written before the last P V was issued
                if (!TWO && whole && slot < 0 && nblk > 0 && bad == 0x7fffffff) {        // the ordinary case, without a branch to wait for
                    if (threadIdx.x == 12 * 32) tma_store_wait_read<0>();                    // what went out before has been read
                    named_bar_sync(BAR, 128);
#pragma unroll
                    for (int e = 0; e < EP; e += 16) {
                        uint32_t o[16], w[8];
                        tmem_ld16(o_tmem + e, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int u = 0; u < 8; ++u) {
                            float a, b;
                            unpack2(mul2(pack2(__uint_as_float(o[2 * u]), __uint_as_float(o[2 * u + 1])), pack2(f, f)), a, b);
                            const __half2 h = __floats2half2_rn(a, b);
                            w[u] = *reinterpret_cast<const uint32_t*>(&h);
                        }
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            st_shared_v4(out + (e >> 6) * PK_ATOM + row * 128 + ((uint32_t)((e & 48) * 2 | c << 4) ^ swz), w + 4 * c);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&o_empty[t]);
                    fence_proxy_async_smem();
                    named_bar_sync(BAR, 128);
                    if (threadIdx.x == 12 * 32) {
                        tma_store_3d(&tmapO, smem + Cfg::S_OUT, 0, head0, row0);
                        if (E > 64) tma_store_3d(&tmapO, smem + Cfg::S_OUT + PK_ATOM, 64, head0, row0);
                        tma_store_commit();
                    }
                    continue;
                }
#pragma unroll 1
                for (int e = 0; e < E; e += 32) {
                    uint32_t o[32];
                    __syncwarp();
                    if (nblk > 0) {
                        tmem_ld32(o_tmem + e, o);
                        tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int u = 0; u < 32; ++u) o[u] = 0;
                    }
#pragma unroll
                    for (int u = 0; u < 32; u += 2) {
                        float a, b;
                        unpack2(mul2(pack2(__uint_as_float(o[u]), __uint_as_float(o[u + 1])), pack2(f, f)), a, b);
                        o[u] = __float_as_uint(a), o[u + 1] = __float_as_uint(b);
                    }
                    if (bad != 0x7fffffff) {        // what was taken out, for those who see it
                        const int end = live ? min((it.j0 + it.nblk) * PK_KEYS - 1, last_key(t, l0)) : -1;
#pragma unroll 1
                        for (int key = max(bad * PK_KEYS, as_it_is() + 1); key <= end; ++key) {
                            const __half* q = p.v + (int64_t)(it.k0 + key) * p.vN + it.h * p.vH + e;
#pragma unroll
                            for (int u = 0; u < 32; ++u) {
                                if (e + u >= E) break;
                                const float y = __half2float(q[u]);
                                if (!(fabsf(y) < INFINITY)) o[u] = __float_as_uint(__uint_as_float(o[u]) + y);
                            }
                        }
                    }
                    if (e + 32 >= E) {          // all of O is in registers or on its way
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&o_empty[t]);
                    }
                    if (slot >= 0) {
                        float4* d = reinterpret_cast<float4*>(p.part + (int64_t)slot * (2 * PK_ROWS * EP)) + e * (PK_ROWS / 2) + t * PK_ROWS + row;
                        if (live)
#pragma unroll
                            for (int u = 0; u < 8; ++u)
                                if (e + 4 * u < E) d[u * 2 * PK_ROWS] = make_float4(__uint_as_float(o[4 * u]), __uint_as_float(o[4 * u + 1]), __uint_as_float(o[4 * u + 2]), __uint_as_float(o[4 * u + 3]));
                        continue;
                    }
                    // a row a lane
                    if (!live) continue;
                    char* to = (char*)p.out + (at + e) * (TWO ? 4 : 2);
                    const bool vectors = p.out_whole && e + 32 <= E;
                    if (TWO) {
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            if (vectors || (p.out_whole && e + 4 * c + 4 <= E)) reinterpret_cast<uint4*>(to)[c] = make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
                            else
#pragma unroll
                                for (int u = 0; u < 4; ++u)
                                    if (e + 4 * c + u < E) reinterpret_cast<uint32_t*>(to)[4 * c + u] = o[4 * c + u];
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t w[4];
#pragma unroll
                            for (int u = 0; u < 4; ++u) {
                                const __half2 h = __floats2half2_rn(__uint_as_float(o[8 * c + 2 * u]), __uint_as_float(o[8 * c + 2 * u + 1]));
                                w[u] = *reinterpret_cast<const uint32_t*>(&h);
                            }
                            if (vectors || (p.out_whole && e + 8 * c + 8 <= E)) reinterpret_cast<uint4*>(to)[c] = make_uint4(w[0], w[1], w[2], w[3]);
                            else
#pragma unroll
                                for (int u = 0; u < 8; ++u)
                                    if (e + 8 * c + u < E) reinterpret_cast<uint16_t*>(to)[8 * c + u] = (uint16_t)(w[u / 2] >> (u % 2 * 16));
                        }
                    }
                }
                if (live && it.slot >= 0) *reinterpret_cast<float2*>(p.part_ml + ((int64_t)it.slot * 2 * PK_ROWS + t * PK_ROWS + row) * 2) = stat;
            }
            if (!ok) break;
            done_with(s);
        }
        if (threadIdx.x == 12 * 32) tma_store_wait_all<0>();
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PK_OTHER_REGS));
        if (warp == 8) {
            // -------------------------------------------------- the work, and its operands
            int unit = blockIdx.x, i = 0, tiles0 = 0, tiles1 = 0;       // sides asked for so far; parts of a tile
            bool ok = true;
            PackedUnit u = {};
            u.next = -1;
            bool some = p.planned ? pk_listed(p, unit, u) : pk_direct(p, unit, u);
#pragma unroll 1
            for (int n = 0; ok; ++n) {
                if (some) pk_part(p, it, u);
                it.more = some;
                const int s = n % PK_PARTS;
                if (!wait(&a_empty[s], (uint32_t)((n / PK_PARTS) & 1) ^ 1, KST_WAIT_EMPTY)) break;
                if (lane == 0) {
                    part[s] = it;
                    odd[s] = 0x7fffffff;
                    mbar_arrive(&a_full[s]);
                }
                __syncwarp();
                if (!some) break;
                some = false;
                if (p.planned && u.next == PK_DEALT && lane == 0) unit = gridDim.x + atomicAdd(&p.counts->w, 1);      // on its way under this part's first loads
                const int sides = 2 * it.nblk;
                auto load_q = [&](int t, int& tiles) {
                    if (it.token + t * p.T >= it.n || sides == 0) return;
                    ok = ok && wait(&q_empty[t], (uint32_t)(tiles & 1) ^ 1, KST_WAIT_EMPTY);
                    ++tiles;
                    if (ok && elect_one()) {
                        mbar_arrive_expect_tx(&q_full[t], Cfg::SIDE);
#pragma unroll
                        for (int a = 0; a < ATOMS; ++a)
                            tma_load_3d(smem + Cfg::S_Q + t * Cfg::SIDE + a * PK_ATOM, &tmapQ, &q_full[t], a * 64, it.h * p.share + it.g0,
                                        it.q0 + it.token + t * p.T);
                    }
                    __syncwarp();
                };
                load_q(0, tiles0);
#pragma unroll 1
                for (int j = 0; ok && (j < sides || j == 0); ++j) {
                    // What comes next is looked up once this part's first sides are asked for.
                    if (p.planned && j == (sides > STAGES ? STAGES : sides >> 1)) {
                        unit = __shfl_sync(0xffffffffu, unit, 0);
                        some = pk_listed(p, unit, u);
                    }
                    if (j >= sides) break;
                    if (j == 1) load_q(1, tiles1);          // tile 1 is the later one to be done with its last part
                    const int st = i % STAGES;
                    ok = wait(&empty[st], (uint32_t)((i / STAGES) & 1) ^ 1, KST_WAIT_EMPTY);
                    if (ok && elect_one()) {
                        mbar_arrive_expect_tx(&full[st], Cfg::SIDE);
#pragma unroll
                        for (int a = 0; a < ATOMS; ++a)
                            tma_load_3d(smem + Cfg::S_KV + st * Cfg::SIDE + a * PK_ATOM, j & 1 ? &tmapV : &tmapK, &full[st], a * 64, it.h,
                                        it.k0 + (it.j0 + (j >> 1)) * PK_KEYS);
                    }
                    __syncwarp();
                    ++i;
                }
            }
        } else if (warp == 11) {
            // -------------------------------------------------- values that may be multiplied
            int i = 0;
            bool ok = true;
#pragma unroll 1
            for (int s; ok && (s = take()) >= 0; done_with(s)) {
                const int see = as_it_is();
                int first = 0x7fffffff;
#pragma unroll 1
                for (int j = 0; ok && j < it.nblk; ++j, i += 2) {
                    const int st = (i + 1) % STAGES, key0 = (it.j0 + j) * PK_KEYS;
                    // Not K's, which is filled again without this warp's say; V's stage only once this block has been handed on
                    ok = wait(&full[st], (uint32_t)(((i + 1) / STAGES) & 1), KST_WAIT_FULL);
                    if (!ok) break;
                    if (key0 + PK_KEYS - 1 > see) {       // some row's weight may be 0, of which what is not finite makes a NaN
                        // Keys from here on.  A number times 0 is 0, anything else a NaN that stays one in a sum.
                        const int from = see < key0 ? 0 : see + 1 - key0;
                        uint8_t* tile = smem + Cfg::S_KV + st * Cfg::SIDE;
                        const __half2 zero = __half2half2(__ushort_as_half(0));
                        __half2 sum[4] = {zero, zero, zero, zero};
#pragma unroll 1
                        for (int a = 0; a < ATOMS; ++a) {
                            const uint4* row = reinterpret_cast<const uint4*>(tile + a * PK_ATOM);
#pragma unroll 4
                            for (int c = from * 8 + lane; c < 128 * 8; c += 32) {
                                const uint4 x = row[c];
                                sum[0] = __hfma2(*reinterpret_cast<const __half2*>(&x.x), zero, sum[0]);
                                sum[1] = __hfma2(*reinterpret_cast<const __half2*>(&x.y), zero, sum[1]);
                                sum[2] = __hfma2(*reinterpret_cast<const __half2*>(&x.z), zero, sum[2]);
                                sum[3] = __hfma2(*reinterpret_cast<const __half2*>(&x.w), zero, sum[3]);
                            }
                        }
                        const __half2 any = __hadd2(__hadd2(sum[0], sum[1]), __hadd2(sum[2], sum[3]));
                        if (__any_sync(0xffffffffu, __hisnan(__low2half(any)) || __hisnan(__high2half(any)))) {
                            bool mine = false;
#pragma unroll 1
                            for (int i2 = from * 32 + lane; i2 < 128 * 32; i2 += 32)       // by words of two
#pragma unroll
                                for (int a = 0; a < ATOMS; ++a) {
                                    uint32_t* w = reinterpret_cast<uint32_t*>(tile + a * PK_ATOM) + i2;
                                    const uint32_t bad = ((*w & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;
                                    if (bad) {
                                        *w &= ~((bad >> 15) * 0xffffu);
                                        mine |= key0 + i2 / 32 < it.m;      // a key of this sequence
                                    }
                                }
                            if (__any_sync(0xffffffffu, mine) && key0 < first) {
                                first = key0;
                                if (lane == 0) odd[s] = it.j0 + j;
                            }
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    if (lane == 0) mbar_arrive(&ready[(i >> 1) % STAGES]);
                }
            }
        } else {
            // -------------------------------------------------- issuers: the whole warp waits, one thread issues
            const int t = warp - 9;
            constexpr uint32_t idesc_s = make_idesc_f16(PK_ROWS, PK_KEYS, 0, 0);
            const int steps = (p.E + 15) / 16;                       // past the head dim both operands are zeros
            const uint32_t idesc_o = make_idesc_f16(PK_ROWS, 16 * steps, 0, 1);
            constexpr uint64_t kdesc0 = make_smem_desc(16, 1024);
            constexpr uint64_t vdesc0 = make_smem_desc(PK_ATOM, 1024);
            const uint32_t q_addr = smem_u32(smem + Cfg::S_Q + t * Cfg::SIDE), kv_addr = smem_u32(smem + Cfg::S_KV);
            const uint32_t s_tmem = tmem_base + t * PK_KEYS, o_tmem = tmem_base + Cfg::O_COL + t * EP;
            const uint32_t p_tmem = OWN_P ? tmem_base + Cfg::P_COL + t * 64 : s_tmem;
            int i = 0, busy = 0, parts = 0, lives = 0;      // sides of the ring before this part; blocks of this tile; parts of it with keys; all of its parts
            auto issue_qk = [&](int j) -> bool {
                const int st = (i + 2 * j) % STAGES;
                if (!wait(&full[st], (uint32_t)(((i + 2 * j) / STAGES) & 1), KST_WAIT_FULL)) return false;
                if (OWN_P && busy + j > 0 && !wait(&s_empty[t], (uint32_t)((busy + j - 1) & 1), KST_WAIT_SOFTMAX)) return false;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t k_addr = kv_addr + st * Cfg::SIDE;
#pragma unroll
                    for (int k = 0; k < EP / 16; ++k) {
                        if (k >= steps) break;
                        const uint32_t in = (uint32_t)(k >> 2) * PK_ATOM + (uint32_t)(k & 3) * 32;
                        umma_ss(s_tmem, smem_desc_at(kdesc0, q_addr + in), smem_desc_at(kdesc0, k_addr + in), idesc_s, k != 0);
                    }
                    umma_commit(&s_full[t]);
                    umma_commit(&empty[st]);
                    if (j == it.nblk - 1) umma_commit(&q_empty[t]);
                }
                __syncwarp();
                return true;
            };
            auto issue_pv = [&](int j, int st, int k0, int k1) {
                const uint32_t v_addr = kv_addr + st * Cfg::SIDE;
#pragma unroll
                for (int k = k0; k < k1; ++k) {
                    umma_ts(o_tmem, p_tmem + k * 8, smem_desc_at(vdesc0, v_addr + k * 2048), idesc_o, (j | k) != 0);
                    if (TWO) umma_ts(o_tmem, p_tmem + 64 + k * 8, smem_desc_at(vdesc0, v_addr + k * 2048), idesc_o, true);
                }
            };
            bool ok = true;
#pragma unroll 1
            for (int s; ok && (s = take()) >= 0; done_with(s)) {
                if (it.token + t * p.T >= it.n) {      // no rows: what the other tile reads is released from here too
#pragma unroll 1
                    for (int j = 0; ok && j < 2 * it.nblk; ++j) {
                        const int st = (i + j) % STAGES;
                        const int vb = (i + j) >> 1;
                        ok = j & 1 ? wait(&ready[vb % STAGES], (uint32_t)((vb / STAGES) & 1), KST_WAIT_FULL)
                                   : wait(&full[st], (uint32_t)(((i + j) / STAGES) & 1), KST_WAIT_FULL);
                        if (ok && elect_one()) mbar_arrive(&empty[st]);
                        __syncwarp();
                    }
                    i += 2 * it.nblk;
                    continue;
                }
                ++lives;
                if (it.nblk == 0) continue;
                ok = wait(&q_full[t], (uint32_t)(parts & 1), KST_WAIT_FULL) && issue_qk(0);
#pragma unroll 1
                for (int j = 0; ok && j < it.nblk; ++j) {
                    if (OWN_P && j + 1 < it.nblk && !issue_qk(j + 1)) { ok = false; break; }
                    const int st = (i + 2 * j + 1) % STAGES, vb = (i >> 1) + j;
                    const uint32_t ph = (uint32_t)((busy + j) & 1);
                    if (j == 0 && !wait(&o_empty[t], (uint32_t)(lives & 1), KST_WAIT_TMEM_EMPTY)) { ok = false; break; }   // of the part before
                    ok = wait(&ready[vb % STAGES], (uint32_t)((vb / STAGES) & 1), KST_WAIT_FULL);
                    if (ok && HALVES) {
                        ok = wait(&p_half[t], ph, KST_WAIT_SOFTMAX);
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one()) issue_pv(j, st, 0, 2 * Cfg::FIRST);
                        __syncwarp();
                    }
                    ok = ok && wait(&p_full[t], ph, KST_WAIT_SOFTMAX);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        issue_pv(j, st, HALVES ? 2 * Cfg::FIRST : 0, 8);
                        umma_commit(&pv_done[t]);
                        umma_commit(&empty[st]);
                    }
                    __syncwarp();
                    if (!OWN_P && j + 1 < it.nblk) ok = issue_qk(j + 1);   // over P(j): after the product that reads it, in issue order
                }
                i += 2 * it.nblk, busy += it.nblk, ++parts;
            }
        }
    } else {
        // ------------------------------------------------------ softmax and results
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PK_SOFTMAX_REGS));
        const int t = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
        const uint32_t lane_base = uint32_t(quad * 32) << 16;
        const uint32_t s_tmem = tmem_base + lane_base + t * PK_KEYS, o_tmem = tmem_base + lane_base + Cfg::O_COL + t * EP;
        const uint32_t p_tmem = OWN_P ? tmem_base + lane_base + Cfg::P_COL + t * 64 : s_tmem;
        const int l0 = row >> p.log_g;        // the row's token in its tile
        int busy = 0, turns = 0, lives = 0;          // blocks of this tile, turns of both, parts of this tile before this one
        bool ok = true;
#pragma unroll 1
        for (int s; ok && (s = take()) >= 0; done_with(s)) {
            if (it.token + t * p.T >= it.n) continue;
            const int last = last_key(t, l0);
            const int see = all_see(it.token + t * p.T);
            float m_run = -INFINITY, l_run = 0.f;
            const bool pingpong = it.token + p.T < it.n;
            const uint64_t k2 = pack2(p.scale_log2, p.scale_log2);
#pragma unroll 1
            for (int j = 0; ok && j < it.nblk; ++j, ++busy) {
                const int key0 = (it.j0 + j) * PK_KEYS;
                ok = wait(&s_full[t], (uint32_t)(busy & 1), KST_WAIT_TMEM_FULL);
                if (!ok) break;
                tc_fence_after();
                uint32_t x[4][32];
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld32(s_tmem + i * 32, x[i]);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int u = 0; u < 32; ++u) asm volatile("" : "+r"(x[i][u]));   // in registers from here on
                if (OWN_P) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_empty[t]);
                }
                if (key0 + PK_KEYS - 1 > see) {
                    const int seen = last - key0;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (key0 + i * 32 + 31 > see) {
#pragma unroll
                            for (int u = 0; u < 32; ++u)
                                if (i * 32 + u > seen) x[i][u] = 0xff800000u;
                        }
                }
                auto highest = [&]() -> float {
                    float a = -INFINITY, b = -INFINITY, c = -INFINITY, d = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int u = 0; u < 32; u += 8) {
                            a = pk_max3(a, __uint_as_float(x[i][u]), __uint_as_float(x[i][u + 1]));
                            b = pk_max3(b, __uint_as_float(x[i][u + 2]), __uint_as_float(x[i][u + 3]));
                            c = pk_max3(c, __uint_as_float(x[i][u + 4]), __uint_as_float(x[i][u + 5]));
                            d = pk_max3(d, __uint_as_float(x[i][u + 6]), __uint_as_float(x[i][u + 7]));
                        }
                    return fmaxf(fmaxf(a, b), fmaxf(c, d)) * p.scale_log2;
                };
                // Any reference point m gives the same quotient; it follows the maximum lazily, only when that has grown by more than 2^8.
                // P goes in times 2^7, so that fp16 holds weights down to 2^-31 of the heaviest key's.  Where the result is rounded to fp16 anyhow, each
                // weight is rounded once to fp16, half a step 2^-11 of itself, as the product's operand; where the caller asks for fp32 it goes in as
                // two fp16 numbers, off by 2^-22, in twice the products (error against 64 bits 1.7e-4 -> 9e-6 and 2090 us -> 3130 for 16384 rows, 1.6e-4 ->
                // 1e-6 and 775 -> 925 for 37 sequences of up to 2000, 2e-4 -> 3e-6 and 173 -> 240 for 16 of up to 1500).  The sum that divides takes
                // the weights as they were, in fp32.
                const float top = highest();
                const float m_new = top > m_run + 8.f ? top : m_run;
                if (OWN_P && busy > 0) ok = wait(&pv_done[t], (uint32_t)((busy - 1) & 1), KST_WAIT_SOFTMAX);     // P and O are free
                if (!ok) break;
                if (__any_sync(0xffffffffu, m_new != m_run)) {
                    const float alpha = m_run == m_new ? 1.f : pk_ex2(m_run - m_new);
                    l_run *= alpha;
                    if (j > 0) {          // the last P V is done: these scores were issued after it, or it has been waited for
                        tc_fence_after();
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
                // In a part's first block the tiles take turns at the exponentials, so that one's run under the other's products; from there on they
                // fall into step by themselves (turns at every block: 599 us for 594 of 37 sequences of up to 2000, 2059 for 1994 of 16384 rows).
                if (pingpong && j == 0 && (t == 1 || turns > 0) &&
                    !wait(&exp_turn[t], (uint32_t)((t == 1 ? turns : turns - 1) & 1), KST_WAIT_SOFTMAX)) { ok = false; break; }
                const float m_sub = m_new == -INFINITY ? 0.f : 7.f - m_new;
                const uint64_t a2 = pack2(m_sub, m_sub);
                uint64_t sum0 = pack2(0.f, 0.f), sum1 = pack2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t pk[16];
#pragma unroll
                    for (int u = 0; u < 16; ++u) {
                        float e0, e1;
                        unpack2(fma2(pack2(__uint_as_float(x[i][2 * u]), __uint_as_float(x[i][2 * u + 1])), k2, a2), e0, e1);
                        // All by the exponential unit: a polynomial for every fourth pair takes 2 to 4 % fewer clocks and, under the power limit,
                        // 594 us for 585 (E = 128) and 166 for 162 (E = 64).
                        e0 = pk_ex2(e0), e1 = pk_ex2(e1);
                        if (u & 1) sum1 = add2(sum1, pack2(e0, e1));
                        else sum0 = add2(sum0, pack2(e0, e1));
                        const __half2 h = __floats2half2_rn(e0, e1);
                        pk[u] = *reinterpret_cast<const uint32_t*>(&h);
                        if (TWO) x[i][2 * u] = __float_as_uint(e0), x[i][2 * u + 1] = __float_as_uint(e1);
                    }
                    pk_tmem_st16(p_tmem + i * 16, pk);
                    if (TWO) {
#pragma unroll
                        for (int u = 0; u < 16; ++u) {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pk[u]));
                            const __half2 h = __floats2half2_rn(__uint_as_float(x[i][2 * u]) - f.x, __uint_as_float(x[i][2 * u + 1]) - f.y);
                            pk[u] = *reinterpret_cast<const uint32_t*>(&h);
                        }
                        pk_tmem_st16(p_tmem + 64 + i * 16, pk);
                    }
                    if (HALVES && i == Cfg::FIRST - 1) {
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_half[t]);
                    }
                }
                if (pingpong && j == 0) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&exp_turn[1 - t]);
                    ++turns;
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
                float s0, s1;
                unpack2(add2(sum0, sum1), s0, s1);
                l_run += s0 + s1;
            }
            if (ok) ok = wait(&o_empty[t], (uint32_t)(lives & 1) ^ 1, KST_WAIT_TMEM_EMPTY);      // the part before's have been read
            if (!ok) break;
            stats[t * PK_ROWS + row] = make_float2(m_run, l_run);
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_full[t]);
            ++lives;
        }
    }
    if (*why) {
        for (int i = 0; i < 4; ++i) __nanosleep(1000000);
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *why) atomicCAS(p.d_status, 0, *why);
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// The parts of what was cut, sixteen elements of a row a thread, in the order of the keys.
template <int EP>
__global__ void __launch_bounds__(256)
packed_join_kernel(const PackedParams p) {
    grid_dep_wait();
    grid_dep_launch();
    const int i = blockIdx.x / (EP / 16), e = (int)(blockIdx.x % (EP / 16)) * 16, prow = threadIdx.x;
    const int4 counts = *p.counts;
    const PackedCut x = p.cut[i];                 // there is room for as many as there are blocks of this launch
    if (i >= counts.z || e >= p.E) return;
    const int h = x.head / p.groups, g0 = (x.head - h * p.groups) * p.G;
    const int t = prow / PK_ROWS, row = prow - t * PK_ROWS, l0 = row >> p.log_g, g = row & (p.G - 1), l = x.token + t * p.T + l0;
    if (l >= x.n) return;
    auto slot = [&](int w) -> int64_t { return w == 0 ? x.slot : 2 * (x.slot / 2 + w); };
    auto stat = [&](int w) { return *reinterpret_cast<const float2*>(p.part_ml + (slot(w) * 2 * PK_ROWS + prow) * 2); };
    float M = -INFINITY, sum = 0.f, v[2][8] = {};
    for (int w = 0; w < x.parts; ++w) M = fmaxf(M, stat(w).x);
    for (int w = 0; w < x.parts; ++w) {
        const float2 ml = stat(w);
        const float f = ml.x == M ? 1.f : exp2f(ml.x - M);
        const float4* y = reinterpret_cast<const float4*>(p.part + slot(w) * (2 * PK_ROWS * EP)) + e / 4 * (2 * PK_ROWS) + prow;
        sum = fmaf(ml.y, f, sum);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float4 a = y[u * 2 * PK_ROWS];
            float* d = &v[u >> 1][(u & 1) * 4];
            d[0] = fmaf(a.x, f, d[0]), d[1] = fmaf(a.y, f, d[1]), d[2] = fmaf(a.z, f, d[2]), d[3] = fmaf(a.w, f, d[3]);
        }
    }
    const float inv = sum == 0.f ? 1.f : 1.f / sum;
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k >> 3][k & 7] *= inv;
    const int64_t to = (int64_t)(x.q0 + l) * p.oN + (int64_t)(h * p.share + g0 + g) * p.oH + e;
    pk_store8(p, to, p.E - e, v[0]);
    pk_store8(p, to + 8, p.E - e - 8, v[1]);
}

// An operand whose rows a tensor map cannot express, brought to rows of E8 elements: eight elements a thread.
__global__ void __launch_bounds__(256)
packed_rows_kernel(const __half* x, int64_t xN, int64_t xH, __half* to, int E, int E8, int H, int64_t total) {
    grid_dep_wait();
    grid_dep_launch();
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int per = E8 / 8, c = (int)(i % per);
    const int64_t row = i / per, n = row / H;
    const __half* q = x + n * xN + (row - n * H) * xH + c * 8;
    __align__(16) __half v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c * 8 + k < E ? q[k] : __half(0.f);
    *reinterpret_cast<uint4*>(to + row * E8 + c * 8) = *reinterpret_cast<const uint4*>(v);
}

// Heads of a tile: the largest power of two that divides those of a key head, so that every row of a tile is some token's and head's, and every tile of a
// key head has as many.  Of 3, 5 or 7 heads each is then a unit of its own and reads the keys again.
constexpr int pk_heads(int share) {
    int g = 1;
    while (g < PK_ROWS && share % (2 * g) == 0) g *= 2;
    return g;
}
static_assert(pk_heads(1) == 1 && pk_heads(5) == 1 && pk_heads(6) == 2 && pk_heads(12) == 4 && pk_heads(130) == 2 && pk_heads(384) == 128 && pk_heads(512) == 128,
              "what stands above");

struct PackedOperand {
    const __half* ptr;
    int64_t sN, sH;
};

template <int EP, bool TWO>
static int pk_launch(b200_ctx* ctx, PackedParams& p, const PackedOperand& q, const PackedOperand& k, const PackedOperand& v, int64_t items, int64_t entries) {
    using Cfg = PkCfg<EP, TWO>;
    auto kern = attention_packed_kernel<EP, TWO>;
    static std::atomic<uint64_t> asked{0};
    B200_CUDA(allow_smem(ctx, kern, Cfg::SMEM, asked));
    CUtensorMap tq, tk, tv, to;
    auto map = [&](CUtensorMap* m, const PackedOperand& a, int64_t heads, int64_t rows, uint32_t box_h, uint32_t box_n) {
        const uint64_t dims[3] = {(uint64_t)p.E, (uint64_t)heads, (uint64_t)rows};
        const uint64_t strides[2] = {(uint64_t)a.sH * 2, (uint64_t)a.sN * 2};
        const uint32_t box[3] = {64, box_h, box_n};
        return make_tmap(ctx, m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, a.ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    const int64_t Nk = p.Nk > 0 ? p.Nk : 1;           // without keys the maps are over q, and not read through
    int rc = map(&tq, q, p.Hq, p.N, p.G, p.T);
    if (!rc) rc = map(&tk, k, p.H, Nk, 1, PK_KEYS);
    if (!rc) rc = map(&tv, v, p.H, Nk, 1, PK_KEYS);
    to = tq;
    if (!rc && p.out_whole && !p.out_f32) {
        const uint64_t dims[3] = {(uint64_t)p.E, (uint64_t)p.Hq, (uint64_t)p.N}, strides[2] = {(uint64_t)p.oH * 2, (uint64_t)p.oN * 2};
        const uint32_t box[3] = {64, (uint32_t)p.G, (uint32_t)p.T};
        rc = make_tmap(ctx, &to, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, p.out, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    }
    if (rc) return rc;
    const int64_t sms = ctx->prop.multiProcessorCount;
    p.sms = (int)sms, p.most = (int)entries;
    // The list and the second launch cost 2 to 6 us (20 heads of 64 over 77 keys 7.4 us without, 13.0 with), cut keys save more where there are many
    // (16 heads of 128 on 8, 100 rows over 1800 keys 24.2 without, 26.2 with; over 3100 35.9 and 29.8).
    p.planned = items > sms || p.Nk > 16 * PK_KEYS;
    const int64_t slots = 2 * sms, rows = slots * 2 * PK_ROWS;
    if (p.planned) {
        void* ws = nullptr;
        // 36 bytes an entry, of which there are one and a half a row at most (a token a tile, a row a sequence)
        const int64_t firsts = p.B > PL_SEQS ? p.B : 0;
        const size_t list = (size_t)entries * (sizeof(PackedEntry) + sizeof(int)) + firsts * sizeof(int) + sms * sizeof(PackedCut) + 2 * sizeof(int4) + 16 * 8;
        rc = ws_scratch(ctx, rows * (EP + 2) * sizeof(float) + list, &ws);
        if (rc) return rc;
        uint8_t* at = static_cast<uint8_t*>(ws);
        auto room = [&](size_t bytes) {
            uint8_t* r = at;
            at += (bytes + 15) / 16 * 16;
            return (void*)r;
        };
        p.part = (float*)room(rows * EP * sizeof(float));
        p.part_ml = (float*)room(rows * 2 * sizeof(float));
        p.entry = (PackedEntry*)room(entries * sizeof(PackedEntry));
        p.cut = (PackedCut*)room(sms * sizeof(PackedCut));
        p.counts = (int4*)room(2 * sizeof(int4));
        p.before = (int*)room(entries * sizeof(int));
        p.first = (int*)room(firsts * sizeof(int));
        B200_CUDA(launch_dep(packed_plan_kernel, dim3(1), dim3(PL_THREADS), 0, ctx->stream, 1, p));
        ctx->launches++;
    }
    const int64_t grid = p.planned ? sms : items;
    B200_CUDA(launch_dep(kern, dim3((unsigned)grid), dim3(PK_THREADS), Cfg::SMEM, ctx->stream, 1, tq, tk, tv, to, p));
    ctx->launches++;
    if (p.planned) {
        B200_CUDA(launch_dep(packed_join_kernel<EP>, dim3((unsigned)(sms * (EP / 16))), dim3(256), 0, ctx->stream, 1, p));
        ctx->launches++;
    }
    return B200_OK;
}

} // namespace b200

using namespace b200;

extern "C" {

int b200_attention_packed_f16(b200_ctx* ctx, int64_t E, int64_t N, int64_t Nk, int64_t Hq, int64_t H, int64_t B, const b200_strided4* q,
                              const b200_strided4* k, const b200_strided4* v, const b200_strided4* out, int out_dtype, float scale,
                              int causal, const int32_t* starts, const int32_t* kstarts) {
    B200_REQUIRE(ctx && q && k && v && out, B200_EINVAL, "attention_packed: null argument");
    B200_REQUIRE(E >= 0 && N >= 0 && Nk >= 0 && Hq >= 0 && H >= 0 && B >= 0, B200_EINVAL, "attention_packed: E=%lld N=%lld Nk=%lld Hq=%lld H=%lld B=%lld",
                 (long long)E, (long long)N, (long long)Nk, (long long)Hq, (long long)H, (long long)B);
    B200_REQUIRE(out_dtype == B200_F16 || out_dtype == B200_F32, B200_DECLINE_ELTYPE, "attention_packed: result type %d", out_dtype);
    B200_REQUIRE(scale >= 0.f && scale < INFINITY, B200_EINVAL, "attention_packed: scale %g", scale);
    B200_REQUIRE(H > 0 ? Hq % H == 0 : Hq == 0, B200_DECLINE_EXTENT, "attention_packed: %lld heads over %lld", (long long)Hq, (long long)H);
    B200_REQUIRE(E <= 128, B200_DECLINE_TILING, "attention_packed: heads of %lld elements (at most 128)", (long long)E);
    B200_REQUIRE(N < (1ll << 30) && Nk < (1ll << 30) && Hq < 65536 && B < (1ll << 24), B200_DECLINE_EXTENT,
                 "attention_packed: N=%lld Nk=%lld Hq=%lld B=%lld", (long long)N, (long long)Nk, (long long)Hq, (long long)B);
    for (const b200_strided4* a : {q, k, v, out})
        B200_REQUIRE(E <= 1 || a->stride[0] == 1, B200_DECLINE_ALIGN, "attention_packed: E is not contiguous");
    if (E == 0 || N == 0 || Hq == 0 || B == 0) return B200_OK;
    B200_REQUIRE(q->ptr && out->ptr && starts && kstarts && (Nk == 0 || (k->ptr && v->ptr)), B200_EINVAL, "attention_packed: null array");
    B200_CUDA(cudaSetDevice(ctx->device));
    PackedParams p = {};
    p.starts = starts, p.kstarts = kstarts;
    p.N = (int)N, p.Nk = (int)Nk, p.B = (int)B, p.H = (int)H, p.Hq = (int)Hq, p.E = (int)E;
    p.causal = causal, p.out_f32 = out_dtype == B200_F32;
    p.out = const_cast<void*>(out->ptr);
    p.oN = out->stride[1], p.oH = out->stride[2];
    if (N == 1 && p.oN <= 0) p.oN = 8;         // strides that nothing is reached through
    if (Hq == 1 && p.oH <= 0) p.oH = 8;
    const int64_t size = p.out_f32 ? 4 : 2;
    p.out_whole = ((uintptr_t)p.out | (uint64_t)(p.oN * size) | (uint64_t)(p.oH * size)) % 16 == 0 && p.oN > 0 && p.oH > 0;
    p.scale_log2 = fmaxf((float)((double)scale * 1.4426950408889634), 0x1p-100f);   // above 0, so that a hidden score of -inf stays that
    p.d_status = ctx->d_status;
    p.share = (int)(Hq / H);
    p.G = pk_heads(p.share);
    for (p.log_g = 0; 1 << p.log_g < p.G;) ++p.log_g;
    p.T = PK_ROWS / p.G;
    p.groups = p.share / p.G;
    p.heads = (int)(p.H * p.groups);
    const int64_t entries = N / (2 * p.T) + (B < N ? B : N), items = entries * p.heads;    // at most
    B200_REQUIRE(items < (1ll << 30), B200_DECLINE_EXTENT, "attention_packed: %lld row tiles", (long long)items);
    PackedOperand op[3];
    const b200_strided4* in[3] = {q, k, v};
    int64_t E8 = (E + 7) / 8 * 8;
    for (int i = 0; i < 3; ++i) {
        const int64_t rows = i ? Nk : N, heads = i ? H : Hq;
        op[i] = {(const __half*)in[i]->ptr, in[i]->stride[1], in[i]->stride[2]};
        if (heads == 1) op[i].sH = E8;         // a stride that nothing is read through
        if (rows == 1) op[i].sN = E8;
        if (rows == 0) {                       // no keys at all: the maps are over something that is there
            op[i] = op[0];
            continue;
        }
        if (((uintptr_t)op[i].ptr % 16 | (uint64_t)op[i].sN % 8 | (uint64_t)op[i].sH % 8) == 0 && op[i].sN > 0 && op[i].sH > 0) continue;
        void* ws = nullptr;
        int rc = ws_scratch(ctx, (size_t)(rows * heads * E8) * sizeof(__half), &ws);
        if (rc) return rc;
        const int64_t total = rows * heads * (E8 / 8);
        B200_REQUIRE(cdiv(total, 256) < (1ll << 31), B200_DECLINE_EXTENT, "attention_packed: %lld rows to copy", (long long)rows);
        B200_CUDA(launch_dep(packed_rows_kernel, dim3((unsigned)cdiv(total, 256)), dim3(256), 0, ctx->stream, 1, op[i].ptr, op[i].sN, op[i].sH, (__half*)ws,
                             (int)E, (int)E8, (int)heads, total));
        ctx->launches++;
        op[i] = {(const __half*)ws, heads * E8, E8};
    }
    p.v = op[2].ptr, p.vN = op[2].sN, p.vH = op[2].sH;
    auto launch = [&](auto run) { return run(ctx, p, op[0], op[1], op[2], items, entries); };
    if (p.out_f32) return E <= 64 ? launch(pk_launch<64, true>) : launch(pk_launch<128, true>);
    return E <= 64 ? launch(pk_launch<64, false>) : launch(pk_launch<128, false>);
}

} // extern "C"
