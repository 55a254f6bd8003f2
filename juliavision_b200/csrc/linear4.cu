// Products with 4-bit weights and a scale for each group of `group` inputs of an output:
//     out[m, n] = epi(T(bias[m] + sum_k s[m, k / group] (q[m, k] - z[m, k / group]) x[k, n])),  q and z in 0 .. 15, z = 8 without zeros.
//
// For few tokens the weights are what is read, half a byte each, once; so they are laid out (b200_q4_pack) as the warp-level
// m16n8k16 tile wants them in registers.  A unit is 16 outputs x 64 inputs, 512 bytes, one 16-byte load a lane: word s of lane
// (g, t) holds inputs 32 (s / 2) + 8 t + 4 (s % 2) + (0 .. 3) of rows g and g + 8, which the sums' free order makes columns
// (2 t, 2 t + 1, 2 t + 8, 2 t + 9) of step s; x is read in the same order, eight contiguous inputs a lane and half.  Steps 0, 1
// and steps 2, 3 are 32 inputs each, so a group of 32 is two steps.  Nibbles (0,4) (1,5) (2,6) (3,7) are the four operand
// registers: a nibble under 0x64 is the fp16 number 1024 + q (or, in the upper half of its byte, 1024 + 16 q), and q - z comes
// out exactly of one subtraction (or one multiply-add by 1 / 16).  A group's sum is fp32, and so is its product by the scale.
// Four row tiles lie side by side, unit by unit, so that 64 rows are one stream of 2 KB a k block.
//
// Two kernels.  A small weight, whose rows do not fill the GPU for long, is a chain of round trips: a block takes 16
// rows, or 32 for up to 40 tokens at a time (each weight is made into fp16 once for all of them), its warps share K and have all
// their loads in flight at once (linear4_kernel).  A large one is bandwidth-bound: the list of
// (64 rows, 8 or 16 tokens, k block) is dealt out to all warps in equal contiguous shares, each streamed by bulk copies through a ring
// of its own; parts of rows meet at the ends of blocks and in a second launch (linear4_stream_kernel, shares.cuh).  Past 512 tokens
// the weight is laid out as fp16, exactly, for the GEMM (linear4_unpack_kernel).
#include <cuda_fp16.h>

#include <type_traits>

#include "act.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "shares.cuh"

namespace b200 {

constexpr int L4_WARPS = 8;      // of a block, which share K
// Tokens the two kernels take; more go through fp16 weights in the workspace, which are made once for all tokens and cost twice the
// products, since an exact weight is two fp16 numbers.  us, kernels / fp16 weights: 384, 512 and 768 tokens of 4096 x 4096 62 / 78, 79 / 78,
// 123 / 92; of 28672 x 8192 720 / 785, 951 / 818, 1415 / 968; of 5120 x 1280 34 / 62, 50 / 51, 70 / 52; 1024 and 2048 of 1280 x 1280 25 / 32, 49 / 54.
// (Weights rounded to one fp16 number: 512 tokens of 4096 x 4096 32 us, of 28672 x 8192 427; 2.8e-4 of the result off for 2.1e-4.)
constexpr int L4_TOKENS = 512;
// What fp16 weights and their fp32 sums take at a time: past it the next product's rows.
constexpr int64_t L4_DENSE_BYTES = 256ll << 20, L4_DENSE_TOKENS = 2048;
// Tiles of 64 rows, 16 tokens and 64 inputs from which on up to 16 tokens go by a list for all warps.  us, blocks / list, 16 tokens: 4096 x 2048
// (2048 tiles) 6.4 / 7.9, 4096 x 4096 (4096) 9.3 / 9.9, 5120 x 5120 (6400) 17 / 11; one token: 4096 x 4096 5.9 / 8.5, 5120 x 5120 11.3 / 9.7,
// 8192 x 4096 (8192) 10.4 / 10.2, 8192 x 8192 (16384) 19 / 14.
constexpr double L4_STREAM_TILES = 4608;
// More than 16 tokens: rounds of loads, times token tiles a block, up to which the blocks that have all of them at once are faster than
// the list.  us, blocks / list: 37 x 5120 x 1280 (15) 8.4 / 10.4, 24 x 4096 x 4096 (24) 11.1 / 12.2, 24 x 8192 x 4096 (24) 14.3 / 16.1,
// 64 x 5120 x 1280 (24) 12.5 / 11.8, 17 x 1280 x 5120 (30) 12.7 / 9.6, 17 x 5120 x 5120 (30) 16.7 / 14.4, 64 x 4096 x 4096 (32) 16.6 / 16.1,
// 37 x 4096 x 4096 (40) 13.8 / 14.1, 37 x 5120 x 5120 (50) 22 / 18, 200 x 4096 x 4096 (120) 45 / 37.
constexpr int64_t L4_ROUNDS = 24;

struct Linear4Params {
    const uint4* data;            // [four row tiles][k block][row tile][lane]
    const uint32_t* scales;       // [four row tiles][group][row tile][8]: fp16 scales of rows g and g + 8
    const uint8_t* zeros;         // the same: zero points of rows g (low) and g + 8 (high), or null
    const __half *x, *bias;
    void* out;
    int64_t ldx, ldo, M;
    int N, K, KB, NG, MT;         // k blocks of 64, groups a row, row tiles
    int logg;                     // log2 of the group size
    int out_f32, epi, whole;
    float* part;                  // [place][row tile, token tile][lane][4] (linear4_stream_kernel)
    int* d_status;

    __device__ __forceinline__ int64_t unit(int mt, int kb) const { return ((int64_t)(mt >> 2) * KB + kb) * 4 + (mt & 3); }
    __device__ __forceinline__ int64_t group8(int mt, int grp) const { return (((int64_t)(mt >> 2) * NG + grp) * 4 + (mt & 3)) * 8; }
};

// (v & M) | magic in one instruction: of two constants one has to be a register
template <uint32_t M> __device__ __forceinline__ uint32_t l4_and_or(uint32_t v, uint32_t magic) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "n"(M), "r"(magic));
    return r;
}
__device__ __forceinline__ uint32_t l4_sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t l4_fma16(uint32_t a, uint32_t b) {   // a / 16 + b
    const __half2 s = __half2half2(__ushort_as_half(0x2c00));
    const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), s, *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// The four operand registers of a word: q - z for rows g (z0 = 1024 + z, twice) and g + 8 (z1 = -(64 + z), twice).
__device__ __forceinline__ void l4_weights(uint32_t v, uint32_t z0, uint32_t z1, uint32_t (&a)[4]) {
    const uint32_t magic = 0x64006400u;
    a[0] = l4_sub(l4_and_or<0x000f000fu>(v, magic), z0);
    a[1] = l4_fma16(l4_and_or<0x00f000f0u>(v, magic), z1);
    v >>= 8;
    a[2] = l4_sub(l4_and_or<0x000f000fu>(v, magic), z0);
    a[3] = l4_fma16(l4_and_or<0x00f000f0u>(v, magic), z1);
}
__device__ __forceinline__ void l4_zero(uint32_t z, uint32_t& z0, uint32_t& z1) {   // two zero points of a byte
    z0 = (0x6400u | (z & 15u)) * 0x10001u;
    z1 = (0xd400u | (z & 0xf0u)) * 0x10001u;
}

// A lane's inputs of token n in k block kb: eight from 8 t on and eight from 32 + 8 t on, zeros past the ends.
__device__ __forceinline__ void l4_input(const Linear4Params& p, int n, int kb, int t, uint32_t (&w)[8]) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int k = kb * 64 + half * 32 + t * 8;
        uint4 a = make_uint4(0, 0, 0, 0);
        if (n < p.N && k < p.K) {   // K is a multiple of 32, so all eight are there or none is
            const __half* x = p.x + n * p.ldx + k;
            if (p.whole) {
                a = __ldg(reinterpret_cast<const uint4*>(x));
            } else {
                const unsigned short* u = reinterpret_cast<const unsigned short*>(x);
                a = make_uint4(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16, u[4] | (uint32_t)u[5] << 16, u[6] | (uint32_t)u[7] << 16);
            }
        }
        w[4 * half] = a.x, w[4 * half + 1] = a.y, w[4 * half + 2] = a.z, w[4 * half + 3] = a.w;
    }
}

// A k block of a row tile: acc += the products of its groups by their scales.
template <int NT, bool SMALL>
__device__ __forceinline__ void l4_block(float (&acc)[NT][4], const uint4& w, const uint32_t* sc, const uint32_t* zb, const uint32_t (&x)[NT][8]) {
    constexpr int GROUPS = SMALL ? 2 : 1, STEPS = 4 / GROUPS;   // groups a k block, steps a group
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
        uint32_t z0, z1;
        l4_zero(zb[j], z0, z1);
        const float2 s = __half22float2(*reinterpret_cast<const __half2*>(&sc[j]));
        float c[NT][4];
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            uint32_t a[4];
            l4_weights(v[j * STEPS + k], z0, z1, a);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t b0 = x[n][2 * (j * STEPS + k)], b1 = x[n][2 * (j * STEPS + k) + 1];
                if (k == 0) mma_16816_first(c[n], a[0], a[1], a[2], a[3], b0, b1);
                else mma_16816_free(c[n], a[0], a[1], a[2], a[3], b0, b1);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            acc[n][0] = fmaf(c[n][0], s.x, acc[n][0]);
            acc[n][1] = fmaf(c[n][1], s.x, acc[n][1]);
            acc[n][2] = fmaf(c[n][2], s.y, acc[n][2]);
            acc[n][3] = fmaf(c[n][3], s.y, acc[n][3]);
        }
    }
}
__device__ __forceinline__ void l4_store(const Linear4Params& p, int64_t m, int n, float v) {
    if (m >= p.M || n >= p.N) return;
    if (p.bias != nullptr) v += __half2float(p.bias[m]);
    // the activation sees the value rounded to the output type, as in the GEMM's store
    if (p.out_f32) ((float*)p.out)[n * p.ldo + m] = apply_act(p.epi, v);
    else ((__half*)p.out)[n * p.ldo + m] = __float2half_rn(apply_act(p.epi, __half2float(__float2half_rn(v))));
}

// ROWS row tiles and NT tiles of 8 tokens a block; the warps take every L4_WARPS-th k block, AT_ONCE of them at a time.  SMALL: groups of 32.
template <int ROWS, int NT, bool SMALL>
__global__ void __launch_bounds__(32 * L4_WARPS, ROWS == 1 ? 1 : 2)
linear4_kernel(const Linear4Params p) {
    constexpr int COLS = 8 * NT + 1, GROUPS = SMALL ? 2 : 1, AT_ONCE = ROWS > 1 ? 1 : NT == 1 ? 4 : 3;
    __shared__ float red[L4_WARPS][16][COLS];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int mt0 = blockIdx.x * ROWS, n0 = blockIdx.y * 8 * NT;
    grid_dep_wait();
    grid_dep_launch();
    float acc[ROWS][NT][4];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[r][n][0] = acc[r][n][1] = acc[r][n][2] = acc[r][n][3] = 0.f;
    for (int kb0 = warp; kb0 < p.KB; kb0 += L4_WARPS * AT_ONCE) {
        uint4 w[AT_ONCE][ROWS];
        uint32_t sc[AT_ONCE][ROWS][GROUPS], zb[AT_ONCE][ROWS][GROUPS], x[AT_ONCE][NT][8];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int kb = kb0 + u * L4_WARPS;
            const bool in = kb < p.KB;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                w[u][r] = in ? __ldg(p.data + p.unit(mt0 + r, kb) * 32 + lane) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < GROUPS; ++j) {
                    const int grp = (kb * 64 + j * 32) >> p.logg;
                    const bool live = in && grp < p.NG;    // the last k block may be half empty
                    sc[u][r][j] = live ? __ldg(p.scales + p.group8(mt0 + r, grp) + g) : 0;
                    zb[u][r][j] = live && p.zeros != nullptr ? __ldg(p.zeros + p.group8(mt0 + r, grp) + g) : 0x88u;
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) l4_input(p, n0 + n * 8 + g, in ? kb : p.KB, t, x[u][n]);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) l4_block<NT, SMALL>(acc[r], w[u][r], sc[u][r], zb[u][r], x[u]);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (r > 0) __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) red[warp][g + (k >> 1) * 8][n * 8 + 2 * t + (k & 1)] = acc[r][n][k];
        __syncthreads();
        for (int i = tid; i < 16 * 8 * NT; i += 32 * L4_WARPS) {
            const int row = i % 16, col = i / 16;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < L4_WARPS; ++w) v += red[w][row][col];
            l4_store(p, (int64_t)(mt0 + r) * 16 + row, n0 + col, v);
        }
    }
}

constexpr int L4_STAGES = 3;     // k blocks of 64 rows in flight, a warp
__device__ __forceinline__ void l4_bulk(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
                 "r"(smem_u32(bar)) : "memory");
}

template <int NT, bool SMALL> struct L4Cfg {
    static constexpr int GROUPS = SMALL ? 2 : 1;
    static constexpr int SCALES = 2048, ZEROS = SCALES + GROUPS * 128, END = ZEROS + GROUPS * 32;   // 64 rows' weights, scales, zero points
    static constexpr int STAGE = (END + 127) / 128 * 128, X_STAGE = NT * 1024;   // the tokens' inputs apart, where the swizzle wants them
    static constexpr int X_RING = L4_WARPS * L4_STAGES * X_STAGE, RING = L4_WARPS * L4_STAGES * STAGE;
    static constexpr int SMEM = X_RING + RING + 1024;
    static constexpr int FLOATS = 4 * NT * 128;      // a warp's results of 64 rows
    static_assert(L4_WARPS * FLOATS * 4 <= RING, "the warps' results fit over the ring");
    static constexpr int CTAS = 2;
};

// Results of row tile i, token tile n of piece q as lane ln of the warp has them.
template <int NT> __device__ __forceinline__ void l4_finish(const Linear4Params& p, int tgs, long long q, int i, int n, const float4& v, int ln) {
    const int rg = (int)q / tgs, tg = (int)q % tgs;
    const int64_t m = (int64_t)(rg * 4 + i) * 16 + (ln >> 2);
    const int c = (tg * NT + n) * 8 + 2 * (ln & 3);
    l4_store(p, m, c, v.x);
    l4_store(p, m, c + 1, v.y);
    l4_store(p, m + 8, c, v.z);
    l4_store(p, m + 8, c + 1, v.w);
}

// NT tiles of 8 tokens.  Tiles of the list: (64 rows, NT token tiles, k block), the k block fastest.  ZP: there are zero points.
template <int NT, bool SMALL, bool ZP>
__global__ void __launch_bounds__(32 * L4_WARPS, L4Cfg<NT, SMALL>::CTAS)
linear4_stream_kernel(const __grid_constant__ CUtensorMap tmapX, const Linear4Params p) {
    using Cfg = L4Cfg<NT, SMALL>;
    constexpr int GROUPS = Cfg::GROUPS;
    extern __shared__ uint8_t l4_raw[];
    __shared__ __align__(8) uint64_t full_s[L4_WARPS][L4_STAGES];
    __shared__ PieceParts parts_s[2 * L4_WARPS];
    __shared__ long long piece_s[2 * L4_WARPS];                    // the pieces this block's warps have parts of: ended, last; -1: none
    __shared__ int abort_s;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t* const l4_x = l4_raw + ((1024 - (smem_u32(l4_raw) & 1023)) & 1023);
    uint8_t* const l4_ring = l4_x + Cfg::X_RING;
    if (lane == 0) {
        for (int i = 0; i < L4_STAGES; ++i) mbar_init(&full_s[warp][i], 1);
        fence_barrier_init();
    }
    if (tid == 0) {
        abort_s = 0;
        prefetch_tmap(&tmapX);
    }
    if (tid < 2 * L4_WARPS) piece_s[tid] = -1;
    __syncthreads();
    grid_dep_wait();
    grid_dep_launch();
    const int tgs = (p.N + 8 * NT - 1) / (8 * NT);
    const Shares shares((long long)(p.MT + 3) / 4 * tgs * p.KB, gridDim.x * L4_WARPS);
    const int me = blockIdx.x * L4_WARPS + warp;
    // the same for all lanes, which the compiler sees: the loop's addresses stay in the warp's own registers (42.4 to 38.9 us at 28672 x 8192 x 16)
    const long long from = __shfl_sync(0xffffffffu, me < shares.warps ? shares.begin(me) : 0, 0);
    const long long to = __shfl_sync(0xffffffffu, me < shares.warps ? shares.begin(me + 1) : 0, 0);
    uint8_t* const ring = l4_ring + warp * L4_STAGES * Cfg::STAGE;
    uint8_t* const xring = l4_x + warp * L4_STAGES * Cfg::X_STAGE;

    // The tile to be asked for next, everything about it carried along: a division for each would cost more than the tile's products.
    // One lane asks for all of it, the inputs through a tensor map: copied 16 bytes a lane they cost a fifth of the loop's instructions.
    const int tiles = (int)(to - from);
    int asked = 0, ask_s = 0, ask_kb, ask_tg;
    const uint8_t *ask_data, *ask_scales, *ask_zeros;
    {
        const int piece = (int)floor_div(from, p.KB), rg = piece / tgs;
        ask_kb = (int)(from - (long long)piece * p.KB);
        ask_tg = piece - rg * tgs;
        ask_data = reinterpret_cast<const uint8_t*>(p.data) + ((int64_t)rg * p.KB + ask_kb) * 2048;
        ask_scales = reinterpret_cast<const uint8_t*>(p.scales) + (int64_t)rg * p.NG * 128;      // of the rows
        ask_zeros = p.zeros + (int64_t)rg * p.NG * 32;
    }
    auto fetch = [&]() {
        if (asked >= tiles) return;
        if (elect_one()) {
            const uint32_t dst = smem_u32(ring + ask_s * Cfg::STAGE);
            const int g0 = (ask_kb * 64) >> p.logg, groups = SMALL && p.NG - g0 < GROUPS ? 1 : GROUPS;
            uint64_t* bar = &full_s[warp][ask_s];
            mbar_arrive_expect_tx(bar, 2048 + groups * (ZP ? 160 : 128) + Cfg::X_STAGE);
            l4_bulk(dst, ask_data, 2048, bar);
            l4_bulk(dst + Cfg::SCALES, ask_scales + g0 * 128, groups * 128, bar);
            if (ZP) l4_bulk(dst + Cfg::ZEROS, ask_zeros + g0 * 32, groups * 32, bar);
            tma_load_2d(xring + ask_s * Cfg::X_STAGE, &tmapX, bar, ask_kb * 64, ask_tg * NT * 8);
        }
        ++asked;
        if (++ask_s == L4_STAGES) ask_s = 0;
        ask_data += 2048;
        if (++ask_kb == p.KB) {      // the next piece: other tokens with the same rows, or the next rows
            ask_kb = 0;
            if (++ask_tg == tgs) {
                ask_tg = 0;
                ask_scales += (int64_t)p.NG * 128;
                ask_zeros += (int64_t)p.NG * 32;
            } else {
                ask_data -= (int64_t)p.KB * 2048;
            }
        }
    };
    for (int i = 0; i < L4_STAGES - 1; ++i) fetch();

    int piece = (int)floor_div(from, p.KB), kb = (int)(from - (long long)piece * p.KB);
    float acc[4][NT][4];
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[i][n][0] = acc[i][n][1] = acc[i][n][2] = acc[i][n][3] = 0.f;
    };
    auto finish = [&](long long q, int i, int n, const float4& v, int ln) { l4_finish<NT>(p, tgs, q, i, n, v, ln); };
    auto keep = [&](float* to_p) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) *reinterpret_cast<float4*>(to_p + ((i * NT + n) * 32 + lane) * 4) = make_float4(acc[i][n][0], acc[i][n][1], acc[i][n][2], acc[i][n][3]);
    };
    clear();
    int s = 0;
    uint32_t phase = 0;
    bool first = true;            // the piece at hand may have begun before this share
    for (int at = 0; at < tiles; ++at) {
        if (!__all_sync(0xffffffffu, mbar_wait(&full_s[warp][s], phase, p.d_status, KST_WAIT_FULL, &abort_s))) {
            for (int i = 0; i < 4; ++i) __nanosleep(1000000);   // copies may still land
            break;
        }
        __syncwarp();             // every lane has read the stage that is asked for now; a vote alone orders no memory
        fetch();
        const uint8_t* st = ring + s * Cfg::STAGE;
        const uint8_t* xs = xring + s * Cfg::X_STAGE + g * 128;
        if (++s == L4_STAGES) s = 0, phase ^= 1;
        uint32_t x[NT][8];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint4 v = *reinterpret_cast<const uint4*>(xs + n * 1024 + (((half * 4 + t) ^ g) << 4));
                x[n][4 * half] = v.x, x[n][4 * half + 1] = v.y, x[n][4 * half + 2] = v.z, x[n][4 * half + 3] = v.w;
            }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 w = *reinterpret_cast<const uint4*>(st + i * 512 + lane * 16);
            uint32_t sc[GROUPS], zb[GROUPS];
#pragma unroll
            for (int j = 0; j < GROUPS; ++j) {
                const bool live = j == 0 || kb * 2 + j < p.NG;
                sc[j] = live ? *reinterpret_cast<const uint32_t*>(st + Cfg::SCALES + j * 128 + i * 32 + g * 4) : 0;
                zb[j] = ZP && live ? st[Cfg::ZEROS + j * 32 + i * 8 + g] : 0x88u;
            }
            l4_block<NT, SMALL>(acc[i], w, sc, zb, x);
        }
        if (++kb == p.KB || at + 1 == tiles) {
            const long long start = (long long)piece * p.KB;
            const bool mine = kb == p.KB && (!first || from == start);
            if (mine) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n) finish(piece, i, n, make_float4(acc[i][n][0], acc[i][n][1], acc[i][n][2], acc[i][n][3]), lane);
            } else {
                if (at + 1 < tiles) keep(p.part + (int64_t)(2 * me) * Cfg::FLOATS);
                if (lane == 0) piece_s[2 * warp + (at + 1 == tiles)] = piece;
            }
            if (at + 1 < tiles) {
                clear();
                first = false;
                kb = 0, ++piece;
            }
        }
    }

    // ---- the block's parts of pieces
    __syncthreads();              // the ring is free: every copy that was asked for has been waited for
    float* rows_s = reinterpret_cast<float*>(l4_ring);
    if (piece_s[2 * warp + 1] >= 0) keep(rows_s + warp * Cfg::FLOATS);
    if (tid < 2 * L4_WARPS && piece_s[tid] >= 0) parts_s[tid] = PieceParts::of<L4_WARPS>(shares, piece_s[tid] * p.KB, (piece_s[tid] + 1) * p.KB);
    __syncthreads();
    auto same = [&](int w) { return w + 1 < L4_WARPS && piece_s[2 * w + 1] >= 0 && piece_s[2 * w + 1] == piece_s[2 * w + 3]; };
    for (int w = 0, end; w < L4_WARPS; w = end) {
        end = w + 1;
        while (same(end - 1)) ++end;
        const long long q = piece_s[2 * w + 1];
        if (q < 0) continue;
        const bool all = parts_s[2 * w + 1].count == 1;
        float* part = p.part + (int64_t)(2 * (blockIdx.x * L4_WARPS + w) + 1) * Cfg::FLOATS;
        for (int i = tid; i < Cfg::FLOATS / 4; i += 32 * L4_WARPS) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k = w; k < end; ++k) {
                const float4 x = *reinterpret_cast<const float4*>(rows_s + k * Cfg::FLOATS + i * 4);
                v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
            }
            if (all) finish(q, i / 32 / NT, i / 32 % NT, v, i % 32);
            else *reinterpret_cast<float4*>(part + i * 4) = v;
        }
    }
}

// One block a piece: the sum of its parts, in the order of the list, where they lie in several places.
template <int NT, bool SMALL>
__global__ void __launch_bounds__(32 * NT * 4)
linear4_join_kernel(const Linear4Params p, int64_t warps) {
    using Cfg = L4Cfg<NT, SMALL>;
    __shared__ PieceParts parts_s;
    const long long q = blockIdx.x;
    const int i = threadIdx.x, tgs = (p.N + 8 * NT - 1) / (8 * NT);
    if (i == 0) parts_s = PieceParts::of<L4_WARPS>(Shares((long long)(p.MT + 3) / 4 * tgs * p.KB, (int)warps), q * p.KB, (q + 1) * p.KB);
    __syncthreads();
    grid_dep_wait();
    grid_dep_launch();
    const PieceParts r = parts_s;
    if (r.w0 == r.w1 || r.count == 1) return;     // a warp or a block had it whole
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int u = 0; u < r.count; ++u) {
        const float4 x = *reinterpret_cast<const float4*>(p.part + r.place<L4_WARPS>(u) * Cfg::FLOATS + i * 4);
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
    }
    l4_finish<NT>(p, tgs, q, i / 32 / NT, i / 32 % NT, v, i % 32);
}

// For many tokens the weights of a block of rows become fp16 in the workspace, exactly: (q - z) s has 16 bits at most and is a whole
// multiple of 2^-24, so what the nearest fp16 number leaves of it is one too.  Rows 0 .. R - 1 of the dense weight hold the upper parts,
// rows R .. 2 R - 1 the lower ones, of 64-row units [four0, four0 + R / 64); one GEMM multiplies both and linear4_finish_kernel adds them.
// (q - z) s may pass fp16's range: a row with a scale above 4096 is stored 2^4 smaller, whole multiples of 2^-20 of the weight, and
// `shift` says so.
constexpr int L4_UNPACK_PITCH = 64 + 8;
constexpr int L4_UNPACK_STEPS = 4;       // of two k blocks, a block: the look at its rows' scales is paid once for them
__global__ void __launch_bounds__(256)
linear4_unpack_kernel(const Linear4Params p, int64_t four0, __half* out, int64_t R, uint8_t* shift) {
    __shared__ __align__(16) __half tile[2][2][64][L4_UNPACK_PITCH];   // [upper, lower][k block][input][row]
    __shared__ uint32_t tops[8][32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int mt0 = (int)(four0 + blockIdx.x) * 4, mt = mt0 + (warp & 3);
    grid_dep_wait();
    grid_dep_launch();
    uint32_t top = 0;                    // largest magnitudes of a row's and its neighbour's scales, as fp16 bits
    for (int grp = warp; grp < p.NG; grp += 8) top = __vmaxu2(top, __ldg(p.scales + p.group8(mt0, grp) + lane) & 0x7fff7fffu);
    tops[warp][lane] = top;
    __syncthreads();
    auto most = [&](int word) {          // bits 0 .. 15 of rows g, 16 .. 31 of rows g + 8
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = __vmaxu2(m, tops[i][word]);
        return m;
    };
    constexpr uint32_t LIMIT = 0x6c00;   // 4096: 15 of it are within the range
    const uint32_t mine = most((warp & 3) * 8 + g);
    const float f0 = (mine & 0xffffu) > LIMIT ? 0x1p-4f : 1.f, f1 = (mine >> 16) > LIMIT ? 0x1p-4f : 1.f;
    if (blockIdx.y == 0 && tid < 64) shift[(int64_t)blockIdx.x * 64 + tid] = (most((tid >> 4) * 8 + (tid & 7)) >> (tid & 8 ? 16 : 0) & 0xffffu) > LIMIT ? 4 : 0;
    for (int step = 0; step < L4_UNPACK_STEPS; ++step) {
        const int kb0 = (blockIdx.y * L4_UNPACK_STEPS + step) * 2, kb = kb0 + (warp >> 2);
        if (kb0 >= p.KB) break;
        if (step > 0) __syncthreads();
        if (kb < p.KB) {
            const uint4 w = __ldg(p.data + p.unit(mt, kb) * 32 + lane);
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int grp = (kb * 64 + (s >> 1) * 32) >> p.logg;
                const bool live = grp < p.NG;
                const uint32_t sc = live ? __ldg(p.scales + p.group8(mt, grp) + g) : 0;
                uint32_t z0, z1, a[4];
                l4_zero(live && p.zeros != nullptr ? __ldg(p.zeros + p.group8(mt, grp) + g) : 0x88u, z0, z1);
                l4_weights(v[s], z0, z1, a);
                float2 s2 = __half22float2(*reinterpret_cast<const __half2*>(&sc));
                s2.x *= f0, s2.y *= f1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&a[i]));
                    const float sv = i & 1 ? s2.y : s2.x, w0 = q.x * sv, w1 = q.y * sv;
                    const __half2 hi = __floats2half2_rn(w0, w1);
                    const float2 back = __half22float2(hi);
                    const __half2 lo = __floats2half2_rn(w0 - back.x, w1 - back.y);
                    const int k = (s >> 1) * 32 + t * 8 + (s & 1) * 4 + (i >> 1) * 2, row = (warp & 3) * 16 + g + (i & 1) * 8;
                    tile[0][warp >> 2][k][row] = __low2half(hi);
                    tile[0][warp >> 2][k + 1][row] = __high2half(hi);
                    tile[1][warp >> 2][k][row] = __low2half(lo);
                    tile[1][warp >> 2][k + 1][row] = __high2half(lo);
                }
            }
        }
        __syncthreads();
        for (int i = tid; i < 2 * 2 * 64 * 8; i += 256) {
            const int part = i >> 10, in = i >> 3 & 127, k = kb0 * 64 + in;
            if (k < p.K)
                *reinterpret_cast<uint4*>(out + (int64_t)k * 2 * R + part * R + blockIdx.x * 64 + (i & 7) * 8) =
                    *reinterpret_cast<const uint4*>(&tile[part][in >> 6][in & 63][(i & 7) * 8]);
        }
    }
}

// Results of `rows` rows from m0 and `tokens` tokens from n0: both parts' sums, brought back to scale.  Where the upper parts' is not
// finite it is the result: what is infinite times a lower part of 0 is no number.
constexpr int L4_FINISH_TOKENS = 8;      // a thread
__global__ void __launch_bounds__(128)
linear4_finish_kernel(const Linear4Params p, const float* __restrict__ y, int64_t R, const uint8_t* __restrict__ shift, int64_t m0, int rows, int n0, int tokens) {
    grid_dep_wait();
    grid_dep_launch();
    const int r = blockIdx.x * 128 + threadIdx.x, at = blockIdx.y * L4_FINISH_TOKENS;
    if (r >= rows) return;
    const float f = shift[r] ? 16.f : 1.f;
    float v[L4_FINISH_TOKENS][2];
#pragma unroll
    for (int i = 0; i < L4_FINISH_TOKENS; ++i)
#pragma unroll
        for (int part = 0; part < 2; ++part) v[i][part] = at + i < tokens ? y[(at + i) * 2 * R + part * R + r] : 0.f;
#pragma unroll
    for (int i = 0; i < L4_FINISH_TOKENS; ++i)
        if (at + i < tokens) l4_store(p, m0 + r, n0 + at + i, (v[i][0] + (isfinite(v[i][0]) ? v[i][1] : 0.f)) * f);
}

struct PackParams {
    const uint8_t *q, *zeros;
    const __half* scales;
    int64_t qM, qK, sM, sG, zM, zG, M;
    int K, KB, NG, M4;      // M4: fours of row tiles
    uint32_t *data, *oscales;
    uint8_t* ozeros;
};

// One thread a word of weights; the first threads of the grid also lay out the scales.
__global__ void __launch_bounds__(256)
linear4_pack_kernel(const PackParams p) {
    grid_dep_wait();
    grid_dep_launch();
    const int64_t words = (int64_t)p.M4 * p.KB * 512, pairs = (int64_t)p.M4 * p.NG * 32;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
        const int s = (int)(i & 3), lane = (int)(i >> 2 & 31), g = lane >> 2, t = lane & 3;
        const int64_t unit = i >> 9, m4 = unit / p.KB, mt = m4 * 4 + (i >> 7 & 3);
        const int kb = (int)(unit - m4 * p.KB);
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {   // nibble j: register j % 4, half j / 4
            const int reg = j & 3, k = kb * 64 + (s >> 1) * 32 + t * 8 + (s & 1) * 4 + (reg >> 1) * 2 + (j >> 2);
            const int64_t m = mt * 16 + g + (reg & 1) * 8;
            const uint32_t v = m < p.M && k < p.K ? p.q[m * p.qM + k * p.qK] & 15u : 8u;
            w |= v << (4 * j);
        }
        p.data[i] = w;
    }
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pairs; i += (int64_t)gridDim.x * 256) {
        const int g = (int)(i & 7);
        const int64_t unit = i >> 5, m4 = unit / p.NG, grp = unit - m4 * p.NG, mt = m4 * 4 + (i >> 3 & 3);
        uint32_t s = 0, z = 0;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int64_t m = mt * 16 + g + r * 8;
            const bool in = m < p.M;
            s |= (in ? (uint32_t)__half_as_ushort(p.scales[m * p.sM + grp * p.sG]) : 0u) << (16 * r);
            z |= (in && p.zeros != nullptr ? p.zeros[m * p.zM + grp * p.zG] & 15u : 8u) << (4 * r);
        }
        p.oscales[i] = s;
        if (p.ozeros != nullptr) p.ozeros[i] = (uint8_t)z;
    }
}

template <int ROWS, int NT>
static int l4_launch(b200_ctx* ctx, const Linear4Params& p) {
    B200_REQUIRE(cdiv(p.N, 8 * NT) < 65536, B200_DECLINE_EXTENT, "matmul_q4: %d tokens off 16-byte boundaries", p.N);
    auto kern = p.logg == 5 ? linear4_kernel<ROWS, NT, true> : linear4_kernel<ROWS, NT, false>;
    B200_CUDA(launch_dep(kern, dim3((unsigned)cdiv(p.MT, ROWS), (unsigned)cdiv(p.N, 8 * NT)), dim3(32 * L4_WARPS), 0, ctx->stream, 1, p));
    ctx->launches++;
    return B200_OK;
}
template <int NT, bool SMALL, bool ZP>
static int l4_stream_launch(b200_ctx* ctx, Linear4Params& p) {
    using Cfg = L4Cfg<NT, SMALL>;
    auto kern = linear4_stream_kernel<NT, SMALL, ZP>;
    static std::atomic<uint64_t> asked{0};
    B200_CUDA(allow_smem(ctx, kern, Cfg::SMEM, asked));
    CUtensorMap mx;               // rows of 64 inputs, zeros past the ends
    const uint64_t dims[2] = {(uint64_t)p.K, (uint64_t)p.N}, strides[1] = {(uint64_t)p.ldx * 2};
    const uint32_t box[2] = {64, 8 * NT};
    int rc = make_tmap(ctx, &mx, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, p.x, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    int64_t grid = (int64_t)ctx->prop.multiProcessorCount * Cfg::CTAS;
    void* ws = nullptr;
    rc = ws_scratch(ctx, (size_t)grid * L4_WARPS * 2 * Cfg::FLOATS * sizeof(float), &ws);
    if (rc) return rc;
    p.part = static_cast<float*>(ws);
    B200_CUDA(launch_dep(kern, dim3((unsigned)grid), dim3(32 * L4_WARPS), Cfg::SMEM, ctx->stream, 1, mx, p));
    const int64_t pieces = cdiv(p.MT, 4) * cdiv(p.N, 8 * NT);
    B200_CUDA(launch_dep(linear4_join_kernel<NT, SMALL>, dim3((unsigned)pieces), dim3(32 * NT * 4), 0, ctx->stream, 1, p, grid * L4_WARPS));
    ctx->launches += 2;
    return B200_OK;
}

// Many tokens: the weight as fp16, a block of rows at a time, and the GEMM.
static int l4_dense(b200_ctx* ctx, const b200_q4* A, const Linear4Params& p, const void* B, int64_t ldb) {
    const int64_t K = A->K, units = cdiv(A->M, 64), parts = cdiv(p.KB, 2 * L4_UNPACK_STEPS);
    B200_REQUIRE(parts < 65536, B200_DECLINE_EXTENT, "matmul_q4: K=%lld", (long long)K);
    const int64_t most = p.N < L4_DENSE_TOKENS ? p.N : L4_DENSE_TOKENS, row = 4 * K + 8 * most + 1;   // two parts of two bytes, their sums, a shift
    int64_t block = L4_DENSE_BYTES / (64 * row);           // units of 64 rows
    if (block < 4) block = 4;
    block = cdiv(units, cdiv(units, block));               // blocks of like sizes
    const int64_t R = block * 64;
    void* ws = nullptr;
    int rc = ws_scratch(ctx, (size_t)(R * row), &ws);
    if (rc) return rc;
    __half* w = static_cast<__half*>(ws);
    float* y = reinterpret_cast<float*>(w + 2 * R * K);
    uint8_t* shift = reinterpret_cast<uint8_t*>(y + 2 * R * most);
    const size_t mark = ctx->ws_used;
    for (int64_t n0 = 0; n0 < p.N; n0 += most) {
        const int64_t tokens = p.N - n0 < most ? p.N - n0 : most;
        for (int64_t u0 = 0; u0 < units; u0 += block) {
            const int64_t have = units - u0 < block ? units - u0 : block, r = have * 64, rows = A->M - u0 * 64 < r ? A->M - u0 * 64 : r;
            if (n0 == 0 || block < units) {
                B200_CUDA(launch_dep(linear4_unpack_kernel, dim3((unsigned)have, (unsigned)parts), dim3(256), 0, ctx->stream, 1, p, u0, w, r, shift));
                ctx->launches++;
            }
            rc = gemm_f16_run(ctx, 2 * r, tokens, K, w, 2 * r, (const __half*)B + n0 * ldb, ldb, nullptr, 0, y, 2 * r, B200_F32, B200_EPI_NONE, 1, 0, 0, 0);
            if (rc) return rc;
            ctx->ws_used = mark;                           // what the GEMM took; the next one runs behind it
            B200_CUDA(launch_dep(linear4_finish_kernel, dim3((unsigned)cdiv(rows, 128), (unsigned)cdiv(tokens, L4_FINISH_TOKENS)), dim3(128), 0, ctx->stream, 1,
                                 p, (const float*)y, r, (const uint8_t*)shift, u0 * 64, (int)rows, (int)n0, (int)tokens));
            ctx->launches++;
        }
    }
    return B200_OK;
}

static int l4_shape(const char* op, int64_t M, int64_t K, int64_t group) {
    B200_REQUIRE(M >= 1 && K >= 1 && M < (1ll << 31) - 64 && K < (1ll << 31) - 128, B200_DECLINE_EXTENT, "%s: M=%lld K=%lld", op, (long long)M, (long long)K);
    B200_REQUIRE(group == 32 || group == 64 || group == 128, B200_DECLINE_EXTENT, "%s: groups of %lld (32, 64 or 128)", op, (long long)group);
    B200_REQUIRE(K % group == 0, B200_DECLINE_EXTENT, "%s: K=%lld is not whole groups of %lld", op, (long long)K, (long long)group);
    return B200_OK;
}

} // namespace b200

using namespace b200;

extern "C" {

int b200_q4_sizes(int64_t M, int64_t K, int64_t group, int64_t* data_bytes, int64_t* scale_bytes, int64_t* zero_bytes) {
    int rc = l4_shape("q4_sizes", M, K, group);
    if (rc) return rc;
    B200_REQUIRE(data_bytes && scale_bytes && zero_bytes, B200_EINVAL, "q4_sizes: null argument");
    const int64_t fours = cdiv(M, 64);
    *data_bytes = fours * cdiv(K, 64) * 2048;
    *scale_bytes = fours * (K / group) * 128;
    *zero_bytes = fours * (K / group) * 32;
    return B200_OK;
}

int b200_q4_pack(b200_ctx* ctx, const void* q, int64_t q_m, int64_t q_k, const void* scales, int64_t s_m, int64_t s_g, const void* zeros,
                 int64_t z_m, int64_t z_g, const b200_q4* out) {
    B200_REQUIRE(ctx && out, B200_EINVAL, "q4_pack: null argument");
    int rc = l4_shape("q4_pack", out->M, out->K, out->group);
    if (rc) return rc;
    B200_REQUIRE(q && scales && out->data && out->scales && (!zeros == !out->zeros), B200_EINVAL, "q4_pack: null array");
    B200_REQUIRE((uintptr_t)out->data % 16 == 0 && (uintptr_t)out->scales % 16 == 0 && (uintptr_t)out->zeros % 16 == 0, B200_DECLINE_ALIGN, "q4_pack: the packed arrays' alignment");
    B200_CUDA(cudaSetDevice(ctx->device));
    PackParams p = {};
    p.q = (const uint8_t*)q, p.scales = (const __half*)scales, p.zeros = (const uint8_t*)zeros;
    p.qM = q_m, p.qK = q_k, p.sM = s_m, p.sG = s_g, p.zM = z_m, p.zG = z_g;
    p.M = out->M, p.K = (int)out->K, p.KB = (int)cdiv(out->K, 64), p.NG = (int)(out->K / out->group), p.M4 = (int)cdiv(out->M, 64);
    p.data = (uint32_t*)out->data, p.oscales = (uint32_t*)out->scales, p.ozeros = (uint8_t*)out->zeros;
    const int64_t blocks = cdiv((int64_t)p.M4 * p.KB * 512, 256), most = (int64_t)ctx->prop.multiProcessorCount * 16;
    B200_CUDA(launch_dep(linear4_pack_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, ctx->stream, 1, p));
    ctx->launches++;
    return B200_OK;
}

int b200_matmul_q4(b200_ctx* ctx, const b200_q4* A, int64_t N, const void* B, int64_t ldb, const void* bias, void* out, int64_t ldo,
                   int out_dtype, int epilogue) {
    B200_REQUIRE(ctx && A, B200_EINVAL, "matmul_q4: null argument");
    int rc = l4_shape("matmul_q4", A->M, A->K, A->group);
    if (rc) return rc;
    B200_REQUIRE(N >= 0 && N < (1ll << 31) - 64 && ldb >= A->K && ldo >= A->M, B200_EINVAL, "matmul_q4: N=%lld ldb=%lld ldo=%lld", (long long)N,
                 (long long)ldb, (long long)ldo);
    B200_REQUIRE(out_dtype == B200_F16 || out_dtype == B200_F32, B200_DECLINE_ELTYPE, "matmul_q4: out dtype %d", out_dtype);
    B200_REQUIRE(epilogue >= B200_EPI_NONE && epilogue <= B200_EPI_GELU_TANH, B200_EINVAL, "matmul_q4: epilogue %d", epilogue);
    if (N == 0) return B200_OK;
    B200_REQUIRE(A->data && A->scales && B && out, B200_EINVAL, "matmul_q4: null array");
    B200_REQUIRE((uintptr_t)A->data % 16 == 0 && (uintptr_t)A->scales % 16 == 0 && (uintptr_t)A->zeros % 16 == 0, B200_DECLINE_ALIGN, "matmul_q4: the packed arrays' alignment");
    B200_CUDA(cudaSetDevice(ctx->device));
    Linear4Params p = {};
    p.data = (const uint4*)A->data, p.scales = (const uint32_t*)A->scales, p.zeros = (const uint8_t*)A->zeros;
    p.x = (const __half*)B, p.bias = (const __half*)bias, p.out = out;
    p.ldx = ldb, p.ldo = ldo, p.M = A->M;
    p.N = (int)N, p.K = (int)A->K, p.KB = (int)cdiv(A->K, 64), p.NG = (int)(A->K / A->group), p.MT = (int)cdiv(A->M, 16);
    p.logg = A->group == 32 ? 5 : A->group == 64 ? 6 : 7;
    p.out_f32 = out_dtype == B200_F32, p.epi = epilogue;
    p.whole = (uintptr_t)B % 16 == 0 && ldb % 8 == 0;
    // Inputs off 16-byte boundaries keep to the kernels, where the GEMM would read them one by one (1000 tokens of 4096 x 4096 403 us and 1153).
    if (N > L4_TOKENS && p.whole) return l4_dense(ctx, A, p, B, ldb);
    p.d_status = ctx->d_status;
    const int nt = N <= 8 ? 1 : 2;
    // More than 16 tokens: up to 40 to a block of linear4_kernel, whose warps take a round trip of loads a k block.
    const int64_t groups = N <= 16 ? 1 : cdiv(N, 40), many = N <= 16 ? nt : cdiv(cdiv(N, 8), groups);
    const int64_t rounds = cdiv(p.KB, L4_WARPS) * cdiv(cdiv(p.MT, 2) * groups, 2 * (int64_t)ctx->prop.multiProcessorCount);
    const double tiles = (double)cdiv(p.MT, 4) * (double)cdiv(N, 8 * nt) * p.KB;
    if (p.whole && (N <= 16 ? tiles >= L4_STREAM_TILES : rounds * many > L4_ROUNDS)) {
        const auto go = [&](auto small, auto zp) {
            return nt == 1 ? l4_stream_launch<1, decltype(small)::value, decltype(zp)::value>(ctx, p)
                           : l4_stream_launch<2, decltype(small)::value, decltype(zp)::value>(ctx, p);
        };
        using yes = std::true_type;
        using no = std::false_type;
        if (p.logg == 5) return p.zeros ? go(yes(), yes()) : go(yes(), no());
        return p.zeros ? go(no(), yes()) : go(no(), no());
    }
    switch (many) {
    case 1: return l4_launch<1, 1>(ctx, p);
    case 2: return l4_launch<1, 2>(ctx, p);
    case 3: return l4_launch<2, 3>(ctx, p);
    case 4: return l4_launch<2, 4>(ctx, p);
    default: return l4_launch<2, 5>(ctx, p);
    }
}

} // extern "C"
