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
#include <cuda_fp16.h>

#include "act.cuh"
#include "internal.h"
#include "ptx.cuh"

namespace b200 {

constexpr int L4_WARPS = 8;      // of a block, which share K
constexpr int L4_TOKENS = 64;    // tokens the kernel takes; more go through fp16 weights in the workspace

struct Linear4Params {
    const uint4* data;            // [row tile][k block][lane]
    const uint32_t* scales;       // [row tile][group][8]: fp16 scales of rows g and g + 8
    const uint8_t* zeros;         // [row tile][group][8]: zero points of rows g (low) and g + 8 (high), or null
    const __half *x, *bias;
    void* out;
    int64_t ldx, ldo, M;
    int N, K, KB, NG, MT;         // k blocks of 64, groups a row, row tiles
    int logg;                     // log2 of the group size
    int out_f32, epi, whole;
};

__device__ __forceinline__ uint32_t l4_and_or(uint32_t v, uint32_t m, uint32_t o) { return (v & m) | o; }
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
    a[0] = l4_sub(l4_and_or(v, 0x000f000fu, 0x64006400u), z0);
    a[1] = l4_fma16(l4_and_or(v, 0x00f000f0u, 0x64006400u), z1);
    v >>= 8;
    a[2] = l4_sub(l4_and_or(v, 0x000f000fu, 0x64006400u), z0);
    a[3] = l4_fma16(l4_and_or(v, 0x00f000f0u, 0x64006400u), z1);
}
__device__ __forceinline__ void l4_zero(const uint8_t* zeros, int64_t at, uint32_t& z0, uint32_t& z1) {
    const uint32_t z = zeros != nullptr ? __ldg(zeros + at) : 0x88u;
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

// MT row tiles and NT tiles of 8 tokens a block; the warps take every L4_WARPS-th k block.  SMALL: groups of 32.
template <int MT, int NT, bool SMALL>
__global__ void __launch_bounds__(32 * L4_WARPS)
linear4_kernel(const Linear4Params p) {
    extern __shared__ __align__(16) float l4_red[];   // [warp][row][token]
    constexpr int COLS = 8 * NT + 1, ROWS = 16 * MT, GROUPS = SMALL ? 2 : 1, STEPS = 4 / GROUPS;   // groups a k block, steps a group
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int mt0 = blockIdx.x * MT, n0 = blockIdx.y * 8 * NT;
    grid_dep_wait();
    grid_dep_launch();
    float acc[MT][NT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[i][n][0] = acc[i][n][1] = acc[i][n][2] = acc[i][n][3] = 0.f;
    for (int kb = warp; kb < p.KB; kb += L4_WARPS) {
        uint4 w[MT];
        uint32_t sc[MT][GROUPS];
        uint32_t z0[MT][GROUPS], z1[MT][GROUPS];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const bool in = mt0 + i < p.MT;
            w[i] = in ? __ldg(p.data + ((int64_t)(mt0 + i) * p.KB + kb) * 32 + lane) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < GROUPS; ++j) {
                const int grp = (kb * 64 + j * 32) >> p.logg;
                const bool live = in && grp < p.NG;    // the last k block may be half empty
                const int64_t at = ((int64_t)(mt0 + i) * p.NG + grp) * 8 + g;
                sc[i][j] = live ? __ldg(p.scales + at) : 0;
                l4_zero(live ? p.zeros : nullptr, at, z0[i][j], z1[i][j]);
            }
        }
        uint32_t x[NT][8];
#pragma unroll
        for (int n = 0; n < NT; ++n) l4_input(p, n0 + n * 8 + g, kb, t, x[n]);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int j = 0; j < GROUPS; ++j) {
                const float2 s = __half22float2(*reinterpret_cast<const __half2*>(&sc[i][j]));
                float c[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    uint32_t a[4];
                    l4_weights(v[j * STEPS + k], z0[i][j], z1[i][j], a);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816(c[n], a, x[n][2 * (j * STEPS + k)], x[n][2 * (j * STEPS + k) + 1]);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    acc[i][n][0] = fmaf(c[n][0], s.x, acc[i][n][0]);
                    acc[i][n][1] = fmaf(c[n][1], s.x, acc[i][n][1]);
                    acc[i][n][2] = fmaf(c[n][2], s.y, acc[i][n][2]);
                    acc[i][n][3] = fmaf(c[n][3], s.y, acc[i][n][3]);
                }
            }
        }
    }
    float* mine = l4_red + warp * ROWS * COLS;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) mine[(i * 16 + g + (k >> 1) * 8) * COLS + n * 8 + 2 * t + (k & 1)] = acc[i][n][k];
    __syncthreads();
    for (int i = tid; i < ROWS * 8 * NT; i += 32 * L4_WARPS) {
        const int row = i % ROWS, col = i / ROWS, n = n0 + col;
        const int64_t m = (int64_t)mt0 * 16 + row;
        if (m >= p.M || n >= p.N) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < L4_WARPS; ++w) v += l4_red[(w * ROWS + row) * COLS + col];
        if (p.bias != nullptr) v += __half2float(p.bias[m]);
        // the activation sees the value rounded to the output type, as in the GEMM's store
        if (p.out_f32) ((float*)p.out)[n * p.ldo + m] = apply_act(p.epi, v);
        else ((__half*)p.out)[n * p.ldo + m] = __float2half_rn(apply_act(p.epi, __half2float(__float2half_rn(v))));
    }
}

// The weight as dense fp16 (M, K), for many tokens: a block writes 64 rows of two k blocks through shared memory.
constexpr int L4_UNPACK_PITCH = 64 + 8;
__global__ void __launch_bounds__(256)
linear4_unpack_kernel(const Linear4Params p, __half* out, int64_t ld) {
    __shared__ __align__(16) __half tile[2][64][L4_UNPACK_PITCH];   // [k block][input][row]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int mt = blockIdx.x * 4 + (warp & 3), kb = blockIdx.y * 2 + (warp >> 2);
    grid_dep_wait();
    grid_dep_launch();
    if (mt < p.MT && kb < p.KB) {
        const uint4 w = __ldg(p.data + ((int64_t)mt * p.KB + kb) * 32 + lane);
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int grp = (kb * 64 + (s >> 1) * 32) >> p.logg;
            const bool live = grp < p.NG;
            const int64_t at = ((int64_t)mt * p.NG + grp) * 8 + g;
            const uint32_t sc = live ? __ldg(p.scales + at) : 0;
            uint32_t z0, z1, a[4];
            l4_zero(live ? p.zeros : nullptr, at, z0, z1);
            l4_weights(v[s], z0, z1, a);
            const __half2 s2 = *reinterpret_cast<const __half2*>(&sc);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a[i]), i & 1 ? __high2half2(s2) : __low2half2(s2));
                const int k = (s >> 1) * 32 + t * 8 + (s & 1) * 4 + (i >> 1) * 2, row = (warp & 3) * 16 + g + (i & 1) * 8;
                tile[warp >> 2][k][row] = __low2half(r);
                tile[warp >> 2][k + 1][row] = __high2half(r);
            }
        }
    }
    __syncthreads();
    const int64_t m0 = (int64_t)blockIdx.x * 64;
    for (int i = tid; i < 2 * 64 * 8; i += 256) {
        const int k = blockIdx.y * 128 + i / 8;
        const int64_t m = m0 + i % 8 * 8;
        if (k < p.K && m < ld) *reinterpret_cast<uint4*>(out + k * ld + m) = *reinterpret_cast<const uint4*>(&tile[i / 512][i / 8 % 64][i % 8 * 8]);
    }
}

struct PackParams {
    const uint8_t *q, *zeros;
    const __half* scales;
    int64_t qM, qK, sM, sG, zM, zG, M;
    int K, KB, NG, MT;
    uint32_t *data, *oscales;
    uint8_t* ozeros;
};

// One thread a word of weights; the first threads of the grid also lay out the scales.
__global__ void __launch_bounds__(256)
linear4_pack_kernel(const PackParams p) {
    grid_dep_wait();
    grid_dep_launch();
    const int64_t words = (int64_t)p.MT * p.KB * 128, pairs = (int64_t)p.MT * p.NG * 8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
        const int s = (int)(i & 3), lane = (int)(i >> 2 & 31), g = lane >> 2, t = lane & 3;
        const int64_t unit = i >> 7, mt = unit / p.KB;
        const int kb = (int)(unit - mt * p.KB);
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
        const int64_t unit = i >> 3, mt = unit / p.NG, grp = unit - mt * p.NG;
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

template <int MT, int NT>
static int l4_launch(b200_ctx* ctx, const Linear4Params& p) {
    constexpr int SMEM = L4_WARPS * 16 * MT * (8 * NT + 1) * 4;
    auto kern = p.logg == 5 ? linear4_kernel<MT, NT, true> : linear4_kernel<MT, NT, false>;
    if (SMEM > 48 * 1024) B200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    B200_CUDA(launch_dep(kern, dim3((unsigned)cdiv(p.MT, MT), (unsigned)cdiv(p.N, 8 * NT)), dim3(32 * L4_WARPS), SMEM, ctx->stream, 1, p));
    ctx->launches++;
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
    const int64_t tiles = cdiv(M, 16);
    *data_bytes = tiles * cdiv(K, 64) * 512;
    *scale_bytes = tiles * (K / group) * 32;
    *zero_bytes = tiles * (K / group) * 8;
    return B200_OK;
}

int b200_q4_pack(b200_ctx* ctx, const void* q, int64_t q_m, int64_t q_k, const void* scales, int64_t s_m, int64_t s_g, const void* zeros,
                 int64_t z_m, int64_t z_g, const b200_q4* out) {
    B200_REQUIRE(ctx && out, B200_EINVAL, "q4_pack: null argument");
    int rc = l4_shape("q4_pack", out->M, out->K, out->group);
    if (rc) return rc;
    B200_REQUIRE(q && scales && out->data && out->scales && (!zeros == !out->zeros), B200_EINVAL, "q4_pack: null array");
    B200_REQUIRE((uintptr_t)out->data % 16 == 0 && (uintptr_t)out->scales % 4 == 0, B200_DECLINE_ALIGN, "q4_pack: the packed arrays' alignment");
    B200_CUDA(cudaSetDevice(ctx->device));
    PackParams p = {};
    p.q = (const uint8_t*)q, p.scales = (const __half*)scales, p.zeros = (const uint8_t*)zeros;
    p.qM = q_m, p.qK = q_k, p.sM = s_m, p.sG = s_g, p.zM = z_m, p.zG = z_g;
    p.M = out->M, p.K = (int)out->K, p.KB = (int)cdiv(out->K, 64), p.NG = (int)(out->K / out->group), p.MT = (int)cdiv(out->M, 16);
    p.data = (uint32_t*)out->data, p.oscales = (uint32_t*)out->scales, p.ozeros = (uint8_t*)out->zeros;
    const int64_t blocks = cdiv((int64_t)p.MT * p.KB * 128, 256), most = (int64_t)ctx->prop.multiProcessorCount * 16;
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
    B200_REQUIRE((uintptr_t)A->data % 16 == 0 && (uintptr_t)A->scales % 4 == 0, B200_DECLINE_ALIGN, "matmul_q4: the packed arrays' alignment");
    B200_CUDA(cudaSetDevice(ctx->device));
    Linear4Params p = {};
    p.data = (const uint4*)A->data, p.scales = (const uint32_t*)A->scales, p.zeros = (const uint8_t*)A->zeros;
    p.x = (const __half*)B, p.bias = (const __half*)bias, p.out = out;
    p.ldx = ldb, p.ldo = ldo, p.M = A->M;
    p.N = (int)N, p.K = (int)A->K, p.KB = (int)cdiv(A->K, 64), p.NG = (int)(A->K / A->group), p.MT = (int)cdiv(A->M, 16);
    p.logg = A->group == 32 ? 5 : A->group == 64 ? 6 : 7;
    p.out_f32 = out_dtype == B200_F32, p.epi = epilogue;
    p.whole = (uintptr_t)B % 16 == 0 && ldb % 8 == 0;
    if (N > L4_TOKENS) {
        const int64_t ld = cdiv(A->M, 8) * 8;
        void* w = nullptr;
        rc = ws_scratch(ctx, (size_t)ld * A->K * 2, &w);
        if (rc) return rc;
        B200_REQUIRE(cdiv(p.KB, 2) < 65536, B200_DECLINE_EXTENT, "matmul_q4: K=%lld", (long long)A->K);
        B200_CUDA(launch_dep(linear4_unpack_kernel, dim3((unsigned)cdiv(p.MT, 4), (unsigned)cdiv(p.KB, 2)), dim3(256), 0, ctx->stream, 1, p,
                             (__half*)w, ld));
        ctx->launches++;
        return gemm_f16_run(ctx, A->M, N, A->K, w, ld, B, ldb, bias, 0, out, ldo, out_dtype, epilogue, 1, 0, 0, 0);
    }
    const bool wide = p.MT >= 8 * ctx->prop.multiProcessorCount;   // enough row tiles to give a block four
    if (N <= 8) return wide ? l4_launch<4, 1>(ctx, p) : l4_launch<1, 1>(ctx, p);
    if (N <= 16) return wide ? l4_launch<4, 2>(ctx, p) : l4_launch<1, 2>(ctx, p);
    if (N <= 32) return l4_launch<1, 4>(ctx, p);
    return l4_launch<1, 8>(ctx, p);
}

} // extern "C"
