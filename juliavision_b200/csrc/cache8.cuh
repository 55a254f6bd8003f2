// The paged cache of 8-bit values as its kernels see it: pages of T tokens (a power of two), each (E, T) for every key head, and
// one fp32 number a (page, head), the largest magnitude m among the page's values when it was written.  An element stands for
// q m / 127 (int8) or q m / 448 (e4m3, whose largest value is 448).
//
// m is kept rather than m / 127 so that writing is exact but for its one rounding: for fp16 x, 127 x and 448 x have at most 18
// significant bits, and so does q m when a page's values are brought to a larger m; their fp32 quotient by m is then within
// 2^-24 of the true one, while a true quotient that is not itself a point half way between two 8-bit values is at least 2^-20
// away from one.  The 8-bit values are therefore those of exact arithmetic.
#pragma once
#include <cuda_fp16.h>

#include "internal.h"
#include "ptx.cuh"

namespace b200 {

struct CacheView {
    uint8_t *k, *v;
    int64_t kT, kH, kP, vT, vH, vP;   // strides in bytes
    float *kmax, *vmax;               // (H, P)
    const int32_t* table;             // (width, B)
    int64_t table_ld, P;
    int E, T, logT, H, width;
    int* d_status;

    // The three look-ups every kernel goes through; whatever the device arrays hold, what they return is inside the cache.
    __host__ __device__ __forceinline__ void report(int code) const {
#ifdef __CUDA_ARCH__
        atomicCAS(d_status, 0, code);
#else
        if (*d_status == 0) *d_status = code;
#endif
    }
    __host__ __device__ __forceinline__ int tokens(int b, const int32_t* lens) const {   // of sequence b, no more than its pages hold
        const int n = lens[b], most = width << logT;
        if (n < 0 || n > most) report(KST_CACHE_LENGTH);
        return n < 0 ? 0 : n > most ? most : n;
    }
    __host__ __device__ __forceinline__ int fresh(int b, const int32_t* news, int L) const {   // rows of sequence b that count
        const int m = news != nullptr ? news[b] : L;
        if (m < 0 || m > L) report(KST_CACHE_LENGTH);
        return m < 0 ? 0 : m > L ? L : m;
    }
    __host__ __device__ __forceinline__ int64_t page(int b, int i) const {   // the page of tokens i T ... of sequence b, or -1
        const int pg = table[b * table_ld + i];
        if (pg >= 0 && pg < P) return pg;
        report(KST_CACHE_PAGE);
        return -1;
    }
};

constexpr int CACHE_MOST_T = 128;

// Checks what the host can see; fills `out`.
int cache_view(b200_ctx* ctx, const b200_cache8* c, const char* op, CacheView* out);

// Attention of many query rows a key head (cache8_prompt.cu); what cache_view checks has been checked, and the operands too.
int cache_prompt_run(b200_ctx* ctx, const CacheView& c, int64_t L, int64_t B, int64_t G, const b200_strided4* q, const b200_strided4* out,
                     int out_dtype, float scale, bool fp8, int causal, const int32_t* lens, const int32_t* news);

template <bool FP8> __device__ __forceinline__ constexpr float cache_top() { return FP8 ? 448.f : 127.f; }

// Four 8-bit values as fp16, exactly: (0, 1) and (2, 3).  A byte u under 0x64 is the fp16 number 1024 + u.
template <bool FP8> __device__ __forceinline__ void cache_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (FP8) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi) : "r"(w));
    } else {
        w ^= 0x80808080u;
        const __half2 off = __half2half2(__ushort_as_half(0x6480));   // 1152
        uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 ha = __hsub2(*reinterpret_cast<__half2*>(&a), off), hb = __hsub2(*reinterpret_cast<__half2*>(&b), off);
        lo = *reinterpret_cast<const uint32_t*>(&ha);
        hi = *reinterpret_cast<const uint32_t*>(&hb);
    }
}

} // namespace b200
