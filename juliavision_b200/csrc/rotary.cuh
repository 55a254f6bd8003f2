// What the kernels that turn heads by their positions share (rotary.cu, norm_rotary.cu).
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

constexpr int ROT_PAIRS = 512;     // pairs of a head at most

// The position of token l of sequence b, and whether it is a token.
struct RotPositions {
    const int32_t *positions, *lens, *news;
    int64_t posL, posB;
    int L;
    __device__ __forceinline__ int at(int64_t l, int64_t b, bool& live) const {
        if (positions != nullptr) {
            live = true;
            return positions[l * posL + b * posB];
        }
        const int m = news != nullptr ? news[b] : L;
        live = l < m;
        return (int)((unsigned)lens[b] - (unsigned)m + (unsigned)l);
    }
};

// Sine and cosine of position * f, f in units of 2^-64 turns.
__device__ __forceinline__ void rot_turn(int position, unsigned long long f, float& s, float& c) {
    const unsigned long long turns = (unsigned long long)(long long)position * f;
    sincospif((float)(int)(turns >> 32) * 0x1p-31f, &s, &c);
}

__device__ __forceinline__ uint32_t rot_pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 rot_unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

} // namespace b200
