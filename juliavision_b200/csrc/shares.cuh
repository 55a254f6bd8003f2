// A list of equal tiles, cut into pieces (one result each), dealt out to the warps of a launch in equal contiguous shares; and
// where the parts of a piece that several warps hold come to lie.  A part that ends inside a warp's share has a place of its
// own; the last pieces of a block's warps are joined in the block, whose first warp of a piece gives them their place.
#pragma once
#include <cuda_runtime.h>

namespace b200 {

// floor(a / b), 0 <= a < 2^52: an integer division of 64 bits takes ten times as long, and the ends of a share wait for several.
__device__ __forceinline__ long long floor_div(long long a, long long b) {
    long long q = (long long)((double)a / (double)b);
    const long long r = a - q * b;
    if (r < 0) --q;
    else if (r >= b) ++q;
    return q;
}

struct Shares {
    long long total;      // tiles
    int warps;            // that have a share

    __device__ __forceinline__ Shares(long long tiles, int all) : total(tiles), warps(tiles < all ? (int)tiles : all) {}
    __device__ __forceinline__ long long begin(long long warp) const { return floor_div(warp * total, warps); }
    __device__ __forceinline__ int holder(long long tile) const { return (int)floor_div((tile + 1) * warps - 1, total); }
};

struct PieceParts {       // a piece's first and last warp, blocks with a part of it, parts in all
    int w0, w1, blocks, count;

    template <int BLOCK_WARPS> static __device__ __forceinline__ PieceParts of(const Shares& s, long long start, long long end) {
        PieceParts r;
        r.w0 = s.holder(start);
        r.w1 = s.holder(end - 1);
        const bool inside = s.begin(r.w1 + 1) > end;      // it ends before its last warp's share does
        r.blocks = (r.w1 - (inside ? 1 : 0)) / BLOCK_WARPS - r.w0 / BLOCK_WARPS + 1;
        r.count = r.blocks + (inside ? 1 : 0);
        return r;
    }
    // The place of part i, in the order of the list; place 2 w is what ended inside warp w's share, 2 w + 1 what warp w leads.
    template <int BLOCK_WARPS> __device__ __forceinline__ long long place(int i) const {
        return i == blocks ? 2ll * w1 : 2ll * (i == 0 ? w0 : w0 / BLOCK_WARPS * BLOCK_WARPS + i * BLOCK_WARPS) + 1;
    }
};

} // namespace b200
