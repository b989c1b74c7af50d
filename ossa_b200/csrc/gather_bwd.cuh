// What the files of the gathered attention's backward pass share (gather_bwd.cu: the turned lists, the
// passes for every shape, the join; gather_bwd_mma.cu: the tensor-core passes).
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace ossa {

// The tensor-core key pass takes blocks of 8 neighbouring keys (one MMA's columns): a turned list then
// holds rows with the block's keys that they list as bits, r | bits << 24.  The other key pass
// takes single keys, its list plain rows r.
constexpr int kKeyBlockShift = 3;
constexpr int kKeyBlock = 1 << kKeyBlockShift;

struct BwdShape {
    int B, H, Hkv, G, Nq, N, D, K, q0, causal;
    int shift, NB;                  // keys per block as a shift, key blocks
    int chunks, chunk_rows, units;  // units = chunks * G per (b, kv head)
    long long cap;                  // entries per (b, kv head) at most
    int tile;                       // entries that a warp of the key pass takes
    long long tiles;                // key-pass tiles per (b, kv head) at most
};

struct BwdBuffers {
    int* keys;          // (B*H*Nq, K) normalised lists: words as list_word makes them, -1 where masked
    int* counts;        // (B*Hkv, units, NB)
    int* base;          // (B*Hkv, NB + 1) start of each key block's run
    int* list;          // (B*Hkv, cap) rows r = g * Nq + il, block by block
    float* delta;       // (B*H*Nq,) sum of p dP
    float* part;        // (B*Hkv, tiles, 2, 2, keys per block, D) sums of runs that a tile's border cuts
    float* slope_rows;  // (B*H*Nq,) or nullptr
};

cudaError_t launch_row_pass_mma(const GatherBwdArgs& a, const BwdShape& s, const BwdBuffers& w, cudaStream_t stream);
cudaError_t launch_key_pass_mma(const GatherBwdArgs& a, const BwdShape& s, const BwdBuffers& w, cudaStream_t stream);

// What a row's sums give: Delta, and its share of -dslope, sum p (dP - Delta) far.  The rounding of the row's
// statistic and of p keeps the sum of p from being 1, so both are divided by it.  xf is sum p (dP - d0) far with d0
// near Delta: as the difference of sum p dP far and Delta sum p far the share lost three quarters of its accuracy.
struct RowSums {
    float delta, slope;
    __device__ __forceinline__ RowSums(float p, float pd, float f, float xf, float d0) {
        const float inv = p == 0.f ? 0.f : 1.f / p;
        delta = pd * inv;
        slope = p == 0.f ? 0.f : ((delta - d0) * f - xf) * inv;  // a row that sees nothing may have any dO
    }
};

// The block whose run holds position pos (base[block] <= pos < base[block + 1]).
__device__ __forceinline__ int block_at(const int* __restrict__ base, int NB, int pos) {
    int lo = 0, hi = NB;  // base[lo] <= pos < base[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(base + mid) <= pos) lo = mid;
        else hi = mid;
    }
    return lo;
}

}  // namespace ossa
