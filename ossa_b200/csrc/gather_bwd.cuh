// What the files of the gathered attention's backward pass share (gather_bwd.cu: the turned lists, the
// passes for every shape, the join; gather_bwd_mma.cu: the tensor-core passes).
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace ossa {

constexpr int kBwdTile = 256;  // entries that a warp of the key pass takes

struct BwdShape {
    int B, H, Hkv, G, Nq, N, D, K, q0, causal;
    int chunks, chunk_rows, units;  // units = chunks * G per (b, kv head)
    long long cap;                  // entries per (b, kv head) at most
    long long tiles;                // key-pass tiles per (b, kv head) at most
};

struct BwdBuffers {
    int* keys;          // (B*H*Nq, K) lists, -1 where masked
    int* counts;        // (B*Hkv, units, N)
    int* base;          // (B*Hkv, N + 1) start of each key's run
    int* list;          // (B*Hkv, cap) rows g * Nq + il, key by key
    float* delta;       // (B*H*Nq,) sum of p dP
    float* part;        // (B*Hkv, tiles, 2, 2, D) sums of runs that a tile's border cuts
    float* slope_rows;  // (B*H*Nq,) or nullptr
};

cudaError_t launch_row_pass_mma(const GatherBwdArgs& a, const BwdShape& s, const BwdBuffers& w, cudaStream_t stream);
cudaError_t launch_key_pass_mma(const GatherBwdArgs& a, const BwdShape& s, const BwdBuffers& w, cudaStream_t stream);

// The key whose run holds position pos (base[key] <= pos < base[key + 1]).
__device__ __forceinline__ int key_at(const int* __restrict__ base, int N, int pos) {
    int lo = 0, hi = N;  // base[lo] <= pos < base[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(base + mid) <= pos) lo = mid;
        else hi = mid;
    }
    return lo;
}

}  // namespace ossa
