// Modifiers of the gathered attention's scores, shared by its forward and backward kernels.
//
// With x = (q_i . k_j) * scale the score in base 2 is
//   s2 = (cap tanh(x / cap) - slope_h |i - j|) * log2(e)     (no cap: x itself)
// and key j is seen by the query at position i of batch element b when
//   (not causal, or j <= i, or j < prefix_len[b])  and  segments[b][j] == segments[b][i].
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace ossa {

constexpr float kLog2E = 1.4426950408889634f;

struct TanhExact {
    __device__ __forceinline__ float operator()(float x) const { return tanhf(x); }
};

// What one query row needs of the modifiers (kMods = false: nothing but the causal rule).
template <bool kMods>
struct RowMods {
    __device__ __forceinline__ RowMods(const ScoreMods&, int, int, int, int) {}
    __device__ __forceinline__ bool sees(long long j, int i, int causal) const { return !causal || j <= i; }
    __device__ __forceinline__ float score2(float x, int, int) const { return x; }
};

template <>
struct RowMods<true> {
    const int* seg;  // of batch element b, nullptr: one document
    int seg_i, prefix;
    float slope;
    const ScoreMods& m;
    __device__ __forceinline__ RowMods(const ScoreMods& mods, int b, int h, int N, int i) : m(mods) {
        seg = mods.segments ? mods.segments + (size_t)b * N : nullptr;
        seg_i = seg ? __ldg(seg + i) : 0;
        prefix = mods.prefix_len ? __ldg(mods.prefix_len + b) : 0;
        slope = mods.slopes ? __ldg(mods.slopes + h) : 0.f;
    }
    // j in [0, N)
    __device__ __forceinline__ bool sees(long long j, int i, int causal) const {
        return (!causal || j <= i || j < prefix) && (!seg || __ldg(seg + j) == seg_i);
    }
    // x[t][e] = -1 for the keys in [0, N) that the row does not see; entries with 32 e >= K are -1.
    template <int G>
    __device__ __forceinline__ void hide(int (&x)[G][4], int K, int i, int causal) const {
        const int last = causal ? max(i, max(prefix, 0) - 1) : 0x7fffffff;  // j <= i or j < prefix
#pragma unroll
        for (int t = 0; t < G; ++t) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[t][e] = x[t][e] > last ? -1 : x[t][e];
        }
        if (!seg) return;  // the same for the whole grid
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (32 * e >= K) continue;  // warp-uniform
            int of[G];
#pragma unroll
            for (int t = 0; t < G; ++t) of[t] = __ldg(seg + max(x[t][e], 0));
#pragma unroll
            for (int t = 0; t < G; ++t) x[t][e] = of[t] == seg_i ? x[t][e] : -1;
        }
    }
    __device__ __forceinline__ float score2(float dot, int i, int j) const {
        return m.score2(dot, slope, fabsf((float)(i - j)), TanhExact());
    }
};

}  // namespace ossa
