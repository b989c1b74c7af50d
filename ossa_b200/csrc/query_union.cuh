// The keys that the heads of one kv head list for one query, each key once with its heads, and their
// staging in shared memory: what the tensor-core forms of the modified gather and of its backward
// row pass share (bf16, D = 128, G query heads per kv head, at most 128 listed keys per head).
//
// A warp owns a query.  Keys come as x[t][e], entry lane + 32 e of head t, -1 where the entry is
// masked.  The list holds key | heads << 24.  It is made in the order (head, entry) of the lowest head
// that lists a key, so it does not depend on the order in which lanes run.
#pragma once

#include "common.cuh"

namespace ossa {

constexpr int kUnionCap = 512;           // keys a list holds
constexpr int kUnionDirectKeys = 12288;  // keys covered by the direct form, a byte of head bits per key
constexpr int kUnionSlots = 1024;        // hash slots otherwise; at least G * K, so every key finds one
constexpr int kUnionArea = 12288;        // bytes of shared memory the build needs besides the list
constexpr int kUnionMaxKeys = 1 << 24;   // the list's key field
static_assert(kUnionDirectKeys <= kUnionArea && 5 * kUnionSlots <= kUnionArea, "the head bits fit");

// Returns the list's length, or -1 when a head lists a key twice or the list would not fit: the
// caller then takes the heads one by one (single_list).
//
// The heads set their bits one after another, so a plain read and write of a key's byte does: the lanes of
// one head differ in their keys, or write the same.  A key that one head lists twice shows in its own bit, or
// among the 32 entries taken together: these differ if they ascend without a gap, as the selectors leave
// them, and are compared with one another otherwise.
template <int G, bool kDirect>
__device__ __forceinline__ int build_union(const int (&x)[G][4], int K, int N, uint8_t* area, uint32_t* list, int lane) {
    const unsigned lt = lanemask_lt();
    uint8_t* bits = area;                                  // direct: of key j; hash: of a slot
    int* skey = reinterpret_cast<int*>(area + kUnionSlots);  // hash: the slot's key
    if constexpr (kDirect) {
        for (int w = lane; w < (N + 15) >> 4; w += 32) reinterpret_cast<uint4*>(bits)[w] = make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
        for (int u = 0; u < kUnionSlots / 512; ++u) reinterpret_cast<uint4*>(bits)[lane + 32 * u] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int u = 0; u < kUnionSlots / 128; ++u) reinterpret_cast<int4*>(skey)[lane + 32 * u] = make_int4(-1, -1, -1, -1);
    }
    __syncwarp();
    int U = 0;
    bool twice = false;
#pragma unroll
    for (int t = 0; t < G; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (32 * e >= K) continue;  // warp-uniform
            const int xv = x[t][e];
            int at = xv;
            if constexpr (!kDirect) {
                if (xv >= 0) {
                    at = (int)(((uint32_t)xv * 2654435761u) >> 22);  // 10 bits
                    for (int probe = 0; probe < kUnionSlots; ++probe) {
                        int cur = *reinterpret_cast<volatile int*>(skey + at);
                        if (cur == -1) cur = atomicCAS(skey + at, -1, xv);
                        if (cur == -1 || cur == xv) break;
                        at = (at + 1) & (kUnionSlots - 1);
                    }
                }
                __syncwarp();
            }
            const int before = __shfl_up_sync(kFull, xv, 1);
            const unsigned valid = __ballot_sync(kFull, xv >= 0);
            const unsigned after = __ballot_sync(kFull, xv >= 0 && lane > 0 && before >= 0 && before < xv);
            if (__popc(valid & ~after) > 1) {  // warp-uniform
                const unsigned same = __match_any_sync(kFull, xv >= 0 ? xv : -1 - lane);
                twice = twice || same != 1u << lane;
            }
            const unsigned old = xv >= 0 ? bits[at] : 1u;
            twice = twice || (xv >= 0 && ((old >> t) & 1u) != 0u);
            __syncwarp();
            if (xv >= 0) bits[at] = (uint8_t)(old | 1u << t);
            const unsigned own = __ballot_sync(kFull, old == 0u);  // no head before lists it
            const int pos = U + __popc(own & lt);
            // the list holds the place of the head bits until they are complete
            if (old == 0u && pos < kUnionCap) list[pos] = (uint32_t)at;
            U += __popc(own);
            __syncwarp();
        }
    }
    if (__any_sync(kFull, twice) || U > kUnionCap) return -1;
    for (int u = lane; u < U; u += 32) {
        const uint32_t at = list[u];
        list[u] = (kDirect ? at : (uint32_t)skey[at]) | (uint32_t)bits[at] << 24;
    }
    return U;
}

// One head's keys as a list of their own, in the order listed (key(e): entry e of the head, -1 masked).
template <typename Key>
__device__ __forceinline__ int single_list(Key key, int t, int K, uint32_t* list, int lane) {
    const unsigned lt = lanemask_lt();
    int U = 0;
    for (int e0 = 0; e0 < K; e0 += 32) {
        const int xv = e0 + lane < K ? key(e0 + lane) : -1;
        const unsigned bal = __ballot_sync(kFull, xv >= 0);
        if (xv >= 0) list[U + __popc(bal & lt)] = (uint32_t)xv | (1u << t) << 24;
        U += __popc(bal);
    }
    return U;
}

// Chunks of 16 rows of 128 bf16 values in shared memory, 16-byte pieces XOR-swizzled by the row: piece c
// of row r lies at r * 256 + ((c ^ (r & 7)) << 4).  The pieces c and c + 8 of a row are 128 bytes apart,
// rows r and r + 8 2048, so four offsets per lane and compile-time distances reach every access.
constexpr int kStageRow = 256;
constexpr int kStageRows = 16;
constexpr int kStageChunk = kStageRows * kStageRow;

// This lane's places in a chunk.
struct StageLane {
    uint32_t a[4];   // ldmatrix, rows as they lie: k-step t reads a[t & 3] + 128 * (t >> 2)
    uint32_t at[4];  // ldmatrix.trans: 16-column step t likewise
    uint32_t w[4];   // copy of piece lane & 15 of rows 2 t + lane / 16: w[t & 3] + 2048 * (t >> 2)
    __device__ __forceinline__ explicit StageLane(int lane) {
        const int ar = (lane & 7) + ((lane >> 3) & 1) * 8, ac = lane >> 4;
        const int tr = (lane & 7) + (lane >> 4) * 8, tc = (lane >> 3) & 1;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            a[t] = (uint32_t)(ar * kStageRow + (((2 * t + ac) ^ (ar & 7)) << 4));
            at[t] = (uint32_t)(tr * kStageRow + (((2 * t + tc) ^ (tr & 7)) << 4));
            const int wr = 2 * t + (lane >> 4);
            w[t] = (uint32_t)(wr * kStageRow + (((lane & 15) ^ (wr & 7)) << 4));
        }
    }
};

template <int kOff>
__device__ __forceinline__ void stage_copy(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0 + %2], [%1], 16;" ::"r"(dst), "l"(src), "n"(kOff) : "memory");
}

__device__ __forceinline__ void stage_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// Copies the rows of list entries c0 .. c0 + 15 of one tensor; past the list's end its last row again
// (finite where the list's rows are, and given no weight).
__device__ __forceinline__ void stage_listed(uint32_t dst, const __nv_bfloat16* base, const uint32_t* list, int c0, int U,
                                             const StageLane& sl, int lane) {
    const char* col = reinterpret_cast<const char*>(base) + (lane & 15) * 16;
#pragma unroll
    for (int t = 0; t < kStageRows / 2; ++t) {
        const uint32_t key = list[min(c0 + 2 * t + (lane >> 4), U - 1)] & 0xffffffu;
        const void* src = col + (size_t)key * kStageRow;
        if (t < 4) stage_copy<0>(dst + sl.w[t & 3], src);
        else stage_copy<2048>(dst + sl.w[t & 3], src);
    }
}

// 2^x and tanh for the tensor-core forms.  ex2.approx: two units in the last place.  tanh x = 1 - 2 / (1 + e^2x)
// is good to 2^-22 in absolute terms, which a score of size cap turns into cap * 2^-22; below 1, where most
// scores of a cap lie, x times a polynomial in x^2 (least maximal relative error there, 2^-22.6) takes its place.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float tanh_fast(float x) {
    const float u = x * x;
    float p = fmaf(0.0010410227114334702f, u, -0.0062033794820308685f);
    p = fmaf(p, u, 0.020289981737732887f);
    p = fmaf(p, u, -0.05345702916383743f);
    p = fmaf(p, u, 0.13325203955173492f);
    p = fmaf(p, u, -0.33332839608192444f);
    p = fmaf(p, u, 0.9999999403953552f);
    return u < 1.f ? p * x : 1.f - __fdividef(2.f, 1.f + exp2_fast(x * 2.885390081777927f));
}

}  // namespace ossa
