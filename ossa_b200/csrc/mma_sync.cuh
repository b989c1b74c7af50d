// Warp-level tensor-core and shuffle helpers of the gather kernels (forward and backward).
#pragma once

#include "common.cuh"

namespace ossa {

// Sums part[0..31] across the warp so that lane m ends with the total of part[m].
__device__ __forceinline__ float transpose_reduce32(float (&part)[32], int lane) {
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) {
        const bool upper = (lane & w) != 0;
#pragma unroll
        for (int t = 0; t < w; ++t) {
            const float a = part[t], b = part[t + w];
            const float send = upper ? a : b;
            const float keep = upper ? b : a;
            part[t] = keep + __shfl_xor_sync(kFull, send, w);
        }
    }
    return part[0];
}

// Whether some lane's score is NaN.  A maximum passes over NaN, so scores whose maximum is -inf may hold it beside
// masked ones: taken against 0 then, they make the row's sum and output NaN.
__device__ __forceinline__ bool shows_nan(float s) { return __any_sync(kFull, s != s); }

// mma.sync m16n8k16 with all four A registers (rows 0..15).
__device__ __forceinline__ void mma_bf16_16816_a4(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                  uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transpose of an 8 x 8 bf16 matrix held one 32-bit pair per lane (lane 4 r + c holds
// row r, columns 2 c, 2 c + 1; afterwards the same for the transpose).
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// What rounding x to bf16 leaves of it.
__device__ __forceinline__ float bf16_rest(float x) { return x - __bfloat162float(__float2bfloat16_rn(x)); }

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <int kPending>
__device__ __forceinline__ void cp_async_wait_pending() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// ldmatrix of the address plus a compile-time offset (no address arithmetic per load).
template <int kOff>
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr), "n"(kOff));
}

template <int kOff>
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr), "n"(kOff));
}

// Weights as MMA operands: their bf16 value and what that rounding left (2^-17 of the weight stays), each
// 8 x 8 half of a (rows x columns) tile transposed across the warp.
struct Weights {
    uint32_t hi[2], lo[2];
    __device__ __forceinline__ explicit Weights(const float (&w)[2][2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t top = pack_bf16x2(w[h][0], w[h][1]);
            float t0, t1;
            unpack_bf16x2(top, t0, t1);
            hi[h] = movmatrix_trans(top);
            lo[h] = movmatrix_trans(pack_bf16x2(w[h][0] - t0, w[h][1] - t1));
        }
    }
    // acc += A W
    __device__ __forceinline__ void mma(float (&acc)[4], const uint32_t (&a)[4]) const {
        mma_bf16_16816_a4(acc, a[0], a[1], a[2], a[3], hi[0], hi[1]);
        mma_bf16_16816_a4(acc, a[0], a[1], a[2], a[3], lo[0], lo[1]);
    }
};

}  // namespace ossa
