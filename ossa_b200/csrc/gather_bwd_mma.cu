// Tensor-core passes of the gathered attention's backward (bf16, D = 128; gather_bwd.cu has the
// mathematics and the other shapes).  mma.sync m16n8k16: the operands are gathered rows that a warp
// stages for itself, 16 at a time, too few and too scattered for a tcgen05 tile.
//
// Measured (B=2, 12/2 heads, N=4096, K=64, half of a row's keys recent: 6.3 M entries): row pass 156 us, of
// which 57 us for the rows' q, dO, output and lists and the union of keys (144 of 384 on average), key pass
// 183 us (3.6 M turned entries); the per-head forms of gather_bwd.cu took 752 and 1147 us here.
// A group of 16 entries of the key pass moves 24 KB through shared memory (8 KB in, 16 KB out as operands): 5.4 GB, 145 us
// at 128 bytes a cycle and SM and 1965 MHz, the nearest bound.  Counted, the shared-memory pipe is busy for 51 % of the
// key pass (67 % of the row pass), the tensor pipe for 26 (15), issue slots for 44 (43): with 12 warps an SM (registers)
// a group's steps, each waiting for the one before, are not covered whole, and blocks of keys differ in their lists.
#include <algorithm>
#include <cstdint>

#include "common.cuh"
#include "gather_bwd.cuh"
#include "kernels.h"
#include "mma_sync.cuh"
#include "query_union.cuh"

namespace ossa {

namespace {

constexpr int D = 128;

struct TanhFast {
    __device__ __forceinline__ float operator()(float x) const { return tanh_fast(x); }
};

__device__ __forceinline__ float dot_bf16x2(uint32_t a, uint32_t b, float c) {
    float a0, a1, b0, b1;
    unpack_bf16x2(a, a0, a1);
    unpack_bf16x2(b, b0, b1);
    return fmaf(a1, b1, fmaf(a0, b0, c));
}

// ------------------------------------------------------------------ row pass
//
// One warp per query and kv head, all heads of the group, over the union of their keys
// (query_union.cuh).  In chunks of 16 keys: S^T = K Q^T and dP^T = V dO^T (keys as MMA rows, heads as
// columns), p, dS and the weights dX per (key, head), then dq^T += K^T dX^T from the same staged key
// rows.  dX enters that product as a bf16 value and its rest (Weights); p, dP, the sums and Delta stay
// fp32.  The rows of chunk c + 1 are in flight while chunk c is computed.  Where the list has no room, or
// the result is not finite (0 times the key row of another head), the heads go one by one, as in the forward.
constexpr int kRowWarps = 6;
constexpr int kRowWarpBytes = 4 * kStageChunk + kUnionCap * 4;  // key and value rows of two chunks; the list
constexpr int kRowBytes = kRowWarps * kRowWarpBytes;
static_assert(kUnionArea <= 4 * kStageChunk, "the list is built in the staging area");
static_assert(2 * (kRowBytes + 1024) <= 233472, "two CTAs per SM");

template <int G, bool kDirect>
__global__ void __launch_bounds__(kRowWarps * 32, 2)
row_pass_mma_kernel(const __nv_bfloat16* __restrict__ q, const __nv_bfloat16* __restrict__ k,
                    const __nv_bfloat16* __restrict__ v, const int* __restrict__ keys,
                    const __nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ dout, const BwdShape s,
                    const ScoreMods mods, __nv_bfloat16* __restrict__ dq, float* __restrict__ delta,
                    float* __restrict__ slope_rows) {
    extern __shared__ __align__(128) uint8_t msm[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int gq = lane >> 2, c4 = lane & 3;
    const int kv = blockIdx.y;
    const int b = kv / s.Hkv, g = kv - b * s.Hkv;
    const int il = blockIdx.x * kRowWarps + warp;
    if (il >= s.Nq) return;  // warp-uniform; no CTA-wide barrier follows
    const int i = s.q0 + il;
    uint8_t* stage = msm + (size_t)warp * kRowWarpBytes;
    uint32_t* list = reinterpret_cast<uint32_t*>(stage + 4 * kStageChunk);
    const __nv_bfloat16* kb = k + (size_t)kv * s.N * D;
    const __nv_bfloat16* vb = v + (size_t)kv * s.N * D;
    const size_t row0 = ((size_t)b * s.H + (size_t)g * G) * s.Nq + il;  // head t: row0 + t * Nq
    const size_t mine = (row0 + (size_t)(gq < G ? gq : 0) * s.Nq) * D;  // head gq's row

    // q and dO rows as B operands of head gq; Delta from the stored output (and its rest)
    uint32_t qa[16], da[16];
    float d0[2];
    {
        const uint32_t* qw = reinterpret_cast<const uint32_t*>(q + mine);
        const uint32_t* dw = reinterpret_cast<const uint32_t*>(dout + mine);
        const uint32_t* ow = reinterpret_cast<const uint32_t*>(out + mine);
        float d = 0.f;
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            qa[t] = gq < G ? __ldg(qw + 4 * t + c4) : 0u;
            da[t] = gq < G ? __ldg(dw + 4 * t + c4) : 0u;
            d = dot_bf16x2(da[t], gq < G ? __ldg(ow + 4 * t + c4) : 0u, d);
        }
        if (mods.rest) {
            const uint32_t* rw = reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(mods.rest) + mine);
#pragma unroll
            for (int t = 0; t < 16; ++t) d = dot_bf16x2(da[t], gq < G ? __ldg(rw + 4 * t + c4) : 0u, d);
        }
        d += __shfl_xor_sync(kFull, d, 1);
        d += __shfl_xor_sync(kFull, d, 2);
        d0[0] = __shfl_sync(kFull, d, 8 * c4);  // heads 2 c4, 2 c4 + 1
        d0[1] = __shfl_sync(kFull, d, 8 * c4 + 4);
    }
    float lse2[2], slope[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int t = 2 * c4 + e;
        lse2[e] = t < G ? mods.lse2[row0 + (size_t)t * s.Nq] : -INFINITY;
        slope[e] = mods.slopes && t < G ? mods.slopes[g * G + t] : 0.f;
    }
    auto key_of = [&](int t, int e) {
        const int w = keys[(row0 + (size_t)t * s.Nq) * s.K + e];
        return w == -1 ? -1 : w & 0xffffff;
    };
    int U;
    {
        int x[G][4];
#pragma unroll
        for (int t = 0; t < G; ++t) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[t][e] = lane + 32 * e < s.K ? key_of(t, lane + 32 * e) : -1;
        }
        U = build_union<G, kDirect>(x, s.K, s.N, stage, list, lane);
    }
    bool single = U < 0;  // the heads one by one
    const uint32_t st = (uint32_t)__cvta_generic_to_shared(stage);
    const StageLane sl(lane);
    auto stage_both = [&](int c) {
        const uint32_t at = st + (uint32_t)((c & 1) * 2 * kStageChunk);
        stage_listed(at, kb, list, c * kStageRows, U, sl, lane);
        stage_listed(at + kStageChunk, vb, list, c * kStageRows, U, sl, lane);
        stage_commit();
    };
#pragma unroll 1
    for (int pass = 0;;) {
        float acc[8][4];  // dq^T: dims 16 mt + gq (+8) of heads 2 c4, 2 c4 + 1
#pragma unroll
        for (int n = 0; n < 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        // sums of p, p dP, p far, p (dP - d0) far
        float a_p[2] = {0.f, 0.f}, a_pd[2] = {0.f, 0.f}, a_f[2] = {0.f, 0.f}, a_xf[2] = {0.f, 0.f};
        __syncwarp();
        if (single) U = single_list([&](int e) { return key_of(pass, e); }, pass, s.K, list, lane);
        __syncwarp();  // the list is complete, the staging area is free
        const int nch = (U + kStageRows - 1) / kStageRows;
        if (nch > 0) stage_both(0);
#pragma unroll 1
        for (int c = 0; c < nch; ++c) {
            const int c0 = c * kStageRows;
            __syncwarp();  // chunk c - 1 is done with its buffers
            if (c + 1 < nch) {
                stage_both(c + 1);
                cp_async_wait_pending<1>();
            } else {
                cp_async_wait_pending<0>();
            }
            __syncwarp();
            const uint32_t kst = st + (uint32_t)((c & 1) * 2 * kStageChunk);  // the value rows a chunk behind
            float sacc[4] = {0.f, 0.f, 0.f, 0.f}, pacc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                uint32_t a[4];
                ldmatrix_x4<0>(a, kst + sl.a[t]);
                mma_bf16_16816_a4(sacc, a[0], a[1], a[2], a[3], qa[2 * t], qa[2 * t + 1]);
                ldmatrix_x4<kStageChunk>(a, kst + sl.a[t]);
                mma_bf16_16816_a4(pacc, a[0], a[1], a[2], a[3], da[2 * t], da[2 * t + 1]);
                ldmatrix_x4<128>(a, kst + sl.a[t]);
                mma_bf16_16816_a4(sacc, a[0], a[1], a[2], a[3], qa[2 * t + 8], qa[2 * t + 9]);
                ldmatrix_x4<kStageChunk + 128>(a, kst + sl.a[t]);
                mma_bf16_16816_a4(pacc, a[0], a[1], a[2], a[3], da[2 * t + 8], da[2 * t + 9]);
            }
            // keys c0 + gq, c0 + gq + 8 x heads 2 c4, 2 c4 + 1
            float w[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = c0 + gq + 8 * h;
                const uint32_t entry = at < U ? list[at] : 0u;
                const float far = fabsf((float)(i - (int)(entry & 0xffffffu)));
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    // selects, no branch: what a masked place computes may not be finite and is dropped
                    const bool on = ((entry >> (24 + 2 * c4 + e)) & 1u) && lse2[e] != -INFINITY;
                    float dx;
                    const float x = mods.log2_p(sacc[2 * h + e], slope[e], far, lse2[e], dx, TanhFast());
                    const float p = on ? exp2_fast(x) : 0.f;
                    const float pd = on ? p * pacc[2 * h + e] : 0.f;
                    const float ds = on ? pd - p * d0[e] : 0.f;
                    w[h][e] = on ? dx * ds : 0.f;
                    a_p[e] += p;
                    a_pd[e] += pd;
                    a_f[e] = fmaf(p, far, a_f[e]);
                    a_xf[e] = fmaf(ds, far, a_xf[e]);
                }
            }
            const Weights wt(w);
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                uint32_t a[4];
                ldmatrix_x4_trans<0>(a, kst + sl.at[mt]);
                wt.mma(acc[mt], a);
                ldmatrix_x4_trans<128>(a, kst + sl.at[mt]);
                wt.mma(acc[mt + 4], a);
            }
        }
        if (G > 1 && !single) {
            float bad = 0.f;  // 0 while every sum is finite
#pragma unroll
            for (int n = 0; n < 8; ++n) {
#pragma unroll
                for (int x = 0; x < 4; ++x) bad = fmaf(acc[n][x], 0.f, bad);
            }
            if (__any_sync(kFull, bad != 0.f)) {
                single = true;
                continue;
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) {
                a_p[e] += __shfl_xor_sync(kFull, a_p[e], o);
                a_pd[e] += __shfl_xor_sync(kFull, a_pd[e], o);
                a_f[e] += __shfl_xor_sync(kFull, a_f[e], o);
                a_xf[e] += __shfl_xor_sync(kFull, a_xf[e], o);
            }
            const int t = 2 * c4 + e;
            if (gq == 0 && (single ? t == pass : t < G)) {
                const size_t row = row0 + (size_t)t * s.Nq;
                const RowSums sums(a_p[e], a_pd[e], a_f[e], a_xf[e], d0[e]);
                delta[row] = sums.delta;
                if (slope_rows) slope_rows[row] = sums.slope;
            }
        }
        __nv_bfloat16* orow = dq + mine + 2 * c4;
        const bool own = single ? gq == pass : gq < G;
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
            const uint32_t lo = movmatrix_trans(pack_bf16x2(acc[mt][0], acc[mt][1]));
            const uint32_t hi = movmatrix_trans(pack_bf16x2(acc[mt][2], acc[mt][3]));
            if (own) {
                *reinterpret_cast<uint32_t*>(orow + 16 * mt) = lo;
                *reinterpret_cast<uint32_t*>(orow + 16 * mt + 8) = hi;
            }
        }
        if (!single || ++pass == G) break;
    }
}

// ------------------------------------------------------------------ key pass
//
// One warp per `tile` entries of a turned list (rows with the keys of one block of 8 that they list),
// in groups of 16 entries whose q and dO rows are staged while the group before is computed.  For
// the part of a group that lies in one block's run: S = Q K^T and dP = dO V^T (entries as MMA rows,
// the block's keys as columns), p and dX per (entry, key) where the mask has the key's bit, then
// dv^T += dO^T P and dk^T += Q^T dX from the same rows, P and dX as bf16 values and their rests (Weights),
// the sums fp32.  A group with a row that is not finite (its products with every key of the block are not)
// is summed entry by entry instead: 0 times such a row must be 0 for the keys that it does not list.
constexpr int kKeyWarps = 4;
constexpr int kKeyWarpBytes = 4 * kStageChunk;  // q and dO rows of two groups
constexpr int kKeyBytes = kKeyWarps * kKeyWarpBytes;
static_assert(3 * (kKeyBytes + 1024) <= 233472, "three CTAs per SM");

// A block's key or value rows as the B operand: column gq is row gq (zeros past the last key).
__device__ __forceinline__ void load_block(const __nv_bfloat16* rows, bool in, int gq, int c4, uint32_t (&r)[16]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(rows + (in ? gq : 0) * D);
#pragma unroll
    for (int t = 0; t < 16; ++t) r[t] = in ? __ldg(w + 4 * t + c4) : 0u;
}

__global__ void __launch_bounds__(kKeyWarps * 32, 3)
key_pass_mma_kernel(const __nv_bfloat16* __restrict__ q, const __nv_bfloat16* __restrict__ k,
                    const __nv_bfloat16* __restrict__ v, const __nv_bfloat16* __restrict__ dout, const BwdShape s,
                    const ScoreMods mods, const int* __restrict__ base, const int* __restrict__ list,
                    const float* __restrict__ delta, __nv_bfloat16* __restrict__ dk, __nv_bfloat16* __restrict__ dv,
                    float* __restrict__ part) {
    extern __shared__ __align__(128) uint8_t msm[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int gq = lane >> 2, c4 = lane & 3, kv = blockIdx.y;
    const long long tile = (long long)blockIdx.x * kKeyWarps + warp;
    const int* bs = base + (size_t)kv * (s.NB + 1);
    const int total = bs[s.NB];
    if (tile * s.tile >= total) return;  // warp-uniform; no CTA-wide barrier follows
    const int t0 = (int)(tile * s.tile), t1 = min(total, t0 + s.tile);
    const int b = kv / s.Hkv, h0 = (kv - b * s.Hkv) * s.G;
    const size_t rows0 = ((size_t)b * s.H + h0) * s.Nq;  // row of list entry r: rows0 + r
    const uint32_t* ls = reinterpret_cast<const uint32_t*>(list) + (size_t)kv * s.cap;
    const char* qb = reinterpret_cast<const char*>(q + rows0 * D) + (lane & 15) * 16;
    const char* db = reinterpret_cast<const char*>(dout + rows0 * D) + (lane & 15) * 16;
    const uint32_t st = (uint32_t)__cvta_generic_to_shared(msm + (size_t)warp * kKeyWarpBytes);
    const StageLane sl(lane);

    // entry lane & 15 of the group at pos; past the tile its last entry again (and given no weight)
    auto entry = [&](int pos) { return ls[min(pos + (lane & 15), t1 - 1)]; };
    auto stage_rows = [&](uint32_t r, int buf) {
        const uint32_t at = st + (uint32_t)(buf * 2 * kStageChunk);
#pragma unroll
        for (int t = 0; t < kStageRows / 2; ++t) {
            const uint32_t row = __shfl_sync(kFull, r, 2 * t + (lane >> 4)) & 0xffffffu;
            const void *qs = qb + (size_t)row * kStageRow, *ds = db + (size_t)row * kStageRow;
            if (t < 4) {
                stage_copy<0>(at + sl.w[t & 3], qs);
                stage_copy<kStageChunk>(at + sl.w[t & 3], ds);
            } else {
                stage_copy<2048>(at + sl.w[t & 3], qs);
                stage_copy<kStageChunk + 2048>(at + sl.w[t & 3], ds);
            }
        }
        stage_commit();
    };
    float ak[8][4], av[8][4];  // dims 16 mt + gq (+8) of the block's keys 2 c4, 2 c4 + 1
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        ak[n][0] = ak[n][1] = ak[n][2] = ak[n][3] = 0.f;
        av[n][0] = av[n][1] = av[n][2] = av[n][3] = 0.f;
    }
    int blk = block_at(bs, s.NB, t0);
    int run0 = bs[blk], run1 = bs[blk + 1];
    uint32_t kf[16], vf[16];
    auto load_keys = [&] {
        const size_t at = ((size_t)kv * s.N + (size_t)blk * kKeyBlock) * D;
        const bool in = blk * kKeyBlock + gq < s.N;
        load_block(k + at, in, gq, c4, kf);
        load_block(v + at, in, gq, c4, vf);
    };
    load_keys();
    uint32_t r = entry(t0), r_next = entry(t0 + kStageRows);
    stage_rows(r, 0);
#pragma unroll 1
    for (int pos = t0, buf = 0; pos < t1; pos += kStageRows, buf ^= 1) {
        const uint32_t r_after = entry(pos + 2 * kStageRows);
        // this lane's entry: statistic, Delta, position and slope
        const uint32_t row = r & 0xffffffu;
        const float lse2 = mods.lse2[rows0 + row], dl = delta[rows0 + row];
        float slope = 0.f;
        int i = 0;
        if (mods.slopes) {
            const int g = (int)row / s.Nq;
            i = s.q0 + (int)row - g * s.Nq;
            slope = mods.slopes[h0 + g];
        }
        __syncwarp();  // the group before is done with its buffer
        if (pos + kStageRows < t1) {
            stage_rows(r_next, buf ^ 1);
            cp_async_wait_pending<1>();
        } else {
            cp_async_wait_pending<0>();
        }
        __syncwarp();
        const uint32_t qst = st + (uint32_t)(buf * 2 * kStageChunk);  // the dO rows a chunk behind
        const int end = min(pos + kStageRows, t1);
#pragma unroll 1
        for (int p0 = pos; p0 < end;) {
            const int p1 = min(end, run1);  // entries p0 .. p1 - 1 are of this block
            float sacc[4] = {0.f, 0.f, 0.f, 0.f}, pacc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                uint32_t a[4];
                ldmatrix_x4<0>(a, qst + sl.a[t]);
                mma_bf16_16816_a4(sacc, a[0], a[1], a[2], a[3], kf[2 * t], kf[2 * t + 1]);
                ldmatrix_x4<kStageChunk>(a, qst + sl.a[t]);
                mma_bf16_16816_a4(pacc, a[0], a[1], a[2], a[3], vf[2 * t], vf[2 * t + 1]);
                ldmatrix_x4<128>(a, qst + sl.a[t]);
                mma_bf16_16816_a4(sacc, a[0], a[1], a[2], a[3], kf[2 * t + 8], kf[2 * t + 9]);
                ldmatrix_x4<kStageChunk + 128>(a, qst + sl.a[t]);
                mma_bf16_16816_a4(pacc, a[0], a[1], a[2], a[3], vf[2 * t + 8], vf[2 * t + 9]);
            }
            float p[2][2], w[2][2];
            unsigned stray = 0u;  // entries (bit 4 e) whose products with every key of the block are not finite
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // entry gq + 8 h x keys 2 c4, 2 c4 + 1
                const int e = gq + 8 * h;
                const float l = __shfl_sync(kFull, lse2, e), d = __shfl_sync(kFull, dl, e);
                uint32_t mask = __shfl_sync(kFull, r, e) >> 24;
                if (pos + e < p0 || pos + e >= p1 || l == -INFINITY) mask = 0u;
                float sp = 0.f;
                int ie = 0;
                if (mods.slopes) {  // warp-uniform
                    sp = __shfl_sync(kFull, slope, e);
                    ie = __shfl_sync(kFull, i, e) - blk * kKeyBlock;
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float dx;
                    const float y = mods.log2_p(sacc[2 * h + x], sp, fabsf((float)(ie - 2 * c4 - x)), l, dx, TanhFast());
                    const bool on = (mask >> (2 * c4 + x)) & 1u;
                    p[h][x] = on ? exp2_fast(y) : 0.f;
                    w[h][x] = on ? dx * p[h][x] * (pacc[2 * h + x] - d) : 0.f;
                }
                const float both = fminf(fabsf(sacc[2 * h] + pacc[2 * h]), fabsf(sacc[2 * h + 1] + pacc[2 * h + 1]));
                const unsigned b4 = __ballot_sync(kFull, !(both < INFINITY));
                stray |= b4 & b4 >> 1 & b4 >> 2 & b4 >> 3 & 0x11111111u;
            }
            if (stray == 0u) {  // warp-uniform
                const Weights pt(p), wt(w);
#pragma unroll
                for (int mt = 0; mt < 4; ++mt) {
                    uint32_t a[4];
                    ldmatrix_x4_trans<kStageChunk>(a, qst + sl.at[mt]);
                    pt.mma(av[mt], a);
                    ldmatrix_x4_trans<0>(a, qst + sl.at[mt]);
                    wt.mma(ak[mt], a);
                    ldmatrix_x4_trans<kStageChunk + 128>(a, qst + sl.at[mt]);
                    pt.mma(av[mt + 4], a);
                    ldmatrix_x4_trans<128>(a, qst + sl.at[mt]);
                    wt.mma(ak[mt + 4], a);
                }
            } else {
                const uint8_t* rows = msm + (size_t)warp * kKeyWarpBytes + buf * 2 * kStageChunk;
#pragma unroll 1
                for (int e = 0; e < kStageRows; ++e) {
                    const float l = __shfl_sync(kFull, lse2, e);
                    uint32_t mask = __shfl_sync(kFull, r, e) >> 24;
                    if (pos + e < p0 || pos + e >= p1 || l == -INFINITY) mask = 0u;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int from = (e & 7) * 4 + c4;  // the lane with this entry's weights
                        const float pe = __shfl_sync(kFull, e < 8 ? p[0][x] : p[1][x], from);
                        const float we = __shfl_sync(kFull, e < 8 ? w[0][x] : w[1][x], from);
                        if (!((mask >> (2 * c4 + x)) & 1u)) continue;
#pragma unroll
                        for (int n = 0; n < 16; ++n) {  // dim 8 n + gq
                            const __nv_bfloat16* at = reinterpret_cast<const __nv_bfloat16*>(
                                rows + e * kStageRow + ((n ^ (e & 7)) << 4)) + gq;
                            float& k_sum = ak[n >> 1][2 * (n & 1) + x];
                            float& v_sum = av[n >> 1][2 * (n & 1) + x];
                            k_sum = fmaf(we, to_f32(at[0]), k_sum);
                            v_sum = fmaf(pe, to_f32(at[kStageChunk / 2]), v_sum);
                        }
                    }
                }
            }
            p0 = p1;
            if (p1 < run1 && p1 < t1) continue;  // the run goes on in the next group
            // the run, or the tile, ends here
            if (run0 >= t0 && run1 <= t1) {
                const bool in = blk * kKeyBlock + gq < s.N;  // after the transpose lane (gq, c4) holds key gq
                const size_t at = ((size_t)kv * s.N + (size_t)blk * kKeyBlock + gq) * D + 2 * c4;
#pragma unroll
                for (int mt = 0; mt < 8; ++mt) {
                    const uint32_t k0 = movmatrix_trans(pack_bf16x2(ak[mt][0], ak[mt][1]));
                    const uint32_t k1 = movmatrix_trans(pack_bf16x2(ak[mt][2], ak[mt][3]));
                    const uint32_t v0 = movmatrix_trans(pack_bf16x2(av[mt][0], av[mt][1]));
                    const uint32_t v1 = movmatrix_trans(pack_bf16x2(av[mt][2], av[mt][3]));
                    if (in) {
                        *reinterpret_cast<uint32_t*>(dk + at + 16 * mt) = k0;
                        *reinterpret_cast<uint32_t*>(dk + at + 16 * mt + 8) = k1;
                        *reinterpret_cast<uint32_t*>(dv + at + 16 * mt) = v0;
                        *reinterpret_cast<uint32_t*>(dv + at + 16 * mt + 8) = v1;
                    }
                }
            } else {  // slot 0: the run began before this tile; slot 1: it begins here and goes on
                float* ps = part + (((size_t)kv * s.tiles + tile) * 2 + (run0 < t0 ? 0 : 1)) * 2 * kKeyBlock * D +
                            2 * c4 * D + gq;
#pragma unroll
                for (int mt = 0; mt < 8; ++mt) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int at = (x & 1) * D + 16 * mt + (x >> 1) * 8;
                        ps[at] = ak[mt][x];
                        ps[kKeyBlock * D + at] = av[mt][x];
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                ak[n][0] = ak[n][1] = ak[n][2] = ak[n][3] = 0.f;
                av[n][0] = av[n][1] = av[n][2] = av[n][3] = 0.f;
            }
            if (p1 < t1) {  // on to the next listed block
                do {
                    ++blk;
                    run0 = run1;
                    run1 = bs[blk + 1];
                } while (run1 <= p1);
                load_keys();
            }
        }
        r = r_next;
        r_next = r_after;
    }
}

}  // namespace

cudaError_t launch_row_pass_mma(const GatherBwdArgs& a, const BwdShape& s, const BwdBuffers& w, cudaStream_t stream) {
    const bool direct = s.N <= kUnionDirectKeys;
#define OSSA_ROW_PICK(GG) (direct ? row_pass_mma_kernel<GG, true> : row_pass_mma_kernel<GG, false>)
    auto kern = s.G == 1 ? OSSA_ROW_PICK(1)
              : s.G == 2 ? OSSA_ROW_PICK(2)
              : s.G == 3 ? OSSA_ROW_PICK(3)
              : s.G == 4 ? OSSA_ROW_PICK(4)
              : s.G == 5 ? OSSA_ROW_PICK(5)
              : s.G == 6 ? OSSA_ROW_PICK(6)
              : s.G == 7 ? OSSA_ROW_PICK(7)
                         : OSSA_ROW_PICK(8);
#undef OSSA_ROW_PICK
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowBytes);
    if (e != cudaSuccess) return e;
    using T = __nv_bfloat16;
    kern<<<dim3((s.Nq + kRowWarps - 1) / kRowWarps, s.B * s.Hkv), kRowWarps * 32, kRowBytes, stream>>>(
        static_cast<const T*>(a.f.q), static_cast<const T*>(a.f.k), static_cast<const T*>(a.f.v), w.keys,
        static_cast<const T*>(a.f.out), static_cast<const T*>(a.dout), s, a.f.mods, static_cast<T*>(a.dq), w.delta,
        w.slope_rows);
    e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e;
}

cudaError_t launch_key_pass_mma(const GatherBwdArgs& a, const BwdShape& s, const BwdBuffers& w, cudaStream_t stream) {
    cudaError_t e =
        cudaFuncSetAttribute(key_pass_mma_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kKeyBytes);
    if (e != cudaSuccess) return e;
    using T = __nv_bfloat16;
    key_pass_mma_kernel<<<dim3((unsigned)((s.tiles + kKeyWarps - 1) / kKeyWarps), (unsigned)(s.B * s.Hkv)),
                          kKeyWarps * 32, kKeyBytes, stream>>>(
        static_cast<const T*>(a.f.q), static_cast<const T*>(a.f.k), static_cast<const T*>(a.f.v),
        static_cast<const T*>(a.dout), s, a.f.mods, w.base, w.list, w.delta, static_cast<T*>(a.dk),
        static_cast<T*>(a.dv), w.part);
    e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e;
}

}  // namespace ossa
