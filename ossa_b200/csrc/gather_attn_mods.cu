// Gathered top-K attention forward with score modifiers (score_mods.cuh), and the row statistic
// that its backward pass reads.  Also the training form of the unmodified gather.
//
// bf16 rows of head_dim 128: few of them take a CTA per row and head (mod_attn_few_kernel); with 2-8
// query heads per kv head and at most 128 listed keys more of them take the tensor-core form; everything
// else takes the per-head forms of gather_attn_kernels.cuh.
//
// Tensor-core form: one warp per query and kv head, all G heads of the group at once (query_union.cuh): every key
// that some head lists is fetched once.  In chunks of 16 keys: S^T = K Q^T with the keys as MMA
// rows and the heads as columns, scores and masks per (key, head), online softmax per head, then
// O^T += V^T P^T with P^T moved into operand layout by movmatrix.  The key rows of chunk c + 1 are in
// flight while chunk c is scored, its value rows while its softmax runs.  p enters the product with the
// bf16 values as a bf16 value and its rest (Weights); sums and statistics are fp32.
// A query with a key listed twice by one head, or with more than 512 different keys, takes its heads
// one after another through the same loop.  So does one whose result is not finite: a key that only some of
// the heads list has no weight for the others, and 0 times its value row must be 0 there.
//
// Bound: shared-memory traffic and issue (16 KB a chunk of 16 keys, 12 KB of it operands): the pipes are busy for 61 % and
// 52 % of the time, the rest is waits between a chunk's steps.  Measured: packed
// prefill B=2, 12/2 heads, N=4096, K=64, slopes: 111 us, 39 us of it for the lists, documents and the union of
// keys (144 of 384 on average, 1.2 GB of key and value rows from L2); N=8192, K=128, B=1: 230 us.
#include "gather_attn_kernels.cuh"
#include <algorithm>
#include "query_union.cuh"

namespace ossa {

namespace {

struct TanhFast {
    __device__ __forceinline__ float operator()(float x) const { return tanh_fast(x); }
};

constexpr int kModWarps = 8;
constexpr float kSlack = 8.f;  // p stays below 2^8 (its rounding is relative) and above what 2^-126 cuts off
constexpr int kModWarpBytes = 3 * kStageChunk + kUnionCap * 4;  // key rows of two chunks, value rows of one; the list
constexpr int kModBytes = kModWarps * kModWarpBytes;
static_assert(kUnionArea <= 3 * kStageChunk, "the list is built in the staging area");
static_assert(2 * (kModBytes + 1024) <= 233472, "two CTAs per SM");

template <typename IdxT, int G, bool kDirect>
__global__ void __launch_bounds__(kModWarps * 32, 2)
mod_attn_mma_kernel(const __nv_bfloat16* __restrict__ q, const __nv_bfloat16* __restrict__ k,
                    const __nv_bfloat16* __restrict__ v, const IdxT* __restrict__ idx, __nv_bfloat16* __restrict__ out,
                    int H, int Hkv, int N, int Nq, int q0, int K, int causal, const ScoreMods mods) {
    constexpr int D = 128;
    extern __shared__ __align__(128) uint8_t msm[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int gq = lane >> 2, c4 = lane & 3;
    const int bg = blockIdx.y;
    const int b = bg / Hkv, g = bg - b * Hkv;
    const int il = blockIdx.x * kModWarps + warp;
    if (il >= Nq) return;  // warp-uniform; no CTA-wide barrier follows
    const int i = q0 + il;
    uint8_t* stage = msm + (size_t)warp * kModWarpBytes;
    uint32_t* list = reinterpret_cast<uint32_t*>(stage + 3 * kStageChunk);
    const __nv_bfloat16* kb = k + (size_t)bg * N * D;
    const __nv_bfloat16* vb = v + (size_t)bg * N * D;
    const size_t row0 = ((size_t)b * H + (size_t)g * G) * Nq + il;  // head t: row0 + t * Nq

    uint32_t qa[16];  // q rows as the MMA's B operand: head gq
    {
        const uint32_t* qw = reinterpret_cast<const uint32_t*>(q + (row0 + (size_t)(gq < G ? gq : 0) * Nq) * D);
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            qa[2 * s] = gq < G ? __ldg(qw + 8 * s + c4) : 0u;
            qa[2 * s + 1] = gq < G ? __ldg(qw + 8 * s + 4 + c4) : 0u;
        }
    }
    const RowMods<true> rm(mods, b, g * G, N, i);  // whether a key is seen does not depend on the head
    auto key_of = [&](int t, int e) {
        const long long j = (long long)idx[(row0 + (size_t)t * Nq) * K + e];
        return j >= 0 && j < N && rm.sees(j, i, causal) ? (int)j : -1;
    };
    int U;
    {
        // all heads' entries, then what hides them, in steps without branches between the loads: a wait for
        // each entry's segment in turn took a third of the kernel's time
        int x[G][4];
#pragma unroll
        for (int t = 0; t < G; ++t) {
            const IdxT* irow = idx + (row0 + (size_t)t * Nq) * K + lane;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const IdxT j = lane + 32 * e < K ? irow[32 * e] : (IdxT)-1;
                x[t][e] = j >= 0 && j < (IdxT)N ? (int)j : -1;
            }
        }
        rm.hide(x, K, i, causal);
        U = build_union<G, kDirect>(x, K, N, stage, list, lane);
    }
    bool single = U < 0;  // the heads one by one
    const uint32_t st = (uint32_t)__cvta_generic_to_shared(stage), vst = st + 2u * kStageChunk;
    const StageLane sl(lane);
    float slope[2] = {0.f, 0.f};
    if (mods.slopes) {
#pragma unroll
        for (int e = 0; e < 2; ++e) slope[e] = 2 * c4 + e < G ? mods.slopes[g * G + 2 * c4 + e] : 0.f;
    }
#pragma unroll 1
    for (int pass = 0;;) {
        float oacc[8][4];  // O^T: dims 16 mt + gq (+8) of heads 2 c4, 2 c4 + 1
#pragma unroll
        for (int n = 0; n < 8; ++n) oacc[n][0] = oacc[n][1] = oacc[n][2] = oacc[n][3] = 0.f;
        float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
        __syncwarp();
        if (single) U = single_list([&](int e) { return key_of(pass, e); }, pass, K, list, lane);
        __syncwarp();  // the list is complete, the staging area is free
        const int nch = (U + kStageRows - 1) / kStageRows;
        if (nch > 0) {
            stage_listed(st, kb, list, 0, U, sl, lane);
            stage_commit();
        }
#pragma unroll 1
        for (int c = 0; c < nch; ++c) {
            const int c0 = c * kStageRows;
            const bool more = c + 1 < nch;  // warp-uniform
            __syncwarp();                   // chunk c - 1 is done with the value rows and key buffer (c + 1) & 1
            stage_listed(vst, vb, list, c0, U, sl, lane);
            stage_commit();
            if (more) {
                stage_listed(st + (uint32_t)(((c + 1) & 1) * kStageChunk), kb, list, c0 + kStageRows, U, sl, lane);
                stage_commit();
                cp_async_wait_pending<2>();
            } else {
                cp_async_wait_pending<1>();
            }
            __syncwarp();
            const uint32_t kst = st + (uint32_t)((c & 1) * kStageChunk);
            float sacc[4] = {0.f, 0.f, 0.f, 0.f}, sacc2[4] = {0.f, 0.f, 0.f, 0.f};  // two chains of half the length
#pragma unroll
            for (int s = 0; s < 4; ++s) {  // keys as the A operand
                uint32_t a[4];
                ldmatrix_x4<0>(a, kst + sl.a[s]);
                mma_bf16_16816_a4(sacc, a[0], a[1], a[2], a[3], qa[2 * s], qa[2 * s + 1]);
                ldmatrix_x4<128>(a, kst + sl.a[s]);
                mma_bf16_16816_a4(sacc2, a[0], a[1], a[2], a[3], qa[2 * s + 8], qa[2 * s + 9]);
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) sacc[s] += sacc2[s];
            // keys c0 + gq, c0 + gq + 8 x heads 2 c4, 2 c4 + 1; a head's scores sit in the lanes of equal c4
            float sc[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = c0 + gq + 8 * h;
                const uint32_t entry = at < U ? list[at] : 0u;
                const float far = fabsf((float)(i - (int)(entry & 0xffffffu)));
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    sc[h][e] = (entry >> (24 + 2 * c4 + e)) & 1u
                                   ? mods.score2(sacc[2 * h + e], slope[e], far, TanhFast()) : -INFINITY;
            }
            // p is taken against m_run, which need not be the maximum: it moves (to the maximum, with what is
            // summed so far rescaled) only where a score exceeds it by more than 2^kSlack allows.  l_run is this
            // lane's share of the sum; the lanes add up at the end.
            float pr[2][2];
            const float t0 = fmaxf(sc[0][0], sc[1][0]), t1 = fmaxf(sc[0][1], sc[1][1]);
            if (__any_sync(kFull, t0 > m_run[0] + kSlack || t1 > m_run[1] + kSlack)) {
                float top[2] = {t0, t1};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int o = 4; o <= 16; o <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(kFull, top[e], o));
                    const float mx = fmaxf(m_run[e], top[e]);
                    const float alpha = mx == -INFINITY ? 1.f : exp2_fast(m_run[e] - mx);
                    l_run[e] *= alpha;
                    m_run[e] = mx;
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        oacc[n][e] *= alpha;
                        oacc[n][2 + e] *= alpha;
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float ref = m_run[e] == -INFINITY ? 0.f : m_run[e];  // nothing seen yet: every score is -inf
                pr[0][e] = exp2_fast(sc[0][e] - ref);
                pr[1][e] = exp2_fast(sc[1][e] - ref);
                l_run[e] += pr[0][e] + pr[1][e];
            }
            const Weights pw(pr);
            if (more) cp_async_wait_pending<1>();
            else cp_async_wait_pending<0>();
            __syncwarp();
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {  // values transposed as the A operand
                uint32_t a[4];
                ldmatrix_x4_trans<0>(a, vst + sl.at[mt]);
                pw.mma(oacc[mt], a);
                ldmatrix_x4_trans<128>(a, vst + sl.at[mt]);
                pw.mma(oacc[mt + 4], a);
            }
        }
        if (!single) {
            float bad = 0.f;  // 0 while every sum is finite
#pragma unroll
            for (int n = 0; n < 8; ++n) {
#pragma unroll
                for (int x = 0; x < 4; ++x) bad = fmaf(oacc[n][x], 0.f, bad);
            }
            if (__any_sync(kFull, bad != 0.f)) {
                single = true;
                continue;
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) l_run[e] += __shfl_xor_sync(kFull, l_run[e], o);
        }
        // each head's row divided by its sum and transposed back: lane (gq, c4) stores dims 2 c4, 2 c4 + 1 of head gq
        const float inv0 = l_run[0] == 0.f ? 0.f : 1.f / l_run[0], inv1 = l_run[1] == 0.f ? 0.f : 1.f / l_run[1];
        __nv_bfloat16* orow = out + (row0 + (size_t)(gq < G ? gq : 0) * Nq) * D + 2 * c4;
        const bool mine = single ? gq == pass : gq < G;
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
            const uint32_t lo = movmatrix_trans(pack_bf16x2(oacc[mt][0] * inv0, oacc[mt][1] * inv1));
            const uint32_t hi = movmatrix_trans(pack_bf16x2(oacc[mt][2] * inv0, oacc[mt][3] * inv1));
            if (mine) {
                *reinterpret_cast<uint32_t*>(orow + 16 * mt) = lo;
                *reinterpret_cast<uint32_t*>(orow + 16 * mt + 8) = hi;
            }
        }
        if (mods.rest) {
            __nv_bfloat16* rrow = static_cast<__nv_bfloat16*>(mods.rest) + (orow - out);
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) {
                const uint32_t lo = movmatrix_trans(pack_bf16x2(bf16_rest(oacc[mt][0] * inv0), bf16_rest(oacc[mt][1] * inv1)));
                const uint32_t hi = movmatrix_trans(pack_bf16x2(bf16_rest(oacc[mt][2] * inv0), bf16_rest(oacc[mt][3] * inv1)));
                if (mine) {
                    *reinterpret_cast<uint32_t*>(rrow + 16 * mt) = lo;
                    *reinterpret_cast<uint32_t*>(rrow + 16 * mt + 8) = hi;
                }
            }
        }
        if (mods.lse2 && gq == 0) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int t = 2 * c4 + e;
                if (single ? t == pass : t < G) mods.lse2[row0 + (size_t)t * Nq] = m_run[e] + log2f(l_run[e]);
            }
        }
        if (!single || ++pass == G) break;
    }
}

// Few rows (single tokens): a CTA per (query, head), a warp per 16 listed keys, so that a row is two trips
// to memory (its list, then all its key and value rows at once) and one join through shared memory.  Half a
// warp holds a key row, 16 bytes a lane.  Longer lists go round again with the running maximum and sum.
constexpr int kFewKeys = 16;     // keys a warp has in flight
constexpr int kFewMaxWarps = 8;
// Up to this many listed keys in all (B * H * Nq * K).  12/2 heads, K = 64: single tokens against 32768 keys,
// batch 8 3.8 us here, 18.5 us on the tensor-core form; batch 128: 11.7, 19.1; neighbouring
// queries of one sequence, 256 of them (196,608): 21.0, 20.6.  K = 16, 1024 queries (196,608): 20.9, 12.7.
constexpr long long kFewEntries = 1 << 17;

template <typename IdxT>
__global__ void __launch_bounds__(kFewMaxWarps * 32)
mod_attn_few_kernel(const __nv_bfloat16* __restrict__ q, const __nv_bfloat16* __restrict__ k,
                    const __nv_bfloat16* __restrict__ v, const IdxT* __restrict__ idx, __nv_bfloat16* __restrict__ out,
                    int H, int Hkv, int N, int Nq, int q0, int K, int causal, const ScoreMods mods) {
    constexpr int D = 128;
    __shared__ float2 s_ml[kFewMaxWarps];
    __shared__ float s_acc[kFewMaxWarps][D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int half = lane >> 4, hl = lane & 15, slot = lane & 7;  // this lane ends with the score of key 8 half + slot
    const size_t row = blockIdx.x;
    const int bh = (int)(row / Nq), i = q0 + (int)(row - (size_t)bh * Nq);
    const int b = bh / H, h = bh - b * H;
    const size_t kv = (size_t)b * Hkv + h / (H / Hkv);
    const uint4* kb = reinterpret_cast<const uint4*>(k + kv * N * D) + hl;
    const uint4* vb = reinterpret_cast<const uint4*>(v + kv * N * D) + hl;
    const uint4 qv = __ldg(reinterpret_cast<const uint4*>(q + row * D) + hl);
    const RowMods<true> rm(mods, b, h, N, i);
    float m_run = -INFINITY, l_run = 0.f, acc[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) acc[t] = 0.f;
    for (int k0 = warp * kFewKeys; k0 < K; k0 += warps * kFewKeys) {
        const int e = k0 + 8 * half + slot;
        const long long jl = e < K ? (long long)idx[row * K + e] : -1;
        const int j = jl >= 0 && jl < N && rm.sees(jl, i, causal) ? (int)jl : -1;
        uint4 kr[8], vr[8];
        int js[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            js[t] = __shfl_sync(kFull, j, 16 * half + t);
            const size_t at = (size_t)max(js[t], 0) * (D / 8);
            kr[t] = __ldg(kb + at);
            vr[t] = __ldg(vb + at);
        }
        float part[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) part[t] = dot8_bf16(qv, kr[t]);
#pragma unroll
        for (int w = 4; w >= 1; w >>= 1) {  // sums over the half-warp; lane l keeps key l & 7
            const bool upper = (lane & w) != 0;
#pragma unroll
            for (int t = 0; t < w; ++t) {
                const float send = upper ? part[t] : part[t + w], keep = upper ? part[t + w] : part[t];
                part[t] = keep + __shfl_xor_sync(kFull, send, w);
            }
        }
        const float dot = part[0] + __shfl_xor_sync(kFull, part[0], 8);
        const float s2 = j >= 0 ? rm.score2(dot, i, j) : -INFINITY;
        const float m_new = fmaxf(m_run, warp_max(s2));
        if (m_new == -INFINITY && !shows_nan(s2)) continue;  // warp-uniform: nothing seen so far
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        const float p = j >= 0 ? exp2f(s2 - ref) : 0.f;
        const float alpha = exp2f(m_run - ref);
        l_run = l_run * alpha + 0.5f * warp_sum(p);  // every key's p sits in two lanes
        m_run = m_new;
#pragma unroll
        for (int t = 0; t < 8; ++t) acc[t] *= alpha;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const float pt = __shfl_sync(kFull, p, 16 * half + t);
            if (js[t] < 0) continue;  // uniform over the half-warp; key 0 in its place may hold anything
            float x[8];
            unpack_bf16x2(vr[t].x, x[0], x[1]);
            unpack_bf16x2(vr[t].y, x[2], x[3]);
            unpack_bf16x2(vr[t].z, x[4], x[5]);
            unpack_bf16x2(vr[t].w, x[6], x[7]);
#pragma unroll
            for (int d = 0; d < 8; ++d) acc[d] = fmaf(pt, x[d], acc[d]);
        }
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) acc[t] += __shfl_xor_sync(kFull, acc[t], 16);
    if (half == 0) {
#pragma unroll
        for (int t = 0; t < 8; ++t) s_acc[warp][8 * hl + t] = acc[t];
    }
    if (lane == 0) s_ml[warp] = make_float2(m_run, l_run);
    __syncthreads();
    float top = -INFINITY;
    for (int w = 0; w < warps; ++w) top = fmaxf(top, s_ml[w].x);
    float l = 0.f;
    for (int w = 0; w < warps; ++w) l += s_ml[w].x == -INFINITY ? s_ml[w].y : s_ml[w].y * exp2f(s_ml[w].x - top);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
        float t = 0.f;
        for (int w = 0; w < warps; ++w) t += s_ml[w].x == -INFINITY ? s_acc[w][d] : s_acc[w][d] * exp2f(s_ml[w].x - top);
        out[row * D + d] = __float2bfloat16_rn(t * inv);
        if (mods.rest) static_cast<__nv_bfloat16*>(mods.rest)[row * D + d] = __float2bfloat16_rn(bf16_rest(t * inv));
    }
    if (mods.lse2 && threadIdx.x == 0) mods.lse2[row] = top + log2f(l);
}

template <typename IdxT>
cudaError_t launch_few(const GatherArgs& a, cudaStream_t stream) {
    const int warps = std::max(1, std::min(kFewMaxWarps, (a.K + kFewKeys - 1) / kFewKeys));
    mod_attn_few_kernel<IdxT><<<(unsigned)((long long)a.B * a.H * a.Nq), warps * 32, 0, stream>>>(
        static_cast<const __nv_bfloat16*>(a.q), static_cast<const __nv_bfloat16*>(a.k),
        static_cast<const __nv_bfloat16*>(a.v), static_cast<const IdxT*>(a.idx), static_cast<__nv_bfloat16*>(a.out), a.H,
        a.Hkv, a.N, a.Nq, a.q0, a.K, a.causal, a.mods);
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e;
}

template <typename IdxT>
cudaError_t launch_mma(const GatherArgs& a, cudaStream_t stream) {
    const int G = a.H / a.Hkv;
    const bool direct = a.N <= kUnionDirectKeys;
#define OSSA_MOD_PICK(GG) (direct ? mod_attn_mma_kernel<IdxT, GG, true> : mod_attn_mma_kernel<IdxT, GG, false>)
    auto kern = G == 2 ? OSSA_MOD_PICK(2)
              : G == 3 ? OSSA_MOD_PICK(3)
              : G == 4 ? OSSA_MOD_PICK(4)
              : G == 5 ? OSSA_MOD_PICK(5)
              : G == 6 ? OSSA_MOD_PICK(6)
              : G == 7 ? OSSA_MOD_PICK(7)
                       : OSSA_MOD_PICK(8);
#undef OSSA_MOD_PICK
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kModBytes);
    if (e != cudaSuccess) return e;
    kern<<<dim3((a.Nq + kModWarps - 1) / kModWarps, a.B * a.Hkv), kModWarps * 32, kModBytes, stream>>>(
        static_cast<const __nv_bfloat16*>(a.q), static_cast<const __nv_bfloat16*>(a.k),
        static_cast<const __nv_bfloat16*>(a.v), static_cast<const IdxT*>(a.idx), static_cast<__nv_bfloat16*>(a.out), a.H,
        a.Hkv, a.N, a.Nq, a.q0, a.K, a.causal, a.mods);
    e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e;
}

}  // namespace

bool gather_union_serves(int dtype, int H, int Hkv, int N, int D, int K) {
    return dtype == kBF16 && D == 128 && K >= 1 && K <= 128 && N <= kUnionMaxKeys && H / Hkv <= 8;
}

cudaError_t launch_gather_attn_mods(const GatherArgs& a, cudaStream_t stream) {
    if (a.dtype == kBF16 && a.D == 128 && (long long)a.B * a.H * a.Nq * a.K <= kFewEntries)
        return a.idx_is_64 ? launch_few<int64_t>(a, stream) : launch_few<int32_t>(a, stream);
    if (a.H > a.Hkv && gather_union_serves(a.dtype, a.H, a.Hkv, a.N, a.D, a.K))
        return a.idx_is_64 ? launch_mma<int64_t>(a, stream) : launch_mma<int32_t>(a, stream);
    if (a.dtype == kF32)
        return a.idx_is_64 ? launch_typed<float, int64_t, true>(a, stream) : launch_typed<float, int32_t, true>(a, stream);
    return a.idx_is_64 ? launch_typed<__nv_bfloat16, int64_t, true>(a, stream)
                       : launch_typed<__nv_bfloat16, int32_t, true>(a, stream);
}

}  // namespace ossa
