// Backward pass of the gathered top-K attention.
//
// Per query row i with listed keys j (score_mods.cuh), row statistic L = log2 sum 2^s2:
//   p_j = 2^(s2_j - L),  dP_j = dO_i . v_j,  Delta_i = sum_j p_j dP_j
//   dS_j = p_j (dP_j - Delta_i),  dX_j = dS_j * d score / d (q.k)
//   dq_i = sum_j dX_j k_j,  dk_j = sum_i dX_ij q_i,  dv_j = sum_i p_ij dO_i
//   dslope_h = -sum dS_ij |i - j|
// Nothing per (row, entry) is kept by the forward: both passes here recompute s2 and dP.
//
//  1. The index lists are turned round: for every (b, kv head) the rows that list a key,
//     key by key, in a fixed order (a counting sort: units of (row chunk, head) count their
//     entries per key, the counts are scanned, every unit then writes its rows).  For the
//     tensor-core key pass "key" is a block of 8 keys: neighbouring entries of an ascending list
//     that fall into one block make one turned entry with a bit per key.
//  2. Row pass, one warp per row: dq_i, Delta_i and the row's share of dslope.
//  3. Key pass, one warp per `tile` consecutive entries of a turned list, which may begin and
//     end inside a key's run: whole runs are stored, cut ones go to per-tile partial sums.
//  4. Join: keys whose run is cut add their partial sums in tile order; keys that nobody
//     lists get zeros.
// No float atomics, and the sort's places do not depend on the order in which atomics run (entry_place):
// repeated calls give the same bits.
//
// Bound: L2-to-SM traffic.  Either pass reads two rows of D values per entry (the row pass's tensor-core form
// per key of the heads' union, the key pass's per row and key block), which no tile keeps: the rows that list
// a key are scattered.
#include <algorithm>
#include <cstdint>

#include "common.cuh"
#include "kernels.h"
#include "gather_bwd.cuh"
#include "mma_sync.cuh"
#include "score_mods.cuh"

namespace ossa {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kKeyRange = 8192;  // key blocks that one CTA of the counting sort covers (32 KB of counters)
constexpr int kMaxChunks = 128;   // row chunks of the counting sort per head
constexpr int kMinChunkRows = 32;
constexpr int kCountRows = 4;    // rows whose entries a warp of the counting sort's first step has in flight
constexpr int kPlaceRows = 8;    // and of its last step

BwdShape make_shape(int dtype, int B, int H, int Hkv, int Nq, int N, int D, int K) {
    BwdShape s{};
    s.B = B;
    s.H = H;
    s.Hkv = Hkv;
    s.G = H / Hkv;
    s.Nq = Nq;
    s.N = N;
    s.D = D;
    s.K = K;
    // the tensor-core key pass: bf16 rows of 128, rows and keys in 24 bits each
    const bool mma = dtype == kBF16 && D == 128 && N <= (1 << 24) && (long long)s.G * Nq < (1ll << 24);
    s.shift = mma ? kKeyBlockShift : 0;
    s.NB = (N + (1 << s.shift) - 1) >> s.shift;
    const long long kv = (long long)B * Hkv;
    // One warp per unit in the sort's last step: enough units for 24 warps per SM, rows permitting.  Fewer
    // leave it waiting, more cost in the scan over units (count + place + scan, us, at 16, 32, 64, 128, 256
    // chunks: B=2, 12/2 heads, N=4096, K=64: 92, 68, 56, 59, 82; B=1, N=8192, K=128: 305, 174, 133, 126, 137).
    const long long want = 24ll * device_sm_count() / std::max(kv * s.G, 1ll);
    s.chunks = (int)std::max(1ll, std::min({want, (long long)kMaxChunks, (long long)Nq / kMinChunkRows}));
    s.chunk_rows = (Nq + s.chunks - 1) / s.chunks;
    s.units = s.chunks * s.G;
    s.cap = (long long)s.G * Nq * K;
    // Tiles: long ones store fewer cut runs, short ones fill the device (key pass + join, us, at tiles of 128,
    // 256, 512, 1024: the two shapes above 241, 198, 186, 219 and 617, 488, 432, 404; fp32 B=2, 6/3 heads, N=517,
    // K=33, at 64, 128, 256, 512: 59, 58, 84, 151).  84 tiles per SM fit all three.
    const long long fair = kv * s.cap / (84ll * device_sm_count());
    s.tile = (int)std::min(std::max((fair + 15) / 16 * 16, 64ll), mma ? 1024ll : 256ll);
    s.tiles = (s.cap + s.tile - 1) / s.tile;
    return s;
}

struct Layout {
    size_t keys, counts, base, list, delta, part, slope_rows, total;
};

Layout make_layout(const BwdShape& s, bool dslopes) {
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    const size_t kv = (size_t)s.B * s.Hkv, rows = (size_t)s.B * s.H * s.Nq;
    Layout l;
    l.keys = 0;
    l.counts = l.keys + up(rows * s.K * 4);
    l.base = l.counts + up(kv * s.units * s.NB * 4);
    l.list = l.base + up(kv * ((size_t)s.NB + 1) * 4);
    l.delta = l.list + up(kv * s.cap * 4);
    l.part = l.delta + up(rows * 4);
    l.slope_rows = l.part + up(kv * s.tiles * 4 * ((size_t)s.D << s.shift) * 4);
    l.total = l.slope_rows + (dslopes ? up(rows * 4) : 0);
    return l;
}

// ------------------------------------------------------------------ 1. turned lists

// A row's entries 32 e .. 32 e + 31, one per lane (key, -1: masked), as the words of the normalised lists.
// Blocks of one key: the key.  Blocks of 8: an entry follows the one before it when its key is greater
// and in the same block; the first of such a chain stands for all and carries a bit per key of the block,
// key | bits << 24, the others have no bits.  (-1 is no such word: a chain of 8 begins at key 0 of a block.)
__device__ __forceinline__ int list_word(int key, int shift, int lane) {
    if (shift == 0) return key;  // warp-uniform
    const int prev = __shfl_up_sync(kFull, key, 1);
    const bool follows = lane > 0 && key >= 0 && prev >= 0 && prev < key && ((prev ^ key) >> shift) == 0;
    const unsigned tails = __ballot_sync(kFull, follows) >> 1 >> lane;  // bit t: lane + 1 + t follows
    uint32_t bits = key >= 0 ? 1u << (key & (kKeyBlock - 1)) : 0u;
    // OR over the chain behind this lane: at most kKeyBlock entries, so three doublings
#pragma unroll
    for (int o = 1; o < kKeyBlock; o <<= 1) {
        const uint32_t other = __shfl_down_sync(kFull, bits, o);
        const unsigned all = (1u << o) - 1u;
        if ((tails & all) == all) bits |= other;
    }
    return key < 0 ? -1 : (int)((uint32_t)key | (follows ? 0u : bits << 24));
}

// The block that an entry stands for, -1 where it is masked or follows another.
__device__ __forceinline__ int word_block(int w, int shift) {
    if (shift == 0 || w == -1) return w;
    return (uint32_t)w >> 24 ? (w & 0xffffff) >> shift : -1;
}

// keys: the normalised lists.
// counts[kv][unit][block]: the unit's entries of the key block's turned list.
// A warp has the entries of kCountRows rows in flight.
template <typename IdxT>
__global__ void __launch_bounds__(kThreads)
count_kernel(const IdxT* __restrict__ idx, const BwdShape s, const ScoreMods mods, int* __restrict__ keys,
             int* __restrict__ counts) {
    extern __shared__ int hist[];  // min(NB, kKeyRange)
    const int unit = blockIdx.x, kv = blockIdx.y, k0 = blockIdx.z * kKeyRange;
    const int nk = min(kKeyRange, s.NB - k0);
    const int b = kv / s.Hkv, h = (kv - b * s.Hkv) * s.G + unit % s.G;
    const int r0 = unit / s.G * s.chunk_rows, r1 = min(s.Nq, r0 + s.chunk_rows);
    for (int t = threadIdx.x; t < nk; t += kThreads) hist[t] = 0;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const int* seg = mods.segments ? mods.segments + (size_t)b * s.N : nullptr;
    const int prefix = mods.prefix_len ? mods.prefix_len[b] : 0;
    const size_t row0 = ((size_t)b * s.H + h) * s.Nq;
    const IdxT* ib = idx + row0 * s.K;
    int* kb = keys + row0 * s.K;
    for (int il0 = r0 + (threadIdx.x >> 5) * kCountRows; il0 < r1; il0 += kWarps * kCountRows) {
        int si[kCountRows];
#pragma unroll
        for (int t = 0; t < kCountRows; ++t) si[t] = seg && il0 + t < r1 ? seg[s.q0 + il0 + t] : 0;
        for (int e = lane; e - lane < s.K; e += 32) {
            int j[kCountRows];
#pragma unroll
            for (int t = 0; t < kCountRows; ++t) {
                const IdxT x = e < s.K && il0 + t < r1 ? ib[(size_t)(il0 + t) * s.K + e] : (IdxT)-1;
                j[t] = x >= 0 && x < (IdxT)s.N ? (int)x : -1;
                if (s.causal && j[t] > s.q0 + il0 + t && j[t] >= prefix) j[t] = -1;
            }
            if (seg) {
#pragma unroll
                for (int t = 0; t < kCountRows; ++t)
                    if (j[t] >= 0 && seg[j[t]] != si[t]) j[t] = -1;
            }
#pragma unroll
            for (int t = 0; t < kCountRows; ++t) {
                const int w = list_word(j[t], s.shift, lane);
                if (blockIdx.z == 0 && e < s.K && il0 + t < r1) kb[(size_t)(il0 + t) * s.K + e] = w;
                const int at = word_block(w, s.shift) - k0;
                if (w != -1 && (unsigned)at < (unsigned)nk) atomicAdd(&hist[at], 1);
            }
        }
    }
    __syncthreads();
    int* out = counts + ((size_t)kv * s.units + unit) * s.NB + k0;
    for (int t = threadIdx.x; t < nk; t += kThreads) out[t] = hist[t];
}

// counts -> exclusive prefix over the units, and the block's total in base[kv][block].  A CTA takes 32
// blocks; each of its 8 warps a contiguous part of the units, summed first and then written.
__global__ void __launch_bounds__(kThreads)
unit_scan_kernel(const BwdShape s, int* __restrict__ counts, int* __restrict__ base) {
    constexpr int kAhead = 8;  // loads in flight
    __shared__ int sums[kWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kv = blockIdx.y;
    const int key = blockIdx.x * 32 + lane;
    const bool on = key < s.NB;
    int* c = counts + (size_t)kv * s.units * s.NB + (on ? key : 0);
    const int per = (s.units + kWarps - 1) / kWarps;
    const int u0 = min(warp * per, s.units), u1 = min(u0 + per, s.units);
    int sum = 0;
    for (int u = u0; u < u1; u += kAhead) {
#pragma unroll
        for (int t = 0; t < kAhead; ++t) sum += u + t < u1 ? c[(size_t)(u + t) * s.NB] : 0;
    }
    sums[warp][lane] = sum;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += sums[w][lane];
    if (on && warp == kWarps - 1) base[(size_t)kv * (s.NB + 1) + key] = before + sum;
    for (int u = u0; u < u1; u += kAhead) {
        int x[kAhead];
#pragma unroll
        for (int t = 0; t < kAhead; ++t) x[t] = u + t < u1 ? c[(size_t)(u + t) * s.NB] : 0;
#pragma unroll
        for (int t = 0; t < kAhead; ++t) {
            if (on && u + t < u1) c[(size_t)(u + t) * s.NB] = before;
            before += x[t];
        }
    }
}

// base[kv][0..NB]: exclusive prefix of the totals over the blocks.
__global__ void __launch_bounds__(1024) key_scan_kernel(const BwdShape s, int* __restrict__ base) {
    __shared__ int wsum[32];
    __shared__ int carry;
    int* p = base + (size_t)blockIdx.x * (s.NB + 1);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) carry = 0;
    __syncthreads();
    for (int k0 = 0; k0 < s.NB; k0 += 1024) {
        const int k = k0 + threadIdx.x;
        const int x = k < s.NB ? p[k] : 0;
        int y = x;  // inclusive over the warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(kFull, y, o);
            if (lane >= o) y += t;
        }
        if (lane == 31) wsum[warp] = y;
        __syncthreads();
        if (warp == 0) {
            int w = wsum[lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(kFull, w, o);
                if (lane >= o) w += t;
            }
            wsum[lane] = w;
        }
        __syncthreads();
        const int before = carry + (warp ? wsum[warp - 1] : 0) + y - x;
        if (k < s.NB) p[k] = before;
        __syncthreads();
        if (threadIdx.x == 1023) carry = before + x;
        __syncthreads();
    }
    if (threadIdx.x == 0) p[s.NB] = carry;
}

// The place of this lane's entry (block at, on: it has one) behind the counter of its block.  Entries of one
// row that share a block take theirs in lane order: ascending lists have none (`some`, `follow`: lanes that
// hold a key, those whose key exceeds the lane's before), others are matched.
__device__ __forceinline__ int entry_place(int* next, int at, bool on, unsigned some, unsigned follow, int lane) {
    if (__popc(some & ~follow) <= 1) return on ? atomicAdd(&next[at], 1) : -1;  // warp-uniform; no block twice
    const unsigned same = __match_any_sync(kFull, on ? at : -1 - lane);
    const int rank = __popc(same & lanemask_lt()), first = on ? next[at] : 0;
    __syncwarp();
    if (on && rank == 0) next[at] = first + __popc(same);
    return on ? first + rank : -1;
}

// list[kv][position] = r (| bits << 24) with r = g * Nq + il of the rows that list a key block, block by
// block.  One warp walks the unit's rows in a fixed order, the counters of its key range in shared memory; the entries of
// kPlaceRows rows are loaded together, and the next ones while these are placed, so a step costs
// one trip to L2 and not one per row.
__global__ void __launch_bounds__(32)
place_kernel(const int* __restrict__ keys, const BwdShape s, const int* __restrict__ counts,
             const int* __restrict__ base, int* __restrict__ list) {
    extern __shared__ int next[];  // min(NB, kKeyRange)
    const int unit = blockIdx.x, kv = blockIdx.y, k0 = blockIdx.z * kKeyRange;
    const int nk = min(kKeyRange, s.NB - k0);
    const int g = unit % s.G;
    const int b = kv / s.Hkv, h = (kv - b * s.Hkv) * s.G + g;
    const int r0 = unit / s.G * s.chunk_rows, r1 = min(s.Nq, r0 + s.chunk_rows);
    const int lane = threadIdx.x;
    const int* c = counts + ((size_t)kv * s.units + unit) * s.NB + k0;
    const int* bs = base + (size_t)kv * (s.NB + 1) + k0;
    for (int t = lane; t < nk; t += 32) next[t] = c[t] + bs[t];
    __syncwarp();
    int* out = list + (size_t)kv * s.cap;
    const int* rows = keys + ((size_t)b * s.H + h) * s.Nq * s.K;
    // a step: 32 entries of kPlaceRows rows; il, e: where the step after the loaded one begins
    int il = r0, e = lane;
    int w[kPlaceRows], ahead[kPlaceRows];
    auto load = [&](int (&x)[kPlaceRows]) {
#pragma unroll
        for (int t = 0; t < kPlaceRows; ++t) x[t] = il + t < r1 && e < s.K ? rows[(size_t)(il + t) * s.K + e] : -1;
        e += 32;
        if (e - lane >= s.K) {
            e = lane;
            il += kPlaceRows;
        }
    };
    int at_row = r0;
    load(w);
    while (at_row < r1) {
        const int row = at_row;
        at_row = il;  // the row group of the next step
        load(ahead);
        int pos[kPlaceRows];
#pragma unroll
        for (int t = 0; t < kPlaceRows; ++t) {
            const int at = word_block(w[t], s.shift) - k0;
            const int key = w[t] == -1 || s.shift == 0 ? w[t] : w[t] & 0xffffff, before = __shfl_up_sync(kFull, key, 1);
            const unsigned some = __ballot_sync(kFull, key >= 0);
            const unsigned follow = __ballot_sync(kFull, key >= 0 && lane > 0 && before >= 0 && before < key);
            pos[t] = entry_place(next, at, w[t] != -1 && (unsigned)at < (unsigned)nk, some, follow, lane);
            __syncwarp();  // a row's places before the next row's
        }
#pragma unroll
        for (int t = 0; t < kPlaceRows; ++t) {
            const uint32_t bits = s.shift ? (uint32_t)w[t] & 0xff000000u : 0u;
            if (pos[t] >= 0) out[pos[t]] = (int)((uint32_t)(g * s.Nq + row + t) | bits);
            w[t] = ahead[t];
        }
    }
}

// ------------------------------------------------------------------ 2. row pass

template <typename T, int D>
struct RowLoad {
    static constexpr int kPer = D >= 32 ? D / 32 : 1;  // values of a row that one lane owns
    static constexpr int kActive = D / kPer;
    static __device__ __forceinline__ void load(const T* row, int lane, float (&v)[kPer]) {
        if (lane < kActive) {
            VecLoad<T, kPer>::load(row + lane * kPer, v);
        } else {
#pragma unroll
            for (int t = 0; t < kPer; ++t) v[t] = 0.f;
        }
    }
    static __device__ __forceinline__ void store(T* row, int lane, const float (&v)[kPer]) {
        if (lane < kActive) {
#pragma unroll
            for (int t = 0; t < kPer; ++t) store_from_f32(row + lane * kPer + t, v[t]);
        }
    }
};

// Rows that a warp holds in registers at once in the passes below: each is fetched once for its dot product
// and its weighted sum (fp32, 12/2 heads, N=4096, K=64: fetched again for the sum, 32 at a time, the key
// pass took 1199 us, the row pass 328; held 8 at a time 259 and 208).
template <int D>
constexpr int kHeld = RowLoad<float, D>::kPer <= 4 ? 8 : 4;

// Sums x[0..n-1] over the warp; lane l ends with the total of x[l % n].
template <int n>
__device__ __forceinline__ float reduce_held(float (&x)[n], int lane) {
#pragma unroll
    for (int w = n / 2; w >= 1; w >>= 1) {
        const bool upper = (lane & w) != 0;
#pragma unroll
        for (int t = 0; t < w; ++t) {
            const float send = upper ? x[t] : x[t + w], keep = upper ? x[t + w] : x[t];
            x[t] = keep + __shfl_xor_sync(kFull, send, w);
        }
    }
#pragma unroll
    for (int o = n; o < 32; o <<= 1) x[0] += __shfl_xor_sync(kFull, x[0], o);
    return x[0];
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads)
row_pass_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const int* __restrict__ keys,
                const T* __restrict__ out, const T* __restrict__ dout, const BwdShape s, const ScoreMods mods,
                T* __restrict__ dq, float* __restrict__ delta, float* __restrict__ slope_rows) {
    using R = RowLoad<T, D>;
    constexpr int B = kHeld<D>;
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (row >= (long long)s.B * s.H * s.Nq) return;  // warp-uniform
    const int bh = (int)(row / s.Nq), il = (int)(row - (long long)bh * s.Nq);
    const int batch = bh / s.H, h = bh - batch * s.H, i = s.q0 + il;
    const size_t kv = (size_t)batch * s.Hkv + h / s.G;
    const T* kb = k + kv * s.N * D;
    const T* vb = v + kv * s.N * D;
    const float slope = mods.slopes ? mods.slopes[h] : 0.f;
    const float lse2 = mods.lse2[row];
    float qv[R::kPer], dv[R::kPer], acc[R::kPer];
    R::load(q + row * D, lane, qv);
    R::load(dout + row * D, lane, dv);
    float d0 = 0.f;  // Delta from the stored output (and its rest), for dq
    {
        float o[R::kPer];
        R::load(out + row * D, lane, o);
        if constexpr (sizeof(T) == 2) {
            if (mods.rest) {
                float rest[R::kPer];
                R::load(static_cast<const T*>(mods.rest) + row * D, lane, rest);
#pragma unroll
                for (int t = 0; t < R::kPer; ++t) o[t] += rest[t];
            }
        }
#pragma unroll
        for (int t = 0; t < R::kPer; ++t) {
            d0 = fmaf(o[t], dv[t], d0);
            acc[t] = 0.f;
        }
        d0 = warp_sum(d0);
    }
    float a_p = 0.f, a_pd = 0.f, a_f = 0.f, a_xf = 0.f;  // sums of p, p dP, p far, p (dP - d0) far
    const int* krow = keys + row * s.K;
    for (int kc = 0; kc < s.K; kc += 32) {
        const int kk = kc + lane;
        int j = kk < s.K ? krow[kk] : -1;
        if (s.shift && j != -1) j &= 0xffffff;  // the key of a word (list_word)
        const unsigned some = __ballot_sync(kFull, j >= 0);
        for (int m0 = 0; m0 < 32; m0 += B) {
            if (((some >> m0) & ((1u << B) - 1u)) == 0u) continue;  // warp-uniform
            float kr[B][R::kPer], x[B], y[B];
#pragma unroll
            for (int t = 0; t < B; ++t) {
                const int jt = max(__shfl_sync(kFull, j, m0 + t), 0);
                R::load(kb + (size_t)jt * D, lane, kr[t]);
            }
#pragma unroll
            for (int t = 0; t < B; ++t) {
                const int jt = max(__shfl_sync(kFull, j, m0 + t), 0);
                float r[R::kPer];
                R::load(vb + (size_t)jt * D, lane, r);
                x[t] = y[t] = 0.f;
#pragma unroll
                for (int d = 0; d < R::kPer; ++d) {
                    x[t] = fmaf(qv[d], kr[t][d], x[t]);
                    y[t] = fmaf(dv[d], r[d], y[t]);
                }
            }
            const float dot = reduce_held<B>(x, lane), dp = reduce_held<B>(y, lane);
            const int je = __shfl_sync(kFull, j, m0 + lane % B);  // this lane's entry
            float p = 0.f, dx = 0.f;
            if (je >= 0 && lse2 != -INFINITY) {  // -inf: every score of the row is, its output was 0
                const float far = fabsf((float)(i - je));
                p = exp2f(mods.log2_p(dot, slope, far, lse2, dx, TanhExact()));
                const float ds = p * (dp - d0);
                dx *= ds;
                if (lane < B) {
                    a_p += p;
                    a_pd = fmaf(p, dp, a_pd);
                    a_f = fmaf(p, far, a_f);
                    a_xf = fmaf(ds, far, a_xf);
                }
            }
#pragma unroll
            for (int t = 0; t < B; ++t) {
                const float w = __shfl_sync(kFull, dx, t);
                if (__shfl_sync(kFull, j, m0 + t) < 0) continue;  // warp-uniform; key 0 in its place may hold anything
#pragma unroll
                for (int d = 0; d < R::kPer; ++d) acc[d] = fmaf(w, kr[t][d], acc[d]);
            }
        }
    }
    R::store(dq + row * D, lane, acc);
    const RowSums sums(warp_sum(a_p), warp_sum(a_pd), warp_sum(a_f), warp_sum(a_xf), d0);
    if (lane == 0) {
        delta[row] = sums.delta;
        if (slope_rows) slope_rows[row] = sums.slope;
    }
}

// ------------------------------------------------------------------ 3. key pass

// Blocks of one key (shift 0).
template <typename T, int D>
__global__ void __launch_bounds__(kThreads)
key_pass_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ dout,
                const BwdShape s, const ScoreMods mods, const int* __restrict__ base, const int* __restrict__ list,
                const float* __restrict__ delta, T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part) {
    using R = RowLoad<T, D>;
    constexpr int B = kHeld<D>;
    const int lane = threadIdx.x & 31, kv = blockIdx.y;
    const long long tile = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int* bs = base + (size_t)kv * (s.N + 1);
    const int total = bs[s.N];
    if (tile * s.tile >= total) return;  // warp-uniform
    const int t0 = (int)(tile * s.tile), t1 = min(total, t0 + s.tile);
    const int batch = kv / s.Hkv, h0 = (kv - batch * s.Hkv) * s.G;
    const size_t rows0 = ((size_t)batch * s.H + h0) * s.Nq;  // row of list entry r: rows0 + r
    const int* ls = list + (size_t)kv * s.cap;
    int key = block_at(bs, s.N, t0);
    for (int pos = t0; pos < t1; ++key) {
        const int run0 = bs[key], run1 = bs[key + 1];
        const int end = min(run1, t1);
        if (end <= pos) continue;  // nobody lists this key
        float kr[R::kPer], vr[R::kPer], ak[R::kPer], av[R::kPer];
        R::load(k + ((size_t)kv * s.N + key) * D, lane, kr);
        R::load(v + ((size_t)kv * s.N + key) * D, lane, vr);
#pragma unroll
        for (int t = 0; t < R::kPer; ++t) ak[t] = av[t] = 0.f;
        for (; pos < end; pos += 32) {
            const int n = min(32, end - pos);
            const int r = ls[pos + min(lane, n - 1)];  // past the run its last row again, without weight
            const int g = r / s.Nq, i = s.q0 + r - g * s.Nq;
            const float lse2 = lane < n ? mods.lse2[rows0 + r] : -INFINITY, dl = delta[rows0 + r];
            const float slope = mods.slopes ? mods.slopes[h0 + g] : 0.f;
            for (int m0 = 0; m0 < n; m0 += B) {
                float qr[B][R::kPer], dr[B][R::kPer], x[B], y[B];
#pragma unroll
                for (int t = 0; t < B; ++t) {
                    const size_t row = rows0 + __shfl_sync(kFull, r, m0 + t);
                    R::load(q + row * D, lane, qr[t]);
                    R::load(dout + row * D, lane, dr[t]);
                }
#pragma unroll
                for (int t = 0; t < B; ++t) {
                    x[t] = y[t] = 0.f;
#pragma unroll
                    for (int d = 0; d < R::kPer; ++d) {
                        x[t] = fmaf(qr[t][d], kr[d], x[t]);
                        y[t] = fmaf(dr[t][d], vr[d], y[t]);
                    }
                }
                const float dot = reduce_held<B>(x, lane), dp = reduce_held<B>(y, lane);
                const int e = m0 + lane % B;  // this lane's entry
                const float le = __shfl_sync(kFull, lse2, e), de = __shfl_sync(kFull, dl, e);
                const float se = __shfl_sync(kFull, slope, e), far = fabsf((float)(__shfl_sync(kFull, i, e) - key));
                float p = 0.f, dx = 0.f;
                if (le != -INFINITY) {
                    p = exp2f(mods.log2_p(dot, se, far, le, dx, TanhExact()));
                    dx *= p * (dp - de);
                }
#pragma unroll
                for (int t = 0; t < B; ++t) {
                    const float pt = __shfl_sync(kFull, p, t), xt = __shfl_sync(kFull, dx, t);
#pragma unroll
                    for (int d = 0; d < R::kPer; ++d) {
                        ak[d] = fmaf(xt, qr[t][d], ak[d]);
                        av[d] = fmaf(pt, dr[t][d], av[d]);
                    }
                }
            }
        }
        pos = end;
        if (run0 >= t0 && run1 <= t1) {
            R::store(dk + ((size_t)kv * s.N + key) * D, lane, ak);
            R::store(dv + ((size_t)kv * s.N + key) * D, lane, av);
        } else {  // slot 0: the run began before this tile; slot 1: it begins here and goes on
            float* ps = part + (((size_t)kv * s.tiles + tile) * 2 + (run0 < t0 ? 0 : 1)) * 2 * D;
            RowLoad<float, D>::store(ps, lane, ak);
            RowLoad<float, D>::store(ps + D, lane, av);
        }
    }
}

// ------------------------------------------------------------------ 4. join

template <typename T>
__global__ void __launch_bounds__(kThreads)
join_kernel(const BwdShape s, const int* __restrict__ base, const float* __restrict__ part, T* __restrict__ dk,
            T* __restrict__ dv) {
    const int lane = threadIdx.x & 31, kv = blockIdx.y;
    const int key = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (key >= s.N) return;
    const int* bs = base + (size_t)kv * (s.NB + 1);
    const int blk = key >> s.shift, kk = key - (blk << s.shift);
    const int run0 = bs[blk], run1 = bs[blk + 1];
    const int first = run0 / s.tile, last = run1 > run0 ? (run1 - 1) / s.tile : first;
    if (run1 > run0 && first == last) return;  // stored by the key pass
    const size_t slot = (size_t)2 * (s.D << s.shift);  // floats of a tile's slot
    const float* ps = part + (size_t)kv * s.tiles * 2 * slot + (size_t)kk * s.D;
    T* ok = dk + ((size_t)kv * s.N + key) * s.D;
    T* ov = dv + ((size_t)kv * s.N + key) * s.D;
    for (int d = 4 * lane; d < s.D; d += 128) {
        float k4[4] = {0.f, 0.f, 0.f, 0.f}, v4[4] = {0.f, 0.f, 0.f, 0.f};
        auto add = [&](const float* at) {
            const float4 x = *reinterpret_cast<const float4*>(at + d);
            const float4 y = *reinterpret_cast<const float4*>(at + (s.D << s.shift) + d);
            k4[0] += x.x;
            k4[1] += x.y;
            k4[2] += x.z;
            k4[3] += x.w;
            v4[0] += y.x;
            v4[1] += y.y;
            v4[2] += y.z;
            v4[3] += y.w;
        };
        if (run1 > run0) {
            add(ps + ((size_t)first * 2 + 1) * slot);
#pragma unroll 4
            for (int i = first + 1; i <= last; ++i) add(ps + (size_t)i * 2 * slot);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            store_from_f32(ok + d + t, k4[t]);
            store_from_f32(ov + d + t, v4[t]);
        }
    }
}

// dslopes[h]: the rows' shares, each thread's in row order, then a fixed tree.
__global__ void __launch_bounds__(1024) slope_join_kernel(const BwdShape s, const float* __restrict__ rows, float* dslopes) {
    __shared__ double sums[32];
    const int h = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double t = 0.0;
    for (int b = 0; b < s.B; ++b)
        for (int i = threadIdx.x; i < s.Nq; i += 1024) t += rows[((size_t)b * s.H + h) * s.Nq + i];
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) t += __shfl_xor_sync(kFull, t, o);
    if (lane == 0) sums[warp] = t;
    __syncthreads();
    if (threadIdx.x == 0) {
        double a = 0.0;
        for (int i = 0; i < 32; ++i) a += sums[i];
        dslopes[h] = (float)a;
    }
}

cudaError_t launched() {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e;
}

template <typename IdxT>
cudaError_t sort_lists(const GatherBwdArgs& a, const BwdShape& s, const BwdBuffers& w, cudaStream_t stream) {
    const unsigned kvs = (unsigned)(s.B * s.Hkv);
    const dim3 grid((unsigned)s.units, kvs, (unsigned)((s.NB + kKeyRange - 1) / kKeyRange));
    const size_t smem = (size_t)std::min(s.NB, kKeyRange) * sizeof(int);
    cudaError_t e;
    count_kernel<IdxT><<<grid, kThreads, smem, stream>>>(static_cast<const IdxT*>(a.f.idx), s, a.f.mods, w.keys, w.counts);
    if ((e = launched()) != cudaSuccess) return e;
    unit_scan_kernel<<<dim3((unsigned)((s.NB + 31) / 32), kvs), kThreads, 0, stream>>>(s, w.counts, w.base);
    if ((e = launched()) != cudaSuccess) return e;
    key_scan_kernel<<<kvs, 1024, 0, stream>>>(s, w.base);
    if ((e = launched()) != cudaSuccess) return e;
    place_kernel<<<grid, 32, smem, stream>>>(w.keys, s, w.counts, w.base, w.list);
    return launched();
}

template <typename T>
cudaError_t passes_typed(const GatherBwdArgs& a, const BwdShape& s, const BwdBuffers& w, cudaStream_t stream) {
    const T *q = static_cast<const T*>(a.f.q), *k = static_cast<const T*>(a.f.k), *v = static_cast<const T*>(a.f.v);
    const T *out = static_cast<const T*>(a.f.out), *dout = static_cast<const T*>(a.dout);
    T *dq = static_cast<T*>(a.dq), *dk = static_cast<T*>(a.dk), *dv = static_cast<T*>(a.dv);
    const ScoreMods& m = a.f.mods;
    const unsigned kvs = (unsigned)(s.B * s.Hkv);
    const long long rows = (long long)s.B * s.H * s.Nq;
    const unsigned row_grid = (unsigned)((rows + kWarps - 1) / kWarps);
    const dim3 key_grid((unsigned)((s.tiles + kWarps - 1) / kWarps), kvs);
    cudaError_t e;
    if (s.shift > 0 && gather_union_serves(a.f.dtype, s.H, s.Hkv, s.N, s.D, s.K)) {
        e = launch_row_pass_mma(a, s, w, stream);
    } else {
        switch (s.D) {
#define OSSA_BWD_CASE(DD)                                                                                        \
    case DD:                                                                                                     \
        row_pass_kernel<T, DD><<<row_grid, kThreads, 0, stream>>>(q, k, v, w.keys, out, dout, s, m, dq, w.delta, \
                                                                  w.slope_rows);                                 \
        break;
            OSSA_BWD_CASE(16)
            OSSA_BWD_CASE(32)
            OSSA_BWD_CASE(64)
            OSSA_BWD_CASE(128)
            OSSA_BWD_CASE(256)
#undef OSSA_BWD_CASE
            default: return cudaErrorInvalidValue;
        }
        e = launched();
    }
    if (e != cudaSuccess) return e;
    if (s.shift > 0) {
        e = launch_key_pass_mma(a, s, w, stream);
    } else {
        switch (s.D) {
#define OSSA_BWD_CASE(DD)                                                                                               \
    case DD:                                                                                                            \
        key_pass_kernel<T, DD><<<key_grid, kThreads, 0, stream>>>(q, k, v, dout, s, m, w.base, w.list, w.delta, dk, dv, \
                                                                  w.part);                                              \
        break;
            OSSA_BWD_CASE(16)
            OSSA_BWD_CASE(32)
            OSSA_BWD_CASE(64)
            OSSA_BWD_CASE(128)
            OSSA_BWD_CASE(256)
#undef OSSA_BWD_CASE
            default: return cudaErrorInvalidValue;
        }
        e = launched();
    }
    if (e != cudaSuccess) return e;
    join_kernel<T><<<dim3((unsigned)((s.N + kWarps - 1) / kWarps), kvs), kThreads, 0, stream>>>(s, w.base, w.part, dk, dv);
    if ((e = launched()) != cudaSuccess || !a.dslopes) return e;
    slope_join_kernel<<<s.H, 1024, 0, stream>>>(s, w.slope_rows, a.dslopes);
    return launched();
}

}  // namespace

size_t gather_bwd_workspace_bytes(int dtype, int B, int H, int Hkv, int Nq, int N, int D, int K, bool dslopes) {
    return make_layout(make_shape(dtype, B, H, Hkv, Nq, N, D, K), dslopes).total;
}

cudaError_t launch_gather_attn_bwd(const GatherBwdArgs& a, cudaStream_t stream) {
    BwdShape s = make_shape(a.f.dtype, a.f.B, a.f.H, a.f.Hkv, a.f.Nq, a.f.N, a.f.D, a.f.K);
    s.q0 = a.f.q0;
    s.causal = a.f.causal;
    const Layout l = make_layout(s, a.dslopes != nullptr);
    char* ws = static_cast<char*>(a.ws);
    BwdBuffers w{};
    w.keys = reinterpret_cast<int*>(ws + l.keys);
    w.counts = reinterpret_cast<int*>(ws + l.counts);
    w.base = reinterpret_cast<int*>(ws + l.base);
    w.list = reinterpret_cast<int*>(ws + l.list);
    w.delta = reinterpret_cast<float*>(ws + l.delta);
    w.part = reinterpret_cast<float*>(ws + l.part);
    w.slope_rows = a.dslopes ? reinterpret_cast<float*>(ws + l.slope_rows) : nullptr;
    const cudaError_t e = a.f.idx_is_64 ? sort_lists<int64_t>(a, s, w, stream) : sort_lists<int32_t>(a, s, w, stream);
    if (e != cudaSuccess) return e;
    return a.f.dtype == kF32 ? passes_typed<float>(a, s, w, stream) : passes_typed<__nv_bfloat16>(a, s, w, stream);
}

}  // namespace ossa
