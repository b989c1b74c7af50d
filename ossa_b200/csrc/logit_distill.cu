// Distillation from a teacher's top logits: loss and gradient over the vocabulary.
//
// Per row, student logits z (V values), teacher logits t at K listed entries:
//   p = softmax(t / tau) over the listed entries inside [0, V) (repeats count each time)
//   loss = tau^2 sum_k p_k (log p_k - (z_k / tau - lse(z / tau)))
//   dz_v = scale * tau * (softmax(z / tau)_v - sum of p_k listed at v)
// scale = row weight (/ the rows' weight sum for the mean) * incoming gradient.  A row
// without a listed entry weighs nothing; a row of weight 0 is not read, its loss and
// gradient are 0 whatever it holds.
//
// Bound: HBM, z read once and dz written once.  A cluster of C CTAs holds one row in registers (kNV 16-byte
// vectors a thread), so the row's maximum and sum and then the gradient come from one read; the CTAs exchange
// (max, sum) pairs through distributed shared memory (st.async on an mbarrier: a cluster barrier would wait
// for the CTA's stores of the row before).  The next row is on its way into shared memory meanwhile.  Clusters
// walk the rows with a fixed stride, as many as run at once.  Rows too long for that are read twice (kNV = 0).
// Exponents are taken as exp2((z - max) * log2(e) / tau), the difference first, so that entries at the
// type's lowest value and rows of them stay finite.
// Measured, loss and gradient: 4096 x 151936 bf16 (2.49 GB) 600 us, 4.1 TB/s; 4096 x 32000 fp32 211 us, 5.0 TB/s;
// 16 x 151936 bf16 15 us.  No unit bounds the 600: DRAM is busy for 44 % of its peak, the exponentials' unit for 53 % (two a
// value are 267 us of it at 16 a cycle and SM), issue slots for 45 %.  A CTA's warps take a row's sum, its exchange
// and its gradient in step, so each of these waits for the others.  Without the exponentials (a probe) 100 us go; a polynomial
// on the fp32 pipe for a quarter of them gave no change, for half of them +21 %; the first pass's exponentials kept
// for the gradient in 2 of a thread's 10 vectors -2 %, in 4 (spills) +7 %; neither is worth its code.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cstdint>

#include "bf16_dot.cuh"
#include "common.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace ossa {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;               // of the row kernel that hold a row's values
constexpr int kBlock = kThreads + 32;       // and a warp for the listed entries,
constexpr int kEntries = 4;                 // that many a lane in registers
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBatch = 4;  // vectors a thread has in flight where a row is read twice
constexpr int kMaxDevices = 64;
constexpr int kPrepThreads = 256;
constexpr int kPrepBlocks = 512;
constexpr float kLog2e = 1.4426950408889634f;

// Workspace: [counter 16 B][weight sums of the prep CTAs, double][row weight, T][row loss, T]
// [(p, p log p), T x K][p summed over equal entries, T x K][ids as int32, -1 outside [0, V), T x K]
struct Layout {
    size_t wsum, weight, loss, plogp, ptot, ids, total;
};

Layout layout(long long T, int K) {
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    Layout l;
    l.wsum = 256;
    l.weight = l.wsum + up(kPrepBlocks * sizeof(double));
    l.loss = l.weight + up((size_t)T * 4);
    l.plogp = l.loss + up((size_t)T * 4);
    l.ptot = l.plogp + up((size_t)T * K * 8);
    l.ids = l.ptot + up((size_t)T * K * 4);
    l.total = l.ids + up((size_t)T * K * 4);
    return l;
}

// The teacher's rows: p, p log p and the p of each entry summed over its repeats, the row's
// weight, and the CTA's share of the weight sum (rows in a fixed order).  A warp per row.
// log p = (t - max) / tau - log sum, the difference first and divided: neither a common offset of the row's logits nor
// their size costs p any of its digits, and rows of the type's lowest value stay finite.
template <typename IdT>
__global__ void __launch_bounds__(kPrepThreads)
distill_prep_kernel(const float* __restrict__ teacher, const IdT* __restrict__ ids, const float* __restrict__ row_weight,
                    int T, int V, int K, float tau, unsigned* counter, double* __restrict__ wsum,
                    float* __restrict__ weight, float2* __restrict__ plogp, float* __restrict__ ptot,
                    int* __restrict__ ids32) {
    constexpr int kPrepWarps = kPrepThreads / 32;
    __shared__ double s_sum[kPrepWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x == 0 && threadIdx.x == 0) *counter = 0u;
    double mine = 0.0;
    for (int r = blockIdx.x * kPrepWarps + warp; r < T; r += gridDim.x * kPrepWarps) {
        const size_t rk = (size_t)r * K;
        const float w = row_weight ? row_weight[r] : 1.f;
        float m = -INFINITY;
        bool any = false;
        for (int k = lane; k < K; k += 32) {
            const IdT id = ids[rk + k];
            const bool ok = id >= 0 && id < (IdT)V;
            ids32[rk + k] = ok ? (int)id : -1;
            if (ok) m = fmaxf(m, teacher[rk + k]);
            any = any || ok;
        }
        m = warp_max(m);
        any = __any_sync(kFull, any);
        __syncwarp();  // this row's ids32 are read by other lanes below
        float sum = 0.f;
        for (int k = lane; k < K; k += 32)
            if (ids32[rk + k] >= 0) sum += expf((teacher[rk + k] - m) / tau);
        sum = warp_sum(sum);
        const float log_sum = logf(sum);
        for (int k = lane; k < K; k += 32) {
            const bool ok = ids32[rk + k] >= 0;
            const float d = ok ? (teacher[rk + k] - m) / tau : 0.f, p = ok ? expf(d) / sum : 0.f;
            plogp[rk + k] = make_float2(p, p == 0.f ? 0.f : p * (d - log_sum));
        }
        __syncwarp();
        // p of equal entries summed in list order (every repeat gets the same sum)
        for (int k0 = 0; k0 < K; k0 += 32) {
            const int k = k0 + lane;
            const int id = k < K ? ids32[rk + k] : -2;
            float tot = 0.f;
            for (int j0 = 0; j0 < K; j0 += 32) {
                const bool in = j0 + lane < K;
                const int jd = in ? ids32[rk + j0 + lane] : -1;
                const float pj = in ? plogp[rk + j0 + lane].x : 0.f;
                const int n = min(32, K - j0);
                for (int i = 0; i < n; ++i) {
                    const int other = __shfl_sync(kFull, jd, i);
                    const float po = __shfl_sync(kFull, pj, i);
                    if (other == id) tot += po;
                }
            }
            if (k < K) ptot[rk + k] = tot;
        }
        const float we = any ? w : 0.f;
        if (lane == 0) weight[r] = we;
        mine += we;
    }
    if (lane == 0) s_sum[warp] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < kPrepWarps; ++i) t += s_sum[i];
        wsum[blockIdx.x] = t;
    }
}

struct Rows {
    const void* z;
    long long sb, st;  // row r: z + (r / inner) * sb + (r % inner) * st
    int inner, T, V, K;  // T rows
    const float* grad;  // nullptr: 1
    int grad_step;      // 0: one value, 1: one per row
    int skip_if_one;
    int mean;
    int prep_blocks;
    float tau;
    unsigned* counter;
    const double* wsum;
    const float *weight, *ptot;
    const float2* plogp;
    const int* ids;
    float *loss_rows, *loss;  // nullptr: not wanted
    void* dz;                 // (T, V) contiguous, nullptr: not wanted
};

template <typename T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int n = 4;
    static constexpr uint32_t neg = 0xff800000u;  // -inf
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x);
        x[1] = __uint_as_float(v.y);
        x[2] = __uint_as_float(v.z);
        x[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ float top(const uint4& v) {
        return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
    // value - m
    static __device__ __forceinline__ void minus(const uint4& v, float m, float (&x)[4]) {
        unpack(v, x);
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] -= m;
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[4]) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int n = 8;
    static constexpr uint32_t neg = 0xff80ff80u;
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
        unpack_bf16x2(v.x, x[0], x[1]);
        unpack_bf16x2(v.y, x[2], x[3]);
        unpack_bf16x2(v.z, x[4], x[5]);
        unpack_bf16x2(v.w, x[6], x[7]);
    }
    static __device__ __forceinline__ float top(const uint4& v) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
        const __nv_bfloat162 t = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(__low2float(t), __high2float(t));
    }
    // value - m as value * 1 + (-m): one mixed-precision fma each, nothing to convert
    static __device__ __forceinline__ void minus(const uint4& v, float m, float (&x)[8]) {
        constexpr uint32_t one = 0x3f803f80u;
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            x[2 * t] = fma_bf16<false>(w[t], one, -m);
            x[2 * t + 1] = fma_bf16<true>(w[t], one, -m);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
        uint4 o;
        uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * t], x[2 * t + 1]);
            w[t] = *reinterpret_cast<const uint32_t*>(&b);
        }
        return o;
    }
};

// Where a row is read twice: the first read keeps it in L2, the second and the gradient's stores let go.
__device__ __forceinline__ uint64_t policy_keep() {
    uint64_t p;
    asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
    return p;
}

__device__ __forceinline__ uint64_t policy_drop() {
    uint64_t p;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}

__device__ __forceinline__ uint4 load_hint(const uint4* p, uint64_t policy) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p), "l"(policy));
    return v;
}

__device__ __forceinline__ void store_hint(uint4* p, const uint4& v, uint64_t policy) {
    asm volatile("st.global.L2::cache_hint.v4.u32 [%0], {%1, %2, %3, %4}, %5;" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z),
                 "r"(v.w), "l"(policy)
                 : "memory");
}

// 2^x, two units in the last place; below 2^-126 it is 0.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// x *= c, two lanes of the fp32 pipe per instruction; each product rounded as a plain one.
template <int E>
__device__ __forceinline__ void scale_pairs(float (&x)[E], float c) {
    uint64_t cc;
    asm("mov.b64 %0, {%1, %1};" : "=l"(cc) : "f"(c));
#pragma unroll
    for (int t = 0; t < E; t += 2) {
        uint64_t v;
        asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x[t]), "f"(x[t + 1]));
        asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(cc));
        asm("mov.b64 {%0, %1}, %2;" : "=f"(x[t]), "=f"(x[t + 1]) : "l"(v));
    }
}

// exp2((value - m) c) of a vector.
template <typename V, int E>
__device__ __forceinline__ void exp_of(const uint4& v, float m, float c, float (&x)[E]) {
    V::minus(v, m, x);
    scale_pairs(x, c);
#pragma unroll
    for (int t = 0; t < E; ++t) x[t] = exp2_fast(x[t]);
}

// Pairwise sum.
template <int E>
__device__ __forceinline__ float sum_of(float (&x)[E]) {
#pragma unroll
    for (int w = E / 2; w >= 1; w /= 2) {
#pragma unroll
        for (int t = 0; t < w; ++t) x[t] += x[t + w];
    }
    return x[0];
}

// Where a row's values lie: `head` single values up to a 16-byte boundary, nb vectors, single values.
// kAligned: every row begins on such a boundary and is whole vectors.
template <typename T, bool kAligned>
struct RowAt {
    const T* z;
    int head, nb, tail0;
    __device__ __forceinline__ RowAt(const Rows& a, int r) {
        const int o = a.inner == a.T ? 0 : r / a.inner;
        z = static_cast<const T*>(a.z) + (size_t)(o * a.sb + (r - o * a.inner) * a.st);
        head = kAligned ? 0 : min(a.V, (int)(((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / sizeof(T)));
        nb = (a.V - head) / Vec<T>::n;
        tail0 = head + nb * Vec<T>::n;
    }
    __device__ __forceinline__ const uint4* vec() const { return reinterpret_cast<const uint4*>(z + head); }
};

// (max, sum of exp2((z - max) c)) over lanes that differ in the bits below kLanes.
template <int kLanes>
__device__ __forceinline__ void join_lanes(float& m, float& l, float c) {
    float top = m;
    if constexpr (kLanes == 32) {
        asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(m));
    } else {
#pragma unroll
        for (int o = kLanes / 2; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
    }
    l *= exp2_fast((m - top) * c);
#pragma unroll
    for (int o = kLanes / 2; o >= 1; o >>= 1) l += __shfl_xor_sync(kFull, l, o);
    m = top;
}

// Sum over the CTA in a fixed order, in every thread.
__device__ __forceinline__ double block_sum(double x, double* buf) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = x;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < kBlock / 32; ++i) t += buf[i];
    return t;
}

// CTAs of the row kernel per SM that its registers leave room for.
constexpr int row_ctas(int nv) { return nv >= 1 && nv <= 4 ? 3 : 2; }

// Writes a pair into the shared memory of another CTA of the cluster and counts its bytes there.  Unlike a
// cluster barrier this does not wait for the CTA's own stores to global memory.
__device__ __forceinline__ void send_pair(const float2* slot, const uint64_t* bar, int to, float m, float l) {
    uint32_t at, b;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(sm100::smem_u32(slot)), "r"(to));
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(sm100::smem_u32(bar)), "r"(to));
    const uint64_t v = (uint64_t)__float_as_uint(l) << 32 | __float_as_uint(m);
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(at), "l"(v), "r"(b)
                 : "memory");
}

template <typename T, int kNV, bool kAligned>
__global__ void __launch_bounds__(kBlock, row_ctas(kNV)) distill_rows_kernel(const Rows a) {
    using Row = RowAt<T, kAligned>;
    using V8 = Vec<T>;
    constexpr int E = V8::n;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int clusters = gridDim.x / C, me = blockIdx.x / C;
    if (a.skip_if_one && a.grad && *a.grad == 1.f) return;  // the same for every CTA
    // what a row leaves here is read behind the next row's barrier at the latest: two copies
    __shared__ float2 s_warp[2][kWarps];
    __shared__ float2 s_pair[2][kMaxCluster];  // (max, sum) of every CTA of the cluster
    __shared__ uint64_t s_bar[2];
    __shared__ double s_sum[kBlock / 32];
    __shared__ bool s_last;
    const float c = kLog2e / a.tau;
    // What a unit of row weight counts in the total, times 2^-up: where fp32 does not hold the inverse of the weights' sum,
    // a power of two goes over to the incoming gradient.
    float unit = 1.f;
    int up = 0;
    if (a.mean) {
        double w = 0.0;
        for (int i = tid; i < a.prep_blocks; i += kBlock) w += a.wsum[i];
        w = block_sum(w, s_sum);
        if (w < 0x1p-100) up = 100;
        else if (w > 0x1p+100) up = -100;
        unit = w != 0.0 ? (float)(1.0 / scalbn(w, up)) : 0.f;
    }
    if (C > 1) {
        if (tid == 0) {
            sm100::mbar_init(&s_bar[0], 1);
            sm100::mbar_init(&s_bar[1], 1);
            sm100::fence_mbar_init();
        }
        cluster.sync();  // every CTA has begun: its shared memory may be written from another
    }
    const float g_all = scalbnf(a.grad && a.grad_step == 0 ? *a.grad : 1.f, up);
    auto row_scale = [&](int r, float w) { return (a.grad && a.grad_step ? scalbnf(a.grad[r], up) : g_all) * w * unit * a.tau; };
    auto weight_at = [&](int r) { return r < a.T ? a.weight[r] : 0.f; };
    // The barrier behind a row's sums: the list warp and the others reach it from different places.
    auto row_barrier = [] { asm volatile("bar.sync 1, %0;" ::"n"(kBlock) : "memory"); };
    // Behind it: maximum and sum of the whole row, the same bits in every warp of the cluster.  n: rows before.
    auto row_sums = [&](int n, float& m, float& l) {
        const int copy = n & 1;
        if (C == 1 || warp == 0) {
            const float2 x = s_warp[copy][lane % kWarps];
            m = x.x;
            l = x.y;
            join_lanes<kWarps>(m, l, c);
        }
        if (C > 1) {
            if (tid == 0) sm100::mbar_arrive_expect_tx(&s_bar[copy], 8 * C);
            if (warp == 0 && lane < C) send_pair(&s_pair[copy][rank], &s_bar[copy], lane, m, l);
            const bool ok = sm100::mbar_wait(&s_bar[copy], (n >> 1) & 1);
            const float2 x = lane % kMaxCluster < C ? s_pair[copy][lane % kMaxCluster] : make_float2(-FLT_MAX, 0.f);
            m = x.x;
            l = ok ? x.y : NAN;  // a wait that ran out shows in the loss and the gradient
            join_lanes<kMaxCluster>(m, l, c);
        }
    };
    float w_next = weight_at(me), w_after = weight_at(me + clusters);
    int n = 0;  // rows this cluster has read

    if (warp == kWarps) {
        // ---- the list warp: it holds no values of a row but its listed entries, kEntries a lane, loaded
        // while the others sum up the row.  Behind the sums rank 0 adds up the row's loss; the entries of
        // this CTA's part are written over the gradient behind the next row's barrier, when the others
        // have stored it.  Entries past 32 kEntries are taken there one by one.
        int at_v[kEntries];  // place of the row before, -1: nothing to write here; value
        float at_x[kEntries];
        int late_row = -1;
        float late_m = 0.f, late_inv = 0.f, late_scale = 0.f;
        auto part_of = [&](const Row& row, int v) {
            return v < row.head || v >= row.tail0 ? 0 : ((v - row.head) / E / kThreads) & (C - 1);
        };
        auto write_late = [&] {
            if (late_row < 0) return;
            T* out = static_cast<T*>(a.dz) + (size_t)late_row * a.V;
#pragma unroll
            for (int t = 0; t < kEntries; ++t)
                if (at_v[t] >= 0) store_from_f32(out + at_v[t], at_x[t]);
            if (a.K > 32 * kEntries) {
                const Row row(a, late_row);
                for (int k = 32 * kEntries + lane; k < a.K; k += 32) {
                    const size_t e = (size_t)late_row * a.K + k;
                    const int v = a.ids[e];
                    if (v >= 0 && part_of(row, v) == rank)
                        store_from_f32(out + v, (exp2_fast((to_f32(row.z[v]) - late_m) * c) * late_inv - a.ptot[e]) *
                                                    late_scale);
                }
            }
            late_row = -1;
        };
        for (int r = me; r < a.T; r += clusters) {
            const float w = w_next;
            w_next = w_after;
            w_after = weight_at(r + 2 * clusters);
            if (w == 0.f) continue;
            const Row row(a, r);
            int v[kEntries];
            float z[kEntries], pt[kEntries];
            float2 pl[kEntries];
#pragma unroll
            for (int t = 0; t < kEntries; ++t) {
                const int k = lane + 32 * t;
                const size_t e = (size_t)r * a.K + k;
                v[t] = k < a.K ? a.ids[e] : -1;
                pt[t] = k < a.K ? a.ptot[e] : 0.f;
                pl[t] = k < a.K ? a.plogp[e] : make_float2(0.f, 0.f);
            }
#pragma unroll
            for (int t = 0; t < kEntries; ++t) z[t] = v[t] >= 0 ? to_f32(row.z[v[t]]) : 0.f;
            row_barrier();
            write_late();
            float m = 0.f, l = 0.f;
            row_sums(n, m, l);
            ++n;
            const float inv = 1.f / l, scale = row_scale(r, w);
            if (a.loss_rows && rank == 0) {
                const float log_l = logf(l);
                // tau times an entry's share, which no small tau takes out of range; a teacher's NaN shows, an entry
                // of p = 0 counts nothing
                auto term = [&](float2 x, float zk) {
                    return x.x == 0.f ? 0.f : a.tau * x.y - x.x * ((zk - m) - a.tau * log_l);
                };
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < kEntries; ++t) sum += v[t] >= 0 ? term(pl[t], z[t]) : 0.f;
                for (int k = 32 * kEntries + lane; k < a.K; k += 32) {
                    const size_t e = (size_t)r * a.K + k;
                    const int vk = a.ids[e];
                    if (vk >= 0) sum += term(a.plogp[e], to_f32(row.z[vk]));
                }
                sum = warp_sum(sum);
                if (lane == 0) a.loss_rows[r] = sum * a.tau;
            }
            if (a.dz) {
#pragma unroll
                for (int t = 0; t < kEntries; ++t) {
                    at_v[t] = v[t] >= 0 && part_of(row, v[t]) == rank ? v[t] : -1;
                    at_x[t] = (exp2_fast((z[t] - m) * c) * inv - pt[t]) * scale;
                }
                late_row = r;
                late_m = m;
                late_inv = inv;
                late_scale = scale;
            }
        }
        row_barrier();
        write_late();
    } else {
        // ---- the other warps: the row's values
        const uint64_t keep = policy_keep(), drop = policy_drop();
        const int first = rank * kThreads + tid, stride = C * kThreads;
        // this thread's vectors of the row in work; the next row's are on their way into shared memory (every
        // thread copies and reads its own) from the moment these are in registers
        uint4 d[kNV > 0 ? kNV : 1];
        extern __shared__ __align__(16) uint4 s_ahead[];  // kNV x kThreads
        auto fetch = [&](const Row& row) {
#pragma unroll
            for (int j = 0; j < kNV; ++j) {
                const int i = first + j * stride;
                if (i < row.nb)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                     sm100::smem_u32(s_ahead + j * kThreads + tid)),
                                 "l"(row.vec() + i)
                                 : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        bool loaded = false;
        for (int r = me; r < a.T; r += clusters) {
            const float w = w_next;
            const int r_next = r + clusters;
            w_next = w_after;
            w_after = weight_at(r_next + clusters);
            T* out = a.dz ? static_cast<T*>(a.dz) + (size_t)r * a.V : nullptr;
            if (w == 0.f) {  // the cluster's CTAs agree
                if (rank == 0 && tid == 0 && a.loss_rows) a.loss_rows[r] = 0.f;
                if (out)
                    for (int v = first; v < a.V; v += stride) store_from_f32(out + v, 0.f);
                loaded = false;
                continue;
            }
            const Row at(a, r);
            Row next(a, r_next < a.T ? r_next : r);
            if (w_next == 0.f) next.nb = 0;  // no next row, or one that is not read
            const T* z = at.z;
            const int head = at.head, nb = at.nb, tail0 = at.tail0;
            const uint4* zv = at.vec();
            float m = -FLT_MAX, l = 0.f, zo = -INFINITY;
            int odd = -1;
            if constexpr (kNV > 0) {
                if (!loaded) fetch(at);
                asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
                for (int j = 0; j < kNV; ++j)
                    d[j] = first + j * stride < nb ? s_ahead[j * kThreads + tid] : make_uint4(V8::neg, V8::neg, V8::neg, V8::neg);
            }
            loaded = true;
            // the single values lie with rank 0: threads 0.. the head, threads 32.. the tail
            if (!kAligned && rank == 0 && tid < head) odd = tid;
            if (!kAligned && rank == 0 && tid >= 32 && tail0 + tid - 32 < a.V) odd = tail0 + tid - 32;
            if (odd >= 0) zo = to_f32(z[odd]);

            // ---- maximum and sum of the row
            m = fmaxf(zo, m);
            if constexpr (kNV > 0) {
#pragma unroll
                for (int j = 0; j < kNV; ++j) m = fmaxf(m, V8::top(d[j]));
                fetch(next);  // behind the last use of what it writes over
#pragma unroll
                for (int j = 0; j < kNV; ++j) {
                    float x[E];
                    exp_of<V8>(d[j], m, c, x);
                    l += sum_of(x);
                }
            } else {
                for (int i0 = first; i0 < nb; i0 += kBatch * stride) {
                    uint4 x4[kBatch];
                    float mn = m;
#pragma unroll
                    for (int t = 0; t < kBatch; ++t)
                        x4[t] = i0 + t * stride < nb ? load_hint(zv + i0 + t * stride, keep)
                                                     : make_uint4(V8::neg, V8::neg, V8::neg, V8::neg);
#pragma unroll
                    for (int t = 0; t < kBatch; ++t) mn = fmaxf(mn, V8::top(x4[t]));
                    l *= exp2_fast((m - mn) * c);
                    m = mn;
#pragma unroll
                    for (int t = 0; t < kBatch; ++t) {
                        float x[E];
                        exp_of<V8>(x4[t], m, c, x);
                        l += sum_of(x);
                    }
                }
            }
            if (odd >= 0) l += exp2_fast((zo - m) * c);
            join_lanes<32>(m, l, c);
            if (lane == 0) s_warp[n & 1][warp] = make_float2(m, l);
            row_barrier();
            row_sums(n, m, l);
            ++n;

            // ---- gradient
            if (out) {
                const float scale = row_scale(r, w), inv = 1.f / l;
                const float qs = inv * scale;
                const bool same_phase = kAligned || ((reinterpret_cast<uintptr_t>(out + head)) & 15) == 0;
                auto emit = [&](int i, const uint4& raw) {
                    float x[E];
                    exp_of<V8>(raw, m, c, x);
                    scale_pairs(x, qs);
                    if (same_phase) {
                        store_hint(reinterpret_cast<uint4*>(out + head) + i, V8::pack(x), drop);
                    } else {
#pragma unroll
                        for (int t = 0; t < E; ++t) store_from_f32(out + head + (size_t)i * E + t, x[t]);
                    }
                };
                if constexpr (kNV > 0) {
#pragma unroll
                    for (int j = 0; j < kNV; ++j) {
                        const int i = first + j * stride;
                        if (i < nb) emit(i, d[j]);
                    }
                } else {
                    for (int i0 = first; i0 < nb; i0 += kBatch * stride) {
                        uint4 x4[kBatch];
#pragma unroll
                        for (int t = 0; t < kBatch; ++t)
                            if (i0 + t * stride < nb) x4[t] = load_hint(zv + i0 + t * stride, drop);
#pragma unroll
                        for (int t = 0; t < kBatch; ++t)
                            if (i0 + t * stride < nb) emit(i0 + t * stride, x4[t]);
                    }
                }
                if (odd >= 0) store_from_f32(out + odd, exp2_fast((zo - m) * c) * qs);
            }
        }
        row_barrier();  // the list warp writes the last row's entries behind it
    }
    if (C > 1) cluster.sync();  // no CTA leaves while another may still write to it
    if (!a.loss) return;
    // the CTA that ends last adds the rows' losses, in an order that is always the same
    __syncthreads();  // the last row's loss is written
    if (tid == 0) {
        __threadfence();
        s_last = atomicAdd(a.counter, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    double t = 0.0;
    for (int r = tid; r < a.T; r += kBlock) {
        const float w = __ldcg(a.weight + r);
        if (w != 0.f) t += (double)w * (double)__ldcg(a.loss_rows + r);
    }
    t = block_sum(t, s_sum);
    if (tid == 0) *a.loss = (float)(scalbn(t, up) * (double)unit);
}

// Cluster size and vectors per thread.  A row of `vecs` vectors wants the fewest CTAs that hold it in at
// most 10 vectors a thread; few rows want more CTAs a row, up to 8, while they leave SMs without work (V =
// 151936 bf16, clusters of 1, 2, 4, 8: one row 31, 23, 17, 14 us, 64 rows 32, 24, 21, 21).  Rows of more than 16
// vectors a thread in 8 CTAs (over 262,144 bf16 values) are read twice; where both can run, 4096 x 151936 takes
// 600 us held and 630 read twice (clusters of 2), 4096 x 32000 fp32 211 and 249.
void pick(int T, long long vecs, int sms, int* C, int* nv) {
    int c = 1;
    while (c < kMaxCluster && vecs > (long long)c * kThreads * 10) c *= 2;
    while (c < kMaxCluster && (long long)T * c * 2 <= 2 * sms && vecs > (long long)c * kThreads) c *= 2;
    const long long per = (vecs + (long long)c * kThreads - 1) / ((long long)c * kThreads);
    *C = c;
    *nv = per <= 16 ? (int)std::max<long long>(per, 1) : 0;
}

template <typename T, int kNV, bool kAligned>
cudaError_t launch_nv(const Rows& a, int C, cudaStream_t stream) {
    auto kern = distill_rows_kernel<T, kNV, kAligned>;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)C);
    cfg.blockDim = dim3(kBlock);
    cfg.stream = stream;
    cfg.dynamicSmemBytes = (size_t)kNV * kThreads * 16;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    // as many clusters as run at once (a GPC's SMs do not divide evenly): each walks its share of the rows
    static std::atomic<int> resident[kMaxDevices][4];  // by device and log2 C
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const int lc = C == 1 ? 0 : C == 2 ? 1 : C == 4 ? 2 : 3;
    int n = dev < kMaxDevices ? resident[dev][lc].load(std::memory_order_relaxed) : 0;
    if (n <= 0) {
        if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cfg.dynamicSmemBytes)) !=
            cudaSuccess)
            return e;
        if ((e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg)) != cudaSuccess) return e;
        n = std::max(n, 1);
        if (dev < kMaxDevices) resident[dev][lc].store(n, std::memory_order_relaxed);
    }
    cfg.gridDim = dim3((unsigned)(std::min(a.T, n) * C));
    e = cudaLaunchKernelEx(&cfg, kern, a);
    if (e == cudaSuccess) note_launch();
    return e;
}

template <typename T, bool kAligned>
cudaError_t launch_rows(const Rows& a, cudaStream_t stream) {
    const int sms = device_sm_count();
    int C = 1, nv = 0;
    pick(a.T, (a.V + Vec<T>::n - 1) / Vec<T>::n, sms, &C, &nv);
    switch (nv) {
        case 1: return launch_nv<T, 1, kAligned>(a, C, stream);
        case 2: return launch_nv<T, 2, kAligned>(a, C, stream);
        case 3: return launch_nv<T, 3, kAligned>(a, C, stream);
        case 4: return launch_nv<T, 4, kAligned>(a, C, stream);
        case 5: return launch_nv<T, 5, kAligned>(a, C, stream);
        case 6: return launch_nv<T, 6, kAligned>(a, C, stream);
        case 7: case 8: return launch_nv<T, 8, kAligned>(a, C, stream);
        case 9: case 10: return launch_nv<T, 10, kAligned>(a, C, stream);
        case 11: case 12: return launch_nv<T, 12, kAligned>(a, C, stream);
        case 0: return launch_nv<T, 0, kAligned>(a, C, stream);
        default: return launch_nv<T, 16, kAligned>(a, C, stream);
    }
}

Rows make_rows(const LogitDistillArgs& a) {
    const Layout l = layout((long long)a.outer * a.inner, a.K);
    char* ws = static_cast<char*>(a.ws);
    Rows r{};
    r.z = a.z;
    r.sb = a.sb;
    r.st = a.st;
    r.inner = a.inner;
    r.T = a.outer * a.inner;
    r.V = a.V;
    r.K = a.K;
    r.ids = reinterpret_cast<const int*>(ws + l.ids);
    r.mean = a.mean;
    r.prep_blocks = (int)std::min(kPrepBlocks, (r.T + kPrepThreads / 32 - 1) / (kPrepThreads / 32));
    r.tau = a.tau;
    r.counter = reinterpret_cast<unsigned*>(ws);
    r.wsum = reinterpret_cast<const double*>(ws + l.wsum);
    r.weight = reinterpret_cast<const float*>(ws + l.weight);
    r.plogp = reinterpret_cast<const float2*>(ws + l.plogp);
    r.ptot = reinterpret_cast<const float*>(ws + l.ptot);
    r.loss_rows = a.loss_rows ? a.loss_rows : reinterpret_cast<float*>(ws + l.loss);
    r.loss = a.loss;
    r.dz = a.dz;
    return r;
}

template <typename T>
cudaError_t launch_by_place(const Rows& r, cudaStream_t stream) {
    constexpr int E = Vec<T>::n;
    const bool aligned = r.V % E == 0 && r.sb % E == 0 && r.st % E == 0 && reinterpret_cast<uintptr_t>(r.z) % 16 == 0 &&
                         reinterpret_cast<uintptr_t>(r.dz) % 16 == 0;
    return aligned ? launch_rows<T, true>(r, stream) : launch_rows<T, false>(r, stream);
}

cudaError_t launch_by_type(const LogitDistillArgs& a, const Rows& r, cudaStream_t stream) {
    return a.dtype == kF32 ? launch_by_place<float>(r, stream) : launch_by_place<__nv_bfloat16>(r, stream);
}

}  // namespace

size_t logit_distill_workspace_bytes(long long T, int K) { return layout(T, K).total; }

cudaError_t launch_logit_distill_fwd(const LogitDistillArgs& a, cudaStream_t stream) {
    Rows r = make_rows(a);
    double* wsum = const_cast<double*>(r.wsum);
    float *weight = const_cast<float*>(r.weight), *ptot = const_cast<float*>(r.ptot);
    float2* plogp = const_cast<float2*>(r.plogp);
    if (a.ids_are_64)
        distill_prep_kernel<int64_t><<<r.prep_blocks, kPrepThreads, 0, stream>>>(
            a.teacher, static_cast<const int64_t*>(a.ids), a.row_weight, r.T, a.V, a.K, a.tau, r.counter, wsum, weight,
            plogp, ptot, const_cast<int*>(r.ids));
    else
        distill_prep_kernel<int32_t><<<r.prep_blocks, kPrepThreads, 0, stream>>>(
            a.teacher, static_cast<const int32_t*>(a.ids), a.row_weight, r.T, a.V, a.K, a.tau, r.counter, wsum, weight,
            plogp, ptot, const_cast<int*>(r.ids));
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    note_launch();
    return launch_by_type(a, r, stream);
}

cudaError_t launch_logit_distill_bwd(const LogitDistillArgs& a, cudaStream_t stream) {
    Rows r = make_rows(a);
    r.grad = a.grad;
    r.grad_step = a.grad_per_row;
    r.skip_if_one = a.skip_if_one;
    r.loss_rows = nullptr;
    r.loss = nullptr;
    return launch_by_type(a, r, stream);
}

}  // namespace ossa
