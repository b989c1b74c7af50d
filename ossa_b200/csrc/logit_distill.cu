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
// Bound: HBM, z read once and dz written once.  A cluster of C CTAs holds one row in
// registers (kNV 16-byte vectors a thread), so the row's maximum and sum and then the
// gradient come from one read: the CTAs exchange (max, sum) pairs through distributed
// shared memory.  Clusters walk the rows with a fixed stride.  Rows too long for that are
// read twice (kNV = 0).  Exponents are taken as exp2((z - max) * log2(e) / tau), the
// difference first, so that entries at the type's lowest value and rows of them stay finite.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cstdint>

#include "bf16_dot.cuh"
#include "common.cuh"
#include "kernels.h"

namespace ossa {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxDevices = 64;
constexpr int kPrepThreads = 256;
constexpr int kPrepBlocks = 512;  // at most kThreads: the row kernel adds their weight sums, one per thread
constexpr float kLog2e = 1.4426950408889634f;

// Workspace: [counter 16 B][weight sums of the prep CTAs, double][row weight, T][row loss, T]
// [log p, T x K][p summed over equal entries, T x K]
struct Layout {
    size_t wsum, weight, loss, logp, ptot, total;
};

Layout layout(long long T, int K) {
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    Layout l;
    l.wsum = 256;
    l.weight = l.wsum + up(kPrepBlocks * sizeof(double));
    l.loss = l.weight + up((size_t)T * 4);
    l.logp = l.loss + up((size_t)T * 4);
    l.ptot = l.logp + up((size_t)T * K * 4);
    l.total = l.ptot + up((size_t)T * K * 4);
    return l;
}

// The teacher's rows: log p and the p of each entry summed over its repeats, the row's
// weight, and the CTA's share of the weight sum (rows in a fixed order).  A warp per row.
template <typename IdT>
__global__ void __launch_bounds__(kPrepThreads)
distill_prep_kernel(const float* __restrict__ teacher, const IdT* __restrict__ ids, const float* __restrict__ row_weight,
                    long long T, int V, int K, float inv_tau, unsigned* counter, double* __restrict__ wsum,
                    float* __restrict__ weight, float* __restrict__ logp, float* __restrict__ ptot) {
    __shared__ double s_sum[kPrepThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x == 0 && threadIdx.x == 0) *counter = 0u;
    double mine = 0.0;
    for (long long r = (long long)blockIdx.x * (kPrepThreads / 32) + warp; r < T;
         r += (long long)gridDim.x * (kPrepThreads / 32)) {
        const float* tr = teacher + r * K;
        const IdT* ir = ids + r * K;
        const float w = row_weight ? row_weight[r] : 1.f;
        float m = -INFINITY;
        bool any = false;
        for (int k = lane; k < K; k += 32) {
            const long long id = (long long)ir[k];
            if (id >= 0 && id < V) {
                any = true;
                m = fmaxf(m, tr[k] * inv_tau);
            }
        }
        m = warp_max(m);
        any = __any_sync(kFull, any);
        const float m0 = m == -INFINITY ? 0.f : m;
        float sum = 0.f;
        for (int k = lane; k < K; k += 32) {
            const long long id = (long long)ir[k];
            if (id >= 0 && id < V) sum += expf(tr[k] * inv_tau - m0);
        }
        const float lse = m0 + logf(warp_sum(sum));
        for (int k = lane; k < K; k += 32) {
            const long long id = (long long)ir[k];
            const bool ok = id >= 0 && id < V;
            logp[r * K + k] = ok ? tr[k] * inv_tau - lse : -INFINITY;
        }
        __syncwarp();
        // p of equal entries summed in list order (every repeat gets the same sum)
        for (int k0 = 0; k0 < K; k0 += 32) {
            const int k = k0 + lane;
            const long long id = k < K ? (long long)ir[k] : -1;
            float tot = 0.f;
            for (int j0 = 0; j0 < K; j0 += 32) {
                const bool in = j0 + lane < K;
                const long long jd = in ? (long long)ir[j0 + lane] : -1;
                const float pj = in ? expf(logp[r * K + j0 + lane]) : 0.f;
                const int n = min(32, K - j0);
                for (int i = 0; i < n; ++i) {
                    const long long other = __shfl_sync(kFull, jd, i);
                    const float po = __shfl_sync(kFull, pj, i);
                    if (other == id) tot += po;
                }
            }
            if (k < K) ptot[r * K + k] = tot;
        }
        const float we = any ? w : 0.f;
        if (lane == 0) weight[r] = we;
        mine += we;
    }
    if (lane == 0) s_sum[warp] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < kPrepThreads / 32; ++i) t += s_sum[i];
        wsum[blockIdx.x] = t;
    }
}

struct Rows {
    const void* z;
    long long sb, st;  // row r: z + (r / inner) * sb + (r % inner) * st
    int inner, T, V, K;  // T rows
    const void* ids;
    const float* grad;  // nullptr: 1
    int grad_step;      // 0: one value, 1: one per row
    int skip_if_one;
    int mean;
    int prep_blocks;
    float tau;
    unsigned* counter;
    const double* wsum;
    const float *weight, *logp, *ptot;
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

__device__ __forceinline__ uint4 load_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
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
template <typename T>
struct RowAt {
    const T* z;
    int head, nb, tail0;
    __device__ __forceinline__ RowAt(const Rows& a, int r) {
        const int o = a.inner == a.T ? 0 : r / a.inner;
        z = static_cast<const T*>(a.z) + (size_t)(o * a.sb + (r - o * a.inner) * a.st);
        head = min(a.V, (int)(((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / sizeof(T)));
        nb = (a.V - head) / Vec<T>::n;
        tail0 = head + nb * Vec<T>::n;
    }
    __device__ __forceinline__ const uint4* vec() const { return reinterpret_cast<const uint4*>(z + head); }
};

// (max, sum of exp2((z - max) c)) over lanes that differ in the bits below kLanes.
template <int kLanes>
__device__ __forceinline__ void join_lanes(float& m, float& l, float c) {
    float top = m;
#pragma unroll
    for (int o = kLanes / 2; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
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
    for (int i = 0; i < kWarps; ++i) t += buf[i];
    return t;
}

template <typename T, typename IdT, int kNV>
__global__ void __launch_bounds__(kThreads, kNV <= 6 ? 2 : 1) distill_rows_kernel(const Rows a) {
    using V8 = Vec<T>;
    constexpr int E = V8::n;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int clusters = gridDim.x / C, me = blockIdx.x / C;
    if (a.skip_if_one && a.grad && *a.grad == 1.f) return;  // the same for every CTA
    __shared__ float2 s_warp[kWarps];
    __shared__ float s_part[kWarps];
    __shared__ float2 s_pair[2][kMaxCluster];  // (max, sum) of every CTA of the cluster, by row parity
    __shared__ double s_sum[kWarps];
    __shared__ bool s_last;
    const float c = kLog2e / a.tau;
    float unit = 1.f;  // what a unit of row weight counts in the total
    if (a.mean) {
        const double w = block_sum(tid < a.prep_blocks ? a.wsum[tid] : 0.0, s_sum);
        unit = w != 0.0 ? (float)(1.0 / w) : 0.f;
    }
    cluster.sync();  // every CTA has begun: its shared memory may be written from another
    auto row_scale = [&](int r, float w) {
        return (a.grad ? a.grad[(size_t)r * a.grad_step] : 1.f) * w * unit * a.tau;
    };
    int parity = 0;
    const int first = rank * kThreads + tid, stride = C * kThreads;
    // this thread's vectors of the row in work; each is replaced by the next row's as soon as it is used
    uint4 d[kNV > 0 ? kNV : 1];
    auto load = [&](int j, const RowAt<T>& row) {
        const int i = first + j * stride;
        d[j] = i < row.nb ? load_stream(row.vec() + i) : make_uint4(V8::neg, V8::neg, V8::neg, V8::neg);
    };
    float w_next = me < a.T ? a.weight[me] : 0.f;
    bool loaded = false;
    for (int r = me; r < a.T; r += clusters) {
        const float w = w_next;
        w_next = r + clusters < a.T ? a.weight[r + clusters] : 0.f;
        const RowAt<T> at(a, r);
        RowAt<T> next(a, r + clusters < a.T ? r + clusters : r);
        if (w_next == 0.f) next.nb = 0;  // no next row, or one that is not read
        T* out = a.dz ? static_cast<T*>(a.dz) + (size_t)r * a.V : nullptr;
        if (w == 0.f) {  // the cluster's CTAs agree
            if (rank == 0 && tid == 0 && a.loss_rows) a.loss_rows[r] = 0.f;
            if (out)
                for (int v = first; v < a.V; v += stride) store_from_f32(out + v, 0.f);
            loaded = false;
            continue;
        }
        if (kNV > 0 && !loaded) {
#pragma unroll
            for (int j = 0; j < kNV; ++j) load(j, at);
        }
        loaded = true;
        const T* z = at.z;
        const int head = at.head, nb = at.nb, tail0 = at.tail0;
        const uint4* zv = at.vec();
        // the single values lie with rank 0: threads 0.. the head, threads 32.. the tail
        int odd = -1;
        if (rank == 0 && tid < head) odd = tid;
        if (rank == 0 && tid >= 32 && tail0 + tid - 32 < a.V) odd = tail0 + tid - 32;
        const float zo = odd >= 0 ? to_f32(z[odd]) : -INFINITY;
        // the first kThreads listed entries, one per thread: loaded with the row, used behind its sums
        const size_t rk = (size_t)r * a.K;
        const IdT* ids = static_cast<const IdT*>(a.ids) + rk;
        auto listed = [&](int k) {
            const long long id = k < a.K ? (long long)ids[k] : -1;
            return id >= 0 && id < a.V ? (int)id : -1;
        };
        const int v0 = listed(tid);
        float p0 = 0.f, lp0 = -INFINITY;
        if (v0 >= 0) {
            p0 = a.ptot[rk + tid];
            lp0 = a.logp[rk + tid];
        }
        float m = fmaxf(zo, -FLT_MAX), l = 0.f;
        if constexpr (kNV > 0) {
#pragma unroll
            for (int j = 0; j < kNV; ++j) m = fmaxf(m, V8::top(d[j]));
#pragma unroll
            for (int j = 0; j < kNV; ++j) {
                float x[E];
                exp_of<V8>(d[j], m, c, x);
                l += sum_of(x);
            }
        } else {
            for (int i = first; i < nb; i += stride) {
                const uint4 v = zv[i];
                const float mn = fmaxf(m, V8::top(v));
                float x[E];
                exp_of<V8>(v, mn, c, x);
                l = l * exp2_fast((m - mn) * c) + sum_of(x);
                m = mn;
            }
        }
        if (odd >= 0) l += exp2_fast((zo - m) * c);
        const float z0 = v0 >= 0 ? to_f32(z[v0]) : 0.f;
        join_lanes<32>(m, l, c);
        if (lane == 0) s_warp[warp] = make_float2(m, l);
        __syncthreads();
        if (warp == 0) {
            const float2 x = s_warp[lane % kWarps];
            m = x.x;
            l = x.y;
            join_lanes<kWarps>(m, l, c);
            if (lane < C) *cluster.map_shared_rank(&s_pair[parity][rank], lane) = make_float2(m, l);
        }
        // one barrier a row: a pair is written again two rows on, when every CTA has
        // passed the next row's barrier and so has read it
        cluster.sync();
        {
            const float2 x = lane % kMaxCluster < C ? s_pair[parity][lane % kMaxCluster] : make_float2(-FLT_MAX, 0.f);
            m = x.x;
            l = x.y;
            join_lanes<kMaxCluster>(m, l, c);  // the same bits in every warp
        }
        parity ^= 1;
        const float inv = 1.f / l;
        if (a.loss_rows && rank == 0) {  // added up behind the barrier that follows
            const float log_l = logf(l), inv_tau = 1.f / a.tau;
            auto term = [&](float lp, float zk) {  // NaN teachers show, entries of p = 0 count nothing
                const float p = expf(lp);
                return p == 0.f ? 0.f : p * (lp - ((zk - m) * inv_tau - log_l));
            };
            float t = v0 >= 0 ? term(lp0, z0) : 0.f;
            for (int k = tid + kThreads; k < a.K; k += kThreads) {
                const int v = listed(k);
                if (v >= 0) t += term(a.logp[rk + k], to_f32(z[v]));
            }
            t = warp_sum(t);
            if (lane == 0) s_part[warp] = t;
        }
        if (out) {
            const float qs = inv * row_scale(r, w);
            const bool same_phase = ((reinterpret_cast<uintptr_t>(out + head)) & 15) == 0;
            auto emit = [&](int i, const uint4& raw) {
                float x[E];
                exp_of<V8>(raw, m, c, x);
                scale_pairs(x, qs);
                if (same_phase) {
                    __stcs(reinterpret_cast<uint4*>(out + head) + i, V8::pack(x));
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
                    load(j, next);
                }
            } else {
                for (int i = first; i < nb; i += stride) emit(i, zv[i]);
            }
            if (odd >= 0) store_from_f32(out + odd, exp2_fast((zo - m) * c) * qs);
        } else if constexpr (kNV > 0) {
#pragma unroll
            for (int j = 0; j < kNV; ++j) load(j, next);
        }
        __syncthreads();  // the listed entries of this CTA's part are written over
        if (out) {
            auto owned = [&](int v) {
                return (v < head || v >= tail0 ? 0 : ((v - head) / E / kThreads) & (C - 1)) == rank;
            };
            const float scale = row_scale(r, w);
            if (v0 >= 0 && owned(v0)) store_from_f32(out + v0, (exp2_fast((z0 - m) * c) * inv - p0) * scale);
            for (int k = tid + kThreads; k < a.K; k += kThreads) {
                const int v = listed(k);
                if (v < 0 || !owned(v)) continue;
                store_from_f32(out + v, (exp2_fast((to_f32(z[v]) - m) * c) * inv - a.ptot[rk + k]) * scale);
            }
        }
        if (a.loss_rows && rank == 0 && tid == 0) {
            float sum = 0.f;
            for (int i = 0; i < kWarps; ++i) sum += s_part[i];
            a.loss_rows[r] = sum * a.tau * a.tau;
        }
    }
    cluster.sync();  // no CTA leaves while another may still read its pair
    if (!a.loss) return;
    // the CTA that ends last adds the rows' losses, in an order that is always the same
    if (tid == 0) {
        __threadfence();
        s_last = atomicAdd(a.counter, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    double t = 0.0;
    for (int r = tid; r < a.T; r += kThreads) {
        const float w = __ldcg(a.weight + r);
        if (w != 0.f) t += (double)w * (double)__ldcg(a.loss_rows + r);
    }
    t = block_sum(t, s_sum);
    if (tid == 0) *a.loss = (float)(t * (double)unit);
}

// Cluster size and vectors per thread.  A row of `vecs` vectors wants the fewest CTAs that
// hold it in at most 6 vectors a thread (two CTAs per SM then); few rows want more CTAs a
// row, up to 8, while they leave SMs without work.
void pick(long long T, long long vecs, int sms, int* C, int* nv) {
    int c = 1;
    while (c < kMaxCluster && vecs > (long long)c * kThreads * 6) c *= 2;
    while (c < kMaxCluster && T * c * 2 <= 2 * sms && vecs > (long long)c * kThreads) c *= 2;
    const long long per = (vecs + (long long)c * kThreads - 1) / ((long long)c * kThreads);
    *C = c;
    *nv = per <= 16 ? (int)std::max<long long>(per, 1) : 0;
}

template <typename T, typename IdT, int kNV>
cudaError_t launch_nv(const Rows& a, int C, cudaStream_t stream) {
    auto kern = distill_rows_kernel<T, IdT, kNV>;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)C);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
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
        if ((e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg)) != cudaSuccess) return e;
        n = std::max(n, 1);
        if (dev < kMaxDevices) resident[dev][lc].store(n, std::memory_order_relaxed);
    }
    cfg.gridDim = dim3((unsigned)(std::min(a.T, n) * C));
    e = cudaLaunchKernelEx(&cfg, kern, a);
    if (e == cudaSuccess) note_launch();
    return e;
}

template <typename T, typename IdT>
cudaError_t launch_rows(const Rows& a, cudaStream_t stream) {
    const int sms = device_sm_count();
    int C = 1, nv = 0;
    pick(a.T, (a.V + Vec<T>::n - 1) / Vec<T>::n, sms, &C, &nv);
    switch (nv) {
        case 1: return launch_nv<T, IdT, 1>(a, C, stream);
        case 2: return launch_nv<T, IdT, 2>(a, C, stream);
        case 3: return launch_nv<T, IdT, 3>(a, C, stream);
        case 4: return launch_nv<T, IdT, 4>(a, C, stream);
        case 5: return launch_nv<T, IdT, 5>(a, C, stream);
        case 6: return launch_nv<T, IdT, 6>(a, C, stream);
        case 7: case 8: return launch_nv<T, IdT, 8>(a, C, stream);
        case 9: case 10: return launch_nv<T, IdT, 10>(a, C, stream);
        case 0: return launch_nv<T, IdT, 0>(a, C, stream);
        default: return launch_nv<T, IdT, 16>(a, C, stream);
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
    r.ids = a.ids;
    r.mean = a.mean;
    r.prep_blocks = (int)std::min(kPrepBlocks, (r.T + kPrepThreads / 32 - 1) / (kPrepThreads / 32));
    r.tau = a.tau;
    r.counter = reinterpret_cast<unsigned*>(ws);
    r.wsum = reinterpret_cast<const double*>(ws + l.wsum);
    r.weight = reinterpret_cast<const float*>(ws + l.weight);
    r.logp = reinterpret_cast<const float*>(ws + l.logp);
    r.ptot = reinterpret_cast<const float*>(ws + l.ptot);
    r.loss_rows = a.loss_rows ? a.loss_rows : reinterpret_cast<float*>(ws + l.loss);
    r.loss = a.loss;
    r.dz = a.dz;
    return r;
}

cudaError_t launch_by_type(const LogitDistillArgs& a, const Rows& r, cudaStream_t stream) {
    if (a.dtype == kF32)
        return a.ids_are_64 ? launch_rows<float, int64_t>(r, stream) : launch_rows<float, int32_t>(r, stream);
    return a.ids_are_64 ? launch_rows<__nv_bfloat16, int64_t>(r, stream)
                        : launch_rows<__nv_bfloat16, int32_t>(r, stream);
}

}  // namespace

size_t logit_distill_workspace_bytes(long long T, int K) { return layout(T, K).total; }

cudaError_t launch_logit_distill_fwd(const LogitDistillArgs& a, cudaStream_t stream) {
    Rows r = make_rows(a);
    double* wsum = const_cast<double*>(r.wsum);
    float *weight = const_cast<float*>(r.weight), *logp = const_cast<float*>(r.logp), *ptot = const_cast<float*>(r.ptot);
    const float inv_tau = 1.f / a.tau;
    if (a.ids_are_64)
        distill_prep_kernel<int64_t><<<r.prep_blocks, kPrepThreads, 0, stream>>>(
            a.teacher, static_cast<const int64_t*>(a.ids), a.row_weight, r.T, a.V, a.K, inv_tau, r.counter, wsum, weight,
            logp, ptot);
    else
        distill_prep_kernel<int32_t><<<r.prep_blocks, kPrepThreads, 0, stream>>>(
            a.teacher, static_cast<const int32_t*>(a.ids), a.row_weight, r.T, a.V, a.K, inv_tau, r.counter, wsum, weight,
            logp, ptot);
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
