// Query and key heads of one layer in one pass: the RMS norm of every head row, the
// rotation and the (B, N, Hx, D) -> (B, Hx, N, D) layout change, and its backward pass.
//
// Per head row x (D values), weight w, tables cos, sin of the row's position:
//   r = rsqrt(mean(x^2) + eps),   y = x r w   (y = x where a tensor has no weight)
//   out_lo = y_lo cos_lo - y_hi sin_lo,   out_hi = y_hi cos_hi + y_lo sin_hi
// (lo, hi: the row's halves; out = y without tables).  Backward, g = dL/dout:
//   a_lo = g_lo cos_lo + g_hi sin_hi,   a_hi = g_hi cos_hi - g_lo sin_lo   (dL/dy)
//   dw = sum over rows of a x r,   dx = r (a w - x r^2 mean(a w x))
// Everything is fp32 from the loaded values and rounded once at the stores.
//
// Measured (12 + 2 heads of 128, bf16; a plain copy runs at 6.45 TB/s): forward B=8, N=4096, 252 MB: 48 us,
// 5.2 TB/s; backward B=4, N=4096, 185 MB: 48 us, 3.9 TB/s, and 4 us for the join of the weight gradients.
//
// Bound: HBM, every row read once and written once.  The backward pass does not reach it (60 % of the copy rate): its 16
// warps an SM load, compute and store a step of two head rows one after another, and nothing covers the loads (the
// largest part of a warp's waiting).  Layout: D / 16 lanes hold a row, each
// 8 values of the low and the 8 matching values of the high half (16-byte loads at bf16),
// so the rotation needs no exchange and the row sum log2(D / 16) shuffles; the lanes of a
// row keep the position's cos and sin in registers while they walk the heads of a token.
// Neighbouring lane groups take neighbouring tokens: both the (token, head) reads and the
// (head, token) writes then cover whole 128-byte lines.
#include <algorithm>
#include <cstdint>

#include "common.cuh"
#include "kernels.h"

namespace ossa {

namespace {

constexpr int kThreads = 256;
constexpr int kBwdCtas = 2;  // CTAs of the backward pass per SM

__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
    uint4 o;
    uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * t], v[2 * t + 1]);
        w[t] = *reinterpret_cast<const uint32_t*>(&x);
    }
    *reinterpret_cast<uint4*>(p) = o;
}

// A weight value: fp32 or bf16 storage, whatever the rows' type.
__device__ __forceinline__ float weight_at(const void* w, int w_f32, int d) {
    return w_f32 ? static_cast<const float*>(w)[d]
                 : __bfloat162float(static_cast<const __nv_bfloat16*>(w)[d]);
}

// One of the two tensors (queries or keys) as the kernels see it.
struct Side {
    const void* x;   // rows (b, n, h): x + b * sb + n * sn + h * D
    long long sb, sn;
    const void* w;   // (D,) or nullptr: no norm
    const void* g;   // backward: dL/dout (B, H, N, D)
    void* o;         // forward: out (B, H, N, D); backward: dx (B, N, H, D)
    int H;
};

struct Pass {
    Side s[2];
    const void *cosv, *sinv;  // (1 or B, N, D) or nullptr
    int cs_batched, w_f32;
    int B, N, D;
    float eps;
    int chunk;        // heads that one lane group walks at a token
    int chunks0, chunks;  // head chunks of side 0, of both sides
};

// The unit (token, head chunk) a lane group works on.
struct Unit {
    int b, n, side, h0, h1;
};

__device__ __forceinline__ Unit unit_at(const Pass& p, long long u, long long tokens) {
    Unit r;
    const int c = (int)(u / tokens);
    const long long t = u - (long long)c * tokens;
    r.b = (int)(t / p.N);
    r.n = (int)(t - (long long)r.b * p.N);
    r.side = c < p.chunks0 ? 0 : 1;
    r.h0 = (r.side ? c - p.chunks0 : c) * p.chunk;
    r.h1 = min(r.h0 + p.chunk, p.s[r.side].H);
    return r;
}

// 8 values as loaded (bf16: 4 registers), so that rows ahead and the tables cost little to hold.
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = __ldg(reinterpret_cast<const float4*>(p));
        b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};
template <>
struct Raw8<__nv_bfloat16> {
    uint4 a;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void zero() { a = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        unpack_bf16x2(a.x, v[0], v[1]);
        unpack_bf16x2(a.y, v[2], v[3]);
        unpack_bf16x2(a.z, v[4], v[5]);
        unpack_bf16x2(a.w, v[6], v[7]);
    }
};

// The two halves of a row's piece.
template <typename T>
struct Pair8 {
    Raw8<T> lo, hi;
    __device__ __forceinline__ void load(const T* row, int l, int h, bool on) {
        if (on) {
            lo.load(row + l);
            hi.load(row + h);
        } else {
            lo.zero();
            hi.zero();
        }
    }
    __device__ __forceinline__ void get(float (&a)[8], float (&b)[8]) const {
        lo.get(a);
        hi.get(b);
    }
};

// cos and sin of a position.
template <typename T>
struct Tables {
    Pair8<T> c, s;
    __device__ __forceinline__ void load(const Pass& p, int b, int n, int lo, int hi) {
        const size_t at = ((size_t)(p.cs_batched ? b : 0) * p.N + n) * p.D;
        c.load(static_cast<const T*>(p.cosv) + at, lo, hi, true);
        s.load(static_cast<const T*>(p.sinv) + at, lo, hi, true);
    }
};

// Sum over the L lanes of a row (L a power of two, lanes adjacent).
template <int L>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
    for (int o = L / 2; o >= 1; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
    return x;
}

// Heads whose rows a lane group loads at once: the more bytes in flight, the nearer to HBM's rate
// (B=8, N=4096, 12 + 2 heads, bf16: one head at a time 66 us, four 48 us).
template <typename T>
constexpr int kHeads = sizeof(T) == 2 ? 4 : 2;

// Steps of a lane group's walk over its heads, the most of the warp's groups (the row sums are warp-wide).
__device__ __forceinline__ int warp_heads(const Unit& u) { return __reduce_max_sync(kFull, u.h1 - u.h0); }

template <typename T, int L>
__global__ void __launch_bounds__(kThreads, 2) norm_rope_fwd_kernel(const Pass p) {
    constexpr int D = 16 * L, kH = kHeads<T>;
    const int l = threadIdx.x % L;
    const int lo = 8 * l, hi = D / 2 + 8 * l;
    const long long tokens = (long long)p.B * p.N, units = tokens * p.chunks;
    const long long u0 = (long long)blockIdx.x * (kThreads / L) + threadIdx.x / L;
    const bool live = u0 < units;
    const Unit u = unit_at(p, live ? u0 : units - 1, tokens);
    const Side& s = p.s[u.side];
    const bool rope = p.cosv != nullptr, norm = s.w != nullptr;
    const T* x = static_cast<const T*>(s.x) + (size_t)(u.b * s.sb + u.n * s.sn);
    const int heads = warp_heads(u);
    Pair8<T> rows[kH];
    auto load = [&](int k) {
#pragma unroll
        for (int i = 0; i < kH; ++i) {
            const int h = u.h0 + k + i;
            rows[i].load(x + (size_t)h * D, lo, hi, live && h < u.h1);
        }
    };
    load(0);
    Tables<T> cs;
    if (rope) cs.load(p, u.b, u.n, lo, hi);
    float wl[8], wh[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        wl[t] = norm ? weight_at(s.w, p.w_f32, lo + t) : 1.f;
        wh[t] = norm ? weight_at(s.w, p.w_f32, hi + t) : 1.f;
    }
    for (int k = 0; k < heads; k += kH) {
        if (k > 0) load(k);
#pragma unroll
        for (int i = 0; i < kH; ++i) {
            const int h = u.h0 + k + i;
            const bool on = live && h < u.h1;
            float a[8], b[8];
            rows[i].get(a, b);
            if (norm) {
                float ss = 0.f;
#pragma unroll
                for (int t = 0; t < 8; ++t) ss = fmaf(a[t], a[t], fmaf(b[t], b[t], ss));
                const float r = rsqrtf(row_sum<L>(ss) * (1.f / D) + p.eps);
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    a[t] *= r * wl[t];
                    b[t] *= r * wh[t];
                }
            }
            if (rope) {
                float cl[8], ch[8], sl[8], sh[8];
                cs.c.get(cl, ch);
                cs.s.get(sl, sh);
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    const float y = a[t];
                    a[t] = y * cl[t] - b[t] * sl[t];
                    b[t] = b[t] * ch[t] + y * sh[t];
                }
            }
            if (on) {
                T* o = static_cast<T*>(s.o) + (((size_t)u.b * s.H + h) * p.N + u.n) * D;
                store8(o + lo, a);
                store8(o + hi, b);
            }
        }
    }
}

// Backward.  A CTA belongs to one side and walks the side's units with a fixed stride; its
// sums for dw go to part[block][D] and are joined in block order by dw_join_kernel, so the
// result does not depend on the order in which CTAs run.
template <typename T, int L>
__global__ void __launch_bounds__(kThreads, 2)
norm_rope_bwd_kernel(const Pass p, int blocks0, float* __restrict__ part) {
    constexpr int D = 16 * L, kGroups = kThreads / L, kH = kHeads<T> / 2;
    __shared__ float sums[kGroups > 16 ? 16 : kGroups][D];
    const int l = threadIdx.x % L, grp = threadIdx.x / L;
    const int lo = 8 * l, hi = D / 2 + 8 * l;
    const int side = (int)blockIdx.x < blocks0 ? 0 : 1;
    const Side& s = p.s[side];
    const int blk = side ? blockIdx.x - blocks0 : blockIdx.x;
    const int nblk = side ? gridDim.x - blocks0 : blocks0;
    const bool rope = p.cosv != nullptr, norm = s.w != nullptr;
    float wl[8], wh[8], dl[8], dh[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        wl[t] = norm ? weight_at(s.w, p.w_f32, lo + t) : 1.f;
        wh[t] = norm ? weight_at(s.w, p.w_f32, hi + t) : 1.f;
        dl[t] = dh[t] = 0.f;
    }
    const long long tokens = (long long)p.B * p.N;
    const int chunks = side ? p.chunks - p.chunks0 : p.chunks0;
    const long long units = tokens * chunks, step = (long long)nblk * kGroups;
    const long long first = side ? tokens * p.chunks0 : 0;
    // the CTA's groups take the same number of rounds
    for (long long base = (long long)blk * kGroups; base < units; base += step) {
        const bool live = base + grp < units;
        const Unit u = unit_at(p, first + (live ? base + grp : units - 1), tokens);
        const T* x = static_cast<const T*>(s.x) + (size_t)(u.b * s.sb + u.n * s.sn);
        const T* g = static_cast<const T*>(s.g) + ((size_t)u.b * s.H * p.N + u.n) * D;
        const size_t gh = (size_t)p.N * D;  // from head to head
        const int heads = warp_heads(u);
        Pair8<T> ax[kH], ag[kH];
        auto load = [&](int k) {
#pragma unroll
            for (int i = 0; i < kH; ++i) {
                const int h = u.h0 + k + i;
                const bool on = live && h < u.h1;
                ag[i].load(g + h * gh, lo, hi, on);
                ax[i].load(x + (size_t)h * D, lo, hi, on && norm);
            }
        };
        load(0);
        Tables<T> cs;
        if (rope) cs.load(p, u.b, u.n, lo, hi);
        for (int k = 0; k < heads; k += kH) {
            if (k > 0) load(k);
#pragma unroll
            for (int i = 0; i < kH; ++i) {
                const int h = u.h0 + k + i;
                const bool on = live && h < u.h1;
                float a[8], b[8], ga[8], gb[8];
                ax[i].get(a, b);
                ag[i].get(ga, gb);
                if (rope) {
                    float cl[8], ch[8], sl[8], sh[8];
                    cs.c.get(cl, ch);
                    cs.s.get(sl, sh);
#pragma unroll
                    for (int t = 0; t < 8; ++t) {
                        const float y = ga[t];
                        ga[t] = y * cl[t] + gb[t] * sh[t];
                        gb[t] = gb[t] * ch[t] - y * sl[t];
                    }
                }
                if (norm) {
                    float ss = 0.f, dot = 0.f;
#pragma unroll
                    for (int t = 0; t < 8; ++t) {
                        ss = fmaf(a[t], a[t], fmaf(b[t], b[t], ss));
                        dot = fmaf(a[t], ga[t] * wl[t], fmaf(b[t], gb[t] * wh[t], dot));
                    }
                    ss = row_sum<L>(ss);
                    dot = row_sum<L>(dot);
                    const float r = rsqrtf(ss * (1.f / D) + p.eps);
                    const float c = dot * (1.f / D) * r * r;
#pragma unroll
                    for (int t = 0; t < 8; ++t) {
                        if (on) {  // a dead lane's zero row has r = 1/sqrt(eps), infinite at eps 0
                            dl[t] = fmaf(ga[t], a[t] * r, dl[t]);
                            dh[t] = fmaf(gb[t], b[t] * r, dh[t]);
                        }
                        ga[t] = r * (ga[t] * wl[t] - a[t] * c);
                        gb[t] = r * (gb[t] * wh[t] - b[t] * c);
                    }
                }
                if (on) {
                    T* o = static_cast<T*>(s.o) + (((size_t)u.b * p.N + u.n) * s.H + h) * D;
                    store8(o + lo, ga);
                    store8(o + hi, gb);
                }
            }
        }
    }
    if (!norm) return;  // CTA-uniform
    // the groups' sums in a fixed order, 16 groups at a time
    constexpr int kSlots = kGroups > 16 ? 16 : kGroups;
    for (int round = 0; round < kGroups / kSlots; ++round) {
        if (grp / kSlots == round) {
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                float* q = &sums[grp % kSlots][0];
                q[lo + t] = dl[t] + (round ? q[lo + t] : 0.f);
                q[hi + t] = dh[t] + (round ? q[hi + t] : 0.f);
            }
        }
        __syncthreads();
    }
    for (int d = threadIdx.x; d < D; d += kThreads) {
        float t = 0.f;
        for (int i = 0; i < kSlots; ++i) t += sums[i][d];
        part[(size_t)blockIdx.x * D + d] = t;
    }
}

// Head dims whose sixteenth is no power of two: a warp per row, lane l holding the pairs
// (d, d + D/2) with d = l, l + 32, ... (D <= 512).
constexpr int kAnyPairs = 8;

template <typename T, bool kBackward>
__global__ void __launch_bounds__(kThreads)
norm_rope_any_kernel(const Pass p, int blocks0, float* __restrict__ part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kWarps = kThreads / 32;
    __shared__ float sums[kWarps][512];
    const int D = p.D, half = D / 2;
    const int side = (int)blockIdx.x < blocks0 ? 0 : 1;
    const Side& s = p.s[side];
    const int blk = side ? blockIdx.x - blocks0 : blockIdx.x;
    const int nblk = side ? gridDim.x - blocks0 : blocks0;
    const bool rope = p.cosv != nullptr, norm = s.w != nullptr;
    const long long rows = (long long)p.B * p.N * s.H;
    float dl[kAnyPairs], dh[kAnyPairs];
#pragma unroll
    for (int t = 0; t < kAnyPairs; ++t) dl[t] = dh[t] = 0.f;
    for (long long row = (long long)blk * kWarps + warp; row < rows; row += (long long)nblk * kWarps) {
        const int h = (int)(row % s.H);
        const long long bn = row / s.H;
        const int b = (int)(bn / p.N), n = (int)(bn - (long long)b * p.N);
        const T* x = static_cast<const T*>(s.x) + (size_t)(b * s.sb + n * s.sn) + (size_t)h * D;
        const size_t head_row = (((size_t)b * s.H + h) * p.N + n) * D;
        const size_t cr = ((size_t)(p.cs_batched ? b : 0) * p.N + n) * D;
        const T* c = static_cast<const T*>(p.cosv) + cr;
        const T* sn = static_cast<const T*>(p.sinv) + cr;
        float a[kAnyPairs], e[kAnyPairs], ga[kAnyPairs], gb[kAnyPairs];
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int t = 0; t < kAnyPairs; ++t) {
            const int d = lane + 32 * t;
            a[t] = e[t] = ga[t] = gb[t] = 0.f;
            if (d < half) {
                if (norm || !kBackward) {
                    a[t] = to_f32(x[d]);
                    e[t] = to_f32(x[half + d]);
                }
                ss = fmaf(a[t], a[t], fmaf(e[t], e[t], ss));
                if constexpr (kBackward) {
                    const T* g = static_cast<const T*>(s.g) + head_row;
                    const float gl = to_f32(g[d]), gh = to_f32(g[half + d]);
                    ga[t] = rope ? gl * to_f32(c[d]) + gh * to_f32(sn[half + d]) : gl;
                    gb[t] = rope ? gh * to_f32(c[half + d]) - gl * to_f32(sn[d]) : gh;
                    if (norm)
                        dot = fmaf(a[t], ga[t] * weight_at(s.w, p.w_f32, d),
                                   fmaf(e[t], gb[t] * weight_at(s.w, p.w_f32, half + d), dot));
                }
            }
        }
        ss = warp_sum(ss);
        const float r = norm ? rsqrtf(ss / (float)D + p.eps) : 1.f;
        if constexpr (kBackward) dot = warp_sum(dot);
        const float cc = dot / (float)D * r * r;
#pragma unroll
        for (int t = 0; t < kAnyPairs; ++t) {
            const int d = lane + 32 * t;
            if (d >= half) continue;
            const float wl = norm ? weight_at(s.w, p.w_f32, d) : 1.f;
            const float wh = norm ? weight_at(s.w, p.w_f32, half + d) : 1.f;
            if constexpr (kBackward) {
                T* o = static_cast<T*>(s.o) + (size_t)row * D;
                if (norm) {
                    dl[t] = fmaf(ga[t], a[t] * r, dl[t]);
                    dh[t] = fmaf(gb[t], e[t] * r, dh[t]);
                    ga[t] = r * (ga[t] * wl - a[t] * cc);
                    gb[t] = r * (gb[t] * wh - e[t] * cc);
                }
                store_from_f32(o + d, ga[t]);
                store_from_f32(o + half + d, gb[t]);
            } else {
                const float yl = norm ? a[t] * (r * wl) : a[t], yh = norm ? e[t] * (r * wh) : e[t];
                T* o = static_cast<T*>(s.o) + head_row;
                store_from_f32(o + d, rope ? yl * to_f32(c[d]) - yh * to_f32(sn[d]) : yl);
                store_from_f32(o + half + d, rope ? yh * to_f32(c[half + d]) + yl * to_f32(sn[half + d]) : yh);
            }
        }
    }
    if (!kBackward || !norm) return;
#pragma unroll
    for (int t = 0; t < kAnyPairs; ++t) {
        const int d = lane + 32 * t;
        if (d < half) {
            sums[warp][d] = dl[t];
            sums[warp][half + d] = dh[t];
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kThreads) {
        float t = 0.f;
        for (int i = 0; i < kWarps; ++i) t += sums[i][d];
        part[(size_t)blockIdx.x * D + d] = t;
    }
}

// dw of both sides: a CTA takes 32 columns, each of its 8 warps every eighth block's row of sums in block
// order; the warps' results are added in warp order.
__global__ void __launch_bounds__(kThreads)
dw_join_kernel(const float* __restrict__ part, int blocks0, int blocks, int D, void* dw0, void* dw1, int w_f32) {
    constexpr int kWarps = kThreads / 32;
    __shared__ float sums[kWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, side = blockIdx.y;
    const int d = blockIdx.x * 32 + lane;
    void* out = side ? dw1 : dw0;
    if (!out) return;  // CTA-uniform
    float t = 0.f;
    if (d < D) {
#pragma unroll 8
        for (int i = (side ? blocks0 : 0) + warp; i < (side ? blocks : blocks0); i += kWarps) t += part[(size_t)i * D + d];
    }
    sums[warp][lane] = t;
    __syncthreads();
    if (warp != 0 || d >= D) return;
    t = 0.f;
    for (int w = 0; w < kWarps; ++w) t += sums[w][lane];
    if (w_f32) static_cast<float*>(out)[d] = t;
    else static_cast<__nv_bfloat16*>(out)[d] = __float2bfloat16_rn(t);
}

Pass make_pass(const NormRopeArgs& a, bool backward) {
    Pass p{};
    const void* x[2] = {a.q, a.k};
    const void* w[2] = {a.wq, a.wk};
    const void* g[2] = {a.gq, a.gk};
    void* o[2] = {a.oq, a.ok};
    const int H[2] = {a.Hq, a.Hk};
    const long long sb[2] = {a.q_sb, a.k_sb}, sn[2] = {a.q_sn, a.k_sn};
    for (int i = 0; i < 2; ++i) p.s[i] = Side{x[i], sb[i], sn[i], w[i], backward ? g[i] : nullptr, o[i], H[i]};
    p.cosv = a.cosv;
    p.sinv = a.sinv;
    p.cs_batched = a.cs_batched;
    p.w_f32 = a.w_f32;
    p.B = a.B;
    p.N = a.N;
    p.D = a.D;
    p.eps = a.eps;
    return p;
}

// Head chunks: as many heads per lane group as leave at least `want` groups.
void set_chunks(Pass& p, long long want) {
    const long long tokens = (long long)p.B * p.N;
    int chunk = std::max(p.s[0].H, p.s[1].H);
    auto count = [&](int c) { return (p.s[0].H + c - 1) / c + (p.s[1].H + c - 1) / c; };
    while (chunk > 1 && tokens * count(chunk) < want) chunk = (chunk + 1) / 2;
    p.chunk = chunk;
    p.chunks0 = (p.s[0].H + chunk - 1) / chunk;
    p.chunks = count(chunk);
}

bool lane_layout(int D) { return D == 16 || D == 32 || D == 64 || D == 128 || D == 256; }

// CTAs of the backward pass, and how many of them are side 0's.
void bwd_blocks(const NormRopeArgs& a, int* blocks0, int* blocks) {
    const int most = kBwdCtas * device_sm_count();
    const int per = lane_layout(a.D) ? kThreads / (a.D / 16) : kThreads / 32;
    const long long rq = ((long long)a.B * a.N * a.Hq + per - 1) / per, rk = ((long long)a.B * a.N * a.Hk + per - 1) / per;
    const int H = a.Hq + a.Hk;
    const int share0 = a.Hk == 0 ? most : std::min(most - 1, std::max(1, most * a.Hq / H));
    const int b0 = (int)std::min<long long>(rq, share0);
    const int b1 = (int)std::min<long long>(rk, std::max(most - share0, 0));
    *blocks0 = b0;
    *blocks = b0 + b1;
}

template <typename T>
cudaError_t fwd_t(const NormRopeArgs& a, cudaStream_t stream) {
    Pass p = make_pass(a, false);
    const long long tokens = (long long)a.B * a.N;
    if (!lane_layout(a.D)) {
        int b0 = 0, blocks = 0;
        bwd_blocks(a, &b0, &blocks);
        norm_rope_any_kernel<T, false><<<blocks, kThreads, 0, stream>>>(p, b0, nullptr);
    } else {
        const int L = a.D / 16, groups = kThreads / L;
        set_chunks(p, (long long)device_sm_count() * groups * 2);
        const long long grid = (tokens * p.chunks + groups - 1) / groups;
        if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
        switch (L) {
            case 1: norm_rope_fwd_kernel<T, 1><<<(unsigned)grid, kThreads, 0, stream>>>(p); break;
            case 2: norm_rope_fwd_kernel<T, 2><<<(unsigned)grid, kThreads, 0, stream>>>(p); break;
            case 4: norm_rope_fwd_kernel<T, 4><<<(unsigned)grid, kThreads, 0, stream>>>(p); break;
            case 8: norm_rope_fwd_kernel<T, 8><<<(unsigned)grid, kThreads, 0, stream>>>(p); break;
            default: norm_rope_fwd_kernel<T, 16><<<(unsigned)grid, kThreads, 0, stream>>>(p); break;
        }
    }
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e;
}

template <typename T>
cudaError_t bwd_t(const NormRopeArgs& a, cudaStream_t stream) {
    Pass p = make_pass(a, true);
    int b0 = 0, blocks = 0;
    bwd_blocks(a, &b0, &blocks);
    if (!lane_layout(a.D)) {
        norm_rope_any_kernel<T, true><<<blocks, kThreads, 0, stream>>>(p, b0, a.part);
    } else {
        const int L = a.D / 16;
        set_chunks(p, (long long)blocks * (kThreads / L) * 2);
        switch (L) {
            case 1: norm_rope_bwd_kernel<T, 1><<<blocks, kThreads, 0, stream>>>(p, b0, a.part); break;
            case 2: norm_rope_bwd_kernel<T, 2><<<blocks, kThreads, 0, stream>>>(p, b0, a.part); break;
            case 4: norm_rope_bwd_kernel<T, 4><<<blocks, kThreads, 0, stream>>>(p, b0, a.part); break;
            case 8: norm_rope_bwd_kernel<T, 8><<<blocks, kThreads, 0, stream>>>(p, b0, a.part); break;
            default: norm_rope_bwd_kernel<T, 16><<<blocks, kThreads, 0, stream>>>(p, b0, a.part); break;
        }
    }
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    note_launch();
    if (!a.dwq && !a.dwk) return cudaSuccess;
    dw_join_kernel<<<dim3((a.D + 31) / 32, 2), kThreads, 0, stream>>>(a.part, b0, blocks, a.D, a.dwq, a.dwk, a.w_f32);
    e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e;
}

}  // namespace

size_t norm_rope_workspace_bytes(int D) { return (size_t)kBwdCtas * device_sm_count() * D * sizeof(float); }

cudaError_t launch_norm_rope_fwd(const NormRopeArgs& a, cudaStream_t stream) {
    return a.dtype == kF32 ? fwd_t<float>(a, stream) : fwd_t<__nv_bfloat16>(a, stream);
}

cudaError_t launch_norm_rope_bwd(const NormRopeArgs& a, cudaStream_t stream) {
    return a.dtype == kF32 ? bwd_t<float>(a, stream) : bwd_t<__nv_bfloat16>(a, stream);
}

}  // namespace ossa
