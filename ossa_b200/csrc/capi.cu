// C ABI entry points (declared in include/ossa_b200.h): argument validation,
// workspace carving and kernel dispatch.  Validation happens before any CUDA
// call, so a rejected request never touches the device.
#include "../../include/ossa_b200.h"
#include "kernels.h"

#include <atomic>
#include <float.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string>

namespace ossa {
namespace {
std::atomic<unsigned long long> g_launches{0};
}
void note_launch(int n) { g_launches.fetch_add((unsigned long long)n, std::memory_order_relaxed); }
}  // namespace ossa

namespace {

thread_local std::string g_last_error;

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    g_last_error = buf;
    return code;
}

}  // namespace

namespace ossa {
// Lets other translation units of the library report a message through
// ossa_last_error_string.
void set_error_message(const char* msg) { g_last_error = msg; }

int device_sm_count() {
    constexpr int kMaxDev = 64;
    static std::atomic<int> cached[kMaxDev];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return 148;
    int n = cached[dev].load(std::memory_order_relaxed);
    if (n <= 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
        cached[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}
}  // namespace ossa

namespace {

int cuda_status(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return OSSA_OK;
    return fail(OSSA_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Whether every pointer (NULL too) lies on a boundary of n bytes.
template <typename... P>
bool aligned_to(uintptr_t n, const P*... p) { return (... && (reinterpret_cast<uintptr_t>(p) % n == 0)); }

constexpr size_t kAlign = 256;
size_t align_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

bool valid_dtype(int d) { return d == OSSA_F32 || d == OSSA_BF16; }

int check_heads(int B, int H, int Hkv, int N) {
    if (B < 0 || H <= 0 || Hkv <= 0 || N < 0)
        return fail(OSSA_ERR_INVALID, "bad shape B=%d H=%d Hkv=%d N=%d", B, H, Hkv, N);
    if (H % Hkv != 0)
        return fail(OSSA_ERR_INVALID, "H=%d is not a multiple of Hkv=%d", H, Hkv);
    if ((long long)B * H > (1ll << 30) || N > (1 << 30))
        return fail(OSSA_ERR_UNSUPPORTED, "shape too large B=%d H=%d N=%d", B, H, N);
    return OSSA_OK;
}

// Workspace: [counters 256 B][q' fp32][k' fp32][tensor-core selection scratch]
// [split selection scratch (few query rows only)].  The counters block
// (fallback row count, status word) sits at offset 0 so ossa_router_status can
// find it for any shape.
struct RouterLayout {
    size_t qp_off, kp_off, tc_off, split_off, total;
};

// Fewer query rows than one tensor-core tile against more keys than one split
// range: the split selector (select_split.cu) instead of the CTA-per-128-rows
// one, which would give each row a single thread.
constexpr long long kSplitMaxRows = 128;
constexpr int kSplitMinKeys = 2048;
bool split_shape(int B, int H, int Nq, int Nk) {
    return (long long)B * H * Nq < kSplitMaxRows && Nk >= kSplitMinKeys;
}

constexpr size_t kCountersBytes = 256;

// Nq query rows per (b, h) against Nk keys per (b, kv head); K = 0 for scoring
// without selection.  own_kp = false: the caller holds the projected keys (the
// decode key cache), so the workspace has no k' region.
RouterLayout router_layout(int B, int H, int Hkv, int Nq, int Nk, int r, int K, bool own_kp = true) {
    RouterLayout l;
    const size_t qp = (size_t)B * H * Nq * r * sizeof(float);
    const size_t kp = own_kp ? (size_t)B * Hkv * Nk * r * sizeof(float) : 0;
    l.qp_off = kCountersBytes;
    l.kp_off = l.qp_off + align_up(qp);
    l.tc_off = l.kp_off + align_up(kp);
    l.split_off = l.tc_off + (r == 64 ? align_up(ossa::router_tc_workspace_bytes(B, H, Hkv, Nq, Nk, K)) : 0);
    l.total = l.split_off + (K > 0 && split_shape(B, H, Nq, Nk)
                                 ? align_up(ossa::split_select_workspace_bytes((long long)B * H * Nq, Nk, K))
                                 : 0);
    return l;
}

// The tensor-core selector serves r = 64, K <= 128 and at least one full tile of
// query and key rows; OSSA_ROUTER_SELECT=exact forces the CUDA-core exact selector
// of score_topk.cu in place of it and of the split selector (all produce identical
// indices; the switch exists to cross-check them).
bool use_tensor_core_select(int B, int H, int Hkv, int Nq, int Nk, int r, int K) {
    const char* env = getenv("OSSA_ROUTER_SELECT");
    if (env && env[0] == 'e') return false;
    return ossa::router_tc_supported(r, K) && (long long)B * Hkv * Nk >= 128 && (long long)B * H * Nq >= 128;
}

bool supported_r(int r) { return r == 16 || r == 32 || r == 64 || r == 128; }

// The oracle selection runs on the tensor-core kernel for head_dim 128, K <= 128
// and at least one full tile of query and key rows; OSSA_ORACLE_SELECT=exact
// forces the CUDA-core exact selector (identical indices; the switch exists to
// cross-check them).
bool use_tensor_core_oracle(int B, int H, int Hkv, int N, int D, int K) {
    const char* env = getenv("OSSA_ORACLE_SELECT");
    if (env && env[0] == 'e') return false;
    return ossa::oracle_tc_supported(D, K) && (long long)B * Hkv * N >= 128 && (long long)B * H * N >= 128;
}

size_t oracle_workspace_bytes(int B, int H, int Hkv, int N, int D, int K, int dtype) {
    if (!use_tensor_core_oracle(B, H, Hkv, N, D, K)) return kCountersBytes;
    return kCountersBytes + align_up(ossa::oracle_tc_workspace_bytes(B, H, Hkv, N, K, dtype));
}

int check_rows(int Nq, int Nk, int q0) {
    if (Nq < 0 || q0 < 0 || (long long)q0 + Nq > (1ll << 30))
        return fail(OSSA_ERR_INVALID, "bad query rows Nq=%d q_start=%d (keys %d)", Nq, q0, Nk);
    return OSSA_OK;
}

int check_router(const void* q, const void* k, int dtype, const float* wq, const float* wk,
                 const float* pos_bias, int B, int H, int Hkv, int Nq, int Nk, int q0, int D, int r,
                 int seq_len_cfg, int K, const void* out, void* ws, size_t ws_bytes, bool own_kp = true) {
    int st = check_heads(B, H, Hkv, Nk);
    if (st) return st;
    if ((st = check_rows(Nq, Nk, q0))) return st;
    if (!valid_dtype(dtype)) return fail(OSSA_ERR_INVALID, "bad dtype %d", dtype);
    if (D <= 0) return fail(OSSA_ERR_INVALID, "bad head_dim D=%d", D);
    if (!supported_r(r)) return fail(OSSA_ERR_UNSUPPORTED, "proj_dim r=%d not in {16,32,64,128}", r);
    if (seq_len_cfg <= 0 || seq_len_cfg > (1 << 28))
        return fail(OSSA_ERR_INVALID, "bad seq_len_cfg %d", seq_len_cfg);
    if ((long long)B * H * Nq == 0) return OSSA_OK;
    if (Nk == 0) return fail(OSSA_ERR_INVALID, "query rows need at least one key (Nk=0)");
    if (!q || !k || !wq || !wk || !pos_bias || !out)
        return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (!aligned16(q) || !aligned16(k) || !aligned16(out))
        return fail(OSSA_ERR_INVALID, "q, k and the output must be 16-byte aligned");
    const RouterLayout l = router_layout(B, H, Hkv, Nq, Nk, r, K, own_kp);
    if (!ws || ws_bytes < l.total || !aligned16(ws))
        return fail(OSSA_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) required, got %zu",
                    l.total, ws ? ws_bytes : (size_t)0);
    return OSSA_OK;
}

// Whether the tensor-core selector takes this call with its query operand made
// straight from the bf16 q rows (router_qtc.cu) and canonical q' only for the rows
// that need it.  OSSA_QPROJ=canonical projects every row first (the same indices;
// the switch exists to cross-check the two).
bool lazy_qproj(const ossa::ProjectArgs& pa, int B, int H, int Hkv, int Nq, int Nk, int r, int K) {
    const char* env = getenv("OSSA_QPROJ");
    if (env && env[0] == 'c') return false;
    return use_tensor_core_select(B, H, Hkv, Nq, Nk, r, K) && ossa::qproj_tc_supported(pa);
}

int project_both(const void* q, const void* k, int dtype, const float* wq, const float* wk,
                 int B, int H, int Hkv, int Nq, int Nk, int D, int r, void* ws, cudaStream_t stream,
                 float** qp_out, float** kp_out) {
    const RouterLayout l = router_layout(B, H, Hkv, Nq, Nk, r, 0);  // qp_off, kp_off do not depend on K
    char* base = static_cast<char*>(ws);
    float* qp = reinterpret_cast<float*>(base + l.qp_off);
    float* kp = reinterpret_cast<float*>(base + l.kp_off);
    ossa::ProjectArgs pa{q, wq, qp, (long long)B * H * Nq, D, r, dtype};
    int st = cuda_status(ossa::launch_project(pa, stream), "q projection launch");
    if (st) return st;
    ossa::ProjectArgs pk{k, wk, kp, (long long)B * Hkv * Nk, D, r, dtype};
    st = cuda_status(ossa::launch_project(pk, stream), "k projection launch");
    if (st) return st;
    *qp_out = qp;
    *kp_out = kp;
    return OSSA_OK;
}

// Selection of Nq query rows from projected q' (B*H*Nq, r) and k' (B*Hkv*Nk, r):
// the tensor-core selector, the split selector (few rows, many keys) or the
// CTA selector; `l` is the workspace layout of the call.
// qproj: the q projection, not launched yet, when the caller leaves q' to the
// tensor-core selector (lazy_qproj); any other selector projects it first.
int select_rows(const float* qp, const float* kp, const float* pos_bias, int B, int H, int Hkv, int Nq, int Nk,
                int r, int seq_len_cfg, int K, int causal, int q_start, int32_t* idx_out, void* workspace,
                const RouterLayout& l, cudaStream_t s, const ossa::ProjectArgs* qproj = nullptr) {
    const float scale = (float)(1.0 / sqrt((double)r));
    if (use_tensor_core_select(B, H, Hkv, Nq, Nk, r, K)) {
        ossa::RouterTcArgs a{qp, kp, pos_bias, seq_len_cfg, B, H, Hkv, Nk, K, causal ? 1 : 0, scale,
                             idx_out, static_cast<char*>(workspace) + l.tc_off,
                             reinterpret_cast<int*>(workspace)};
        a.Nq = Nq;
        a.q0 = q_start;
        a.qproj = qproj;
        return cuda_status(ossa::launch_router_tc(a, s), "tensor-core router top-K launch");
    }
    if (qproj) {
        int st = cuda_status(ossa::launch_project(*qproj, s), "q projection launch");
        if (st) return st;
    }
    const char* env = getenv("OSSA_ROUTER_SELECT");
    if (split_shape(B, H, Nq, Nk) && !(env && env[0] == 'e')) {
        ossa::SplitSelectArgs a{qp, kp, pos_bias, seq_len_cfg, B, H, Hkv, Nk, r, K, scale, causal ? 1 : 0,
                                idx_out, Nq, q_start, static_cast<char*>(workspace) + l.split_off};
        return cuda_status(ossa::launch_split_select(a, s), "split router top-K launch");
    }
    ossa::ScoreTopkArgs a{qp, kp, ossa::kF32, pos_bias, seq_len_cfg, B, H, Hkv, Nk, r, K, scale,
                          causal ? 1 : 0, idx_out};
    a.Nq = Nq;
    a.q0 = q_start;
    return cuda_status(ossa::launch_score_topk(a, s), "router top-K launch");
}

}  // namespace

extern "C" {

const char* ossa_version(void) { return "0.1.0"; }

const char* ossa_last_error_string(void) { return g_last_error.c_str(); }

uint64_t ossa_launch_count(void) { return (uint64_t)ossa::g_launches.load(std::memory_order_relaxed); }

int ossa_topk_attention_fwd_rows(const void* q, const void* k, const void* v, const void* indices,
                                 int idx_is_64, int dtype, int B, int H, int Hkv, int Nq, int Nk, int D, int K,
                                 float scale, int causal, int q_start, void* out, ossa_stream_t stream) {
    int st = check_heads(B, H, Hkv, Nk);
    if (st) return st;
    if ((st = check_rows(Nq, Nk, q_start))) return st;
    if (!valid_dtype(dtype)) return fail(OSSA_ERR_INVALID, "bad dtype %d", dtype);
    if (D != 16 && D != 32 && D != 64 && D != 128 && D != 256)
        return fail(OSSA_ERR_UNSUPPORTED, "head_dim D=%d not in {16,32,64,128,256}", D);
    if (K < 0) return fail(OSSA_ERR_INVALID, "bad K=%d", K);
    if (idx_is_64 != 0 && idx_is_64 != 1) return fail(OSSA_ERR_INVALID, "idx_is_64 must be 0 or 1");
    if (!isfinite(scale)) return fail(OSSA_ERR_INVALID, "scale must be finite");
    if ((long long)B * H * Nq == 0) return OSSA_OK;
    if (Nk == 0) return fail(OSSA_ERR_INVALID, "query rows need at least one key (Nk=0)");
    if (!q || !k || !v || !out || (K > 0 && !indices))
        return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
        return fail(OSSA_ERR_INVALID, "q, k, v and out must be 16-byte aligned");
    if (K > 0 && !aligned16(indices)) return fail(OSSA_ERR_INVALID, "indices must be 16-byte aligned");
    ossa::GatherArgs a{q, k, v, indices, out, idx_is_64, dtype, B, H, Hkv, Nk, D, K, scale, causal ? 1 : 0};
    a.Nq = Nq;
    a.q0 = q_start;
    return cuda_status(ossa::launch_gather_attn(a, static_cast<cudaStream_t>(stream)),
                       "topk attention launch");
}

int ossa_topk_attention_fwd(const void* q, const void* k, const void* v, const void* indices,
                            int idx_is_64, int dtype, int B, int H, int Hkv, int N, int D, int K,
                            float scale, int causal, void* out, ossa_stream_t stream) {
    return ossa_topk_attention_fwd_rows(q, k, v, indices, idx_is_64, dtype, B, H, Hkv, N, N, D, K, scale, causal,
                                        0, out, stream);
}

// Listed keys of one kv head that the backward's turned lists hold (32-bit places).
static constexpr long long kMaxTurned = 1ll << 30;

// The checks that the modified gather and its backward share.
static int check_modified(int dtype, int B, int H, int Hkv, int Nq, int Nk, int D, int K, int idx_is_64, float scale,
                          int q_start, float softcap, const float* slopes, const int32_t* segments,
                          const int32_t* prefix_len, const float* lse2) {
    int st = check_heads(B, H, Hkv, Nk);
    if (st) return st;
    if ((st = check_rows(Nq, Nk, q_start))) return st;
    if (!valid_dtype(dtype)) return fail(OSSA_ERR_INVALID, "bad dtype %d", dtype);
    if (D != 16 && D != 32 && D != 64 && D != 128 && D != 256)
        return fail(OSSA_ERR_UNSUPPORTED, "head_dim D=%d not in {16,32,64,128,256}", D);
    if (K < 0) return fail(OSSA_ERR_INVALID, "bad K=%d", K);
    if (idx_is_64 != 0 && idx_is_64 != 1) return fail(OSSA_ERR_INVALID, "idx_is_64 must be 0 or 1");
    if (!isfinite(scale)) return fail(OSSA_ERR_INVALID, "scale must be finite");
    if (!isfinite(softcap) || softcap < 0.f || (softcap > 0.f && softcap < FLT_MIN))  // below, 1 / softcap overflows
        return fail(OSSA_ERR_INVALID, "softcap must be 0, or finite and at least 2^-126");
    if (segments && (long long)q_start + Nq > Nk)
        return fail(OSSA_ERR_INVALID, "segments need every query position below Nk=%d (rows end at %lld)", Nk,
                    (long long)q_start + Nq);
    if ((long long)B * Hkv > 65535) return fail(OSSA_ERR_UNSUPPORTED, "B * Hkv = %lld > 65535", (long long)B * Hkv);
    if (!aligned_to(4, slopes, segments, prefix_len, lse2))
        return fail(OSSA_ERR_INVALID, "slopes, segments, prefix_len and lse2 must be aligned to their types");
    return OSSA_OK;
}

static ossa::ScoreMods make_mods(float scale, float softcap, const float* slopes, const int32_t* segments,
                                 const int32_t* prefix_len, float* lse2, void* out_rest) {
    return ossa::ScoreMods{scale, scale * 1.4426950408889634f, softcap, softcap > 0.f ? 1.f / softcap : 0.f,
                           softcap > 0.f || slopes ? 1 : 0, slopes, segments, prefix_len, lse2, out_rest};
}

int ossa_topk_attention_mod_fwd(const void* q, const void* k, const void* v, const void* indices, int idx_is_64,
                                int dtype, int B, int H, int Hkv, int Nq, int Nk, int D, int K, float scale, int causal,
                                int q_start, float softcap, const float* slopes, const int32_t* segments,
                                const int32_t* prefix_len, void* out, float* lse2, void* out_rest,
                                ossa_stream_t stream) {
    int st = check_modified(dtype, B, H, Hkv, Nq, Nk, D, K, idx_is_64, scale, q_start, softcap, slopes, segments,
                            prefix_len, lse2);
    if (st) return st;
    if ((long long)B * H * Nq == 0) return OSSA_OK;
    if (Nk == 0) return fail(OSSA_ERR_INVALID, "query rows need at least one key (Nk=0)");
    if (!q || !k || !v || !out || (K > 0 && !indices)) return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
        return fail(OSSA_ERR_INVALID, "q, k, v and out must be 16-byte aligned");
    if (K > 0 && reinterpret_cast<uintptr_t>(indices) % (idx_is_64 ? 8 : 4))
        return fail(OSSA_ERR_INVALID, "indices are not aligned to their type");
    ossa::GatherArgs a{q, k, v, indices, out, idx_is_64, dtype, B, H, Hkv, Nk, D, K, scale, causal ? 1 : 0};
    a.Nq = Nq;
    a.q0 = q_start;
    if (out_rest && (dtype != OSSA_BF16 || !aligned16(out_rest)))
        return fail(OSSA_ERR_INVALID, "out_rest goes with bf16 outputs and must be 16-byte aligned");
    a.mods = make_mods(scale, softcap, slopes, segments, prefix_len, lse2, out_rest);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (softcap == 0.f && !slopes && !segments && !prefix_len && !lse2 && !out_rest)
        return cuda_status(ossa::launch_gather_attn(a, s), "topk attention launch");
    return cuda_status(ossa::launch_gather_attn_mods(a, s), "modified topk attention launch");
}

size_t ossa_topk_attention_bwd_workspace_size(int dtype, int B, int H, int Hkv, int Nq, int Nk, int D, int K,
                                              int want_dslopes) {
    if (!valid_dtype(dtype) || B < 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || Nq < 0 || Nk < 0 || D <= 0 || K < 0) return 0;
    if ((long long)(H / Hkv) * Nq * K > kMaxTurned) return 0;  // refused by the backward call
    return ossa::gather_bwd_workspace_bytes(dtype, B, H, Hkv, Nq, Nk, D, K, want_dslopes != 0);
}

int ossa_topk_attention_bwd(const void* q, const void* k, const void* v, const void* indices, int idx_is_64, int dtype,
                            int B, int H, int Hkv, int Nq, int Nk, int D, int K, float scale, int causal, int q_start,
                            float softcap, const float* slopes, const int32_t* segments, const int32_t* prefix_len,
                            const void* out, const float* lse2, const void* out_rest, const void* dout, void* dq,
                            void* dk, void* dv, float* dslopes, void* workspace, size_t workspace_bytes, ossa_stream_t stream) {
    int st = check_modified(dtype, B, H, Hkv, Nq, Nk, D, K, idx_is_64, scale, q_start, softcap, slopes, segments,
                            prefix_len, lse2);
    if (st) return st;
    if (dslopes && !slopes) return fail(OSSA_ERR_INVALID, "dslopes without slopes");
    if (!aligned_to(4, dslopes)) return fail(OSSA_ERR_INVALID, "dslopes is not aligned to its type");
    if ((long long)(H / Hkv) * Nq * K > kMaxTurned)
        return fail(OSSA_ERR_UNSUPPORTED, "(H / Hkv) * Nq * K = %lld > 2^30 listed keys per kv head",
                    (long long)(H / Hkv) * Nq * K);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const size_t es = dtype == OSSA_F32 ? 4 : 2;
    const size_t qn = (size_t)B * H * Nq * D * es, kn = (size_t)B * Hkv * Nk * D * es;
    if ((qn && !dq) || (kn && (!dk || !dv))) return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (qn == 0 || K == 0) {  // nothing listed: every gradient is zero
        if (qn && (st = cuda_status(cudaMemsetAsync(dq, 0, qn, s), "gradient reset"))) return st;
        if (kn && (st = cuda_status(cudaMemsetAsync(dk, 0, kn, s), "gradient reset"))) return st;
        if (kn && (st = cuda_status(cudaMemsetAsync(dv, 0, kn, s), "gradient reset"))) return st;
        if (dslopes && (st = cuda_status(cudaMemsetAsync(dslopes, 0, (size_t)H * 4, s), "gradient reset"))) return st;
        return OSSA_OK;
    }
    if (Nk == 0) return fail(OSSA_ERR_INVALID, "query rows need at least one key (Nk=0)");
    if (!q || !k || !v || !out || !indices || !lse2 || !dout) return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(dout) || !aligned16(dq) ||
        !aligned16(dk) || !aligned16(dv))
        return fail(OSSA_ERR_INVALID, "q, k, v, out, dout, dq, dk and dv must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(indices) % (idx_is_64 ? 8 : 4))
        return fail(OSSA_ERR_INVALID, "indices are not aligned to their type");
    const size_t need = ossa::gather_bwd_workspace_bytes(dtype, B, H, Hkv, Nq, Nk, D, K, dslopes != nullptr);
    if (!workspace || workspace_bytes < need || !aligned16(workspace))
        return fail(OSSA_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) required, got %zu", need,
                    workspace ? workspace_bytes : (size_t)0);
    ossa::GatherBwdArgs a{};
    a.f = ossa::GatherArgs{q, k, v, indices, const_cast<void*>(out), idx_is_64, dtype, B, H, Hkv, Nk, D, K, scale,
                           causal ? 1 : 0};
    a.f.Nq = Nq;
    a.f.q0 = q_start;
    if (out_rest && (dtype != OSSA_BF16 || !aligned16(out_rest)))
        return fail(OSSA_ERR_INVALID, "out_rest goes with bf16 outputs and must be 16-byte aligned");
    a.f.mods = make_mods(scale, softcap, slopes, segments, prefix_len, const_cast<float*>(lse2),
                         const_cast<void*>(out_rest));
    a.dout = dout;
    a.dq = dq;
    a.dk = dk;
    a.dv = dv;
    a.dslopes = dslopes;
    a.ws = workspace;
    return cuda_status(ossa::launch_gather_attn_bwd(a, s), "topk attention backward launch");
}

// The checks that the head norm's forward and backward share.
static int check_norm_rope(const void* q, const void* k, const void* wq, const void* wk, const void* cos, const void* sin,
                           int dtype, int w_dtype, int B, int N, int Hq, int Hk, int D, long long q_sb, long long q_sn,
                           long long k_sb, long long k_sn, float eps) {
    if (!valid_dtype(dtype)) return fail(OSSA_ERR_INVALID, "bad dtype %d", dtype);
    if (!valid_dtype(w_dtype)) return fail(OSSA_ERR_INVALID, "bad weight dtype %d", w_dtype);
    if (B < 0 || N < 0 || Hq <= 0 || Hk < 0 || D <= 0 || D % 8 != 0)
        return fail(OSSA_ERR_INVALID, "bad shape B=%d N=%d heads=%d,%d D=%d (D must be a multiple of 8)", B, N, Hq, Hk, D);
    if (D > 512) return fail(OSSA_ERR_UNSUPPORTED, "head_dim D=%d > 512", D);
    if ((long long)B * N > (1ll << 30) || Hq > (1 << 16) || Hk > (1 << 16))
        return fail(OSSA_ERR_UNSUPPORTED, "shape too large B=%d N=%d heads=%d,%d", B, N, Hq, Hk);
    if (!(eps >= 0.f) || !isfinite(eps)) return fail(OSSA_ERR_INVALID, "eps must be finite and >= 0");
    if ((!cos) != (!sin)) return fail(OSSA_ERR_INVALID, "pass both cos and sin, or neither");
    const int unit = dtype == OSSA_F32 ? 4 : 8;  // elements of 16 bytes
    if (q_sb % unit || q_sn % unit || (Hk && (k_sb % unit || k_sn % unit)))
        return fail(OSSA_ERR_INVALID, "row strides must be multiples of 16 bytes");
    if (!aligned16(q) || !aligned16(k) || !aligned16(cos) || !aligned16(sin))
        return fail(OSSA_ERR_INVALID, "q, k, cos and sin must be 16-byte aligned");
    if (!aligned_to(w_dtype == OSSA_F32 ? 4 : 2, wq, wk)) return fail(OSSA_ERR_INVALID, "weights are not aligned to their type");
    return OSSA_OK;
}

int ossa_qk_norm_rope_fwd(const void* q, const void* k, const void* wq, const void* wk, const void* cos,
                          const void* sin, int cs_batched, int dtype, int w_dtype, int B, int N, int Hq, int Hk, int D,
                          long long q_sb, long long q_sn, long long k_sb, long long k_sn, float eps, void* q_out,
                          void* k_out, ossa_stream_t stream) {
    int st = check_norm_rope(q, k, wq, wk, cos, sin, dtype, w_dtype, B, N, Hq, Hk, D, q_sb, q_sn, k_sb, k_sn, eps);
    if (st) return st;
    if ((long long)B * N == 0) return OSSA_OK;
    if (!q || !q_out || (Hk && (!k || !k_out))) return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (!aligned16(q_out) || !aligned16(k_out)) return fail(OSSA_ERR_INVALID, "outputs must be 16-byte aligned");
    ossa::NormRopeArgs a{};
    a.q = q;
    a.k = k;
    a.q_sb = q_sb;
    a.q_sn = q_sn;
    a.k_sb = k_sb;
    a.k_sn = k_sn;
    a.wq = wq;
    a.wk = wk;
    a.w_f32 = w_dtype == OSSA_F32;
    a.cosv = cos;
    a.sinv = sin;
    a.cs_batched = cs_batched ? 1 : 0;
    a.dtype = dtype;
    a.B = B;
    a.N = N;
    a.Hq = Hq;
    a.Hk = Hk;
    a.D = D;
    a.eps = eps;
    a.oq = q_out;
    a.ok = k_out;
    return cuda_status(ossa::launch_norm_rope_fwd(a, static_cast<cudaStream_t>(stream)), "head norm launch");
}

size_t ossa_qk_norm_rope_bwd_workspace_size(int D) { return D > 0 ? ossa::norm_rope_workspace_bytes(D) : 0; }

int ossa_qk_norm_rope_bwd(const void* q, const void* k, const void* wq, const void* wk, const void* cos,
                          const void* sin, int cs_batched, int dtype, int w_dtype, int B, int N, int Hq, int Hk, int D,
                          long long q_sb, long long q_sn, long long k_sb, long long k_sn, float eps, const void* dq_out,
                          const void* dk_out, void* dq, void* dk, void* dwq, void* dwk, void* workspace,
                          size_t workspace_bytes, ossa_stream_t stream) {
    int st = check_norm_rope(q, k, wq, wk, cos, sin, dtype, w_dtype, B, N, Hq, Hk, D, q_sb, q_sn, k_sb, k_sn, eps);
    if (st) return st;
    if ((dwq && !wq) || (dwk && !wk)) return fail(OSSA_ERR_INVALID, "a weight gradient without its weight");
    if (!aligned_to(w_dtype == OSSA_F32 ? 4 : 2, dwq, dwk))
        return fail(OSSA_ERR_INVALID, "weight gradients are not aligned to their type");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if ((long long)B * N == 0) {
        const size_t wn = (size_t)D * (w_dtype == OSSA_F32 ? 4 : 2);
        if (dwq && (st = cuda_status(cudaMemsetAsync(dwq, 0, wn, s), "gradient reset"))) return st;
        if (dwk && (st = cuda_status(cudaMemsetAsync(dwk, 0, wn, s), "gradient reset"))) return st;
        return OSSA_OK;
    }
    if (!dq_out || !dq || (wq && !q) || (Hk && (!dk_out || !dk || (wk && !k))))
        return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (!aligned16(dq_out) || !aligned16(dk_out) || !aligned16(dq) || !aligned16(dk))
        return fail(OSSA_ERR_INVALID, "gradients must be 16-byte aligned");
    const size_t need = ossa::norm_rope_workspace_bytes(D);
    if ((wq || (Hk && wk)) && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail(OSSA_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) required, got %zu", need,
                    workspace ? workspace_bytes : (size_t)0);
    ossa::NormRopeArgs a{};
    a.q = q;
    a.k = k;
    a.q_sb = q_sb;
    a.q_sn = q_sn;
    a.k_sb = k_sb;
    a.k_sn = k_sn;
    a.wq = wq;
    a.wk = Hk ? wk : nullptr;
    a.w_f32 = w_dtype == OSSA_F32;
    a.cosv = cos;
    a.sinv = sin;
    a.cs_batched = cs_batched ? 1 : 0;
    a.dtype = dtype;
    a.B = B;
    a.N = N;
    a.Hq = Hq;
    a.Hk = Hk;
    a.D = D;
    a.eps = eps;
    a.gq = dq_out;
    a.gk = dk_out;
    a.oq = dq;
    a.ok = dk;
    a.dwq = dwq;
    a.dwk = Hk ? dwk : nullptr;
    a.part = static_cast<float*>(workspace);
    return cuda_status(ossa::launch_norm_rope_bwd(a, s), "head norm backward launch");
}

// The checks that the top-logit distillation's forward and backward share.
static int check_logit_distill(const void* logits, int dtype, int outer, int inner, int V, const void* ids,
                               int ids_are_64, int K, float temperature, const void* dlogits, void* workspace,
                               size_t workspace_bytes) {
    if (!valid_dtype(dtype)) return fail(OSSA_ERR_INVALID, "bad dtype %d", dtype);
    if (outer < 0 || inner < 0 || V <= 0 || K <= 0)
        return fail(OSSA_ERR_INVALID, "bad shape rows=%dx%d V=%d K=%d", outer, inner, V, K);
    if (K > 1024) return fail(OSSA_ERR_UNSUPPORTED, "K=%d > 1024 teacher entries per row", K);
    if (V > (1 << 30) || (long long)outer * inner > (1ll << 30))
        return fail(OSSA_ERR_UNSUPPORTED, "shape too large rows=%dx%d V=%d", outer, inner, V);
    if (ids_are_64 != 0 && ids_are_64 != 1) return fail(OSSA_ERR_INVALID, "ids_are_64 must be 0 or 1");
    if (!(temperature >= FLT_MIN) || !isfinite(temperature))  // below, log2(e) / temperature overflows
        return fail(OSSA_ERR_INVALID, "temperature must be finite and at least 2^-126");
    if ((long long)outer * inner == 0) return fail(OSSA_ERR_INVALID, "empty input (no rows)");
    if (!logits || !ids) return fail(OSSA_ERR_INVALID, "null pointer argument");
    const uintptr_t es = dtype == OSSA_F32 ? 4 : 2;
    if (!aligned_to(es, logits, dlogits)) return fail(OSSA_ERR_INVALID, "logits are not aligned to their type");
    if (!aligned_to(ids_are_64 ? 8 : 4, ids)) return fail(OSSA_ERR_INVALID, "ids are not aligned to their type");
    const size_t need = ossa::logit_distill_workspace_bytes((long long)outer * inner, K);
    if (!workspace || workspace_bytes < need || !aligned16(workspace))
        return fail(OSSA_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) required, got %zu", need,
                    workspace ? workspace_bytes : (size_t)0);
    return OSSA_OK;
}

size_t ossa_top_logit_distill_workspace_size(long long rows, int K) {
    if (rows < 0 || rows > (1ll << 30) || K <= 0 || K > 1024) return 0;  // refused by the calls
    return ossa::logit_distill_workspace_bytes(rows, K);
}

int ossa_top_logit_distill_fwd(const void* logits, int dtype, int outer, int inner, int V, long long stride_outer,
                               long long stride_inner, const float* teacher, const void* ids, int ids_are_64, int K,
                               float temperature, const float* row_weight, int mean, float* loss_rows, float* loss,
                               void* dlogits, void* workspace, size_t workspace_bytes, ossa_stream_t stream) {
    int st = check_logit_distill(logits, dtype, outer, inner, V, ids, ids_are_64, K, temperature, dlogits, workspace,
                                 workspace_bytes);
    if (st) return st;
    if (!teacher || (!loss_rows && !loss)) return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (!aligned_to(4, teacher, row_weight, loss_rows, loss))
        return fail(OSSA_ERR_INVALID, "teacher, row_weight and losses must be aligned to their type");
    ossa::LogitDistillArgs a{};
    a.z = logits;
    a.sb = stride_outer;
    a.st = stride_inner;
    a.dtype = dtype;
    a.outer = outer;
    a.inner = inner;
    a.V = V;
    a.teacher = teacher;
    a.ids = ids;
    a.ids_are_64 = ids_are_64;
    a.K = K;
    a.tau = temperature;
    a.row_weight = row_weight;
    a.mean = mean ? 1 : 0;
    a.loss_rows = loss_rows;
    a.loss = loss;
    a.dz = dlogits;
    a.ws = workspace;
    return cuda_status(ossa::launch_logit_distill_fwd(a, static_cast<cudaStream_t>(stream)),
                       "top-logit distillation launch");
}

int ossa_top_logit_distill_bwd(const void* logits, int dtype, int outer, int inner, int V, long long stride_outer,
                               long long stride_inner, const void* ids, int ids_are_64, int K, float temperature,
                               int mean, const float* grad, int grad_per_row, int skip_if_one, void* dlogits,
                               const void* workspace, size_t workspace_bytes, ossa_stream_t stream) {
    int st = check_logit_distill(logits, dtype, outer, inner, V, ids, ids_are_64, K, temperature, dlogits,
                                 const_cast<void*>(workspace), workspace_bytes);
    if (st) return st;
    if (!grad || !dlogits) return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (!aligned_to(4, grad)) return fail(OSSA_ERR_INVALID, "grad is not aligned to its type");
    if (skip_if_one && grad_per_row) return fail(OSSA_ERR_INVALID, "skip_if_one needs a single gradient value");
    ossa::LogitDistillArgs a{};
    a.z = logits;
    a.sb = stride_outer;
    a.st = stride_inner;
    a.dtype = dtype;
    a.outer = outer;
    a.inner = inner;
    a.V = V;
    a.ids = ids;
    a.ids_are_64 = ids_are_64;
    a.K = K;
    a.tau = temperature;
    a.mean = mean ? 1 : 0;
    a.grad = grad;
    a.grad_per_row = grad_per_row ? 1 : 0;
    a.skip_if_one = skip_if_one ? 1 : 0;
    a.dz = dlogits;
    a.ws = const_cast<void*>(workspace);
    return cuda_status(ossa::launch_logit_distill_bwd(a, static_cast<cudaStream_t>(stream)),
                       "top-logit distillation backward launch");
}

int ossa_router_status(const void* workspace, int* fallback_rows, int* status) {
    if (!workspace || !aligned16(workspace)) return fail(OSSA_ERR_INVALID, "bad workspace pointer");
    int h[2] = {0, 0};
    int st = cuda_status(cudaMemcpy(h, workspace, sizeof(h), cudaMemcpyDeviceToHost), "status read");
    if (st) return st;
    if (fallback_rows) *fallback_rows = h[0];
    if (status) *status = h[1];
    return OSSA_OK;
}

size_t ossa_router_workspace_size_rows(int B, int H, int Hkv, int Nq, int Nk, int r, int K) {
    if (B < 0 || H <= 0 || Hkv <= 0 || Nq < 0 || Nk < 0 || r <= 0) return 0;
    return router_layout(B, H, Hkv, Nq, Nk, r, K).total;
}

size_t ossa_router_workspace_size(int B, int H, int Hkv, int N, int r, int K) {
    return ossa_router_workspace_size_rows(B, H, Hkv, N, N, r, K);
}

int ossa_router_topk_rows(const void* q, const void* k, int dtype, const float* wq, const float* wk,
                          const float* pos_bias, int B, int H, int Hkv, int Nq, int Nk, int D, int r,
                          int seq_len_cfg, int K, int causal, int q_start, int32_t* idx_out, void* workspace,
                          size_t workspace_bytes, ossa_stream_t stream) {
    int st = check_router(q, k, dtype, wq, wk, pos_bias, B, H, Hkv, Nq, Nk, q_start, D, r, seq_len_cfg, K,
                          idx_out, workspace, workspace_bytes);
    if (st) return st;
    if (K <= 0) return fail(OSSA_ERR_INVALID, "bad K=%d", K);
    if (!ossa::score_topk_supported(r, K))
        return fail(OSSA_ERR_UNSUPPORTED, "top-K selection supports K <= 160 (got K=%d)", K);
    if ((long long)B * H * Nq == 0) return OSSA_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    st = cuda_status(cudaMemsetAsync(workspace, 0, kCountersBytes, s), "workspace counters reset");
    if (st) return st;
    const RouterLayout l = router_layout(B, H, Hkv, Nq, Nk, r, K);
    float* qp = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.qp_off);
    float* kp = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.kp_off);
    const ossa::ProjectArgs pa{q, wq, qp, (long long)B * H * Nq, D, r, dtype};
    if (lazy_qproj(pa, B, H, Hkv, Nq, Nk, r, K)) {
        const ossa::ProjectArgs pk{k, wk, kp, (long long)B * Hkv * Nk, D, r, dtype};
        if ((st = cuda_status(ossa::launch_project(pk, s), "k projection launch"))) return st;
        return select_rows(qp, kp, pos_bias, B, H, Hkv, Nq, Nk, r, seq_len_cfg, K, causal, q_start, idx_out,
                           workspace, l, s, &pa);
    }
    st = project_both(q, k, dtype, wq, wk, B, H, Hkv, Nq, Nk, D, r, workspace, s, &qp, &kp);
    if (st) return st;
    return select_rows(qp, kp, pos_bias, B, H, Hkv, Nq, Nk, r, seq_len_cfg, K, causal, q_start, idx_out, workspace,
                       l, s);
}

size_t ossa_router_workspace_size_kp(int B, int H, int Hkv, int Nq, int Nk, int r, int K) {
    if (B < 0 || H <= 0 || Hkv <= 0 || Nq < 0 || Nk < 0 || r <= 0) return 0;
    return router_layout(B, H, Hkv, Nq, Nk, r, K, false).total;
}

int ossa_router_project_keys(const void* k, int dtype, const float* wk, long long rows, int D, int r,
                             float* kp_out, ossa_stream_t stream) {
    if (!valid_dtype(dtype)) return fail(OSSA_ERR_INVALID, "bad dtype %d", dtype);
    if (rows < 0 || D <= 0) return fail(OSSA_ERR_INVALID, "bad shape rows=%lld D=%d", rows, D);
    if (!supported_r(r)) return fail(OSSA_ERR_UNSUPPORTED, "proj_dim r=%d not in {16,32,64,128}", r);
    if (rows == 0) return OSSA_OK;
    if (!k || !wk || !kp_out) return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (!aligned16(k) || !aligned16(kp_out)) return fail(OSSA_ERR_INVALID, "k and kp_out must be 16-byte aligned");
    ossa::ProjectArgs pk{k, wk, kp_out, rows, D, r, dtype};
    return cuda_status(ossa::launch_project(pk, static_cast<cudaStream_t>(stream)), "k projection launch");
}

int ossa_router_topk_rows_kp(const void* q, int dtype, const float* wq, const float* kp, const float* pos_bias,
                             int B, int H, int Hkv, int Nq, int Nk, int D, int r, int seq_len_cfg, int K,
                             int causal, int q_start, int32_t* idx_out, void* workspace, size_t workspace_bytes,
                             ossa_stream_t stream) {
    int st = check_router(q, kp, dtype, wq, wq, pos_bias, B, H, Hkv, Nq, Nk, q_start, D, r, seq_len_cfg, K,
                          idx_out, workspace, workspace_bytes, false);
    if (st) return st;
    if (K <= 0) return fail(OSSA_ERR_INVALID, "bad K=%d", K);
    if (!ossa::score_topk_supported(r, K))
        return fail(OSSA_ERR_UNSUPPORTED, "top-K selection supports K <= 160 (got K=%d)", K);
    if ((long long)B * H * Nq == 0) return OSSA_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    st = cuda_status(cudaMemsetAsync(workspace, 0, kCountersBytes, s), "workspace counters reset");
    if (st) return st;
    const RouterLayout l = router_layout(B, H, Hkv, Nq, Nk, r, K, false);
    float* qp = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.qp_off);
    const ossa::ProjectArgs pa{q, wq, qp, (long long)B * H * Nq, D, r, dtype};
    if (lazy_qproj(pa, B, H, Hkv, Nq, Nk, r, K))
        return select_rows(qp, kp, pos_bias, B, H, Hkv, Nq, Nk, r, seq_len_cfg, K, causal, q_start, idx_out,
                           workspace, l, s, &pa);
    st = cuda_status(ossa::launch_project(pa, s), "q projection launch");
    if (st) return st;
    return select_rows(qp, kp, pos_bias, B, H, Hkv, Nq, Nk, r, seq_len_cfg, K, causal, q_start, idx_out, workspace,
                       l, s);
}

int ossa_router_topk(const void* q, const void* k, int dtype, const float* wq, const float* wk,
                     const float* pos_bias, int B, int H, int Hkv, int N, int D, int r,
                     int seq_len_cfg, int K, int causal, int32_t* idx_out, void* workspace,
                     size_t workspace_bytes, ossa_stream_t stream) {
    return ossa_router_topk_rows(q, k, dtype, wq, wk, pos_bias, B, H, Hkv, N, N, D, r, seq_len_cfg, K, causal, 0,
                                 idx_out, workspace, workspace_bytes, stream);
}

int ossa_router_topk_sorted(const void* q, const void* k, int dtype, const float* wq, const float* wk,
                            const float* pos_bias, int B, int H, int Hkv, int N, int D, int r, int seq_len_cfg,
                            int K, int causal, int32_t* idx_out, void* workspace, size_t workspace_bytes,
                            ossa_stream_t stream) {
    int st = ossa_router_topk(q, k, dtype, wq, wk, pos_bias, B, H, Hkv, N, D, r, seq_len_cfg, K, causal, idx_out,
                              workspace, workspace_bytes, stream);
    if (st) return st;
    if ((long long)B * H * N == 0) return OSSA_OK;
    if (!ossa::sort_rows_supported(r, K))
        return fail(OSSA_ERR_UNSUPPORTED, "score-ordered rows support K <= 256 (got K=%d)", K);
    // the selection left the canonical k' in the workspace, and q' too unless the
    // tensor-core selector made only the rows it needed: then q' is projected here
    const RouterLayout l = router_layout(B, H, Hkv, N, N, r, K);
    char* base = static_cast<char*>(workspace);
    const ossa::ProjectArgs pa{q, wq, reinterpret_cast<float*>(base + l.qp_off), (long long)B * H * N, D, r, dtype};
    if (lazy_qproj(pa, B, H, Hkv, N, N, r, K) &&
        (st = cuda_status(ossa::launch_project(pa, static_cast<cudaStream_t>(stream)), "q projection launch")))
        return st;
    ossa::SortRowsArgs a{reinterpret_cast<const float*>(base + l.qp_off),
                         reinterpret_cast<const float*>(base + l.kp_off),
                         pos_bias, seq_len_cfg, H, Hkv, N, r, K, (float)(1.0 / sqrt((double)r)),
                         (long long)B * H * N, idx_out};
    return cuda_status(ossa::launch_sort_rows(a, static_cast<cudaStream_t>(stream)), "score-order launch");
}

int ossa_router_score(const void* q, const void* k, int dtype, const float* wq, const float* wk,
                      const float* pos_bias, int B, int H, int Hkv, int N, int D, int r,
                      int seq_len_cfg, float* scores_out, void* workspace, size_t workspace_bytes,
                      ossa_stream_t stream) {
    int st = check_router(q, k, dtype, wq, wk, pos_bias, B, H, Hkv, N, N, 0, D, r, seq_len_cfg, 0,
                          scores_out, workspace, workspace_bytes);
    if (st) return st;
    if ((long long)B * H * N == 0) return OSSA_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    float *qp = nullptr, *kp = nullptr;
    st = project_both(q, k, dtype, wq, wk, B, H, Hkv, N, N, D, r, workspace, s, &qp, &kp);
    if (st) return st;
    ossa::ScoreDenseArgs a{qp, kp, pos_bias, seq_len_cfg, B, H, Hkv, N, r,
                           (float)(1.0 / sqrt((double)r)), scores_out};
    return cuda_status(ossa::launch_score_dense(a, s), "router score launch");
}

int ossa_oracle_topk(const void* q, const void* k, int dtype, int B, int H, int Hkv, int N, int D,
                     float scale, int K, int causal, int32_t* idx_out, ossa_stream_t stream) {
    int st = check_heads(B, H, Hkv, N);
    if (st) return st;
    if (!valid_dtype(dtype)) return fail(OSSA_ERR_INVALID, "bad dtype %d", dtype);
    if (!supported_r(D))
        return fail(OSSA_ERR_UNSUPPORTED, "oracle selection supports head_dim in {16,32,64,128}, got %d", D);
    if (K <= 0) return fail(OSSA_ERR_INVALID, "bad K=%d", K);
    if (!ossa::score_topk_supported(D, K))
        return fail(OSSA_ERR_UNSUPPORTED, "top-K selection supports K <= 160 (got K=%d)", K);
    if (!isfinite(scale)) return fail(OSSA_ERR_INVALID, "scale must be finite");
    if ((long long)B * H * N == 0) return OSSA_OK;
    if (!q || !k || !idx_out) return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (!aligned16(q) || !aligned16(k) || !aligned16(idx_out))
        return fail(OSSA_ERR_INVALID, "q, k and the output must be 16-byte aligned");
    ossa::ScoreTopkArgs a{q, k, dtype, nullptr, 1, B, H, Hkv, N, D, K, scale, causal ? 1 : 0, idx_out};
    return cuda_status(ossa::launch_score_topk(a, static_cast<cudaStream_t>(stream)),
                       "oracle top-K launch");
}

size_t ossa_router_distill_workspace_size(int B, int H, int Hkv, int N, int r) {
    if (B < 0 || H <= 0 || Hkv <= 0 || N < 0 || !supported_r(r)) return 0;
    const size_t rq = (size_t)B * H * N * r * sizeof(float), rk = (size_t)B * Hkv * N * r * sizeof(float);
    return kCountersBytes + 2 * align_up(rq) + 2 * align_up(rk) +
           align_up(ossa::distill_loss_parts(B, H, N) * sizeof(float));
}

int ossa_router_distill_grad(const void* q, const void* k, int dtype, const float* wq, const float* wk,
                             const float* pos_bias, int B, int H, int Hkv, int N, int D, int r, int seq_len_cfg,
                             const int32_t* targets, int K, float* loss_out, float* dwq, float* dwk,
                             float* dpos_bias, void* workspace, size_t workspace_bytes, ossa_stream_t stream) {
    int st = check_heads(B, H, Hkv, N);
    if (st) return st;
    if (!valid_dtype(dtype)) return fail(OSSA_ERR_INVALID, "bad dtype %d", dtype);
    if (D <= 0) return fail(OSSA_ERR_INVALID, "bad head_dim D=%d", D);
    if (!supported_r(r)) return fail(OSSA_ERR_UNSUPPORTED, "proj_dim r=%d not in {16,32,64,128}", r);
    if (seq_len_cfg <= 0 || seq_len_cfg > (1 << 28)) return fail(OSSA_ERR_INVALID, "bad seq_len_cfg %d", seq_len_cfg);
    if (K < 0) return fail(OSSA_ERR_INVALID, "bad K=%d", K);
    if ((long long)B * H * N == 0) return fail(OSSA_ERR_INVALID, "empty input (the mean loss is undefined)");
    if (!q || !k || !wq || !wk || !pos_bias || !loss_out || !dwq || !dwk || !dpos_bias || (K > 0 && !targets))
        return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (!aligned16(q) || !aligned16(k)) return fail(OSSA_ERR_INVALID, "q and k must be 16-byte aligned");
    const size_t need = ossa_router_distill_workspace_size(B, H, Hkv, N, r);
    if (!workspace || workspace_bytes < need || !aligned16(workspace))
        return fail(OSSA_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) required, got %zu", need,
                    workspace ? workspace_bytes : (size_t)0);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    char* w = static_cast<char*>(workspace) + kCountersBytes;
    const size_t rq = (size_t)B * H * N * r * sizeof(float), rk = (size_t)B * Hkv * N * r * sizeof(float);
    float* qp = reinterpret_cast<float*>(w);
    float* kp = reinterpret_cast<float*>(w + align_up(rq));
    float* dqp = reinterpret_cast<float*>(w + align_up(rq) + align_up(rk));
    float* dkp = reinterpret_cast<float*>(w + 2 * align_up(rq) + align_up(rk));
    float* parts = reinterpret_cast<float*>(w + 2 * align_up(rq) + 2 * align_up(rk));
    ossa::ProjectArgs pa{q, wq, qp, (long long)B * H * N, D, r, dtype};
    if ((st = cuda_status(ossa::launch_project(pa, s), "q projection launch"))) return st;
    ossa::ProjectArgs pk{k, wk, kp, (long long)B * Hkv * N, D, r, dtype};
    if ((st = cuda_status(ossa::launch_project(pk, s), "k projection launch"))) return st;
    if ((st = cuda_status(cudaMemsetAsync(dwq, 0, (size_t)r * D * sizeof(float), s), "gradient reset"))) return st;
    if ((st = cuda_status(cudaMemsetAsync(dwk, 0, (size_t)r * D * sizeof(float), s), "gradient reset"))) return st;
    if ((st = cuda_status(cudaMemsetAsync(dpos_bias, 0, (size_t)2 * seq_len_cfg * sizeof(float), s),
                          "gradient reset")))
        return st;
    ossa::DistillArgs a{q, k, dtype, qp, kp, pos_bias, seq_len_cfg, B, H, Hkv, N, D, r, targets, K,
                        dqp, dkp, dpos_bias, dwq, dwk, parts, loss_out};
    return cuda_status(ossa::launch_distill(a, s), "router distillation launch");
}

int ossa_rope_to_heads(const void* x, const void* cos, const void* sin, int cs_batched, int dtype, int B, int N,
                       int Hx, int D, void* out, ossa_stream_t stream) {
    if (!valid_dtype(dtype)) return fail(OSSA_ERR_INVALID, "bad dtype %d", dtype);
    if (B < 0 || N < 0 || Hx <= 0 || D <= 0 || D % 8 != 0)
        return fail(OSSA_ERR_INVALID, "bad shape B=%d N=%d heads=%d D=%d (D must be a multiple of 8)", B, N, Hx, D);
    if ((long long)B * N == 0) return OSSA_OK;
    if (!x || !out || (!cos) != (!sin)) return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (!aligned16(x) || !aligned16(out) || (cos && (!aligned16(cos) || !aligned16(sin))))
        return fail(OSSA_ERR_INVALID, "x, cos, sin and out must be 16-byte aligned");
    ossa::RopeArgs a{x, cos, sin, cs_batched ? 1 : 0, dtype, B, N, Hx, D, out};
    return cuda_status(ossa::launch_rope_heads(a, static_cast<cudaStream_t>(stream)), "rope launch");
}

size_t ossa_oracle_workspace_size(int B, int H, int Hkv, int N, int D, int K, int dtype) {
    if (B < 0 || H <= 0 || Hkv <= 0 || N < 0 || D <= 0 || K <= 0 || !valid_dtype(dtype)) return 0;
    return oracle_workspace_bytes(B, H, Hkv, N, D, K, dtype);
}

int ossa_oracle_topk_ws(const void* q, const void* k, int dtype, int B, int H, int Hkv, int N, int D,
                        float scale, int K, int causal, int32_t* idx_out, void* workspace,
                        size_t workspace_bytes, ossa_stream_t stream) {
    int st = check_heads(B, H, Hkv, N);
    if (st) return st;
    if (!valid_dtype(dtype)) return fail(OSSA_ERR_INVALID, "bad dtype %d", dtype);
    if (!supported_r(D))
        return fail(OSSA_ERR_UNSUPPORTED, "oracle selection supports head_dim in {16,32,64,128}, got %d", D);
    if (K <= 0) return fail(OSSA_ERR_INVALID, "bad K=%d", K);
    if (!ossa::score_topk_supported(D, K))
        return fail(OSSA_ERR_UNSUPPORTED, "top-K selection supports K <= 160 (got K=%d)", K);
    if (!isfinite(scale)) return fail(OSSA_ERR_INVALID, "scale must be finite");
    if ((long long)B * H * N == 0) return OSSA_OK;
    if (!q || !k || !idx_out) return fail(OSSA_ERR_INVALID, "null pointer argument");
    if (!aligned16(q) || !aligned16(k) || !aligned16(idx_out))
        return fail(OSSA_ERR_INVALID, "q, k and the output must be 16-byte aligned");
    const size_t need = oracle_workspace_bytes(B, H, Hkv, N, D, K, dtype);
    if (!workspace || workspace_bytes < need || !aligned16(workspace))
        return fail(OSSA_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) required, got %zu", need,
                    workspace ? workspace_bytes : (size_t)0);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    st = cuda_status(cudaMemsetAsync(workspace, 0, kCountersBytes, s), "workspace counters reset");
    if (st) return st;
    if (!use_tensor_core_oracle(B, H, Hkv, N, D, K)) {
        ossa::ScoreTopkArgs a{q, k, dtype, nullptr, 1, B, H, Hkv, N, D, K, scale, causal ? 1 : 0, idx_out};
        return cuda_status(ossa::launch_score_topk(a, s), "oracle top-K launch");
    }
    ossa::OracleTcArgs a{q, k, dtype, B, H, Hkv, N, K, causal ? 1 : 0, scale, idx_out,
                         static_cast<char*>(workspace) + kCountersBytes, reinterpret_cast<int*>(workspace)};
    return cuda_status(ossa::launch_oracle_tc(a, s), "tensor-core oracle top-K launch");
}

}  // extern "C"
