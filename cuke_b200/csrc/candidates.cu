// Losses over the score rows of candidate sets (all entities, all relations, the outgoing edges of a node):
//
//   log_prob     logp = (s_a - m) / T - log S,  m = max_j s_j,  S = sum_j exp((s_j - m) / T),  a the chosen candidate
//   its gradient ds_j = dlogp / T * (1[j = a] - exp((s_j - m) / T) / S)
//   policy loss  ratio = exp(logp - old),  l = -min(ratio A, clip(ratio, 1 - lo, 1 + hi) A) + beta (exp(ref - logp) - (ref - logp) - 1)
//                loss = scale sum_r w_r l_r, and the gradient above with dlogp = scale w dl/dlogp, in the same call
//
// The sum is kept as S = e_a + S', S' over the other candidates: 1 - p_a = S' / S and (where a is the maximum)
// logp = -log1p(S') then keep their digits when the chosen candidate has nearly all the mass.
// Row statistics are fp32; what is left per row (one logarithm, two exponentials) is done in 64 bits, because the ratio
// and the KL term subtract numbers that are nearly equal.
#include "common.cuh"

namespace kge {

struct CandArgs {
    const void* scores; void* dscores;
    long long rows, ld, ldd;
    int n, id64;
    const int* n_cand;               // optional (rows)
    const void* action;              // (rows) int32 / int64, -1: none
    float inv_temp;
    float* logp; float* stats;       // (rows), (rows, 3): m, S', 1 / S (0: a row that takes no part)
    const float* dlogp;              // gradient of log_prob
    const float* old_logp; const float* ref_logp; const float* adv; const float* weight;
    float clip_lo, clip_hi, kl_coef, scale;
    float* kl; double* partial;
    int32_t* err;
};

enum { CM_LOGP = 0, CM_POLICY = 1, CM_GRAD = 2 };

__device__ __forceinline__ float cand_get(const float* p) { return *p; }
__device__ __forceinline__ float cand_get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void cand_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void cand_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ float cand_ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

__device__ __forceinline__ int cand_count(const CandArgs& a, long long row) {
    return a.n_cand ? min(max(__ldg(a.n_cand + row), 0), a.n) : a.n;
}
// The chosen candidate of a row, or -1 where there is none; an id outside the row's candidates is reported and taken as -1.
__device__ __forceinline__ int cand_action(const CandArgs& a, long long row, int cnt, bool report) {
    const long long id = a.id64 ? __ldg(static_cast<const long long*>(a.action) + row) : (long long)__ldg(static_cast<const int*>(a.action) + row);
    if (id >= 0 && id < cnt) return static_cast<int>(id);
    if (id != -1 && report) atomicOr(a.err, KGE_ERR_ID_RANGE);
    return -1;
}

// Logarithm of the chosen candidate's probability from x = (s_a - m) / T and S' (S = e_a + S').
__device__ __forceinline__ double cand_logp(double x, float rest) {
    return x == 0.0 ? -log1p(static_cast<double>(rest)) : x - log(exp(x) + static_cast<double>(rest));
}

// Loss term of one row and, in *g, d(loss) / d(logp); logp and kl are stored by the caller's thread.
__device__ __forceinline__ double policy_term(const CandArgs& a, long long row, double logp, double* g) {
    const double w = a.weight ? a.weight[row] : 1.0;
    const double A = a.adv[row], ratio = exp(logp - static_cast<double>(a.old_logp[row]));
    const double lo = 1.0 - static_cast<double>(a.clip_lo), hi = 1.0 + static_cast<double>(a.clip_hi);
    const bool held = (A > 0.0 && ratio > hi) || (A < 0.0 && ratio < lo);
    double l = -(held ? (A > 0.0 ? hi : lo) : ratio) * A, dl = held ? 0.0 : -ratio * A, kl = 0.0;
    if (a.ref_logp) {
        const double d = static_cast<double>(a.ref_logp[row]) - logp, e = expm1(d);
        kl = e - d;
        l += a.kl_coef * kl;
        dl -= a.kl_coef * e;
    }
    a.logp[row] = static_cast<float>(logp);
    a.kl[row] = static_cast<float>(kl);
    if (w == 0.0) { *g = 0.0; return 0.0; }
    *g = w * a.scale * dl;
    return w * a.scale * l;
}

// One CTA per row: maximum, sum, gradient in three passes over the row.
template <typename T, int MODE>
__global__ void __launch_bounds__(256) cand_row_kernel(CandArgs a) {
    __shared__ float red[8];
    __shared__ float bc[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    double total = 0.0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* s = static_cast<const T*>(a.scores) + row * a.ld;
        const int cnt = cand_count(a, row);
        const int act = cand_action(a, row, cnt, tid == 0 && MODE != CM_GRAD);
        float m, rest;
        if (MODE == CM_GRAD) {
            m = a.stats[3 * row]; rest = a.stats[3 * row + 1];
        } else {
            m = -INFINITY;
            for (int j = tid; j < cnt; j += 256) m = fmaxf(m, cand_get(s + j));
#pragma unroll
            for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
            if (lane == 0) red[warp] = m;
            __syncthreads();
            m = red[0];
            for (int i = 1; i < 8; ++i) m = fmaxf(m, red[i]);
            __syncthreads();
            if (m == -INFINITY) m = 0.f;         // no candidate, or none with a finite score: the sum below says which
        }
        const float c = a.inv_temp * 1.4426950408889634f;
        if (MODE != CM_GRAD) {
            rest = 0.f;
            for (int j = tid; j < cnt; j += 256) if (j != act) rest += cand_ex2((cand_get(s + j) - m) * c);
            rest = warp_sum(rest);
            if (lane == 0) red[warp] = rest;
            __syncthreads();
            rest = 0.f;
            for (int i = 0; i < 8; ++i) rest += red[i];
        }
        if (tid == 0) {
            double g = 0.0;
            float inv = 0.f;
            if (MODE == CM_GRAD) {
                g = a.dlogp[row]; inv = act >= 0 ? a.stats[3 * row + 2] : 0.f;
            } else {
                const float sa = act >= 0 ? cand_get(s + act) : 0.f;
                const double x = act >= 0 ? static_cast<double>(sa - m) * static_cast<double>(a.inv_temp) : 0.0;
                const bool live = act >= 0 && !(sa == -INFINITY && rest == 0.f);
                const double lp = live ? cand_logp(x, rest) : 0.0;
                if (live) inv = static_cast<float>(1.0 / (exp(x) + rest));
                if (MODE == CM_POLICY) {
                    if (live) total += policy_term(a, row, lp, &g);
                    else { a.logp[row] = 0.f; a.kl[row] = 0.f; }
                } else {
                    a.logp[row] = static_cast<float>(lp);
                    a.stats[3 * row] = m; a.stats[3 * row + 1] = rest; a.stats[3 * row + 2] = inv;
                }
            }
            bc[0] = static_cast<float>(g * a.inv_temp); bc[1] = inv;
        }
        if (MODE != CM_LOGP) {
            __syncthreads();
            const float ga = bc[0] == 0.f ? 0.f : bc[0] * bc[1];      // (a row of weight 0 may hold NaN)
            T* d = static_cast<T*>(a.dscores) + row * a.ldd;
            for (int j = tid; j < a.n; j += 256) {
                float v = 0.f;
                if (j < cnt && ga != 0.f) v = j == act ? ga * rest : -ga * cand_ex2((cand_get(s + j) - m) * c);
                cand_put(d + j, v);
            }
        }
        __syncthreads();
    }
    if (MODE == CM_POLICY && tid == 0) a.partial[blockIdx.x] = total;
}

__global__ void __launch_bounds__(256) sum_partials_kernel(const double* partial, int n, float* out) {
    __shared__ double red[256];
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) v += partial[i];
    red[threadIdx.x] = v;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) *out = static_cast<float>(red[0]);
}

int launch_sum_partials(const double* partial, int n, float* out, cudaStream_t s) {
    sum_partials_kernel<<<1, 256, 0, s>>>(partial, n, out);
    KGE_LAUNCH_CHECK("sum_partials_kernel");
    return 0;
}

constexpr int kCandMaxBlocks = 148 * 8;

static int launch_candidates(const CandArgs& a, int dtype, int mode, cudaStream_t s) {
    if (a.rows == 0) return 0;
    const unsigned blocks = static_cast<unsigned>(a.rows < kCandMaxBlocks ? a.rows : kCandMaxBlocks);
#define KGE_CAND(M) do { if (dtype == KGE_F32) cand_row_kernel<float, M><<<blocks, 256, 0, s>>>(a); \
                         else cand_row_kernel<__nv_bfloat16, M><<<blocks, 256, 0, s>>>(a); } while (0)
    if (mode == CM_LOGP) KGE_CAND(CM_LOGP);
    else if (mode == CM_POLICY) KGE_CAND(CM_POLICY);
    else KGE_CAND(CM_GRAD);
#undef KGE_CAND
    KGE_LAUNCH_CHECK("cand_row_kernel");
    return 0;
}

}  // namespace kge

using namespace kge;

static int check_candidates(const char* fn, const void* scores, int32_t dtype, int64_t ld, int64_t rows, int64_t n, const int32_t* n_cand,
                            const void* action, int32_t id_bits, float temperature, CandArgs* a) {
    if (dtype != KGE_F32 && dtype != KGE_BF16) { set_error("%s: unknown dtype %d", fn, dtype); return KGE_E_UNSUPPORTED; }
    if (id_bits != 32 && id_bits != 64) { set_error("%s: id_bits must be 32 or 64, got %d", fn, id_bits); return KGE_E_UNSUPPORTED; }
    if (!(temperature > 0.f) || !(1.f / temperature > 0.f) || isinf(1.f / temperature)) { set_error("%s: temperature %g is not a positive number", fn, temperature); return KGE_E_RANGE; }
    if (rows < 0 || n < 0) { set_error("%s: negative size", fn); return KGE_E_SHAPE; }
    if (n > (1LL << 30) || rows > (1LL << 40)) { set_error("%s: more than 2^30 candidates or 2^40 rows", fn); return KGE_E_RANGE; }
    if (rows > 1 && ld < n) { set_error("%s: row pitch %lld is below n", fn, (long long)ld); return KGE_E_SHAPE; }
    if (ld > (1LL << 40)) { set_error("%s: row pitch above 2^40", fn); return KGE_E_RANGE; }
    if (rows == 0) return 0;
    if (!scores && n > 0) { set_error("%s: scores is NULL", fn); return KGE_E_NULL; }
    if (!action) { set_error("%s: action is NULL", fn); return KGE_E_NULL; }
    if ((reinterpret_cast<uintptr_t>(scores) & (dtype == KGE_F32 ? 3 : 1)) || (reinterpret_cast<uintptr_t>(action) & (id_bits / 8 - 1)) ||
        (reinterpret_cast<uintptr_t>(n_cand) & 3)) { set_error("%s: a pointer is not aligned to its element size", fn); return KGE_E_ALIGN; }
    a->scores = scores; a->ld = ld; a->rows = rows; a->n = static_cast<int>(n); a->n_cand = n_cand; a->action = action; a->id64 = id_bits == 64;
    a->inv_temp = 1.f / temperature;
    a->err = device_error_word();
    if (!a->err) { set_error("%s: no usable device", fn); return KGE_E_DEVICE; }
    return 0;
}
static int check_floats(const char* fn, const char* name, const float* p, bool required) {
    if (!p && required) { set_error("%s: %s is NULL", fn, name); return KGE_E_NULL; }
    if (reinterpret_cast<uintptr_t>(p) & 3) { set_error("%s: %s is not aligned to its element size", fn, name); return KGE_E_ALIGN; }
    return 0;
}
static int check_gradient(const char* fn, void* dscores, int32_t dtype, int64_t ldd, int64_t rows, int64_t n) {
    if (rows > 1 && ldd < n) { set_error("%s: row pitch %lld of dscores is below n", fn, (long long)ldd); return KGE_E_SHAPE; }
    if (ldd > (1LL << 40)) { set_error("%s: row pitch above 2^40", fn); return KGE_E_RANGE; }
    if (!dscores && n > 0) { set_error("%s: dscores is NULL", fn); return KGE_E_NULL; }
    if (reinterpret_cast<uintptr_t>(dscores) & (dtype == KGE_F32 ? 3 : 1)) { set_error("%s: dscores is not aligned to its element size", fn); return KGE_E_ALIGN; }
    return 0;
}

extern "C" {

size_t kge_candidates_workspace_bytes(int64_t rows, int64_t n) {
    (void)rows; (void)n;
    return kCandMaxBlocks * sizeof(double);
}

int kge_log_prob(const void* scores, int32_t dtype, int64_t ld, int64_t rows, int64_t n, const int32_t* n_cand, const void* action,
                 int32_t id_bits, float temperature, float* logp, float* stats, void* workspace, size_t workspace_bytes,
                 kge_stream_t stream) {
    const char* fn = "kge_log_prob";
    CandArgs a = {};
    int rc = check_candidates(fn, scores, dtype, ld, rows, n, n_cand, action, id_bits, temperature, &a);
    if (rc || rows == 0) return rc;
    if ((rc = check_floats(fn, "logp", logp, true)) || (rc = check_floats(fn, "stats", stats, true))) return rc;
    if (workspace_bytes < kge_candidates_workspace_bytes(rows, n)) { set_error("%s: workspace too small", fn); return KGE_E_WORKSPACE; }
    if (!workspace) { set_error("%s: workspace is NULL", fn); return KGE_E_NULL; }
    if (!aligned16(workspace)) { set_error("%s: workspace is not 16-byte aligned", fn); return KGE_E_ALIGN; }
    a.logp = logp; a.stats = stats;
    return launch_candidates(a, dtype, CM_LOGP, reinterpret_cast<cudaStream_t>(stream));
}

int kge_log_prob_backward(const void* scores, int32_t dtype, int64_t ld, int64_t rows, int64_t n, const int32_t* n_cand, const void* action,
                          int32_t id_bits, float temperature, const float* stats, const float* dlogp, void* dscores, int64_t ldd,
                          kge_stream_t stream) {
    const char* fn = "kge_log_prob_backward";
    CandArgs a = {};
    int rc = check_candidates(fn, scores, dtype, ld, rows, n, n_cand, action, id_bits, temperature, &a);
    if (rc || rows == 0) return rc;
    if ((rc = check_floats(fn, "stats", stats, true)) || (rc = check_floats(fn, "dlogp", dlogp, true)) ||
        (rc = check_gradient(fn, dscores, dtype, ldd, rows, n))) return rc;
    a.stats = const_cast<float*>(stats); a.dlogp = dlogp; a.dscores = dscores; a.ldd = ldd;
    return launch_candidates(a, dtype, CM_GRAD, reinterpret_cast<cudaStream_t>(stream));
}

int kge_policy_loss(const void* scores, int32_t dtype, int64_t ld, int64_t rows, int64_t n, const int32_t* n_cand, const void* action,
                    int32_t id_bits, float temperature, const float* old_logp, const float* ref_logp, const float* advantage,
                    const float* weight, float clip_low, float clip_high, float kl_coef, float scale, float* loss, float* logp,
                    float* kl, void* dscores, int64_t ldd, void* workspace, size_t workspace_bytes, kge_stream_t stream) {
    const char* fn = "kge_policy_loss";
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (!(clip_low >= 0.f && clip_low <= 1.f) || !(clip_high >= 0.f)) { set_error("%s: clip range [1 - %g, 1 + %g]", fn, clip_low, clip_high); return KGE_E_RANGE; }
    if (!(kl_coef >= 0.f) || isinf(kl_coef)) { set_error("%s: kl_coef %g", fn, kl_coef); return KGE_E_RANGE; }
    CandArgs a = {};
    int rc = check_candidates(fn, scores, dtype, ld, rows, n, n_cand, action, id_bits, temperature, &a);
    if (rc || (rc = check_floats(fn, "loss", loss, true))) return rc;
    if (rows == 0) return launch_sum_partials(nullptr, 0, loss, s);
    if ((rc = check_floats(fn, "old_logp", old_logp, true)) || (rc = check_floats(fn, "ref_logp", ref_logp, false)) ||
        (rc = check_floats(fn, "advantage", advantage, true)) || (rc = check_floats(fn, "weight", weight, false)) ||
        (rc = check_floats(fn, "logp", logp, true)) || (rc = check_floats(fn, "kl", kl, true)) ||
        (rc = check_gradient(fn, dscores, dtype, ldd, rows, n))) return rc;
    if (workspace_bytes < kge_candidates_workspace_bytes(rows, n)) { set_error("%s: workspace too small", fn); return KGE_E_WORKSPACE; }
    if (!workspace) { set_error("%s: workspace is NULL", fn); return KGE_E_NULL; }
    if (!aligned16(workspace)) { set_error("%s: workspace is not 16-byte aligned", fn); return KGE_E_ALIGN; }
    a.logp = logp; a.kl = kl; a.dscores = dscores; a.ldd = ldd;
    a.old_logp = old_logp; a.ref_logp = ref_logp; a.adv = advantage; a.weight = weight;
    a.clip_lo = clip_low; a.clip_hi = clip_high; a.kl_coef = kl_coef; a.scale = scale;
    a.partial = static_cast<double*>(workspace);
    if ((rc = launch_candidates(a, dtype, CM_POLICY, s))) return rc;
    return launch_sum_partials(a.partial, static_cast<int>(rows < kCandMaxBlocks ? rows : kCandMaxBlocks), loss, s);
}

}  // extern "C"
