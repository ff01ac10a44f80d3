// Preference loss over score differences: every positive against its negatives, relative to a frozen reference scorer.
//
//   z = beta ((pos - ref_pos) - (neg_j - ref_neg_j)) - margin
//   logistic  l = (1 - e) softplus(-z) + e softplus(z),   l' = e sigmoid(z) - (1 - e) sigmoid(-z)
//   square    l = z^2,                                    l' = 2 z
//   loss = scale sum_b w_b / c_b sum_{j valid} l,  dpos_b = scale beta w_b / c_b sum_j l',  dneg_bj = -scale beta w_b / c_b l'
//
// c_b is the number of valid negatives of row b; a row without any contributes nothing and gets zero gradients.
// fp32 per pair (both sigmoids from one exponential of -|z|, so neither side loses its small values), a row's sum in
// fp32, the sum over rows in fp64 and in a fixed order.
#include "common.cuh"

namespace kge {

int launch_sum_partials(const double* partial, int n, float* out, cudaStream_t s);

struct PrefArgs {
    const float* pos; const float* rpos; const float* neg; const float* rneg;
    const unsigned char* mask; const float* weight;
    float* dpos; float* dneg; double* partial;
    long long rows, ldn, ldr, ldm, ldd;
    int n, kind;
    float beta, margin, smooth, scale;
};
enum { PREF_LOGISTIC = 0, PREF_SQUARE = 1 };

__device__ __forceinline__ void pref_pair(const PrefArgs& a, float z, float& l, float& d) {
    if (a.kind == PREF_SQUARE) { l = z * z; d = 2.f * z; return; }
    const float t = __expf(-fabsf(z)), inv = __frcp_rn(1.f + t);
    const float up = z >= 0.f ? inv : t * inv, down = z >= 0.f ? t * inv : inv;      // sigmoid(z), sigmoid(-z)
    const float keep = 1.f - a.smooth;
    l = log1pf(t) + keep * fmaxf(-z, 0.f);
    d = -keep * down;
    if (a.smooth > 0.f) { l += a.smooth * fmaxf(z, 0.f); d += a.smooth * up; }        // (0 x inf without the test)
}

// One warp per row.
__global__ void __launch_bounds__(256) pref_kernel(PrefArgs a) {
    __shared__ double red[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double total = 0.0;
    for (long long row = (long long)blockIdx.x * 8 + warp; row < a.rows; row += (long long)gridDim.x * 8) {
        const float* neg = a.neg + row * a.ldn;
        const float* rneg = a.rneg ? a.rneg + row * a.ldr : nullptr;
        const unsigned char* mask = a.mask ? a.mask + row * a.ldm : nullptr;
        int cnt = a.n;
        if (mask) {
            cnt = 0;
            for (int j = lane; j < a.n; j += 32) cnt += mask[j] != 0;
            cnt = __reduce_add_sync(kFull, cnt);
        }
        const float base = a.pos[row] - (a.rpos ? a.rpos[row] : 0.f);
        const float w = a.weight ? a.weight[row] : 1.f;
        const float cw = cnt > 0 ? a.scale * w / static_cast<float>(cnt) : 0.f;
        float ls = 0.f, ds = 0.f;
        for (int j = lane; j < a.n; j += 32) {
            float l = 0.f, d = 0.f;
            if (!mask || mask[j]) {
                const float h = base - (neg[j] - (rneg ? rneg[j] : 0.f));
                pref_pair(a, a.beta * h - a.margin, l, d);
                d *= a.beta;
                ls += l; ds += d;
            }
            a.dneg[row * a.ldd + j] = cw != 0.f ? -cw * d : 0.f;
        }
        ls = warp_sum(ls); ds = warp_sum(ds);
        if (lane == 0) {
            a.dpos[row] = cw != 0.f ? cw * ds : 0.f;
            if (cw != 0.f) total += static_cast<double>(cw) * ls;
        }
    }
    if (lane == 0) red[warp] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) total += red[i];
        a.partial[blockIdx.x] = total;
    }
}

constexpr int kPrefMaxBlocks = 148 * 8;

static int launch_preference(const PrefArgs& a, float* loss, cudaStream_t s) {
    const long long want = (a.rows + 7) / 8;
    const unsigned blocks = static_cast<unsigned>(want < kPrefMaxBlocks ? want : kPrefMaxBlocks);
    pref_kernel<<<blocks, 256, 0, s>>>(a);
    KGE_LAUNCH_CHECK("pref_kernel");
    return launch_sum_partials(a.partial, static_cast<int>(blocks), loss, s);
}

}  // namespace kge

using namespace kge;

extern "C" {

size_t kge_preference_workspace_bytes(int64_t rows, int64_t n) {
    (void)rows; (void)n;
    return kPrefMaxBlocks * sizeof(double);
}

int kge_preference_loss(const float* pos, const float* ref_pos, const float* neg, int64_t ld_neg, const float* ref_neg, int64_t ld_ref,
                        const uint8_t* mask, int64_t ld_mask, const float* weight, int64_t rows, int64_t n, int32_t kind, float beta,
                        float margin, float smoothing, float scale, float* loss, float* dpos, float* dneg, int64_t ld_dneg,
                        void* workspace, size_t workspace_bytes, kge_stream_t stream) {
    const char* fn = "kge_preference_loss";
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (kind != PREF_LOGISTIC && kind != PREF_SQUARE) { set_error("%s: unknown kind %d", fn, kind); return KGE_E_UNSUPPORTED; }
    if (!(smoothing >= 0.f && smoothing <= 1.f)) { set_error("%s: smoothing %g outside [0, 1]", fn, smoothing); return KGE_E_RANGE; }
    if (kind == PREF_SQUARE && smoothing != 0.f) { set_error("%s: the square loss has no label smoothing", fn); return KGE_E_UNSUPPORTED; }
    if (rows < 0 || n < 0) { set_error("%s: negative size", fn); return KGE_E_SHAPE; }
    if (n > (1LL << 30) || rows > (1LL << 40) || ld_neg > (1LL << 40) || ld_ref > (1LL << 40) || ld_mask > (1LL << 40) || ld_dneg > (1LL << 40)) {
        set_error("%s: more than 2^30 negatives a row, 2^40 rows or a pitch above 2^40", fn); return KGE_E_RANGE; }
    if (rows > 1 && (ld_neg < n || ld_dneg < n || (ref_neg && ld_ref < n) || (mask && ld_mask < n))) { set_error("%s: a row pitch is below n", fn); return KGE_E_SHAPE; }
    if (!loss) { set_error("%s: loss is NULL", fn); return KGE_E_NULL; }
    if (rows > 0 && (!pos || !dpos || (n > 0 && (!neg || !dneg)))) { set_error("%s: pos / neg / dpos / dneg is NULL", fn); return KGE_E_NULL; }
    if (rows > 0 && n > 0 && (ref_pos == nullptr) != (ref_neg == nullptr)) { set_error("%s: ref_pos and ref_neg come together", fn); return KGE_E_NULL; }
    const void* ptrs[] = {pos, ref_pos, neg, ref_neg, weight, loss, dpos, dneg};
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) & 3) { set_error("%s: a pointer is not aligned to its element size", fn); return KGE_E_ALIGN; }
    if (rows == 0) return launch_sum_partials(nullptr, 0, loss, s);
    if (workspace_bytes < kge_preference_workspace_bytes(rows, n)) { set_error("%s: workspace too small", fn); return KGE_E_WORKSPACE; }
    if (!workspace) { set_error("%s: workspace is NULL", fn); return KGE_E_NULL; }
    if (!aligned16(workspace)) { set_error("%s: workspace is not 16-byte aligned", fn); return KGE_E_ALIGN; }
    PrefArgs a = {pos, ref_pos, neg, ref_neg, mask, weight, dpos, dneg, static_cast<double*>(workspace), rows, ld_neg, ld_ref, ld_mask, ld_dneg,
                  static_cast<int>(n), kind, beta, margin, smoothing, scale};
    return launch_preference(a, loss, s);
}

}  // extern "C"
