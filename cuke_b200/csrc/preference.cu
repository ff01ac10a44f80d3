// Preference loss over score differences: every positive against its negatives, relative to a frozen reference scorer.
//
//   z = beta ((pos - ref_pos) - (neg_j - ref_neg_j)) - margin
//   logistic  l = (1 - e) softplus(-z) + e softplus(z),   l' = e sigmoid(z) - (1 - e) sigmoid(-z)
//   square    l = z^2,                                    l' = 2 z
//   loss = scale sum_b w_b / c_b sum_{j valid} l,  dpos_b = scale beta w_b / c_b sum_j l',  dneg_bj = -scale beta w_b / c_b l'
//
// c_b is the number of valid negatives of row b; a row without any contributes nothing and gets zero gradients.
// fp32 per pair (both sigmoids from one exponential of -|z|, so neither side loses its small values).  Sums are taken in a fixed
// order: a row's in fp32 with at most 64 additions behind one another in a thread, longer ones continued in fp64; the sum over
// rows in fp64.
#include "common.cuh"

namespace kge {

int launch_sum_partials(const double* partial, int n, float* out, cudaStream_t s);

struct PrefArgs {
    const float* pos; const float* rpos; const float* neg; const float* rneg;
    const unsigned char* mask; const float* weight;
    float* dpos; float* dneg; float* loss; double* partial;     // loss: written by the only CTA of a launch, else summed from partial
    long long rows, ldn, ldr, ldm, ldd;
    int n, kind;
    float beta, margin, smooth, scale;
};
enum { PREF_LOGISTIC = 0, PREF_SQUARE = 1 };

__device__ __forceinline__ float pref_ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float pref_rcp(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

// Loss and slope of one pair.  With t = exp(-|z|): sigmoid(|z|) = 1 / (1 + t), sigmoid(-|z|) = t / (1 + t), and
// softplus(-|z|) = log1p(t) = 2 atanh(w), w = t / (2 + t) in [0, 1/3]: atanh(w) / w as a polynomial in w^2 (Chebyshev
// interpolation of degree 4 on [0, 1/9], 4e-9 relative), so small terms keep their digits at the cost of one reciprocal and six
// fused multiply-adds: the loss is bound by memory only if a pair stays below some 40 instructions.
// Two pairs at a time: additions, products and the polynomial run on packed fp32 pairs.
__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }
template <bool SQUARE>
__device__ __forceinline__ void pref_pairs(const PrefArgs& a, float keep, float2 z, float2& l, float2& d) {
    if (SQUARE) { l = __fmul2_rn(z, z); d = __fadd2_rn(z, z); return; }
    const float2 t = make_float2(pref_ex2(fabsf(z.x) * -1.4426950408889634f), pref_ex2(fabsf(z.y) * -1.4426950408889634f));
    const float2 t1 = __fadd2_rn(t, f2(1.f)), t2 = __fadd2_rn(t, f2(2.f));
    const float2 inv = make_float2(pref_rcp(t1.x), pref_rcp(t1.y));                        // sigmoid(|z|)
    const float2 w = __fmul2_rn(t, make_float2(pref_rcp(t2.x), pref_rcp(t2.y))), x = __fmul2_rn(w, w);
    float2 q = __ffma2_rn(f2(2.f * 0.14078890f), x, f2(2.f * 0.13982579f));
    q = __ffma2_rn(q, x, f2(2.f * 0.20012298f));
    q = __ffma2_rn(q, x, f2(2.f * 0.33333161f));
    q = __ffma2_rn(q, x, f2(2.f));
    const float2 small = __fmul2_rn(t, inv);                                               // sigmoid(-|z|)
    const bool ux = z.x >= 0.f, uy = z.y >= 0.f;
    const float2 hi = make_float2(ux ? a.smooth : -keep, uy ? a.smooth : -keep), lo = make_float2(ux ? -keep : a.smooth, uy ? -keep : a.smooth);
    d = __ffma2_rn(hi, inv, __fmul2_rn(lo, small));
    l = __ffma2_rn(f2(keep), make_float2(fmaxf(-z.x, 0.f), fmaxf(-z.y, 0.f)), __fmul2_rn(w, q));
    if (a.smooth > 0.f)                                                                    // (0 x inf without the test)
        l = __ffma2_rn(f2(a.smooth), make_float2(fmaxf(z.x, 0.f), fmaxf(z.y, 0.f)), l);
}

// bytes of w that are not zero: the low seven bits carry into the eighth, or it is set already
__device__ __forceinline__ int nonzero_bytes(uint32_t w) { return __popc((((w & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | w) & 0x80808080u); }

template <int G>
__device__ __forceinline__ float pref_group_sum(float v) {
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}
template <int G>
__device__ __forceinline__ int pref_group_sum(int v) {
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

// Turns of a long row after which a thread's fp32 sums, of four terms a turn, go to its 64-bit ones and start again.
constexpr int kPrefFold = 16;
__device__ __forceinline__ void pref_fold(double2& wide, bool more, float2& ls, float2& ds) {
    const double l = static_cast<double>(ls.x) + static_cast<double>(ls.y), d = static_cast<double>(ds.x) + static_cast<double>(ds.y);
    wide = more ? make_double2(wide.x + l, wide.y + d) : make_double2(l, d);
    ls = ds = f2(0.f);
}

// A group of G threads per row: one thread for a handful of negatives, part of a warp, a warp, or a whole CTA.  VEC: four
// negatives per access (all rows of neg, ref_neg, dneg on 16-byte and of mask on 4-byte boundaries).  The valid negatives of
// a row are counted first - the mask is a thirteenth of the traffic and comes from L1 the second time - so that the main pass
// writes final gradients; it requests U accesses of each array before it uses the first.  Without VEC a thread has the same four
// negatives, read one by one: the order of the additions, and so every bit of the result, does not depend on alignment.
template <int G, bool VEC, bool SQUARE, bool MASK, bool LONG>
__global__ void __launch_bounds__(G > 32 ? G : 256) pref_kernel(PrefArgs a) {
    constexpr int BLOCK = G > 32 ? G : 256;
    constexpr int W = 4;                           // consecutive negatives of a thread
    constexpr int U = G == 1 ? 1 : 2;
    constexpr int FOLD = G * W * U * kPrefFold;    // LONG: negatives after which the threads' sums go to 64 bits
    __shared__ double red[32];
    __shared__ float rl[32], rd[32];
    __shared__ int rc[32];
    __shared__ double2 wide[LONG ? G : 1];         // a thread's own
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int gl = threadIdx.x % G;
    let_next_start();
    double total = 0.0;
    const long long step = (long long)gridDim.x * (BLOCK / G);
    // every lane of a warp makes the same number of turns: the shuffles below need all of them
    const long long first = (long long)blockIdx.x * (BLOCK / G) + (G > 32 ? 0 : warp * (32 / G));
    for (long long base_row = first; base_row < a.rows; base_row += step) {
        const long long row = base_row + (G < 32 ? lane / G : 0);
        const bool live = row < a.rows;
        const long long rr = live ? row : a.rows - 1;
        const int n = live ? a.n : 0;
        const float* neg = a.neg + rr * a.ldn;
        const float* rneg = a.rneg ? a.rneg + rr * a.ldr : nullptr;
        const unsigned char* mask = MASK ? a.mask + rr * a.ldm : nullptr;
        float* dneg = a.dneg + rr * a.ldd;
        int cnt = n;
        if (MASK) {
            cnt = 0;
            for (int j = gl * W; j < n; j += G * W) {
                if (VEC) {
                    cnt += nonzero_bytes(*reinterpret_cast<const uint32_t*>(mask + j));
                } else {
#pragma unroll
                    for (int k = 0; k < W; ++k) cnt += j + k < n && mask[j + k] != 0;
                }
            }
            cnt = pref_group_sum<G>(cnt);
            if (G > 32) {
                if (lane == 0) rc[warp] = cnt;
                __syncthreads();
                cnt = 0;
                for (int w = 0; w < G / 32; ++w) cnt += rc[w];
            }
        }
        const float base = a.pos[rr] - (a.rpos ? a.rpos[rr] : 0.f);
        const float weight = a.weight ? a.weight[rr] : 1.f;
        const float cw = cnt > 0 ? a.scale * weight / static_cast<float>(cnt) : 0.f;
        const float dscale = -cw * a.beta, keep = 1.f - a.smooth;
        const bool off = cw == 0.f;                    // nothing valid, or weight 0: zeros, whatever the scores hold
        float2 ls = f2(0.f), ds = f2(0.f);
        for (int s0 = 0; s0 < n; s0 += LONG ? FOLD : n) {
            const int s1 = LONG ? s0 + min(n - s0, FOLD) : n;
            if (LONG && s0 > 0) pref_fold(wide[threadIdx.x], s0 > FOLD, ls, ds);
            for (int j0 = s0 + gl * W; j0 < s1; j0 += G * W * U) {
                float x[U][W], y[U][W];
                uint32_t m[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int j = j0 + u * G * W;
                    m[u] = 0;
                    if (j < n) {
                        if (VEC) {
                            const float4 f = __ldcs(reinterpret_cast<const float4*>(neg + j));
                            float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (rneg) g = __ldcs(reinterpret_cast<const float4*>(rneg + j));
                            if (MASK) m[u] = *reinterpret_cast<const uint32_t*>(mask + j);
                            x[u][0] = f.x; x[u][1] = f.y; x[u][2] = f.z; x[u][3] = f.w;
                            y[u][0] = g.x; y[u][1] = g.y; y[u][2] = g.z; y[u][3] = g.w;
                        } else {
#pragma unroll
                            for (int k = 0; k < W; ++k) {
                                x[u][k] = y[u][k] = 0.f;
                                if (j + k < n) {
                                    x[u][k] = neg[j + k];
                                    if (rneg) y[u][k] = rneg[j + k];
                                    if (!MASK || mask[j + k]) m[u] |= 0xFFu << (8 * k);
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int j = j0 + u * G * W;
                    if (j < n) {
                        float o[W];
#pragma unroll
                        for (int k = 0; k < W; k += 2) {
                            float2 l, d;
                            const float2 gap = __ffma2_rn(make_float2(x[u][k], x[u][k + 1]), f2(-1.f), make_float2(y[u][k], y[u][k + 1]));
                            pref_pairs<SQUARE>(a, keep, __ffma2_rn(f2(a.beta), __fadd2_rn(f2(base), gap), f2(-a.margin)), l, d);
                            if (MASK || !VEC) {
                                if (!(m[u] & (0xFFu << (8 * k)))) { l.x = 0.f; d.x = 0.f; }
                                if (!(m[u] & (0xFFu << (8 * k + 8)))) { l.y = 0.f; d.y = 0.f; }
                            }
                            ls = __fadd2_rn(ls, l);
                            ds = __fadd2_rn(ds, d);
                            const float2 g = __fmul2_rn(f2(dscale), d);
                            o[k] = g.x; o[k + 1] = g.y;
                        }
                        if (off) o[0] = o[1] = o[2] = o[3] = 0.f;
                        if (VEC) {
                            __stcs(reinterpret_cast<float4*>(dneg + j), make_float4(o[0], o[1], o[2], o[3]));
                        } else {
#pragma unroll
                            for (int k = 0; k < W; ++k) if (j + k < n) dneg[j + k] = o[k];
                        }
                    }
                }
            }
        }
        if (LONG) {
            pref_fold(wide[threadIdx.x], n > FOLD, ls, ds);
            ls.x = static_cast<float>(wide[threadIdx.x].x);
            ds.x = static_cast<float>(wide[threadIdx.x].y);
        }
        float lsum = pref_group_sum<G>(ls.x + ls.y), dsum = pref_group_sum<G>(ds.x + ds.y);
        if (G > 32) {
            if (lane == 0) { rl[warp] = lsum; rd[warp] = dsum; }
            __syncthreads();
            if (threadIdx.x == 0)
                for (int w = 1; w < G / 32; ++w) { lsum += rl[w]; dsum += rd[w]; }
        }
        if (gl == 0 && live) {
            a.dpos[row] = cw != 0.f ? -dscale * dsum : 0.f;
            if (cw != 0.f) total += static_cast<double>(cw) * lsum;
        }
        if (G > 32) __syncthreads();               // rc, rl, rd are free for the next row
    }
    if (G > 32) {
        if (threadIdx.x == 0) {
            if (gridDim.x == 1) *a.loss = static_cast<float>(total);
            else a.partial[blockIdx.x] = total;
        }
    } else {
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(kFull, total, o);
        if (lane == 0) red[warp] = total;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < 8; ++w) total += red[w];
            if (gridDim.x == 1) *a.loss = static_cast<float>(total);
            else a.partial[blockIdx.x] = total;
        }
    }
}

// One turn per group as far as the grid allows: CTAs that end leave room for the next one's loads (a loop of eight resident CTAs
// per SM copies at 5.7 TB/s, short CTAs at 6.6).  The cap bounds the partial sums.
constexpr int kPrefMaxBlocks = 1 << 16;
static long long pref_blocks(long long rows, int per) {
    const long long want = (rows + per - 1) / per;
    return want < kPrefMaxBlocks ? want : kPrefMaxBlocks;
}

template <int G, bool VEC, bool SQUARE, bool MASK, bool LONG>
static int pref_go2(const PrefArgs& a, float* loss, cudaStream_t s) {
    constexpr int per = G > 32 ? 1 : 256 / G;
    const unsigned blocks = static_cast<unsigned>(pref_blocks(a.rows, per));
    pref_kernel<G, VEC, SQUARE, MASK, LONG><<<blocks, G > 32 ? G : 256, 0, s>>>(a);
    KGE_LAUNCH_CHECK("pref_kernel");
    // one CTA has written the loss itself (200 x 3: 2.7 us, with a sum 3.7 us; one CTA of 1024 threads for more rows is slower: 500 x 20
    // 5.7 us against 4.2 us)
    return blocks > 1 ? launch_sum_partials(a.partial, static_cast<int>(blocks), loss, s) : 0;
}
template <int G, bool VEC, bool SQUARE>
static int pref_go(const PrefArgs& a, float* loss, cudaStream_t s) {
    // More than kPrefFold turns of eight negatives a thread (fewer than 256 threads never have such rows).  16 x 4000000 with reference
    // 661 us, with mask too 904 us; without the folds 733 and 839 us, but 40,000,001 equal pairs were then off by 7e-5 of their loss;
    // rows of fewer turns, with the folds all the same: up to 7 % slower.
    if (G >= 256 && a.n > G * 8 * kPrefFold) {
        constexpr bool LONG = G >= 256;
        return a.mask ? pref_go2<G, VEC, SQUARE, true, LONG>(a, loss, s) : pref_go2<G, VEC, SQUARE, false, LONG>(a, loss, s);
    }
    return a.mask ? pref_go2<G, VEC, SQUARE, true, false>(a, loss, s) : pref_go2<G, VEC, SQUARE, false, false>(a, loss, s);
}
// Threads per row: the fewest that still fill the GPU, so that a thread has some eight negatives at once and few share a row's own
// scalars and reductions.  us with reference and mask:
//   400000 x 8      2 threads 16.2   4 threads 27.8   8 threads 51.4          100000 x 48   4 threads 15.0   8 threads 20.6
//   60000 x 132     8 threads 24.2   32 threads 47.0        but 2000 x 100    8 threads 5.7    32 threads 4.2
//   40000 x 512    32 threads 51.1    8 threads 54.8        but 25915 x 412   8 threads 28.0   32 threads 35.4
//   1336 x 3356   128 threads 11.9   32 threads 19.0   1024 threads 29.3      500 x 512   128 threads 4.7   32 threads 5.7
//   5000 x 10000  256 threads 111   128 threads 115    32 threads 156         100 x 3000   256 threads 5.2   128 threads 6.3
//   140 x 60000  1024 threads 20.8   256 threads 40    but 300 x 20000  1024 threads 21.7   256 threads 19.1
template <bool VEC, bool SQUARE>
static int pref_pick(const PrefArgs& a, float* loss, cudaStream_t s) {
    if (a.n <= 4) return pref_go<1, false, SQUARE>(a, loss, s);
    if (a.n <= 24) return pref_go<2, VEC, SQUARE>(a, loss, s);
    if (a.n <= 64) return pref_go<4, VEC, SQUARE>(a, loss, s);
    if (a.n <= 448 && a.rows >= 148 * 32) return pref_go<8, VEC, SQUARE>(a, loss, s);
    if (a.n <= 2048 && a.rows >= 148 * 8) return pref_go<32, VEC, SQUARE>(a, loss, s);
    if ((a.n > 4096 && a.rows <= 148) || (a.n > 32768 && a.rows <= 148 * 2)) return pref_go<1024, VEC, SQUARE>(a, loss, s);
    if (a.n <= 512 || (a.n <= 8192 && a.rows >= 148 * 5)) return pref_go<128, VEC, SQUARE>(a, loss, s);
    return pref_go<256, VEC, SQUARE>(a, loss, s);
}

static int launch_preference(const PrefArgs& a, float* loss, cudaStream_t s) {
    const bool vec = a.n % 4 == 0 && aligned16(a.neg) && aligned16(a.dneg) && aligned16(a.rneg) && (reinterpret_cast<uintptr_t>(a.mask) & 3) == 0 &&
                     (a.rows == 1 || ((a.ldn | a.ldd | (a.rneg ? a.ldr : 0) | (a.mask ? a.ldm : 0)) & 3) == 0);
    if (a.kind == PREF_SQUARE) return vec ? pref_pick<true, true>(a, loss, s) : pref_pick<false, true>(a, loss, s);
    return vec ? pref_pick<true, false>(a, loss, s) : pref_pick<false, false>(a, loss, s);
}

}  // namespace kge

using namespace kge;

extern "C" {

size_t kge_preference_workspace_bytes(int64_t rows, int64_t n) {
    (void)n;                                       // at most one partial sum per row (a CTA a row)
    return rows > 0 ? sizeof(double) * static_cast<size_t>(pref_blocks(rows, 1)) : 0;
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
    if (rows > 1 && n > 0 && dneg == neg && ld_dneg != ld_neg) { set_error("%s: dneg may be neg only with the same row pitch", fn); return KGE_E_SHAPE; }
    const void* ptrs[] = {pos, ref_pos, neg, ref_neg, weight, loss, dpos, dneg};
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) & 3) { set_error("%s: a pointer is not aligned to its element size", fn); return KGE_E_ALIGN; }
    if (rows == 0) return launch_sum_partials(nullptr, 0, loss, s);
    if (workspace_bytes < kge_preference_workspace_bytes(rows, n)) { set_error("%s: workspace too small", fn); return KGE_E_WORKSPACE; }
    if (!workspace) { set_error("%s: workspace is NULL", fn); return KGE_E_NULL; }
    if (!aligned16(workspace)) { set_error("%s: workspace is not 16-byte aligned", fn); return KGE_E_ALIGN; }
    PrefArgs a = {pos, ref_pos, neg, ref_neg, mask, weight, dpos, dneg, loss, static_cast<double*>(workspace), rows, ld_neg, ld_ref, ld_mask, ld_dneg,
                  static_cast<int>(n), kind, beta, margin, smoothing, scale};
    if (kind == PREF_LOGISTIC && smoothing == 1.f) {
        // softplus(z) alone, as softplus(-z') of z' = -z: the kernel's factor (1 - smoothing) of max(-z, 0) is never 0, which it could only
        // skip at a cost (a test for it: 65536 x 1024 with reference 156 us instead of 127)
        a.beta = -beta; a.margin = -margin; a.smooth = 0.f;
    }
    return launch_preference(a, loss, s);
}

}  // extern "C"
