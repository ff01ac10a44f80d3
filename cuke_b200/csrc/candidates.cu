// Losses over the score rows of candidate sets (all entities, all relations, the outgoing edges of a node):
//
//   log_prob     logp = (s_a - m) / T - log S,  m = max_j s_j,  S = sum_j exp((s_j - m) / T),  a the chosen candidate
//   its gradient ds_j = dlogp / T * (1[j = a] - exp((s_j - m) / T) / S)
//   policy loss  ratio = exp(logp - old),  l = -min(ratio A, clip(ratio, 1 - lo, 1 + hi) A) + beta (exp(ref - logp) - (ref - logp) - 1)
//                loss = scale sum_r w_r l_r, and the gradient above with dlogp = scale w dl/dlogp, in the same call
//
// The sum is kept as S = e_a + S', S' over the other candidates: 1 - p_a = S' / S and (where a is the maximum)
// logp = -log1p(S') then keep their digits when the chosen candidate has nearly all the mass.
// Row statistics are fp32, the loss is summed over rows in 64 bits.
#include <math.h>
#include "umma.cuh"

namespace kge {

struct CandArgs {
    const void* scores; void* dscores;
    long long rows, ld, ldd;
    int n, id64;
    const int* n_cand;               // optional (rows)
    const void* action;              // (rows) int32 / int64, -1: none
    double inv_temp;
    float c_hi, c_lo;                // log2(e) / T as a sum of two floats: one alone, off by 2^-25, would tilt every sum the same way
    float* logp; float* stats;       // (rows), (rows, 3): m, S', 1 / S (0: a row that takes no part)
    const float* dlogp;              // gradient of log_prob
    const float* old_logp; const float* ref_logp; const float* adv; const float* weight;
    float clip_lo, clip_hi, kl_coef, scale;
    float* kl; float* loss; double* partial;     // loss: written by the only CTA of a launch, else summed from partial
    int32_t* err;
};

enum { CM_LOGP = 0, CM_POLICY = 1 };

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

// The scalars of a row.  Differences of logarithms are subtracted in 64 bits; the functions themselves are fp32, because
// 64-bit ones are a chain of some thousand cycles that a whole row waits for.  log S is one fp32 logarithm y plus the residual
// S exp(-y) - 1 (exact product inside the fma, so what remains is the error of one expf: ~6e-8 absolute whatever log S is).
__device__ __forceinline__ double cand_log_sum(double S) {
    const float s = static_cast<float>(S), y = logf(s);
    const float r = fmaf(s, expf(-y), -1.f) + static_cast<float>(S - static_cast<double>(s)) / s;
    return static_cast<double>(y) + static_cast<double>(r);
}
// e^d - 1 - d: its power series near 0, where the three terms cancel (next term below 2^-24 of the sum for |d| <= 1); e^d - 1 in
// *em1: farther out it cannot be had back as the difference of the two (d = -1e8 has a step of 8)
__device__ __forceinline__ float exp_minus_line(float d, float* em1) {
    if (fabsf(d) > 1.f) {
        *em1 = expm1f(d);
        return d == INFINITY ? d : *em1 - d;             // (a chosen candidate of probability 0)
    }
    float t = 1.f / 479001600.f;
    t = fmaf(t, d, 1.f / 39916800.f); t = fmaf(t, d, 1.f / 3628800.f); t = fmaf(t, d, 1.f / 362880.f); t = fmaf(t, d, 1.f / 40320.f);
    t = fmaf(t, d, 1.f / 5040.f); t = fmaf(t, d, 1.f / 720.f); t = fmaf(t, d, 1.f / 120.f); t = fmaf(t, d, 1.f / 24.f);
    t = fmaf(t, d, 1.f / 6.f); t = fmaf(t, d, 0.5f);
    const float kl = d * d * t;
    *em1 = kl + d;
    return kl;
}

// What follows from a row's statistics: logp, kl, loss term (returned), and the factor ga of the gradient,
// ds_j = ga (rest [j = a] - e_j [j != a]) with e_j = exp((s_j - m) / T).  One thread of a row calls it.
struct RowSide { float w, adv, old, ref; };            // a row's operands of the policy loss
__device__ __forceinline__ float cand_side(const CandArgs& a, long long row, int which) {
    const float* p = which == 0 ? a.weight : which == 1 ? a.adv : which == 2 ? a.old_logp : a.ref_logp;
    return p ? __ldg(p + row) : which == 0 ? 1.f : 0.f;
}
template <int MODE>
__device__ __forceinline__ double cand_finish(const CandArgs& a, long long row, int act, float sa, float m, float rest, bool write,
                                              const RowSide& o, float* ga) {
    const double x = act >= 0 ? (static_cast<double>(sa) - static_cast<double>(m)) * a.inv_temp : 0.0;
    const bool live = act >= 0 && !(sa == -INFINITY && rest == 0.f);
    const double S = static_cast<double>(expf(static_cast<float>(x))) + static_cast<double>(rest);
    const double lp = !live ? 0.0 : x == 0.0 && rest < 0.5f ? -static_cast<double>(log1pf(rest)) : x - cand_log_sum(S);
    const float inv = live ? 1.f / static_cast<float>(S) : 0.f;
    *ga = 0.f;
    if (write) a.logp[row] = static_cast<float>(lp);
    if (MODE == CM_LOGP) {
        if (write) { a.stats[3 * row] = m; a.stats[3 * row + 1] = rest; a.stats[3 * row + 2] = inv; }
        return 0.0;
    }
    if (!live) {
        if (write) a.kl[row] = 0.f;
        return 0.0;
    }
    const float w = o.w * a.scale, A = o.adv;
    const float ratio = expf(static_cast<float>(lp - static_cast<double>(o.old)));
    const float lo = 1.f - a.clip_lo, hi = 1.f + a.clip_hi;
    const bool held = (A > 0.f && ratio > hi) || (A < 0.f && ratio < lo);
    const float gain = A == 0.f && ratio == INFINITY ? 0.f : ratio * A;      // (exp(89) is past fp32; 0 times it is 0)
    float l = held ? -(A > 0.f ? hi : lo) * A : -gain, dl = held ? 0.f : -gain, kl = 0.f;
    if (a.ref_logp) {
        const float d = static_cast<float>(static_cast<double>(o.ref) - lp);
        float em1;
        kl = exp_minus_line(d, &em1);
        if (a.kl_coef > 0.f) {                           // (0 x infinity without the test: kl is only reported then)
            l = fmaf(a.kl_coef, kl, l);
            dl = fmaf(-a.kl_coef, em1, dl);
        }
    }
    if (write) a.kl[row] = kl;
    if (w == 0.f) return 0.0;                            // (a row of weight 0 may hold NaN)
    const float g = w * dl * static_cast<float>(a.inv_temp);
    if (g != 0.f) *ga = g * inv;
    return static_cast<double>(w) * static_cast<double>(l);
}

// ---- 16-byte vectors of a row --------------------------------------------------------------------------------------
// A row is cut into a head of fewer than V elements up to the first 16-byte boundary, whole vectors, and a tail; head and
// tail elements are one extra element each of 16 threads.  Vector v holds the elements head + v V, ...
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int V = 4;
    static constexpr uint32_t kLow = 0xFF800000u;          // a word of -infinity
    __device__ static __forceinline__ float max(uint4 r) {
        return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
    }
    __device__ static __forceinline__ void open(uint4 r, float (&f)[4]) {
        f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
    }
    __device__ static __forceinline__ uint4 close(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int V = 8;
    static constexpr uint32_t kLow = 0xFF80FF80u;
    __device__ static __forceinline__ float max(uint4 r) {
        const __nv_bfloat162 a = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&r.x), *reinterpret_cast<__nv_bfloat162*>(&r.y));
        const __nv_bfloat162 b = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&r.z), *reinterpret_cast<__nv_bfloat162*>(&r.w));
        const float2 f = __bfloat1622float2(__hmax2(a, b));
        return fmaxf(f.x, f.y);
    }
    __device__ static __forceinline__ void open(uint4 r, float (&f)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
    }
    __device__ static __forceinline__ uint4 close(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<uint32_t*>(&p);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
// over groups of G adjacent lanes
template <int G = 32>
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
    return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}
// exp((f - m) / T) of V scores, two at a time (packed fp32 pairs: half the instructions of the subtraction and the product)
struct Scale2 { float hi, lo; };
__device__ __forceinline__ float cand_exp(float x, Scale2 c) { return cand_ex2(fmaf(x, c.hi, x * c.lo)); }      // exp(x / T)
template <int V>
__device__ __forceinline__ void cand_exps(float (&f)[V], float m, Scale2 c) {
    const float2 nm = make_float2(-m, -m), hi = make_float2(c.hi, c.hi), lo = make_float2(c.lo, c.lo);
#pragma unroll
    for (int k = 0; k < V; k += 2) {
        const float2 d = __fadd2_rn(make_float2(f[k], f[k + 1]), nm);
        const float2 p = __ffma2_rn(d, hi, __fmul2_rn(d, lo));
        f[k] = cand_ex2(p.x); f[k + 1] = cand_ex2(p.y);
    }
}
template <int V>
__device__ __forceinline__ void cand_scale(float (&f)[V], float by) {
    const float2 b2 = make_float2(by, by);
#pragma unroll
    for (int k = 0; k < V; k += 2) {
        const float2 p = __fmul2_rn(make_float2(f[k], f[k + 1]), b2);
        f[k] = p.x; f[k + 1] = p.y;
    }
}
// even and odd elements summed side by side
template <int V>
__device__ __forceinline__ void cand_add(float2& sum, const float (&f)[V]) {
    float2 t = __fadd2_rn(make_float2(f[0], f[1]), make_float2(f[2], f[3]));
    if (V == 8) t = __fadd2_rn(t, __fadd2_rn(make_float2(f[V - 4], f[V - 3]), make_float2(f[V - 2], f[V - 1])));
    sum = __fadd2_rn(sum, t);
}
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int n) {
    const int to = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(T));
    return to < n ? to : n;
}
// Elements from `cnt` on read as -infinity.
template <typename T>
__device__ __forceinline__ uint4 mask_past(uint4 r, int first, int cnt) {
    float f[Vec<T>::V];
    Vec<T>::open(r, f);
#pragma unroll
    for (int k = 0; k < Vec<T>::V; ++k) if (first + k >= cnt) f[k] = -INFINITY;
    return Vec<T>::close(f);
}
// (m, rest) of two disjoint parts of a row
__device__ __forceinline__ void merge_parts(float& m, float& rest, float m2, float r2, Scale2 c) {
    const float top = finite_or_zero(fmaxf(m, m2));
    rest = rest * cand_exp(m - top, c) + r2 * cand_exp(m2 - top, c);
    m = fmaxf(m, m2);
}

// ---- rows kept in registers -------------------------------------------------------------------------------------------
// A warp, a CTA or a cluster of CTAs reads a row once, as I vectors a thread, and keeps it until the gradient is written:
// 8 bytes of traffic per fp32 score, 4 per bf16.  Each warp takes its own maximum and sum; the (m, rest) pairs of a row's
// warps are merged after one barrier.  fp32 scores are replaced by their exponentials in place, so the gradient costs one
// multiplication each; bf16 scores stay packed and are exponentiated a second time.
struct Slice {                    // a CTA's part of a row
    int head, nv, v0, v1;         // elements before the first vector, vectors of the row, vectors [v0, v1) of this CTA
};
template <typename T>
__device__ __forceinline__ Slice cand_slice(const T* s, int n, uint32_t rank, uint32_t csize) {
    Slice q;
    q.head = head_of(s, n);
    q.nv = (n - q.head) / Vec<T>::V;
    const int shift = 31 - __clz(static_cast<int>(csize));        // cluster sizes are powers of two
    const int share = (q.nv + static_cast<int>(csize) - 1) >> shift;
    q.v0 = min(q.nv, static_cast<int>(rank) * share);
    q.v1 = min(q.nv, q.v0 + share);
    return q;
}
// The head or tail element that thread tid < 16 of the row's first CTA takes, or -1.
template <typename T>
__device__ __forceinline__ int extra_index(const Slice& q, int n, int tid) {
    if (tid < 8) return tid < q.head ? tid : -1;
    const int j = q.head + q.nv * Vec<T>::V + tid - 8;
    return tid < 16 && j < n ? j : -1;
}

// A thread's part of one row between the loads and the gradient: register i holds vector lane + i G of the row, threads below 8
// also one element of the head and one of the tail.
template <typename T, int G, int I>
struct RowPart {
    static constexpr int V = Vec<T>::V;
    static constexpr bool kKeepExp = sizeof(T) == 4;
    uint4 r[I];
    float xe[2];                  // the head and tail elements
    int xi[2], own;               // their indexes or -1; the register that holds the chosen candidate, or -1
    float mw, mz;                 // maximum of the row, and with 0 in the place of -infinity

    __device__ __forceinline__ void load(const T* s, const Slice& q, int n, int cnt, int lane) {
        const uint4* src = reinterpret_cast<const uint4*>(s + q.head) + lane;
        const int nvc = cnt <= q.head ? 0 : (cnt - q.head + V - 1) / V, left = min(q.nv, nvc) - lane;
#pragma unroll
        for (int i = 0; i < I; ++i) {
            r[i] = make_uint4(Vec<T>::kLow, Vec<T>::kLow, Vec<T>::kLow, Vec<T>::kLow);
            if (i * G < left) r[i] = __ldcs(src + i * G);
        }
        xi[0] = lane < q.head ? lane : -1;
        xi[1] = lane < 8 && q.head + q.nv * V + lane < n ? q.head + q.nv * V + lane : -1;
#pragma unroll
        for (int k = 0; k < 2; ++k) xe[k] = xi[k] >= 0 && xi[k] < cnt ? cand_get(s + xi[k]) : -INFINITY;
    }
    __device__ __forceinline__ float stats(const Slice& q, int n, int cnt, int act, int lane, Scale2 c) {
        const int used = (q.nv + G - 1) / G;                                  // registers that hold anything, the same for all
        if (cnt < n) {
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const int at = q.head + (lane + i * G) * V;
                if (at < cnt && at + V > cnt) r[i] = mask_past<T>(r[i], at, cnt);
            }
        }
        mw = fmaxf(xe[0], xe[1]);
#pragma unroll
        for (int i = 0; i < I; ++i) if (i < used) mw = fmaxf(mw, Vec<T>::max(r[i]));
        mw = warp_max<G>(mw);
        mz = finite_or_zero(mw);
        own = -1;
        if (act >= q.head && act < q.head + q.nv * V) {
            const int v = (act - q.head) / V;
            if (v % G == lane) own = v / G;
        }
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float e = cand_exp(xe[k] - mz, c);
            if (xi[k] != act) sum.x += e;
            if (kKeepExp) xe[k] = e;
        }
#pragma unroll
        for (int i = 0; i < I; ++i) {
            if (i >= used) continue;
            float f[V];
            Vec<T>::open(r[i], f);
            cand_exps<V>(f, mz, c);
            if (kKeepExp) r[i] = Vec<T>::close(f);
            if (i == own) {
#pragma unroll
                for (int k = 0; k < V; ++k) if ((act - q.head) % V == k) f[k] = 0.f;
            }
            cand_add<V>(sum, f);
        }
        if (!kKeepExp) {          // keep the packed words, not their unpacked values, in registers until the gradient
#pragma unroll
            for (int i = 0; i < I; ++i) asm volatile("" : "+r"(r[i].x), "+r"(r[i].y), "+r"(r[i].z), "+r"(r[i].w));
        }
        return group_sum<G>(sum.x + sum.y);
    }
    __device__ __forceinline__ void write(T* d, const Slice& q, int n, int cnt, int act, int lane, Scale2 c, float rest, float ga) const {
        uint4* dv = reinterpret_cast<uint4*>(d + q.head) + lane;
        const int left = q.nv - lane;
        const float f0 = ga == 0.f ? 0.f : -ga, fa = ga == 0.f ? 0.f : ga * rest;
        const bool plain = cnt == n && ga != 0.f;                 // no padding, and something to write
#pragma unroll
        for (int i = 0; i < I; ++i) {
            if (i * G < left) {
                float f[V];
                Vec<T>::open(r[i], f);
                if (!kKeepExp) cand_exps<V>(f, mz, c);
                cand_scale<V>(f, f0);
                if (!plain) {
                    const int at = q.head + (lane + i * G) * V;
#pragma unroll
                    for (int k = 0; k < V; ++k) if (ga == 0.f || at + k >= cnt) f[k] = 0.f;
                }
                __stcs(dv + i * G, Vec<T>::close(f));
            }
        }
        if (own >= 0) cand_put(d + act, fa);                      // over the vector just stored by this thread
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (xi[k] < 0) continue;
            float v = 0.f;
            if (xi[k] < cnt && ga != 0.f) v = xi[k] == act ? fa : f0 * (kKeepExp ? xe[k] : cand_exp(xe[k] - mz, c));
            cand_put(d + xi[k], v);
        }
    }
};

// Short rows: G lanes per row, up to G I vectors.  With one warp a row whatever its length, 10782 rows of 35 took three waves of
// resident warps; four rows a warp also share the instructions of the rows' scalars.
template <typename T, int G, int I, int MODE>
__global__ void __launch_bounds__(256, I <= 4 ? 4 : 3) cand_group_kernel(CandArgs a) {
    constexpr int R = 32 / G;                                     // rows of a warp
    __shared__ double red[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gl = lane % G;
    let_next_start();
    const Scale2 c = {a.c_hi, a.c_lo};
    double total = 0.0;
    for (long long first = ((long long)blockIdx.x * 8 + warp) * R; first < a.rows; first += (long long)gridDim.x * (8 * R)) {
        const bool live = first + lane / G < a.rows;              // (all lanes take part in the shuffles)
        const long long row = live ? first + lane / G : a.rows - 1;
        const T* s = static_cast<const T*>(a.scores) + row * a.ld;
        const int cnt = cand_count(a, row);
        const int act = cand_action(a, row, cnt, live && gl == 0);
        const float sa = act >= 0 && gl == 0 ? cand_get(s + act) : 0.f;
        float side = 0.f;                 // lane k < 4 of a row requests operand k now: its finish must not wait for memory
        if (MODE == CM_POLICY && gl < 4) side = cand_side(a, row, gl);
        const Slice q = cand_slice(s, a.n, 0, 1);
        RowPart<T, G, I> p;
        p.load(s, q, a.n, cnt, gl);
        const float rest = p.stats(q, a.n, cnt, act, gl, c);
        RowSide o = {};
        if (MODE == CM_POLICY) {
            const int l0 = lane - gl;
            o.w = __shfl_sync(kFull, side, l0); o.adv = __shfl_sync(kFull, side, l0 + 1);
            o.old = __shfl_sync(kFull, side, l0 + 2); o.ref = __shfl_sync(kFull, side, l0 + 3);
        }
        float ga = 0.f;
        __syncwarp();                     // (rows written over their scores: every lane of the row has read its own)
        if (gl == 0 && live) total += cand_finish<MODE>(a, row, act, sa, p.mz, rest, true, o, &ga);
        if (MODE == CM_POLICY) {
            ga = __shfl_sync(kFull, ga, lane - gl);
            if (live) p.write(static_cast<T*>(a.dscores) + row * a.ldd, q, a.n, cnt, act, gl, c, rest, ga);
        }
    }
    if (MODE == CM_POLICY) {
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

// ---- rows kept in shared memory -----------------------------------------------------------------------------------------
// A CTA, or a cluster, with one row each.  Its part of the row arrives by one bulk copy (in flight before anything else is
// known about the row), is read twice from shared memory - online maximum and sum, then the gradient - and leaves by 16-byte
// stores.  As many CTAs as shared memory holds (3 at 60 KB) share an SM, so that copies, arithmetic and stores of different
// rows overlap.  Policy loss over 4096 x 15000 fp32 / 1024 x 100000 bf16: 78 / 86 us; a row in the registers of 512 threads
// 95 / 136 us, of 256 threads 93 / 132 us; one CTA per SM with a ring of row slots 122 / 150 us.
// The chosen candidate's place in shared memory reads as -infinity from here on, so that it adds nothing to S'; its score is the
// caller's first maximum.  The thread that works on its vector calls this (one test for each vector instead cost an eighth of the
// instructions).
template <typename T>
__device__ __forceinline__ float take_chosen(T* p) {
    const float x = cand_get(p);
    cand_put(p, -INFINITY);
    return x;
}
// Maximum and sum over the vectors first, first + step, ... below nv; m comes in as the maximum so far.  Two vectors share a test for
// a new maximum (rare after the first ones).
template <typename T>
__device__ __forceinline__ float2 online_sum(const uint4* sv, int first, int nv, int step, float& m, Scale2 c) {
    constexpr int V = Vec<T>::V;
    float2 sum = make_float2(0.f, 0.f);
    float mz = finite_or_zero(m);
    const uint4 low = make_uint4(Vec<T>::kLow, Vec<T>::kLow, Vec<T>::kLow, Vec<T>::kLow);
    for (int v = first; v < nv; v += 2 * step) {
        const uint4 r0 = sv[v], r1 = v + step < nv ? sv[v + step] : low;
        const float vm = fmaxf(Vec<T>::max(r0), Vec<T>::max(r1));
        if (vm > m) {                     // rescale what there is
            mz = finite_or_zero(vm);
            const float by = cand_exp(m - mz, c);
            sum = __fmul2_rn(sum, make_float2(by, by));
            m = vm;
        }
        float f[V], g[V];
        Vec<T>::open(r0, f);
        Vec<T>::open(r1, g);
        cand_exps<V>(f, mz, c);
        cand_exps<V>(g, mz, c);
        cand_add<V>(sum, f);
        cand_add<V>(sum, g);
    }
    return sum;
}
constexpr int kMaxCluster = 8;
constexpr int kRowSlot = 4608, kRowSmem = 216 * 1024;          // vectors of a row per CTA, at most (72 KB: three CTAs per SM)
template <typename T, int THREADS, int ROWS, int CTAS, int MODE>
__global__ void __launch_bounds__(THREADS * ROWS, CTAS) cand_row_kernel(CandArgs a, int slot) {
    constexpr int kWarps = THREADS / 32, V = Vec<T>::V;
    static_assert(ROWS == 1 || THREADS == 32, "rows that share a CTA have a warp each");
    extern __shared__ __align__(128) uint8_t cta_smem[];
    __shared__ __align__(8) uint64_t fulls[ROWS];
    __shared__ float2 parts[kWarps];
    __shared__ float bcast, sides[4];
    const int tid = threadIdx.x % THREADS, lane = tid & 31, warp = tid >> 5, mine_of = threadIdx.x / THREADS;
    uint8_t* row_smem = cta_smem + mine_of * slot * 16;
    uint64_t& full = fulls[mine_of];
    uint32_t rank, csize;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(csize));
    let_next_start();
    const long long row = ROWS > 1 ? (long long)blockIdx.x * ROWS + mine_of : blockIdx.x / csize;
    if (ROWS > 1 && row >= a.rows) return;
    const Scale2 c = {a.c_hi, a.c_lo};
    const T* s = static_cast<const T*>(a.scores) + row * a.ld;
    const int cnt = cand_count(a, row);
    const Slice q = cand_slice(s, a.n, rank, csize);
    const int nvc = cnt <= q.head ? 0 : (cnt - q.head + V - 1) / V;         // vectors of the row that hold a candidate
    const int have = max(0, min(q.v1, nvc) - q.v0);                         // of this CTA
    if (tid == 0) {
        umma::mbar_init(&full, 1);
        umma::fence_barrier_init();
        if (have > 0) {
            umma::mbar_expect_tx(&full, static_cast<uint32_t>(have) * 16u);
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                         ::"r"(umma::smem_u32(row_smem)), "l"(reinterpret_cast<const uint4*>(s + q.head) + q.v0),
                           "r"(static_cast<uint32_t>(have) * 16u), "r"(umma::smem_u32(&full)) : "memory");
        } else {
            umma::mbar_arrive(&full);
        }
    }
    const int act = cand_action(a, row, cnt, tid == 0 && rank == 0);
    const float sa = act >= 0 && tid == 0 ? cand_get(s + act) : 0.f;
    float side = 0.f;                     // thread k < 4 requests operand k now: the finish of the row must not wait for memory
    if (MODE == CM_POLICY && tid < 4) side = cand_side(a, row, tid);
    const int xi = rank == 0 ? extra_index<T>(q, a.n, tid) : -1;
    const float xe = xi >= 0 && xi < cnt ? cand_get(s + xi) : -INFINITY;
    // this CTA's vector that holds the chosen candidate
    const int av = act >= q.head && act < q.head + q.nv * V ? (act - q.head) / V - q.v0 : -1;
    const bool mine_chosen = av >= 0 && av < have && av % THREADS == tid;
    float m = -INFINITY, rest = 0.f, mz;
    if (ROWS > 1) __syncwarp();           // the barrier exists
    else __syncthreads();
    if (!umma::mbar_wait(&full, 0)) {     // (the row's outputs are invalid; its copy is waited for once more)
        atomicOr(a.err, KGE_ERR_WAIT_TIMEOUT);
        umma::mbar_wait(&full, 0);
    }
    const uint4* sv = reinterpret_cast<const uint4*>(row_smem);
    const int whole = cnt >= a.n ? have : min(have, max(0, (cnt - q.head) / V - q.v0));      // vectors without padding in them
    if (mine_chosen) m = take_chosen(reinterpret_cast<T*>(row_smem) + (act - q.head - q.v0 * V));
    if (whole < have && whole % THREADS == tid)             // the vector that the count cuts: padding reads as -infinity
        reinterpret_cast<uint4*>(row_smem)[whole] = mask_past<T>(sv[whole], q.head + (q.v0 + whole) * V, cnt);
    const float2 sum = online_sum<T>(sv, tid, have, THREADS, m, c);
    {
        const float mine = m;
        m = warp_max(fmaxf(m, xe));
        mz = finite_or_zero(m);
        rest = warp_sum((sum.x + sum.y) * cand_exp(mine - mz, c) + (xi != act ? cand_exp(xe - mz, c) : 0.f));
    }
    RowSide o = {};
    if (kWarps == 1) {                    // (one warp: always a row of its own)
        if (MODE == CM_POLICY) {
            o.w = __shfl_sync(kFull, side, 0); o.adv = __shfl_sync(kFull, side, 1);
            o.old = __shfl_sync(kFull, side, 2); o.ref = __shfl_sync(kFull, side, 3);
        }
    } else {
        if (lane == 0) parts[warp] = make_float2(m, rest);
        if (MODE == CM_POLICY && tid < 4) sides[tid] = side;
        if (csize == 1) __syncthreads();
        else asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        // every warp merges all parts of the row, in the same order
        m = -INFINITY;
        rest = 0.f;
        if (csize == 1) {
            if (lane < kWarps) { m = parts[lane].x; rest = parts[lane].y; }
        } else {
            for (int j = lane; j < kWarps * static_cast<int>(csize); j += 32) {
                float2 o;
                uint32_t remote;
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(umma::smem_u32(&parts[j % kWarps])), "r"(static_cast<uint32_t>(j / kWarps)));
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(o.x), "=f"(o.y) : "r"(remote) : "memory");
                merge_parts(m, rest, o.x, o.y, c);
            }
            // the parts have been read: no CTA of the cluster leaves before the others have got here (nothing is handed over)
            asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
        }
        {
            const float mine = m;
            m = warp_max(m);
            mz = finite_or_zero(m);
            rest = warp_sum(rest * cand_exp(mine - mz, c));
        }
        if (MODE == CM_POLICY && tid == 0) o = RowSide{sides[0], sides[1], sides[2], sides[3]};
    }
    float ga = 0.f;
    if (tid == 0) {
        const double l = cand_finish<MODE>(a, row, act, sa, mz, rest, rank == 0, o, &ga);
        if (kWarps > 1) bcast = ga;
        if (MODE == CM_POLICY && rank == 0) a.partial[row] = l;
    }
    if (MODE == CM_POLICY) {
        if (kWarps > 1) {
            __syncthreads();
            ga = bcast;
        } else {
            ga = __shfl_sync(kFull, ga, 0);
        }
        const float fa = ga == 0.f ? 0.f : ga * rest;
        T* d = static_cast<T*>(a.dscores) + row * a.ldd;
        uint4* dv = reinterpret_cast<uint4*>(d + q.head) + q.v0;
        const int mine = q.v1 - q.v0, full_to = ga == 0.f ? 0 : whole;
#pragma unroll 2
        for (int v = tid; v < full_to; v += THREADS) {
            float f[V];
            Vec<T>::open(sv[v], f);
            cand_exps<V>(f, mz, c);
            cand_scale<V>(f, -ga);
            __stcs(dv + v, Vec<T>::close(f));
        }
        const int from = full_to <= tid ? tid : tid + (full_to - tid + THREADS - 1) / THREADS * THREADS;      // (a vector keeps its thread)
        for (int v = from; v < mine; v += THREADS) {                        // the vector that the count cuts, padding, dead rows
            float f[V];
#pragma unroll
            for (int k = 0; k < V; ++k) f[k] = 0.f;
            const int at = q.head + (q.v0 + v) * V;
            if (ga != 0.f && at < cnt) {
                float g[V];
                Vec<T>::open(sv[v], g);
#pragma unroll
                for (int k = 0; k < V; ++k) if (at + k < cnt) f[k] = -ga * cand_exp(g[k] - mz, c);
            }
            __stcs(dv + v, Vec<T>::close(f));
        }
        if (mine_chosen) cand_put(d + act, fa);             // over the vector just stored by this thread
        if (xi >= 0) cand_put(d + xi, xi >= cnt || ga == 0.f ? 0.f : xi == act ? fa : -ga * cand_exp(xe - mz, c));
    }
    if (csize > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- rows cut over several CTAs, in passes ----------------------------------------------------------------------------
// For a few long rows (every SM reads), rows that no cluster can hold, and rows whose gradient lies at another alignment.
// Pass 1: (m, rest) of every chunk of a row; pass 2: a warp per row joins them; pass 3 (policy): the gradient, elementwise.
// A chunk arrives in shared memory by one bulk copy, under way before anything else is known about its row: 16 rows of 4,000,000
// fp32 scores 42 us (6.1 TB/s), with loads into registers instead 66 us; 1024 x 100000 bf16 45 us; CTAs that stay, with two slots each,
// 52 us and 66 us.
constexpr int kChunk = 8192;                                            // fp32 scores of a chunk, at most; bf16: twice as many
template <typename T>
__global__ void __launch_bounds__(256) cand_stats_kernel(CandArgs a, float2* parts, int chunk, int chunks) {
    constexpr int V = Vec<T>::V;
    extern __shared__ __align__(128) uint8_t chunk_smem[];
    __shared__ __align__(8) uint64_t full;
    __shared__ float2 red[8];
    let_next_start();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Scale2 c = {a.c_hi, a.c_lo};
    const uint4* sv = reinterpret_cast<const uint4*>(chunk_smem);
    if (tid == 0) {
        umma::mbar_init(&full, 1);
        umma::fence_barrier_init();
    }
    uint32_t phase = 0;
    for (long long u = blockIdx.x; u < a.rows * chunks; u += gridDim.x, phase ^= 1) {
        const long long row = u / chunks;
        const int k = static_cast<int>(u - row * chunks), j0 = k * chunk;
        const int cnt = cand_count(a, row), n = max(0, min(chunk, cnt - j0));
        const T* s = static_cast<const T*>(a.scores) + row * a.ld + j0;
        const int head = head_of(s, n), nv = (n - head) / V;
        if (tid == 0) {
            if (nv > 0) {
                umma::mbar_expect_tx(&full, static_cast<uint32_t>(nv) * 16u);
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                             ::"r"(umma::smem_u32(chunk_smem)), "l"(s + head), "r"(static_cast<uint32_t>(nv) * 16u), "r"(umma::smem_u32(&full)) : "memory");
            } else {
                umma::mbar_arrive(&full);
            }
        }
        const int act = cand_action(a, row, cnt, tid == 0 && k == 0), la = act - j0;
        const int xi = tid < 8 ? (tid < head ? tid : -1) : tid < 16 && head + nv * V + tid - 8 < n ? head + nv * V + tid - 8 : -1;
        const float xe = xi >= 0 ? cand_get(s + xi) : -INFINITY;
        const int av = act >= 0 && la >= head && la < head + nv * V ? (la - head) / V : -1;
        __syncthreads();                  // the barrier exists
        if (!umma::mbar_wait(&full, phase)) {     // (the call's outputs are invalid; the copy is waited for once more)
            atomicOr(a.err, KGE_ERR_WAIT_TIMEOUT);
            umma::mbar_wait(&full, phase);
        }
        float m = -INFINITY;
        if (av >= 0 && tid == (av & 255)) {
            m = take_chosen(reinterpret_cast<T*>(chunk_smem) + (la - head));
            umma::fence_proxy_async();    // (before the next chunk's copy)
        }
        float2 sum = online_sum<T>(sv, tid, nv, 256, m, c);
        const float mine = m;
        m = warp_max(fmaxf(m, xe));
        const float mz = finite_or_zero(m);
        float rest = warp_sum((sum.x + sum.y) * cand_exp(mine - mz, c) + (act < 0 || xi != la ? cand_exp(xe - mz, c) : 0.f));
        if (lane == 0) red[warp] = make_float2(m, rest);
        __syncthreads();                  // (also: the chunk has been read, the next one may arrive)
        if (warp == 0) {
            m = lane < 8 ? red[lane].x : -INFINITY;
            rest = lane < 8 ? red[lane].y : 0.f;
            const float own = m;
            m = warp_max(m);
            rest = warp_sum(rest * cand_exp(own - finite_or_zero(m), c));
            if (lane == 0) parts[u] = make_float2(m, rest);
        }
    }
}

// WARPS warps per row: one, or the whole CTA for rows of many chunks
template <typename T, int MODE, int WARPS>
__global__ void __launch_bounds__(256) cand_join_kernel(CandArgs a, const float2* parts, int chunks, float* coef) {
    __shared__ double red[8];
    __shared__ float2 merged[8];
    let_next_start();
    after_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = threadIdx.x % (32 * WARPS);
    const Scale2 c = {a.c_hi, a.c_lo};
    double total = 0.0;
    for (long long row = WARPS == 1 ? (long long)blockIdx.x * 8 + warp : blockIdx.x; row < a.rows; row += (long long)gridDim.x * (8 / WARPS)) {
        float m = -INFINITY, rest = 0.f;
#pragma unroll 4
        for (int k = tid; k < chunks; k += 32 * WARPS) {
            const float2 q = parts[row * chunks + k];
            merge_parts(m, rest, q.x, q.y, c);
        }
        float mine = m;
        m = warp_max(m);
        rest = warp_sum(rest * cand_exp(mine - finite_or_zero(m), c));
        if (WARPS > 1) {
            if (lane == 0) merged[warp] = make_float2(m, rest);
            __syncthreads();
            m = lane < WARPS ? merged[lane].x : -INFINITY;
            rest = lane < WARPS ? merged[lane].y : 0.f;
            mine = m;
            m = warp_max(m);
            rest = warp_sum(rest * cand_exp(mine - finite_or_zero(m), c));
            __syncthreads();
        }
        if (tid == 0) {
            const int act = cand_action(a, row, cand_count(a, row), false);
            const float sa = act >= 0 ? cand_get(static_cast<const T*>(a.scores) + row * a.ld + act) : 0.f;
            float ga;
            RowSide o = {};
            if (MODE == CM_POLICY) o = RowSide{cand_side(a, row, 0), cand_side(a, row, 1), cand_side(a, row, 2), cand_side(a, row, 3)};
            total += cand_finish<MODE>(a, row, act, sa, finite_or_zero(m), rest, true, o, &ga);
            if (MODE == CM_POLICY) { coef[3 * row] = finite_or_zero(m); coef[3 * row + 1] = rest; coef[3 * row + 2] = ga; }
        }
    }
    if (MODE == CM_POLICY) {
        if (lane == 0) red[warp] = total;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < 8; ++w) total += red[w];
            a.partial[blockIdx.x] = total;
        }
    }
}

// ds from (m, rest, ga) per row, or, with dlogp, from the stats of log_prob: ga = dlogp / T / S.  ALIGNED (scores and gradient rows
// at the same 16-byte phase): eight lanes take pieces of 32 vectors, so that a warp's scalars serve four of them (100000 x 40 fp32 11.8 us,
// 40000 x 1100 bf16 38.5 us; with a warp a piece of 128 vectors 32.9 and 50.2 us); otherwise a warp takes pieces of 128 elements.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) cand_grad_kernel(CandArgs a, const float* coef, long long pieces) {
    constexpr int V = ALIGNED ? Vec<T>::V : 1, G = ALIGNED ? 8 : 32;
    const int lane = threadIdx.x % G;
    let_next_start();
    after_previous();
    const Scale2 c = {a.c_hi, a.c_lo};
    const long long units = a.rows * pieces, step = (long long)gridDim.x * (256 / G);
    for (long long u = (long long)blockIdx.x * (256 / G) + threadIdx.x / G; u < units; u += step) {
        const long long row = units < (1LL << 32) ? static_cast<uint32_t>(u) / static_cast<uint32_t>(pieces) : u / pieces;
        const int piece = static_cast<int>(u - row * pieces);
        const T* s = static_cast<const T*>(a.scores) + row * a.ld;
        T* d = static_cast<T*>(a.dscores) + row * a.ldd;
        const int cnt = cand_count(a, row), act = cand_action(a, row, cnt, false);
        const float m = coef[3 * row], rest = coef[3 * row + 1];       // (plain loads: the kernel ahead wrote them)
        float ga = coef[3 * row + 2];
        if (a.dlogp) {                    // 1 / S of 0: a row that takes no part, whatever dlogp holds there
            const float g = __ldg(a.dlogp + row) * static_cast<float>(a.inv_temp);
            ga = g == 0.f || act < 0 || ga == 0.f ? 0.f : g * ga;
        }
        const float fa = ga == 0.f ? 0.f : ga * rest;
        auto one = [&](int j, float x) { return j >= cnt || ga == 0.f ? 0.f : j == act ? fa : -ga * cand_exp(x - m, c); };
        if constexpr (ALIGNED) {
            const int head = head_of(s, a.n), nv = (a.n - head) / V;
            const uint4* sv = reinterpret_cast<const uint4*>(s + head);
            uint4* dv = reinterpret_cast<uint4*>(d + head);
            uint4 r[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int v = piece * (4 * G) + i * G + lane;
                if (v < nv && head + v * V < cnt) r[i] = __ldcs(sv + v);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int v = piece * (4 * G) + i * G + lane, at = head + v * V;
                if (v >= nv) continue;
                float f[V];
                if (at >= cnt || ga == 0.f) {
#pragma unroll
                    for (int k = 0; k < V; ++k) f[k] = 0.f;
                } else {
                    Vec<T>::open(r[i], f);
                    if (at + V > cnt || (act >= at && act < at + V)) {
#pragma unroll
                        for (int k = 0; k < V; ++k) f[k] = one(at + k, f[k]);
                    } else {
                        cand_exps<V>(f, m, c);
                        cand_scale<V>(f, -ga);
                    }
                }
                __stcs(dv + v, Vec<T>::close(f));
            }
            if (piece == 0) {             // fewer than 8 elements before the first vector, and behind the last one
                const int tail = head + nv * V + lane;
                if (lane < head) cand_put(d + lane, one(lane, lane < cnt ? cand_get(s + lane) : 0.f));
                if (tail < a.n) cand_put(d + tail, one(tail, tail < cnt ? cand_get(s + tail) : 0.f));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = piece * 128 + i * 32 + lane;
                if (j < a.n) cand_put(d + j, one(j, j < cnt ? cand_get(s + j) : 0.f));
            }
        }
    }
}

__global__ void __launch_bounds__(1024) sum_partials_kernel(const double* partial, int n, float* out) {
    __shared__ double red[32];
    after_previous();
    double v = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += 1024) v += partial[i];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x < 32) {
        v = red[threadIdx.x];
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
        if (threadIdx.x == 0) *out = static_cast<float>(v);
    }
}

int launch_sum_partials(const double* partial, int n, float* out, cudaStream_t s) {
    if (n == 0) {                    // the only kernel of its call
        sum_partials_kernel<<<1, 1024, 0, s>>>(partial, n, out);
        KGE_LAUNCH_CHECK("sum_partials_kernel");
        return 0;
    }
    KGE_LAUNCH_AFTER("sum_partials_kernel", sum_partials_kernel, 1u, 1024u, s, partial, n, out);
    return 0;
}

constexpr int kCandMaxBlocks = 148 * 16;           // groups that take rows in turn; each leaves a partial sum of the loss

// Workspace: partial sums of the loss, then per-chunk (m, rest) and per-row coefficients of the multi-pass form.
struct CandLayout { int chunk, chunks; size_t off_parts, off_coef, total; };
static CandLayout cand_layout(long long rows, long long n) {
    CandLayout L;
    // about eight chunks per SM, of 1024 to 8192 scores
    long long per = (rows * n / (148 * 8) + 1023) / 1024 * 1024;
    per = per < 1024 ? 1024 : per > kChunk ? kChunk : per;
    L.chunk = static_cast<int>(per);
    L.chunks = static_cast<int>((n + per - 1) / per);
    if (L.chunks < 1) L.chunks = 1;
    L.off_parts = sizeof(double) * static_cast<size_t>(rows > kCandMaxBlocks ? rows : kCandMaxBlocks);
    L.off_coef = L.off_parts + sizeof(float2) * static_cast<size_t>(rows) * L.chunks;
    L.total = L.off_coef + 3 * sizeof(float) * static_cast<size_t>(rows);
    return L;
}

template <typename T, int G, int I, int MODE>
static int cand_groups(const CandArgs& a, int* n_partial, cudaStream_t s) {
    constexpr int per = 8 * (32 / G);
    const long long want = (a.rows + per - 1) / per;
    *n_partial = static_cast<int>(want < kCandMaxBlocks ? want : kCandMaxBlocks);
    cand_group_kernel<T, G, I, MODE><<<*n_partial, 256, 0, s>>>(a);
    KGE_LAUNCH_CHECK("cand_group_kernel");
    if (*n_partial == 1) *n_partial = 0;               // (nothing left to sum)
    return 0;
}

// slot: vectors of a row that one CTA holds
template <typename T, int THREADS, int ROWS, int CTAS, int MODE>
static int cand_rows(const CandArgs& a, int cluster, long long slot, int* n_partial, cudaStream_t s) {
    static thread_local unsigned long long opted_in = 0;      // the shared-memory opt-in is per context and kernel
    const unsigned long long here = context_number();
    if (here == 0 || here != opted_in) {
        cudaError_t e = cudaFuncSetAttribute(cand_row_kernel<T, THREADS, ROWS, CTAS, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowSmem);
        if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(cand_row_kernel)");
        opted_in = context_number();
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((a.rows + ROWS - 1) / ROWS * cluster));
    cfg.blockDim = dim3(THREADS * ROWS);
    cfg.dynamicSmemBytes = static_cast<size_t>(slot) * ROWS * 16;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = cluster > 1 ? 1 : 0;
    *n_partial = static_cast<int>(a.rows);
    cudaError_t e = cudaLaunchKernelEx(&cfg, cand_row_kernel<T, THREADS, ROWS, CTAS, MODE>, a, static_cast<int>(slot));
    if (e != cudaSuccess) return cuda_status(e, "cand_row_kernel");
    KGE_LAUNCH_CHECK("cand_row_kernel");
    return 0;
}

template <typename T>
static int cand_gradient(const CandArgs& a, const float* coef, bool aligned, bool first, cudaStream_t s) {
    const int per = aligned ? 32 * Vec<T>::V : 128, groups = aligned ? 32 : 8;          // elements of a piece, pieces of a CTA
    const long long pieces = a.n > 0 ? (a.n + per - 1) / per : 1, want = (a.rows * pieces + groups - 1) / groups;
    const unsigned blocks = static_cast<unsigned>(want < (1 << 30) ? want : (1 << 30));       // (short CTAs copy faster than a loop)
    if (!first) {
        if (aligned) KGE_LAUNCH_AFTER("cand_grad_kernel", cand_grad_kernel<T, true>, blocks, 256u, s, a, coef, pieces);
        else KGE_LAUNCH_AFTER("cand_grad_kernel", cand_grad_kernel<T, false>, blocks, 256u, s, a, coef, pieces);
        return 0;
    }
    if (aligned) cand_grad_kernel<T, true><<<blocks, 256, 0, s>>>(a, coef, pieces);
    else cand_grad_kernel<T, false><<<blocks, 256, 0, s>>>(a, coef, pieces);
    KGE_LAUNCH_CHECK("cand_grad_kernel");
    return 0;
}

template <typename T>
static bool same_phase(const CandArgs& a) {
    const uintptr_t d = reinterpret_cast<uintptr_t>(a.scores) - reinterpret_cast<uintptr_t>(a.dscores);
    return ((d & 15) == 0) && (a.rows == 1 || (((a.ld - a.ldd) * static_cast<long long>(sizeof(T))) & 15) == 0);
}

template <typename T, int MODE>
static int cand_passes(const CandArgs& a, void* ws, int* n_partial, cudaStream_t s) {
    const CandLayout L = cand_layout(a.rows, a.n);
    float2* parts = reinterpret_cast<float2*>(static_cast<char*>(ws) + L.off_parts);
    float* coef = reinterpret_cast<float*>(static_cast<char*>(ws) + L.off_coef);
    const int chunk = L.chunk * (4 / static_cast<int>(sizeof(T))), chunks = a.n > 0 ? (a.n - 1) / chunk + 1 : 1;      // the same bytes of either type
    const long long units = a.rows * chunks;
    cand_stats_kernel<T><<<static_cast<unsigned>(units < (1 << 30) ? units : (1 << 30)), 256, chunk * sizeof(T), s>>>(a, parts, chunk, chunks);
    KGE_LAUNCH_CHECK("cand_stats_kernel");
    const bool wide = chunks > 64;
    const long long jb = wide ? a.rows : (a.rows + 7) / 8;
    *n_partial = static_cast<int>(jb < kCandMaxBlocks ? jb : kCandMaxBlocks);
    if (wide) KGE_LAUNCH_AFTER("cand_join_kernel", (cand_join_kernel<T, MODE, 8>), static_cast<unsigned>(*n_partial), 256u, s, a, parts, chunks, coef);
    else KGE_LAUNCH_AFTER("cand_join_kernel", (cand_join_kernel<T, MODE, 1>), static_cast<unsigned>(*n_partial), 256u, s, a, parts, chunks, coef);
    return MODE == CM_POLICY ? cand_gradient<T>(a, coef, same_phase<T>(a), false, s) : 0;
}

// Which form: the smallest group of lanes that holds a row in registers, then a warp or a CTA a row, the smaller the shorter the
// row; passes where the rows are too long for a cluster, where the groups of all rows would leave most SMs idle, or where the
// gradient's alignment differs.  A row's own scalars cost a warp some 500 issue slots whatever its length, so few lanes a row win
// while the lanes are busy (us, log_prob / policy loss):
//   20000 x 420 fp32   16 lanes 11.4 / 19.0   32 lanes 12.4 / 22.3        but 800 x 900 bf16   16 lanes 4.2 / 7.3   32 lanes 3.7 / 6.3
//   30000 x 300 bf16    8 lanes 11.4 / 18.5   16 lanes 12.4 / 21.1
//   8350 x 923 bf16   a warp, shared memory 7.8 / 14.1   16 lanes 9.3 / 15.1       20000 x 420 fp32   a warp 11.9 / 22.1
//   40000 x 1100 bf16   four warps a CTA, a row each 29.8 / 57.5   CTAs of one warp 42.7 / 59.5   two warps a row 52 / 94
//   12995 x 3297 fp32  64 threads 31.1 / 59.7   128 threads 33.5 / 62.0    32 threads 37.0 / 67.9
//   8000 x 5600 fp32  128 threads 30.3 / 59.1   256 threads 37.5 / 67.0    4000 x 9200 fp32   128 threads 26.9 / 50.7   256 threads 26.0 / 49.8
template <typename T, int MODE>
static int cand_go(const CandArgs& a, void* ws, int* n_partial, cudaStream_t s) {
    const long long nv = a.n / Vec<T>::V;              // vectors of a row, at most
    if (MODE == CM_POLICY && !same_phase<T>(a)) return cand_passes<T, MODE>(a, ws, n_partial, s);
    if (nv <= 8) return cand_groups<T, 8, 1, MODE>(a, n_partial, s);
    if (nv <= 16) return cand_groups<T, 8, 2, MODE>(a, n_partial, s);
    if (nv <= 32) return cand_groups<T, 8, 4, MODE>(a, n_partial, s);
    if (nv <= 64) return cand_groups<T, 8, 8, MODE>(a, n_partial, s);
    if (nv <= 128 && a.rows <= 148 * 16) return cand_groups<T, 32, 4, MODE>(a, n_partial, s);
    if (nv <= (sizeof(T) == 4 ? 128 : 96)) return cand_groups<T, 16, 8, MODE>(a, n_partial, s);
    if (a.rows >= (1LL << 31) / kMaxCluster) return cand_passes<T, MODE>(a, ws, n_partial, s);      // (beyond a grid of one CTA a row)
    if (nv <= 512) return cand_rows<T, 32, 4, 8, MODE>(a, 1, nv, n_partial, s);
    if (nv <= 1024) return cand_rows<T, 64, 1, 16, MODE>(a, 1, nv, n_partial, s);
    if (nv <= 2048) return cand_rows<T, 128, 1, 10, MODE>(a, 1, nv, n_partial, s);
    int cluster = 1;
    while (cluster <= kMaxCluster && nv > cluster * static_cast<long long>(kRowSlot)) cluster *= 2;
    if (cluster > kMaxCluster || a.rows * cluster < 32) return cand_passes<T, MODE>(a, ws, n_partial, s);
    // without a gradient nothing is read twice, and clusters only cost their barriers: 1000 x 100000 fp32 61 us in passes, 84 us in
    // clusters; but 40 x 100000, with its second launch, 7.3 us and 6.7 us
    if (MODE == CM_LOGP && cluster > 1 && a.rows * cluster >= 148 * 3) return cand_passes<T, MODE>(a, ws, n_partial, s);
    return cand_rows<T, 256, 1, 5, MODE>(a, cluster, (nv + cluster - 1) / cluster, n_partial, s);
}

}  // namespace kge

using namespace kge;

static int check_candidates(const char* fn, const void* scores, int32_t dtype, int64_t ld, int64_t rows, int64_t n, const int32_t* n_cand,
                            const void* action, int32_t id_bits, double temperature, CandArgs* a) {
    if (dtype != KGE_F32 && dtype != KGE_BF16) { set_error("%s: unknown dtype %d", fn, dtype); return KGE_E_UNSUPPORTED; }
    if (id_bits != 32 && id_bits != 64) { set_error("%s: id_bits must be 32 or 64, got %d", fn, id_bits); return KGE_E_UNSUPPORTED; }
    if (!(temperature >= 1e-30 && temperature <= 1e30)) { set_error("%s: temperature %g outside [1e-30, 1e30]", fn, temperature); return KGE_E_RANGE; }
    if (rows < 0 || n < 0) { set_error("%s: negative size", fn); return KGE_E_SHAPE; }
    if (n > (1LL << 30) || rows > (1LL << 40)) { set_error("%s: more than 2^30 candidates or 2^40 rows", fn); return KGE_E_RANGE; }
    if (n > 0 && rows > (1LL << 46) / n) { set_error("%s: more than 2^46 scores", fn); return KGE_E_RANGE; }
    if (rows > 1 && ld < n) { set_error("%s: row pitch %lld is below n", fn, (long long)ld); return KGE_E_SHAPE; }
    if (ld > (1LL << 40)) { set_error("%s: row pitch above 2^40", fn); return KGE_E_RANGE; }
    if (rows == 0) return 0;
    if (!scores && n > 0) { set_error("%s: scores is NULL", fn); return KGE_E_NULL; }
    if (!action) { set_error("%s: action is NULL", fn); return KGE_E_NULL; }
    if ((reinterpret_cast<uintptr_t>(scores) & (dtype == KGE_F32 ? 3 : 1)) || (reinterpret_cast<uintptr_t>(action) & (id_bits / 8 - 1)) ||
        (reinterpret_cast<uintptr_t>(n_cand) & 3)) { set_error("%s: a pointer is not aligned to its element size", fn); return KGE_E_ALIGN; }
    a->scores = scores; a->ld = ld; a->rows = rows; a->n = static_cast<int>(n); a->n_cand = n_cand; a->action = action; a->id64 = id_bits == 64;
    a->inv_temp = 1.0 / temperature;
    const double c = 1.4426950408889634073599 / temperature;
    a->c_hi = static_cast<float>(c);
    if (static_cast<double>(a->c_hi) >= c) a->c_hi = nextafterf(a->c_hi, 0.f);     // c_lo > 0: a score of -infinity stays one in both products
    a->c_lo = static_cast<float>(c - static_cast<double>(a->c_hi));
    a->err = device_error_word();
    if (!a->err) { set_error("%s: no usable device", fn); return KGE_E_DEVICE; }
    return 0;
}
static int check_floats(const char* fn, const char* name, const float* p, bool required) {
    if (!p && required) { set_error("%s: %s is NULL", fn, name); return KGE_E_NULL; }
    if (reinterpret_cast<uintptr_t>(p) & 3) { set_error("%s: %s is not aligned to its element size", fn, name); return KGE_E_ALIGN; }
    return 0;
}
static int check_gradient(const char* fn, const void* scores, int64_t ld, void* dscores, int32_t dtype, int64_t ldd, int64_t rows, int64_t n) {
    if (rows > 1 && ldd < n) { set_error("%s: row pitch %lld of dscores is below n", fn, (long long)ldd); return KGE_E_SHAPE; }
    if (ldd > (1LL << 40)) { set_error("%s: row pitch above 2^40", fn); return KGE_E_RANGE; }
    if (!dscores && n > 0) { set_error("%s: dscores is NULL", fn); return KGE_E_NULL; }
    if (dscores == scores && rows > 1 && n > 0 && ldd != ld) { set_error("%s: dscores may be scores only with the same row pitch", fn); return KGE_E_SHAPE; }
    if (reinterpret_cast<uintptr_t>(dscores) & (dtype == KGE_F32 ? 3 : 1)) { set_error("%s: dscores is not aligned to its element size", fn); return KGE_E_ALIGN; }
    return 0;
}

extern "C" {

size_t kge_candidates_workspace_bytes(int64_t rows, int64_t n) {
    if (rows <= 0 || n < 0 || n > (1LL << 30) || rows > (1LL << 40) || (n > 0 && rows > (1LL << 46) / n)) return 0;
    return cand_layout(rows, n).total;
}

int kge_log_prob(const void* scores, int32_t dtype, int64_t ld, int64_t rows, int64_t n, const int32_t* n_cand, const void* action,
                 int32_t id_bits, double temperature, float* logp, float* stats, void* workspace, size_t workspace_bytes,
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
    int parts;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return dtype == KGE_F32 ? cand_go<float, CM_LOGP>(a, workspace, &parts, s) : cand_go<__nv_bfloat16, CM_LOGP>(a, workspace, &parts, s);
}

int kge_log_prob_backward(const void* scores, int32_t dtype, int64_t ld, int64_t rows, int64_t n, const int32_t* n_cand, const void* action,
                          int32_t id_bits, double temperature, const float* stats, const float* dlogp, void* dscores, int64_t ldd,
                          kge_stream_t stream) {
    const char* fn = "kge_log_prob_backward";
    CandArgs a = {};
    int rc = check_candidates(fn, scores, dtype, ld, rows, n, n_cand, action, id_bits, temperature, &a);
    if (rc || rows == 0) return rc;
    if ((rc = check_floats(fn, "stats", stats, true)) || (rc = check_floats(fn, "dlogp", dlogp, true)) ||
        (rc = check_gradient(fn, scores, ld, dscores, dtype, ldd, rows, n))) return rc;
    a.stats = const_cast<float*>(stats); a.dlogp = dlogp; a.dscores = dscores; a.ldd = ldd;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return dtype == KGE_F32 ? cand_gradient<float>(a, stats, same_phase<float>(a), true, s)
                            : cand_gradient<__nv_bfloat16>(a, stats, same_phase<__nv_bfloat16>(a), true, s);
}

int kge_policy_loss(const void* scores, int32_t dtype, int64_t ld, int64_t rows, int64_t n, const int32_t* n_cand, const void* action,
                    int32_t id_bits, double temperature, const float* old_logp, const float* ref_logp, const float* advantage,
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
        (rc = check_gradient(fn, scores, ld, dscores, dtype, ldd, rows, n))) return rc;
    if (workspace_bytes < kge_candidates_workspace_bytes(rows, n)) { set_error("%s: workspace too small", fn); return KGE_E_WORKSPACE; }
    if (!workspace) { set_error("%s: workspace is NULL", fn); return KGE_E_NULL; }
    if (!aligned16(workspace)) { set_error("%s: workspace is not 16-byte aligned", fn); return KGE_E_ALIGN; }
    a.logp = logp; a.kl = kl; a.dscores = dscores; a.ldd = ldd;
    a.old_logp = old_logp; a.ref_logp = ref_logp; a.adv = advantage; a.weight = weight;
    a.clip_lo = clip_low; a.clip_hi = clip_high; a.kl_coef = kl_coef; a.scale = scale;
    a.loss = loss;
    a.partial = static_cast<double*>(workspace);
    int parts = 0;
    rc = dtype == KGE_F32 ? cand_go<float, CM_POLICY>(a, workspace, &parts, s) : cand_go<__nv_bfloat16, CM_POLICY>(a, workspace, &parts, s);
    return rc || parts == 0 ? rc : launch_sum_partials(a.partial, parts, loss, s);
}

}  // extern "C"
