// Dropout from a counter-based generator: out = keep ? x / (1 - p) : 0 (+ residual), the mask is never stored.
//
// Element e = row * dim + column takes word e % 4 of Philox4x32-10 at counter (e / 4 low, e / 4 high, stream, 2^31 | step),
// key = seed, and is kept when that word is >= floor(p 2^32).  The gradient is the same map applied to d(out), so the
// backward call repeats the forward's (seed, stream, step) and nothing but that travels between them.  The id sampler
// uses counter word 3 = 0, so a mask never shares words with the ids drawn under the same seed and stream.
#include "common.cuh"
#include "philox.cuh"

namespace kge {

struct DropoutArgs {
    const void* x; const void* res; void* out;
    long long rows, ldx, ldr, ldo;
    int dim;
    uint32_t threshold, stream, step, k0, k1;
    const long long* step_dev;
    float scale;
};

__device__ __forceinline__ float drop_get(const float* p) { return *p; }
__device__ __forceinline__ float drop_get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void drop_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void drop_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// One thread per quad of elements (one Philox call), any pitch and alignment.
template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(DropoutArgs a) {
    const long long n = a.rows * a.dim, quads = (n + 3) / 4;
    const uint32_t step = 0x80000000u | (a.step_dev ? static_cast<uint32_t>(*a.step_dev) + a.step : a.step);
    const T* x = static_cast<const T*>(a.x);
    const T* res = static_cast<const T*>(a.res);
    T* out = static_cast<T*>(a.out);
    for (long long q = (long long)blockIdx.x * blockDim.x + threadIdx.x; q < quads; q += (long long)gridDim.x * blockDim.x) {
        const Philox4 w = philox4x32_10(static_cast<uint32_t>(q), static_cast<uint32_t>(static_cast<unsigned long long>(q) >> 32), a.stream, step,
                                        a.k0, a.k1);
        long long row = 4 * q / a.dim;
        int col = static_cast<int>(4 * q - row * a.dim);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (4 * q + i < n) {
                // a dropped element is 0 whatever it held (an infinity or NaN included)
                float v = w.x[i] >= a.threshold ? drop_get(x + row * a.ldx + col) * a.scale : 0.f;
                if (res) v += drop_get(res + row * a.ldr + col);
                drop_put(out + row * a.ldo + col, v);
            }
            if (++col == a.dim) { col = 0; ++row; }
        }
    }
}


// Rows of whole 16-byte vectors (or one packed run of them): V elements a vector, V / 4 Philox calls.  The ten round keys are
// computed on the host and read as constants, which leaves two wide multiplications and two xors a round: 12 integer
// instructions an element, below what the memory traffic of bf16 elements allows for.
struct RoundKeys { uint32_t a[10], b[10]; };

template <typename T> struct DropVec;
template <> struct DropVec<float> {
    static constexpr int V = 4;
    __device__ static __forceinline__ void open(uint4 r, float (&f)[4]) {
        f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
    }
    __device__ static __forceinline__ uint4 close(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <> struct DropVec<__nv_bfloat16> {
    static constexpr int V = 8;
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

// Each CTA has 256 x kDropU adjacent vectors and ends: a plain copy in this form runs at 6.6 TB/s, at 5.7 TB/s as a loop of
// eight resident CTAs per SM and at 6.4 TB/s with the vectors of a thread a grid apart.
constexpr int kDropU = 2;
template <typename T, bool PACKED>
__global__ void __launch_bounds__(256) dropout_vec_kernel(DropoutArgs a, RoundKeys keys, long long vectors, int per_row, int tail) {
    constexpr int V = DropVec<T>::V, U = kDropU;
    const uint32_t step = 0x80000000u | (a.step_dev ? static_cast<uint32_t>(*a.step_dev) + a.step : a.step);
    const uint4* x = static_cast<const uint4*>(a.x);
    const uint4* res = static_cast<const uint4*>(a.res);
    uint4* out = static_cast<uint4*>(a.out);
    if (PACKED && tail > 0 && blockIdx.x == gridDim.x - 1 && static_cast<int>(threadIdx.x) < tail) {
        // the elements behind the last whole vector, one a thread
        const long long e = vectors * V + threadIdx.x, q = e >> 2;
        const Philox4 w = philox4x32_10(static_cast<uint32_t>(q), static_cast<uint32_t>(q >> 32), a.stream, step, a.k0, a.k1);
        const uint32_t word = w.x[e & 3];
        float f = word >= a.threshold ? drop_get(static_cast<const T*>(a.x) + e) * a.scale : 0.f;
        if (res) f += drop_get(static_cast<const T*>(a.res) + e);
        drop_put(static_cast<T*>(a.out) + e, f);
    }
    {
        const long long v0 = (long long)blockIdx.x * (256 * U) + threadIdx.x;
        uint4 r[U], q[U];
        long long ox[U], orr[U], oo[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long v = v0 + u * 256;
            if (v >= vectors) break;
            if (PACKED) {
                ox[u] = orr[u] = oo[u] = v;
            } else {
                const long long row = v < (1LL << 32) ? static_cast<uint32_t>(v) / static_cast<uint32_t>(per_row) : v / per_row;
                const long long k = v - row * per_row;
                ox[u] = row * (a.ldx / V) + k; orr[u] = row * (a.ldr / V) + k; oo[u] = row * (a.ldo / V) + k;
            }
            r[u] = __ldcs(x + ox[u]);
            q[u] = make_uint4(0u, 0u, 0u, 0u);
            if (res) q[u] = __ldcs(res + orr[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long v = v0 + u * 256;
            if (v >= vectors) break;
            float f[V], g[V];
            DropVec<T>::open(r[u], f);
            DropVec<T>::open(q[u], g);
#pragma unroll
            for (int h = 0; h < V / 4; ++h) {
                const unsigned long long c = static_cast<unsigned long long>(v) * (V / 4) + h;
                uint32_t c0 = static_cast<uint32_t>(c), c1 = static_cast<uint32_t>(c >> 32), c2 = a.stream, c3 = step;
#pragma unroll
                for (int i = 0; i < 10; ++i) {
                    const unsigned long long p0 = 0xD2511F53ull * c0, p1 = 0xCD9E8D57ull * c2;
                    const uint32_t n0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ keys.a[i], n2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ keys.b[i];
                    c1 = static_cast<uint32_t>(p1); c3 = static_cast<uint32_t>(p0);
                    c0 = n0; c2 = n2;
                }
                const uint32_t w[4] = {c0, c1, c2, c3};
#pragma unroll
                for (int k = 0; k < 4; ++k) f[4 * h + k] = w[k] >= a.threshold ? f[4 * h + k] * a.scale : 0.f;
            }
            if (res) {
#pragma unroll
                for (int k = 0; k < V; ++k) f[k] += g[k];
            }
            __stcs(out + oo[u], DropVec<T>::close(f));
        }
    }
}

template <typename T>
static bool drop_vectors(const DropoutArgs& a, bool* packed) {
    constexpr int V = DropVec<T>::V;
    if (!aligned16(a.x) || !aligned16(a.res) || !aligned16(a.out)) return false;
    *packed = a.rows == 1 || (a.ldx == a.dim && a.ldo == a.dim && (!a.res || a.ldr == a.dim));
    if (*packed) return a.rows * a.dim >= V;
    return a.dim % V == 0 && a.ldx % V == 0 && a.ldo % V == 0 && a.ldr % V == 0;
}

template <typename T>
static int drop_go(const DropoutArgs& a, cudaStream_t s) {
    bool packed = false;
    if (!drop_vectors<T>(a, &packed)) {
        const long long want = ((a.rows * a.dim + 3) / 4 + 255) / 256;
        dropout_kernel<T><<<static_cast<unsigned>(want < 148 * 16 ? want : 148 * 16), 256, 0, s>>>(a);
        KGE_LAUNCH_CHECK("dropout_kernel");
        return 0;
    }
    RoundKeys keys;
    uint32_t k0 = a.k0, k1 = a.k1;
    for (int i = 0; i < 10; ++i, k0 += 0x9E3779B9u, k1 += 0xBB67AE85u) { keys.a[i] = k0; keys.b[i] = k1; }
    const long long vectors = a.rows * a.dim / DropVec<T>::V, want = (vectors + 256 * kDropU - 1) / (256 * kDropU);
    if (want >= (1LL << 31)) { set_error("kge_dropout: more than 2^40 vectors"); return KGE_E_RANGE; }
    const unsigned blocks = static_cast<unsigned>(want);
    const int per_row = a.dim / DropVec<T>::V;
    const int tail = static_cast<int>(a.rows * a.dim - vectors * DropVec<T>::V);
    if (packed) dropout_vec_kernel<T, true><<<blocks, 256, 0, s>>>(a, keys, vectors, per_row, tail);
    else dropout_vec_kernel<T, false><<<blocks, 256, 0, s>>>(a, keys, vectors, per_row, 0);
    KGE_LAUNCH_CHECK("dropout_vec_kernel");
    return 0;
}
int launch_dropout(const DropoutArgs& a, int dtype, cudaStream_t s) {
    return dtype == KGE_F32 ? drop_go<float>(a, s) : drop_go<__nv_bfloat16>(a, s);
}

}  // namespace kge

using namespace kge;

extern "C" int kge_dropout(const void* x, int32_t dtype, int64_t rows, int32_t dim, int64_t ldx, const void* residual, int64_t ldr,
                           void* out, int64_t ldo, double p, uint64_t seed, uint32_t stream_id, int64_t step, const int64_t* step_dev,
                           kge_stream_t stream) {
    const char* fn = "kge_dropout";
    if (dtype != KGE_F32 && dtype != KGE_BF16) { set_error("%s: unknown dtype %d", fn, dtype); return KGE_E_UNSUPPORTED; }
    if (!(p >= 0.0 && p < 1.0)) { set_error("%s: p = %g outside [0, 1)", fn, p); return KGE_E_RANGE; }
    if (rows < 0 || dim < 0) { set_error("%s: negative size", fn); return KGE_E_SHAPE; }
    if (rows == 0 || dim == 0) return 0;
    if (rows > (1LL << 60) / dim) { set_error("%s: rows x dim above 2^60", fn); return KGE_E_RANGE; }
    if (rows > 1 && (ldx < dim || ldo < dim || (residual && ldr < dim))) { set_error("%s: a row pitch is below dim", fn); return KGE_E_SHAPE; }
    if (!x || !out) { set_error("%s: x / out is NULL", fn); return KGE_E_NULL; }
    if (rows > 1 && ((out == x && ldo != ldx) || (out == residual && ldo != ldr))) {
        set_error("%s: out may be x or residual only with the same row pitch", fn); return KGE_E_SHAPE; }
    const uintptr_t m = dtype == KGE_F32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(x) & m) || (reinterpret_cast<uintptr_t>(out) & m) || (reinterpret_cast<uintptr_t>(residual) & m) ||
        (reinterpret_cast<uintptr_t>(step_dev) & 7)) { set_error("%s: a pointer is not aligned to its element size", fn); return KGE_E_ALIGN; }
    DropoutArgs a;
    a.x = x; a.res = residual; a.out = out;
    a.rows = rows; a.dim = dim; a.ldx = ldx; a.ldr = residual ? ldr : 0; a.ldo = ldo;
    a.threshold = static_cast<uint32_t>(p * 4294967296.0);      // p < 1: below 2^32; the product is exact, the cast is its floor
    a.scale = static_cast<float>(1.0 / (1.0 - p));
    a.stream = stream_id; a.step = static_cast<uint32_t>(step); a.step_dev = reinterpret_cast<const long long*>(step_dev);
    a.k0 = static_cast<uint32_t>(seed); a.k1 = static_cast<uint32_t>(seed >> 32);
    return launch_dropout(a, dtype, reinterpret_cast<cudaStream_t>(stream));
}
