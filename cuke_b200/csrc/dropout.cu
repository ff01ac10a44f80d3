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

int launch_dropout(const DropoutArgs& a, int dtype, cudaStream_t s) {
    const long long quads = (a.rows * a.dim + 3) / 4;
    const long long want = (quads + 255) / 256;
    const unsigned blocks = static_cast<unsigned>(want < 148 * 16 ? want : 148 * 16);
    if (dtype == KGE_F32) dropout_kernel<float><<<blocks, 256, 0, s>>>(a);
    else dropout_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>(a);
    KGE_LAUNCH_CHECK("dropout_kernel");
    return 0;
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
