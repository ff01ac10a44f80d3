// Rows from features: out = act(x w + b) (+ residual) and its gradient, bf16 with fp32 accumulation.
//
//   forward   z = x w + b        x (M, K), w (K, N) in the framework's matrix orientation out[j] = sum_i x[i] w[i][j]
//             out = act(z) + residual, and for training slope = act'(z) in fp16 (2^-11 relative, an eighth of a bf16
//             rounding; 2^-25 absolute below 6e-5)
//   backward  dz = dout * slope,  dx = dz w^T,  dw = x^T dz,  db = sum over rows of dz,  d(residual) = dout
//             dz is rounded to bf16, the products' operand type: their results are then off by 0.0024 of their size where the
//             rounding of the results alone gives 0.0017; db sums the unrounded values
//
// The three products run on one persistent tcgen05 kernel over CTA pairs (256-row tiles, cta_group::2): operands are
// used as they lie in memory, K-major or MN-major, so nothing is transposed; two accumulators in tensor memory let a
// tile's epilogue overlap the next tile's main loop.  Bias, activation, residual and slope are applied to the fp32
// accumulator in the epilogue, with one rounding to bf16.  dx and dw are one launch: their tiles share one list of work.
#include <string.h>
#include <atomic>
#include <cuda_fp16.h>
#include "umma.cuh"

namespace kge {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };
enum { LE_FORWARD = 0, LE_PLAIN = 1 };            // the whole forward epilogue; rounding to bf16, or fp32 shares of a split sum

constexpr int LG_BM = 128;                        // rows of a tile per CTA (a pair: 256)
constexpr int LG_BK = 64;                         // contraction per stage: one 128-byte swizzle row of bf16
constexpr int LG_A_BYTES = LG_BM * LG_BK * 2;
constexpr int LG_SLAB = LG_BK * 128;              // MN-major slab: 64 k-rows x 128 bytes
// warp 0: TMA, warp 1: MMA and tensor memory, warps 2..17: epilogue.  An epilogue is a chain of latencies (residual, tensor
// memory, bias, two special functions a value, stores): with eight warps on 32-column chunks it took 12.7 us a tile against 6 us
// of products (65536 x 1024 x 1024 with gelu, residual and slope).  Sixteen warps on 16-column chunks fit the registers.
constexpr int LG_EPI_WARPS = 16;
constexpr int LG_THREADS = 64 + 32 * LG_EPI_WARPS;
constexpr int LG_MAX_SMEM = 227 * 1024;
constexpr int LG_ACC_COLS = 256;
// An epilogue warp works on blocks of 32 rows x 32 columns, staged in shared memory as 64-byte rows: a residual block arrives by
// a tiled load, the finished block and its slope leave by tiled stores.  (Thread-per-row accesses to global memory touch 32 cache
// lines an instruction: with them residual and slope cost 50 us of 172.)  Two residual / output blocks and one slope block a warp.
constexpr int LG_BLOCK = 32 * 64;
constexpr int LG_STRIP = 32 * 4;                  // a block's bias in fp32, read by broadcast
__host__ __device__ constexpr int lin_warp_stage(bool slope) { return (slope ? 3 : 2) * LG_BLOCK; }
__host__ __device__ constexpr int lin_staging(int epi, bool slope) {
    return LG_EPI_WARPS * (lin_warp_stage(slope) + (epi == LE_FORWARD ? LG_STRIP : 0));
}
constexpr int LG_TAIL = 512;                      // barriers and the tensor-memory slot

struct LinEpilogue {
    const __nv_bfloat16* bias; const __nv_bfloat16* res; long long ldr;
    __nv_bfloat16* out; long long ldo;
    __half* slope;                                // (M, N) packed, or NULL
    int act;
};
// One product: work items are (output tile, share of the contraction), all tiles of a share before the next share.
struct LinShape {
    int m, n;                                     // output rows and columns
    int kb;                                       // stages of the whole contraction
    int bn, a_mn, b_mn, splits, tiles_m, tiles_n;
    int items;                                    // tiles x splits
    float* part;                                  // (splits, M, N) fp32 shares, where splits > 1
};
struct LinGemm {
    LinShape q[2];                                // the second one may have no items
    int items, stages, stage_bytes;
    LinEpilogue e;                                // LE_FORWARD (of q[0])
    const float* colpart; long long colblocks; __nv_bfloat16* db; int db_n;      // LE_PLAIN: db = column sums of colpart, if db
    int32_t* err;
};
struct LinMaps { CUtensorMap a[2], b[2], out[2], slope, res; };
struct LinJoin { const float* part; LinEpilogue e; long long m, groups; int n, splits; };       // groups of 8 columns; 0: nothing

// ---- elementwise pieces -------------------------------------------------------------------------------------------
__device__ __forceinline__ float lin_ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float lin_rcp(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float lin_max(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float lin_min(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }
// 1 / (1 + 2^x): 2^x overflows to +inf for large x and the reciprocal is then 0
__device__ __forceinline__ float2 lin_sigmoid2(float2 x) {
    const float2 d = __fadd2_rn(make_float2(lin_ex2(x.x), lin_ex2(x.y)), f2(1.f));
    return make_float2(lin_rcp(d.x), lin_rcp(d.y));
}

// act(z) and, with SLOPE, act'(z) of two values: the epilogue has 13 instructions a value for the tensor core not to wait for it
// (K = 1024), so additions and products are packed fp32 pairs.  gelu is the tanh form, 0.5 z (1 + tanh u) = z s(2 u),
// u = sqrt(2 / pi) (z + 0.044715 z^3).  Far from the origin s rounds to 0 or 1; clamping z there (below at -3e4 for all, above at
// 3e4 for the slope alone) keeps 0 x infinity out of the products and leaves every result as it is; NaN goes through.
template <int ACT, bool SLOPE>
__device__ __forceinline__ float2 lin_act(float2 z, float2& slope) {
    if (ACT == ACT_NONE) { if (SLOPE) slope = f2(1.f); return z; }
    if (ACT == ACT_RELU) {
        if (SLOPE) slope = make_float2(z.x > 0.f ? 1.f : 0.f, z.y > 0.f ? 1.f : 0.f);
        return make_float2(lin_max(z.x, 0.f), lin_max(z.y, 0.f));
    }
    const float lim = 3e4f;
    z = make_float2(lin_max(z.x, -lim), lin_max(z.y, -lim));
    if (ACT == ACT_SILU) {
        const float2 s = lin_sigmoid2(__fmul2_rn(z, f2(-1.4426950408889634f)));
        if (SLOPE) {
            const float2 zc = make_float2(lin_min(z.x, lim), lin_min(z.y, lim));
            slope = __ffma2_rn(__fmul2_rn(zc, s), __ffma2_rn(s, f2(-1.f), f2(1.f)), s);
        }
        return __fmul2_rn(z, s);
    }
    const float c = 1.5957691216057308f, l = -1.4426950408889634f * c;          // 2 sqrt(2 / pi), and times -log2 e
    const float2 zc = make_float2(lin_min(z.x, lim), lin_min(z.y, lim));
    const float2 z2 = __fmul2_rn(zc, zc);
    const float2 s = lin_sigmoid2(__fmul2_rn(zc, __ffma2_rn(z2, f2(0.044715f * l), f2(l))));
    if (SLOPE) {
        const float2 t = __fmul2_rn(__fmul2_rn(zc, s), __ffma2_rn(s, f2(-1.f), f2(1.f)));
        slope = __ffma2_rn(t, __ffma2_rn(z2, f2(3.f * 0.044715f * c), f2(c)), s);
    }
    return __fmul2_rn(z, s);
}
__device__ __forceinline__ uint32_t lin_bf2(float a, float b) {
    __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t lin_h2(float a, float b) {
    __half2 p = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&p);
}
__device__ __forceinline__ float lin_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float lin_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

__device__ __forceinline__ void lin_st8(void* p, const uint32_t* w) {      // 32 bytes, 32-byte aligned
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
// 16 consecutive columns of one output row: fp32 sums in v -> bias, activation, residual -> bf16 row and fp16 slope
template <int ACT, bool SLOPE>
__device__ __forceinline__ void lin_apply(const float (&v)[16], const float4* bias, const uint32_t (&res)[8], uint32_t (&out)[8], uint32_t (&slope)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float4 b = bias[i / 2];
        float2 g0, g1;
        float2 y0 = lin_act<ACT, SLOPE>(__fadd2_rn(make_float2(v[2 * i], v[2 * i + 1]), make_float2(b.x, b.y)), g0);
        float2 y1 = lin_act<ACT, SLOPE>(__fadd2_rn(make_float2(v[2 * i + 2], v[2 * i + 3]), make_float2(b.z, b.w)), g1);
        y0 = __fadd2_rn(y0, make_float2(lin_lo(res[i]), lin_hi(res[i])));
        y1 = __fadd2_rn(y1, make_float2(lin_lo(res[i + 1]), lin_hi(res[i + 1])));
        out[i] = lin_bf2(y0.x, y0.y);
        out[i + 1] = lin_bf2(y1.x, y1.y);
        if (SLOPE) { slope[i] = lin_h2(g0.x, g0.y); slope[i + 1] = lin_h2(g1.x, g1.y); }
    }
}
// tiled store of a staged block, and its bookkeeping (one thread of a warp issues and waits)
__device__ __forceinline__ void lin_store_block(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
                 ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
}
__device__ __forceinline__ void lin_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void lin_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }     // the staged bytes have been read
__device__ __forceinline__ void lin_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// 32 lanes x 16 consecutive fp32 columns of tensor memory, complete on return
__device__ __forceinline__ void lin_tmem16(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// Arrives on the barrier at `bar` (same offset) of both CTAs of the pair once all MMAs issued so far have completed.
__device__ __forceinline__ void lin_commit_both(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}
__device__ __forceinline__ void lin_epilogue_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(32 * LG_EPI_WARPS) : "memory"); }
// One lane of the (converged) warp.
__device__ __forceinline__ bool lin_elect() {
    uint32_t is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
    return is != 0;
}
// Bounded wait by a whole warp on the barrier at a shared address; false = gave up.
__device__ __forceinline__ bool lin_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .u32 n;\n\t"
        "mov.u32 n, %3;\n"
        "WAIT:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "@p bra DONE;\n\t"
        "sub.u32 n, n, 1;\n\t"
        "setp.eq.u32 p, n, 0;\n\t"
        "@!p bra WAIT;\n\t"
        "setp.ne.u32 p, n, n;\n"
        "DONE:\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity), "n"(1 << 22) : "memory");
    return __all_sync(kFull, ok != 0) != 0;
}
// Arrival that hands nothing over but tensor memory, whose reads have completed (wait::ld) and are fenced by the caller: the
// releasing form waits for the warp's stores and copies too, 2500 cycles in the middle of a tile's epilogue.
__device__ __forceinline__ void lin_arrive_relaxed(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void lin_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void lin_tma_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t leader_bar) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(0), "r"(leader_bar) : "memory");
}
// ---- the product ----------------------------------------------------------------------------------------------------
// Items run over the column tiles first, so the pairs working at one time read the same rows of A.  Pair p takes items p,
// p + pairs, ... of q[0] and then q[1].
template <int EPI, int ACT, bool SLOPE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(LG_THREADS, 1)
linear_pair_kernel(const __grid_constant__ LinMaps maps, const __grid_constant__ LinGemm p) {
    extern __shared__ __align__(1024) uint8_t smem[];              // swizzle atoms start on 1024-byte boundaries; no room to round up
    if ((umma::smem_u32(smem) & 1023u) != 0) {                     // (every thread of both CTAs leaves: the launch reports itself)
        if (threadIdx.x == 0) atomicOr(p.err, KGE_ERR_WAIT_TIMEOUT);
        return;
    }
    const int stage_bytes = p.stage_bytes;
    uint8_t* staging = smem + p.stages * stage_bytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + lin_staging(EPI, SLOPE));
    uint64_t* empty = full + p.stages;
    uint64_t* acc_full = empty + p.stages;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* res_full = acc_empty + 2;                            // two per epilogue warp: its residual blocks
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(res_full + 2 * LG_EPI_WARPS);

    // (a shuffle makes the warp number uniform for the compiler too: see the producer)
    const int warp = __shfl_sync(kFull, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t rank = umma::cluster_ctarank();
    const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const int items = p.items;
    auto which = [&](int item) { return EPI == LE_PLAIN && item >= p.q[0].items ? 1 : 0; };

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) { umma::mbar_init(&full[s], 1); umma::mbar_init(&empty[s], 1); }
        for (int s = 0; s < 2; ++s) { umma::mbar_init(&acc_full[s], 1); umma::mbar_init(&acc_empty[s], 2 * LG_EPI_WARPS); }
        for (int s = 0; s < 2 * LG_EPI_WARPS; ++s) umma::mbar_init(&res_full[s], 1);
        umma::fence_barrier_init();
    }
    if (warp == 1) { umma::tmem_alloc_pair(tmem_slot, 2 * LG_ACC_COLS); umma::tmem_relinquish_pair(); }
    umma::tc_fence_before();
    __syncthreads();
    umma::cluster_sync();
    umma::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    let_next_start();
    after_previous();

    const uint32_t smem0 = umma::smem_u32(smem), full0 = umma::smem_u32(full), empty0 = umma::smem_u32(empty);
    const uint32_t acc_full0 = umma::smem_u32(acc_full), acc_empty0 = umma::smem_u32(acc_empty);
    if (warp == 0) {
        // TMA producer.  The whole warp runs the loop and one elected lane issues: inside a branch on the lane the compiler has no
        // uniform registers, every copy and MMA gets its operands through moves, and a stage took its threads 650 cycles where
        // the MMAs take 512.
        const bool elected = lin_elect();
        if (elected) { umma::prefetch_tensormap(&maps.a[0]); umma::prefetch_tensormap(&maps.b[0]); }
        const uint32_t lead0 = umma::map_to_cta(full0, 0);          // the leader's `full` barriers count the bytes of both CTAs
        int s = 0; uint32_t ph = 0;
        bool ok = true;
        for (int item = pair; item < items && ok; item += n_pairs) {
            const int w = which(item);
            const LinShape& q = p.q[w];
            const int half_n = q.bn / 2;                            // B columns staged by each CTA
            const int b_slabs = (half_n + 63) / 64;
            const uint32_t tx_pair = 2u * (LG_A_BYTES + (q.b_mn ? b_slabs * LG_SLAB : half_n * 128));
            const CUtensorMap *map_a = &maps.a[w], *map_b = &maps.b[w];
            const int mine = item - (w ? p.q[0].items : 0), tiles = q.tiles_m * q.tiles_n;
            const int split = mine / tiles, tile = mine - split * tiles;
            const int tm = tile / q.tiles_n;
            const int m0 = tm * 2 * LG_BM + static_cast<int>(rank) * LG_BM;
            const int nb0 = (tile - tm * q.tiles_n) * q.bn + static_cast<int>(rank) * half_n;
            const int kb0 = static_cast<int>(static_cast<long long>(q.kb) * split / q.splits);
            const int kb1 = static_cast<int>(static_cast<long long>(q.kb) * (split + 1) / q.splits);
            const bool a_mn = q.a_mn != 0, b_mn = q.b_mn != 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = lin_wait(empty0 + 8 * s, ph ^ 1);
                if (!ok) break;
                if (elected) {
                    const uint32_t a = smem0 + s * stage_bytes, b = a + LG_A_BYTES, lead = lead0 + 8 * s;
                    if (rank == 0) lin_expect_tx(full0 + 8 * s, tx_pair);
                    const int k0 = kb * LG_BK;
                    if (!a_mn) {
                        lin_tma_pair(a, map_a, k0, m0, lead);
                    } else {
                        lin_tma_pair(a, map_a, m0, k0, lead);
                        lin_tma_pair(a + LG_SLAB, map_a, m0 + 64, k0, lead);
                    }
                    if (!b_mn) {
                        lin_tma_pair(b, map_b, k0, nb0, lead);
                    } else {
                        lin_tma_pair(b, map_b, nb0, k0, lead);
                        if (b_slabs > 1) lin_tma_pair(b + LG_SLAB, map_b, nb0 + 64, k0, lead);
                    }
                }
                __syncwarp();
                if (++s == p.stages) { s = 0; ph ^= 1; }
            }
        }
        for (int i = 0; i < p.stages && ok; ++i) {                  // every commit aimed at this CTA has landed before it may exit
            ok = lin_wait(empty0 + 8 * s, ph ^ 1);
            if (++s == p.stages) { s = 0; ph ^= 1; }
        }
        if (!ok && lane == 0) atomicOr(p.err, KGE_ERR_WAIT_TIMEOUT);
    } else if (warp == 1) {
        if (rank == 0) {
            const bool elected = lin_elect();
            int s = 0, lt = 0; uint32_t ph = 0;
            bool ok = true;
            for (int item = pair; item < items && ok; item += n_pairs, ++lt) {
                const int w = which(item);
                const LinShape& q = p.q[w];
                const uint64_t a_tmpl = q.a_mn ? umma::smem_desc_mn(0, LG_SLAB, 1024u, 2u) : umma::smem_desc_k_sw128(0);
                const uint64_t b_tmpl = q.b_mn ? umma::smem_desc_mn(0, LG_SLAB, 1024u, 2u) : umma::smem_desc_k_sw128(0);
                const uint32_t a_step = (q.a_mn ? 2048u : 32u) >> 4, b_step = (q.b_mn ? 2048u : 32u) >> 4;
                const uint32_t idesc = umma::instr_desc(1u, 2 * LG_BM, static_cast<uint32_t>(q.bn), static_cast<uint32_t>(q.a_mn), static_cast<uint32_t>(q.b_mn));
                const int split = (item - (w ? p.q[0].items : 0)) / (q.tiles_m * q.tiles_n);
                const int nkb = static_cast<int>(static_cast<long long>(q.kb) * (split + 1) / q.splits) -
                                static_cast<int>(static_cast<long long>(q.kb) * split / q.splits);
                const int buf = lt & 1;
                ok = lin_wait(acc_empty0 + 8 * buf, (static_cast<uint32_t>(lt >> 1) & 1) ^ 1);
                if (!ok) break;
                umma::tc_fence_after();
                const uint32_t tmem_d = tmem_base + buf * LG_ACC_COLS;
                for (int kb = 0; kb < nkb; ++kb) {
                    ok = lin_wait(full0 + 8 * s, ph);
                    if (!ok) break;
                    const uint32_t st = ((smem0 + s * stage_bytes) & 0x3FFFFu) >> 4;
                    const uint64_t da = a_tmpl | st, db = b_tmpl | (st + (LG_A_BYTES >> 4));
                    if (elected) {
                        umma::mma_f16_pair(tmem_d, da, db, idesc, kb > 0 ? 1u : 0u);
                        umma::mma_f16_pair(tmem_d, da + a_step, db + b_step, idesc, 1u);
                        umma::mma_f16_pair(tmem_d, da + 2 * a_step, db + 2 * b_step, idesc, 1u);
                        umma::mma_f16_pair(tmem_d, da + 3 * a_step, db + 3 * b_step, idesc, 1u);
                        lin_commit_both(empty0 + 8 * s);
                    }
                    __syncwarp();
                    if (++s == p.stages) { s = 0; ph ^= 1; }
                }
                if (elected) lin_commit_both(acc_full0 + 8 * buf);
                __syncwarp();
            }
            if (!ok && lane == 0) atomicOr(p.err, KGE_ERR_WAIT_TIMEOUT);
        }
    } else {
        // thread = row of a block; the four warps of a lane quarter take the 32-column blocks of their rows in turn
        const int sub = warp & 3, part = (warp - 2) >> 2;
        uint8_t* mine = staging + (warp - 2) * lin_warp_stage(SLOPE);
        uint64_t* res_bar = res_full + 2 * (warp - 2);
        const bool has_res = EPI == LE_FORWARD && p.e.res != nullptr;
        const uint32_t swz = static_cast<uint32_t>(lane >> 1) & 3u;               // 64-byte swizzle: 16-byte piece c of row `lane` lies at c ^ swz
        float* strip = reinterpret_cast<float*>(staging + LG_EPI_WARPS * lin_warp_stage(SLOPE)) + 32 * (warp - 2);
        const uint32_t out_addr = umma::smem_u32(mine);
        const int row_in = static_cast<int>(rank) * LG_BM + sub * 32;
        if (EPI == LE_PLAIN && p.db != nullptr) {
            // db[c] = sum of its partial sums in a fixed order (16 interleaved sums a column, in fp64: each has a million terms at 2^30
            // rows), while the first tiles are multiplied: a kernel of its own took 3 us of the 8191 x 1024 x 400 backward pass
            float* red = reinterpret_cast<float*>(staging);                       // 16 x 33: nothing is staged yet
            for (int c0 = blockIdx.x * 32; c0 < p.db_n; c0 += gridDim.x * 32) {
                const int c = c0 + lane;
                double wide = 0.0;
                if (c < p.db_n) {
#pragma unroll 8
                    for (long long b = warp - 2; b < p.colblocks; b += LG_EPI_WARPS) wide += static_cast<double>(p.colpart[b * p.db_n + c]);
                }
                float t = static_cast<float>(wide);
                red[(warp - 2) * 33 + lane] = t;
                lin_epilogue_barrier();
                if (warp == 2 && c < p.db_n) {
                    for (int w = 1; w < LG_EPI_WARPS; ++w) t += red[w * 33 + lane];
                    p.db[c] = __float2bfloat16_rn(t);
                }
                lin_epilogue_barrier();
            }
        }
        int lt = 0, b = 0;
        uint32_t res_phase = 0, pending = 0;                                      // bit b: parity of buffer b's next load; a load is under way
        float bias_next = 0.f;
        // what the block at (row, col) needs from memory: its residual into buffer b, its bias into a register (whole warp calls)
        auto fetch = [&](bool exists, int row, int col, int b) {
            if (EPI != LE_FORWARD) return;
            bias_next = exists && p.e.bias != nullptr && col + lane < p.q[0].n ? __bfloat162float(p.e.bias[col + lane]) : 0.f;
            if (!has_res || !exists || row >= p.q[0].m || col >= p.q[0].n) return;
            pending |= 1u << b;
            if (lane == 0) {
                umma::mbar_expect_tx(&res_bar[b], LG_BLOCK);
                umma::tma_load_2d(mine + b * LG_BLOCK, &maps.res, col, row, &res_bar[b]);
            }
            __syncwarp();
        };
        // LE_FORWARD: coordinates of this tile and the next, kept by addition
        const int step_m = n_pairs / p.q[0].tiles_n, step_n = n_pairs - step_m * p.q[0].tiles_n;
        int tm = pair / p.q[0].tiles_n, tn = pair - tm * p.q[0].tiles_n;
        fetch(pair < items && part < (p.q[0].bn + 31) / 32, tm * 2 * LG_BM + row_in, tn * p.q[0].bn + part * 32, 0);
        for (int item = pair; item < items; item += n_pairs, ++lt) {
            const int w = which(item);
            const LinShape& q = p.q[w];
            const int qm = q.m, qn = q.n, bn = q.bn, blocks = (bn + 31) / 32;
            int tm_next = tm + step_m, tn_next = tn + step_n, split = 0;
            if (EPI == LE_FORWARD) {
                if (tn_next >= q.tiles_n) { tn_next -= q.tiles_n; ++tm_next; }
            } else {
                const int at = item - (w ? p.q[0].items : 0), tiles = q.tiles_m * q.tiles_n;
                split = at / tiles;
                tm = (at - split * tiles) / q.tiles_n;
                tn = at - split * tiles - tm * q.tiles_n;
            }
            const bool shares = EPI == LE_PLAIN && q.splits > 1;
            const int row = tm * 2 * LG_BM + row_in;
            const int buf = lt & 1;
            const uint32_t taddr = tmem_base + buf * LG_ACC_COLS + (static_cast<uint32_t>(sub * 32) << 16);
            bool ready = false;
            auto wait_full = [&]() { return lin_wait(acc_full0 + 8 * buf, static_cast<uint32_t>(lt >> 1) & 1); };
            auto drained = [&]() {                                                // this warp is done with the accumulator
                umma::tc_fence_before();
                __syncwarp();
                if (lane == 0) lin_arrive_relaxed(umma::map_to_cta(acc_empty0 + 8 * buf, 0));
            };
            bool ok = true;
#pragma unroll 1
            for (int blk = part; blk < blocks; blk += 4, b ^= 1) {
                const int col = tn * bn + blk * 32;
                const bool live = row < qm && col < qn;                         // something of the block exists
                const bool last = blk + 4 >= blocks;
                if (EPI == LE_FORWARD) {
                    strip[lane] = bias_next;
                    if (has_res && live) {
                        ok = lin_wait(umma::smem_u32(&res_bar[b]), (res_phase >> b) & 1u);
                        if (!ok) break;
                        res_phase ^= 1u << b;
                        pending &= ~(1u << b);
                    }
                }
                if (!ready) {
                    ready = ok = wait_full();
                    if (!ready) break;
                    umma::tc_fence_after();
                }
                __syncwarp();                     // the strip is written; tensor-memory reads are warp-collective
                uint8_t* rows = mine + b * LG_BLOCK + lane * 64;
                uint8_t* srow = mine + 2 * LG_BLOCK + lane * 64;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[16];
                    lin_tmem16(taddr + blk * 32 + h * 16, v);
                    if (last && h == 1) drained();
                    if (shares) {
                        const int lim = live && row + lane < qm && blk * 32 + h * 16 < bn ? qn - (col + h * 16) : 0;
                        float* d = q.part + (static_cast<long long>(split) * qm + row + lane) * qn + col + h * 16;
                        if (lim > 0) lin_st8(d, reinterpret_cast<const uint32_t*>(v));
                        if (lim > 8) lin_st8(d + 8, reinterpret_cast<const uint32_t*>(v) + 8);
                        __syncwarp();
                        continue;
                    }
                    uint4* p0 = reinterpret_cast<uint4*>(rows + (((2 * h) ^ swz) << 4));
                    uint4* p1 = reinterpret_cast<uint4*>(rows + (((2 * h + 1) ^ swz) << 4));
                    uint32_t w[8];
                    if (EPI == LE_FORWARD) {
                        uint32_t res[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u}, sl[8];
                        if (has_res) {            // (a block that does not exist reads what lies there and is not stored)
                            const uint4 r0 = *p0, r1 = *p1;
                            res[0] = r0.x; res[1] = r0.y; res[2] = r0.z; res[3] = r0.w; res[4] = r1.x; res[5] = r1.y; res[6] = r1.z; res[7] = r1.w;
                        }
                        lin_apply<ACT, SLOPE>(v, reinterpret_cast<const float4*>(strip) + 4 * h, res, w, sl);
                        if (h == 0) {             // the last block's copies have been read by now: its buffers take the next block
                            if (lane == 0) lin_wait_read();
                            __syncwarp();
                            if (last) fetch(item + n_pairs < items, tm_next * 2 * LG_BM + row_in, tn_next * bn + part * 32, b ^ 1);
                            else fetch(true, row, col + 128, b ^ 1);
                        }
                        if (SLOPE) {
                            *reinterpret_cast<uint4*>(srow + (((2 * h) ^ swz) << 4)) = make_uint4(sl[0], sl[1], sl[2], sl[3]);
                            *reinterpret_cast<uint4*>(srow + (((2 * h + 1) ^ swz) << 4)) = make_uint4(sl[4], sl[5], sl[6], sl[7]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) w[i] = lin_bf2(v[2 * i], v[2 * i + 1]);
                        if (h == 0) {
                            if (lane == 0) lin_wait_read();
                            __syncwarp();
                        }
                    }
                    *p0 = make_uint4(w[0], w[1], w[2], w[3]);
                    *p1 = make_uint4(w[4], w[5], w[6], w[7]);
                }
                if (!shares) {
                    umma::fence_proxy_async();                                    // the staged block is visible to the copy engine
                    __syncwarp();
                    if (lane == 0 && live) {                                      // (rows and columns past the end are not written)
                        lin_store_block(&maps.out[w], out_addr + b * LG_BLOCK, col, row);
                        if (SLOPE) lin_store_block(&maps.slope, out_addr + 2 * LG_BLOCK, col, row);
                        lin_commit();
                    }
                }
                __syncwarp();
            }
            if (part >= blocks) {                                                 // a warp without a block only keeps step
                ok = wait_full();
                drained();
            }
            if (!ok) {
                if (lane == 0) atomicOr(p.err, KGE_ERR_WAIT_TIMEOUT);
                break;
            }
            tm = tm_next; tn = tn_next;
        }
        for (int i = 0; i < 2; ++i)                                               // only after a wait ran out: copies still under way
            if ((pending >> i) & 1u) umma::mbar_wait(&res_bar[i], (res_phase >> i) & 1u);
        if (lane == 0) lin_wait_all();
    }
    umma::tc_fence_before();
    __syncthreads();
    umma::cluster_sync();
    if (warp == 1) { umma::tc_fence_after(); umma::tmem_dealloc_pair(tmem_base, 2 * LG_ACC_COLS); }
}

// Sums of the shares of up to two split products in a fixed order, then the epilogue.  8 columns per group of LANES threads, which
// take the shares in turn: with one thread a group, 64 shares of a 128 x 128 gradient were a chain of 64 loads (11 us).
template <int EPI, int LANES>
__global__ void __launch_bounds__(256) linear_join_kernel(const __grid_constant__ LinJoin j0, const __grid_constant__ LinJoin j1) {
    let_next_start();
    after_previous();
    const long long total = j0.groups + j1.groups;
    const int sub = threadIdx.x % LANES;
    for (long long first = (long long)blockIdx.x * (256 / LANES); first < total; first += (long long)gridDim.x * (256 / LANES)) {
        const bool live = first + threadIdx.x / LANES < total;                  // (all lanes take part in the shuffles)
        const long long i = live ? first + threadIdx.x / LANES : total - 1;
        const bool second = EPI == LE_PLAIN && i >= j0.groups;
        const LinJoin& j = second ? j1 : j0;
        const long long at = second ? i - j0.groups : i, m = j.m;
        const LinEpilogue& e = j.e;
        const int n = j.n, per_row = n / 8, splits = j.splits;
        const long long row = at / per_row;
        const int col = static_cast<int>(at - row * per_row) * 8;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int s = sub; s < splits; s += LANES) {
            const float4* d = reinterpret_cast<const float4*>(j.part + (static_cast<long long>(s) * m + row) * n + col);
            const float4 a = __ldcs(d), b = __ldcs(d + 1);
            v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w; v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
        }
        if (LANES > 1) {
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1)
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] += __shfl_xor_sync(kFull, v[k], o);
        }
        if (!live || sub != 0) continue;
        if (EPI == LE_FORWARD) {
            uint4 bias = make_uint4(0u, 0u, 0u, 0u), res = bias;
            if (e.bias) bias = __ldg(reinterpret_cast<const uint4*>(e.bias + col));
            if (e.res) res = *reinterpret_cast<const uint4*>(e.res + row * e.ldr + col);
            const uint32_t bw[4] = {bias.x, bias.y, bias.z, bias.w}, rw[4] = {res.x, res.y, res.z, res.w};
            uint32_t sl[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float2 g, y;
                const float2 z = make_float2(v[2 * k] + lin_lo(bw[k]), v[2 * k + 1] + lin_hi(bw[k]));
                switch (e.act) {
                    case ACT_NONE: y = lin_act<ACT_NONE, true>(z, g); break;
                    case ACT_RELU: y = lin_act<ACT_RELU, true>(z, g); break;
                    case ACT_SILU: y = lin_act<ACT_SILU, true>(z, g); break;
                    default: y = lin_act<ACT_GELU, true>(z, g); break;
                }
                v[2 * k] = y.x + lin_lo(rw[k]); v[2 * k + 1] = y.y + lin_hi(rw[k]);
                sl[k] = lin_h2(g.x, g.y);
            }
            if (e.slope) *reinterpret_cast<uint4*>(e.slope + row * n + col) = make_uint4(sl[0], sl[1], sl[2], sl[3]);
        }
        *reinterpret_cast<uint4*>(e.out + row * e.ldo + col) =
            make_uint4(lin_bf2(v[0], v[1]), lin_bf2(v[2], v[3]), lin_bf2(v[4], v[5]), lin_bf2(v[6], v[7]));
    }
}

// ---- few rows ------------------------------------------------------------------------------------------------------------
// Up to 8 rows (one entity while serving): bound by reading w once, so w streams past fp32 registers instead of filling a
// 128-row tensor tile.  A CTA has 32 columns (4 lanes of 8 columns, 64-byte pieces of a w row) and a share of K: 8 warps x 8 rows
// of w at a time.  A cluster's CTAs share the columns and sum up over distributed shared memory in rank order.
// One row, K = 1024, N = 512: 4.2 us, against 10.3 us for the split tensor product and its join.
constexpr int LF_ROWS = 8;                        // rows of x, at most
constexpr int LF_KC = 512;                        // k-values of x staged at a time
template <int M>
__global__ void __launch_bounds__(256) linear_few_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, const __nv_bfloat16* __restrict__ w,
                                                         long long ldw, int m, int k, int n, LinEpilogue e) {
    __shared__ float xs[M][LF_KC];
    __shared__ float part[8][M][32];
    __shared__ float sum[M][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t rank, csize;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(csize));
    const int n0 = static_cast<int>(blockIdx.x / csize) * 32, col = n0 + (lane & 3) * 8;
    const int k_lo = static_cast<int>(static_cast<long long>(k) * rank / csize), k_hi = static_cast<int>(static_cast<long long>(k) * (rank + 1) / csize);
    float2 acc[M][4];
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f2(0.f);
    for (int kc = k_lo; kc < k_hi; kc += LF_KC) {
        const int len = min(LF_KC, k_hi - kc);
        for (int i = tid; i < M * LF_KC; i += 256) {
            const int r = i / LF_KC, c = i % LF_KC;
            if (c < len) xs[r][c] = r < m ? __bfloat162float(x[r * ldx + kc + c]) : 0.f;
        }
        __syncthreads();
        if (col < n) {
            const int first = warp * 8 + (lane >> 2);
            for (int c0 = first; c0 < len; c0 += 256) {
                uint4 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    v[u] = make_uint4(0u, 0u, 0u, 0u);
                    if (c0 + 64 * u < len) v[u] = __ldg(reinterpret_cast<const uint4*>(w + (kc + c0 + 64 * u) * ldw + col));
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (c0 + 64 * u >= len) continue;
                    const uint32_t ww[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
                    for (int i = 0; i < M; ++i) {
                        const float2 xi = f2(xs[i][c0 + 64 * u]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[i][j] = __ffma2_rn(xi, make_float2(lin_lo(ww[j]), lin_hi(ww[j])), acc[i][j]);
                    }
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                acc[i][j].x += __shfl_xor_sync(kFull, acc[i][j].x, o);
                acc[i][j].y += __shfl_xor_sync(kFull, acc[i][j].y, o);
            }
            if (lane < 4) {
                part[warp][i][lane * 8 + 2 * j] = acc[i][j].x;
                part[warp][i][lane * 8 + 2 * j + 1] = acc[i][j].y;
            }
        }
    __syncthreads();
    for (int i = tid; i < M * 32; i += 256) {
        float t = 0.f;
#pragma unroll
        for (int v = 0; v < 8; ++v) t += part[v][i / 32][i % 32];
        sum[i / 32][i % 32] = t;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    // pairs of columns, dealt out over the CTAs of the cluster
    for (int i = static_cast<int>(rank) * 256 + tid; i < M * 16; i += static_cast<int>(csize) * 256) {
        const int r = i / 16, c = (i % 16) * 2;
        if (r >= m || n0 + c >= n) continue;
        float2 z = f2(0.f), g, y;
        const uint32_t addr = umma::smem_u32(&sum[r][c]);
        for (uint32_t q = 0; q < csize; ++q) {
            float2 o;
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(o.x), "=f"(o.y) : "r"(umma::map_to_cta(addr, q)) : "memory");
            z.x += o.x; z.y += o.y;
        }
        if (e.bias) {
            const uint32_t b = *reinterpret_cast<const uint32_t*>(e.bias + n0 + c);
            z.x += lin_lo(b); z.y += lin_hi(b);
        }
        switch (e.act) {
            case ACT_NONE: y = lin_act<ACT_NONE, true>(z, g); break;
            case ACT_RELU: y = lin_act<ACT_RELU, true>(z, g); break;
            case ACT_SILU: y = lin_act<ACT_SILU, true>(z, g); break;
            default: y = lin_act<ACT_GELU, true>(z, g); break;
        }
        if (e.res) {
            const uint32_t v = *reinterpret_cast<const uint32_t*>(e.res + r * e.ldr + n0 + c);
            y.x += lin_lo(v); y.y += lin_hi(v);
        }
        *reinterpret_cast<uint32_t*>(e.out + r * e.ldo + n0 + c) = lin_bf2(y.x, y.y);
        if (e.slope) *reinterpret_cast<uint32_t*>(e.slope + static_cast<long long>(r) * n + n0 + c) = lin_h2(g.x, g.y);
    }
    // no CTA leaves while another may still read its sums
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// dz = dout * slope (skipped when slope is NULL: dz is dout itself) and the column sums of dz per block of LZ_ROWS rows.
// A warp has 4 rows of a strip of 256 columns (8 per lane), all requested before the first is used; strips of the same rows
// follow one another, so whole rows leave and arrive together.
constexpr int LZ_ROWS = 64;
__global__ void __launch_bounds__(512) linear_dz_kernel(const __nv_bfloat16* __restrict__ dout, long long ldd, const __half* __restrict__ slope,
                                                        __nv_bfloat16* __restrict__ dz, long long ldz, float* __restrict__ colpart, long long m,
                                                        int n, unsigned strips) {
    constexpr int W = 16, R = LZ_ROWS / W;
    let_next_start();
    __shared__ __align__(16) float red[W][256];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long block = blockIdx.x / strips;
    const int c0 = static_cast<int>(blockIdx.x - block * strips) * 256, col = c0 + lane * 8;
    const long long r0 = block * LZ_ROWS + warp;
    float2 sum[4] = {f2(0.f), f2(0.f), f2(0.f), f2(0.f)};
    if (col < n) {
        uint4 d[R], g[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const long long r = r0 + i * W;
            d[i] = g[i] = make_uint4(0u, 0u, 0u, 0u);
            if (r < m) {
                d[i] = __ldcs(reinterpret_cast<const uint4*>(dout + r * ldd + col));
                if (slope) g[i] = __ldcs(reinterpret_cast<const uint4*>(slope + r * n + col));
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const long long r = r0 + i * W;
            const uint32_t dw[4] = {d[i].x, d[i].y, d[i].z, d[i].w}, gw[4] = {g[i].x, g[i].y, g[i].z, g[i].w};
            uint32_t o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float2 v = make_float2(lin_lo(dw[k]), lin_hi(dw[k]));
                if (slope) v = __fmul2_rn(v, __half22float2(*reinterpret_cast<const __half2*>(&gw[k])));
                o[k] = lin_bf2(v.x, v.y);
                sum[k] = __fadd2_rn(sum[k], v);
            }
            if (slope && r < m) *reinterpret_cast<uint4*>(dz + r * ldz + col) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
    if (!colpart) return;
    float4* mine = reinterpret_cast<float4*>(&red[warp][lane * 8]);
    mine[0] = make_float4(sum[0].x, sum[0].y, sum[1].x, sum[1].y);
    mine[1] = make_float4(sum[2].x, sum[2].y, sum[3].x, sum[3].y);
    __syncthreads();
    const int c = c0 + threadIdx.x;
    if (threadIdx.x < 256 && c < n) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) t += red[w][threadIdx.x];
        colpart[block * n + c] = t;
    }
}
// ---- host -----------------------------------------------------------------------------------------------------------
static int lin_sms() {
    static std::atomic<int> known[128];              // by device
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 128 && (sms = known[dev].load(std::memory_order_relaxed)) > 0) return sms;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 2) {
        cudaGetLastError();
        return 148;
    }
    if (dev >= 0 && dev < 128) known[dev].store(sms, std::memory_order_relaxed);
    return sms;
}
// Columns of a tile when n columns are cut into so many: whole 32-column blocks, or one tile in units of 16.
static int lin_bn(long long n, long long tiles) {
    const long long unit = tiles > 1 ? 32 : 16;
    return static_cast<int>(((n + tiles - 1) / tiles + unit - 1) / unit * unit);
}
constexpr int LIN_MAX_SPLITS = 64;
struct LinDim { long long m, n, k; };       // out (m, n), contraction k
struct LinPlan { int bn[2], splits[2]; };
// Tile widths and shares of the contractions of the products of one launch (one, or dx and dw): the choice with the least estimated
// time.  Widths: the fewest tiles of at most 256 columns, or two or four times as many (64 columns and more) while pairs would be idle.
// Shares: 1, and what fills the pairs half, once or twice.  The first pair of each kind of load is followed through its items
// (longest items first): 0.2 us + 0.2 us per 256 columns for a stage, 1 us for an item; the join 2.5 us and its traffic at 6 TB/s.
// 4000 x 1024 x 512 with gelu, residual and slope: 10.9 us in tiles of 128 columns, 14.0 us of 256; backward 16.5 us of 256,
// 19.6 us of 64.  16 x 2048 x 2048: 9.8 us in 9 shares of 256 columns, 12.9 us in tiles of 64.
static LinPlan lin_plan(const LinDim* d, int count, int sms) {
    const int slots = sms / 2;
    struct Option { double item, join; long long items; int bn, splits; } opt[2][16];
    int n_opt[2] = {0, 0};
    for (int i = 0; i < count; ++i) {
        const long long rows = (d[i].m + 255) / 256, kb = (d[i].k + 63) / 64, least = (d[i].n + 255) / 256;
        for (int times = 1; times <= 4; times *= 2) {
            const long long cols = least * times, tiles = rows * cols;
            if (times > 1 && (cols * 64 > d[i].n + 63 || tiles > slots)) break;
            const int bn = lin_bn(d[i].n, cols);
            long long last = 0;
            for (int half = 0; half <= 4; half = half ? 2 * half : 1) {
                long long s = half ? slots * half / (2 * tiles) : 1;
                s = s < LIN_MAX_SPLITS ? s : LIN_MAX_SPLITS;
                s = s < kb ? s : kb;
                if (s <= last) continue;
                last = s;
                Option& o = opt[i][n_opt[i]++];
                o.bn = bn;
                o.splits = static_cast<int>(s);
                o.item = (0.2 + 0.2 / 256 * bn) * static_cast<double>((kb + s - 1) / s) + 1.0;
                o.join = s > 1 ? 8.0 / 6.0e6 * static_cast<double>(s * d[i].m * d[i].n) : 0.0;
                o.items = tiles * s;
            }
        }
    }
    if (count < 2) opt[1][n_opt[1]++] = {1.0, 0.0, 0, 0, 1};
    LinPlan best = {};
    double least = -1.0;
    for (int a = 0; a < n_opt[0]; ++a)
        for (int b = 0; b < n_opt[1]; ++b) {
            const Option &x = opt[0][a], &y = opt[1][b];
            const Option &lead = y.item > x.item ? y : x, &rest = y.item > x.item ? x : y;
            double t = 0.0;
            for (long long p : {0LL, lead.items % slots}) {
                const long long all = (lead.items + rest.items - p + slots - 1) / slots, longer = (lead.items - p + slots - 1) / slots;
                const double mine = longer * lead.item + (all - longer) * rest.item;
                if (mine > t) t = mine;
            }
            if (x.join + y.join > 0.0) t += x.join + y.join + 2.5;
            if (least < 0.0 || t < least) { least = t; best = {{x.bn, y.bn}, {x.splits, y.splits}}; }
        }
    return best;
}
// dz rows start on 128-byte lines, as the tiled loads read them: backward of 53333 x 520 x 696 123 us, with packed rows 145 us.
static long long lin_dz_pitch(long long n) { return (n + 63) & ~63LL; }
static size_t lin_up(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }
static size_t lin_dz_bytes(long long m, long long n, int act) { return act != ACT_NONE ? lin_up(2 * static_cast<size_t>(m) * lin_dz_pitch(n)) : 0; }
static size_t lin_col_bytes(long long m, long long n) { return lin_up(sizeof(float) * ((m + LZ_ROWS - 1) / LZ_ROWS) * n); }
static size_t lin_part_bytes(const LinDim* d, int count, const LinPlan& plan) {
    size_t bytes = 0;
    for (int i = 0; i < count; ++i)
        if (plan.splits[i] > 1) bytes += lin_up(sizeof(float) * static_cast<size_t>(plan.splits[i]) * d[i].m * d[i].n);
    return bytes;
}

template <int EPI, int ACT, bool SLOPE>
static int lin_launch(const LinMaps& maps, const LinGemm& p, unsigned ctas, size_t smem, bool first, cudaStream_t s) {
    static thread_local unsigned long long opted_in = 0;      // the shared-memory opt-in is per context and kernel
    const unsigned long long here = context_number();
    if (here == 0 || here != opted_in) {
        cudaError_t e = cudaFuncSetAttribute(linear_pair_kernel<EPI, ACT, SLOPE>, cudaFuncAttributeMaxDynamicSharedMemorySize, LG_MAX_SMEM);
        if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(linear_pair_kernel)");
        opted_in = context_number();
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(LG_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = first ? 0 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, linear_pair_kernel<EPI, ACT, SLOPE>, maps, p);
    if (e != cudaSuccess) return cuda_status(e, "linear_pair_kernel");
    KGE_LAUNCH_CHECK("linear_pair_kernel");
    return 0;
}

template <int ACT>
static int lin_launch_forward(const LinMaps& maps, const LinGemm& p, unsigned ctas, size_t smem, cudaStream_t s) {
    return p.e.slope ? lin_launch<LE_FORWARD, ACT, true>(maps, p, ctas, smem, true, s)
                     : lin_launch<LE_FORWARD, ACT, false>(maps, p, ctas, smem, true, s);
}

// out[m][n] = sum_k A[m][k] B[n][k].  a_mn / b_mn: the operand lies as (k rows, m or n columns).
struct LinTask {
    const void* a; long long lda; int a_mn;
    const void* b; long long ldb; int b_mn;
    LinDim d;
    LinEpilogue e;
};
struct LinColumns { const float* colpart; long long blocks; int n; __nv_bfloat16* db; };
// One product with the forward epilogue, or up to two plain ones and the column sums.  `first`: nothing of the call is ahead.
static int lin_gemm(const LinTask* t, int count, const LinPlan& plan, int sms, bool forward, const LinColumns* cols, bool first, void* part,
                    cudaStream_t s) {
    LinDim d[2];
    for (int i = 0; i < count; ++i) d[i] = t[i].d;
    const int (&splits)[2] = plan.splits, (&bn)[2] = plan.bn;
    LinGemm p;
    memset(&p, 0, sizeof(p));
    p.q[0].tiles_m = p.q[0].tiles_n = p.q[1].tiles_m = p.q[1].tiles_n = p.q[0].bn = p.q[1].bn = 1;
    p.err = device_error_word();
    if (!p.err) { set_error("linear: no usable device"); return KGE_E_DEVICE; }
    if (cols) { p.colpart = cols->colpart; p.colblocks = cols->blocks; p.db_n = cols->n; p.db = cols->db; }
    LinMaps maps;
    LinJoin join[2];
    memset(join, 0, sizeof(join));
    memset(&maps, 0, sizeof(maps));
    const bool fused = forward && splits[0] == 1;        // a split product gets its epilogue in the join
    const bool slope = fused && t[0].e.slope != nullptr;
    size_t used = 0;
    long long items = 0, groups = 0;
    // longest items first: what is short evens out the end
    const int lead = count == 2 && (d[1].k + 63) / 64 / splits[1] * bn[1] > (d[0].k + 63) / 64 / splits[0] * bn[0] ? 1 : 0;
    for (int at = 0; at < count; ++at) {
        const int i = at ^ lead;
        const LinTask& c = t[i];
        const long long m = d[i].m, n = d[i].n, k = d[i].k;
        LinShape& q = p.q[at];
        q.m = static_cast<int>(m); q.n = static_cast<int>(n); q.kb = static_cast<int>((k + LG_BK - 1) / LG_BK);
        q.bn = bn[i]; q.a_mn = c.a_mn; q.b_mn = c.b_mn;
        q.tiles_m = static_cast<int>((m + 2 * LG_BM - 1) / (2 * LG_BM));
        q.tiles_n = static_cast<int>((n + q.bn - 1) / q.bn);
        q.splits = splits[i];
        const long long mine = static_cast<long long>(q.tiles_m) * q.tiles_n * q.splits;
        items += mine;
        if (items >= (1LL << 30)) { set_error("linear: %lld tiles exceed the tile index", items); return KGE_E_RANGE; }
        q.items = static_cast<int>(mine);
        int rc;
        if (q.splits > 1) {
            q.part = reinterpret_cast<float*>(static_cast<char*>(part) + used);
            used += lin_up(sizeof(float) * static_cast<size_t>(q.splits) * m * n);
            join[at].part = q.part; join[at].e = c.e; join[at].m = m; join[at].n = q.n; join[at].splits = q.splits;
            join[at].groups = m * (n / 8);
            groups += join[at].groups;
        } else {
            if ((rc = make_tensor_map_64b(&maps.out[at], c.e.out, m, n, static_cast<uint64_t>(c.e.ldo) * 2, 32))) return rc;
            if (slope && (rc = make_tensor_map_64b(&maps.slope, c.e.slope, m, n, static_cast<uint64_t>(n) * 2, 32))) return rc;
            if (fused && c.e.res && (rc = make_tensor_map_64b(&maps.res, c.e.res, m, n, static_cast<uint64_t>(c.e.ldr) * 2, 32))) return rc;
        }
        if (c.a_mn) rc = make_tensor_map_2d(&maps.a[at], c.a, 2, k, m, c.lda * 2, LG_BK, 64);
        else rc = make_tensor_map_2d(&maps.a[at], c.a, 2, m, k, c.lda * 2, LG_BM, LG_BK);
        if (rc) return rc;
        const int half_n = q.bn / 2;
        if (c.b_mn) rc = make_tensor_map_2d(&maps.b[at], c.b, 2, k, n, c.ldb * 2, LG_BK, 64);
        else rc = make_tensor_map_2d(&maps.b[at], c.b, 2, n, k, c.ldb * 2, static_cast<uint32_t>(half_n), LG_BK);
        if (rc) return rc;
        const int b_room = ((c.b_mn ? (half_n + 63) / 64 * LG_SLAB : half_n * 128) + 1023) & ~1023;      // atoms start on 1024-byte boundaries
        if (LG_A_BYTES + b_room > p.stage_bytes) p.stage_bytes = LG_A_BYTES + b_room;
    }
    if (fused) p.e = t[0].e;
    if (p.stage_bytes == 0) p.stage_bytes = LG_A_BYTES;
    p.items = static_cast<int>(items);
    const int staging = lin_staging(fused ? LE_FORWARD : LE_PLAIN, slope);
    p.stages = (LG_MAX_SMEM - LG_TAIL - staging) / p.stage_bytes;          // 4 or 5 at 256 columns; 3 cost 6 %
    if (p.stages > 8) p.stages = 8;
    const size_t smem = static_cast<size_t>(p.stages) * p.stage_bytes + staging + LG_TAIL;
    long long pairs = items;
    if (p.db && pairs < (p.db_n + 63) / 64) pairs = (p.db_n + 63) / 64;    // a CTA sums 32 columns at a time
    const unsigned ctas = 2u * static_cast<unsigned>(pairs < sms / 2 ? pairs : sms / 2);
    if (fused) {
        switch (t[0].e.act) {
            case ACT_NONE: return lin_launch<LE_FORWARD, ACT_NONE, false>(maps, p, ctas, smem, true, s);
            case ACT_RELU: return lin_launch_forward<ACT_RELU>(maps, p, ctas, smem, s);
            case ACT_SILU: return lin_launch_forward<ACT_SILU>(maps, p, ctas, smem, s);
            default: return lin_launch_forward<ACT_GELU>(maps, p, ctas, smem, s);
        }
    }
    int rc = lin_launch<LE_PLAIN, ACT_NONE, false>(maps, p, ctas, smem, first, s);
    if (rc || groups == 0) return rc;
    // (8191 x 1024 x 400, 9 shares of 51200 groups: one thread a group 20.6 us for the backward pass, eight 24.7 us; 39866 x 72 x 440,
    // 37 shares of 3960: 27.3 and 22.8 us)
    const bool many = (splits[0] >= 8 || splits[1] >= 8) && groups <= 148 * 64;
    const long long want = many ? (groups + 31) / 32 : (groups + 255) / 256;
    const unsigned blocks = static_cast<unsigned>(want < 148 * 8 ? want : 148 * 8);
    if (forward && many) KGE_LAUNCH_AFTER("linear_join_kernel", (linear_join_kernel<LE_FORWARD, 8>), blocks, 256u, s, join[0], join[1]);
    else if (forward) KGE_LAUNCH_AFTER("linear_join_kernel", (linear_join_kernel<LE_FORWARD, 1>), blocks, 256u, s, join[0], join[1]);
    else if (many) KGE_LAUNCH_AFTER("linear_join_kernel", (linear_join_kernel<LE_PLAIN, 8>), blocks, 256u, s, join[0], join[1]);
    else KGE_LAUNCH_AFTER("linear_join_kernel", (linear_join_kernel<LE_PLAIN, 1>), blocks, 256u, s, join[0], join[1]);
    return 0;
}

template <int M>
static int lin_few(const void* x, long long ldx, const void* w, long long ldw, long long m, long long k, long long n, const LinEpilogue& e, cudaStream_t s) {
    int cluster = 8;
    while (cluster > 1 && k < cluster * 64) cluster /= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((n + 31) / 32 * cluster));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    cudaError_t err = cudaLaunchKernelEx(&cfg, linear_few_kernel<M>, static_cast<const __nv_bfloat16*>(x), ldx, static_cast<const __nv_bfloat16*>(w), ldw,
                                         static_cast<int>(m), static_cast<int>(k), static_cast<int>(n), e);
    if (err != cudaSuccess) return cuda_status(err, "linear_few_kernel");
    KGE_LAUNCH_CHECK("linear_few_kernel");
    return 0;
}

}  // namespace kge

using namespace kge;

static int check_linear(const char* fn, int64_t m, int64_t k, int64_t n, int32_t act) {
    if (act < ACT_NONE || act > ACT_GELU) { set_error("%s: unknown activation %d", fn, act); return KGE_E_UNSUPPORTED; }
    if (m < 0 || k < 1 || n < 1) { set_error("%s: sizes m = %lld, k = %lld, n = %lld", fn, (long long)m, (long long)k, (long long)n); return KGE_E_SHAPE; }
    if ((k & 7) || (n & 7)) { set_error("%s: bf16 rows need k %% 8 == 0 and n %% 8 == 0 (16-byte rows), got k = %lld, n = %lld", fn, (long long)k, (long long)n); return KGE_E_UNSUPPORTED; }
    if (m > (1LL << 30) || k > (1LL << 20) || n > (1LL << 20)) { set_error("%s: m above 2^30 or k, n above 2^20", fn); return KGE_E_RANGE; }
    return 0;
}
static int check_rows(const char* fn, const char* name, const void* p, int64_t ld, int64_t rows, int64_t cols, bool required) {
    if (!p) {
        if (!required) return 0;
        set_error("%s: %s is NULL", fn, name); return KGE_E_NULL;
    }
    if (!aligned16(p)) { set_error("%s: %s is not 16-byte aligned", fn, name); return KGE_E_ALIGN; }
    if (rows > 1 && ld < cols) { set_error("%s: row pitch %lld of %s is below %lld", fn, (long long)ld, name, (long long)cols); return KGE_E_SHAPE; }
    if (rows > 1 && (ld & 7)) { set_error("%s: row pitch %lld of %s is not a multiple of 8 (16-byte rows)", fn, (long long)ld, name); return KGE_E_ALIGN; }
    if (ld > (1LL << 32)) { set_error("%s: row pitch of %s above 2^32", fn, name); return KGE_E_RANGE; }
    return 0;
}
static int check_workspace(const char* fn, const void* p) {
    if (!p) { set_error("%s: workspace is NULL", fn); return KGE_E_NULL; }
    if (reinterpret_cast<uintptr_t>(p) & 255) { set_error("%s: workspace is not 256-byte aligned", fn); return KGE_E_ALIGN; }
    return 0;
}
// a single row is read through its own length, whatever pitch came with it
static long long pitch_of(int64_t ld, int64_t rows, int64_t cols) { return rows > 1 ? ld : cols; }

extern "C" {

size_t kge_linear_workspace_bytes(int64_t m, int64_t k, int64_t n, int32_t act, int32_t backward) {
    if (m <= 0 || k <= 0 || n <= 0 || check_linear("kge_linear_workspace_bytes", m, k, n, act)) return 0;
    const int sms = lin_sms();
    const LinDim fwd = {m, n, k}, both[2] = {{m, k, n}, {k, n, m}};
    if (!backward) return m <= LF_ROWS ? 0 : lin_part_bytes(&fwd, 1, lin_plan(&fwd, 1, sms));
    size_t part = lin_part_bytes(both, 2, lin_plan(both, 2, sms));           // both gradients, or either alone
    for (int i = 0; i < 2; ++i) {
        const size_t one = lin_part_bytes(&both[i], 1, lin_plan(&both[i], 1, sms));
        if (one > part) part = one;
    }
    return lin_dz_bytes(m, n, act) + lin_col_bytes(m, n) + part;
}

int kge_linear_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* residual, int64_t ldr,
                       int64_t m, int64_t k, int64_t n, int32_t act, void* out, int64_t ldo, void* slope, void* workspace,
                       size_t workspace_bytes, kge_stream_t stream) {
    const char* fn = "kge_linear_forward";
    int rc = check_linear(fn, m, k, n, act);
    if (rc || m == 0) return rc;
    if ((rc = check_rows(fn, "x", x, ldx, m, k, true)) || (rc = check_rows(fn, "w", w, ldw, k, n, true)) ||
        (rc = check_rows(fn, "bias", bias, n, 1, n, false)) || (rc = check_rows(fn, "residual", residual, ldr, m, n, false)) ||
        (rc = check_rows(fn, "out", out, ldo, m, n, true)) || (rc = check_rows(fn, "slope", slope, n, m, n, false))) return rc;
    const int sms = lin_sms();
    const LinDim dim = {m, n, k};
    const LinPlan plan = m <= LF_ROWS ? LinPlan{{0, 0}, {1, 1}} : lin_plan(&dim, 1, sms);
    const size_t need = lin_part_bytes(&dim, 1, plan);
    if (workspace_bytes < need) { set_error("%s: workspace needs %zu bytes, got %zu", fn, need, workspace_bytes); return KGE_E_WORKSPACE; }
    if (need && (rc = check_workspace(fn, workspace))) return rc;
    if (out == x || out == w) { set_error("%s: out lies over an operand of the product", fn); return KGE_E_UNSUPPORTED; }
    if (residual == out && m > 1 && ldr != ldo) { set_error("%s: out may be residual only with the same row pitch", fn); return KGE_E_SHAPE; }
    LinEpilogue e;
    memset(&e, 0, sizeof(e));
    e.bias = static_cast<const __nv_bfloat16*>(bias);
    e.res = static_cast<const __nv_bfloat16*>(residual); e.ldr = pitch_of(ldr, m, n);
    e.out = static_cast<__nv_bfloat16*>(out); e.ldo = pitch_of(ldo, m, n);
    e.slope = act == ACT_NONE ? nullptr : static_cast<__half*>(slope);
    e.act = act;
    if (m <= LF_ROWS) {
        cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
        ldx = pitch_of(ldx, m, k); ldw = pitch_of(ldw, k, n);
        if (m == 1) return lin_few<1>(x, ldx, w, ldw, m, k, n, e, s);
        if (m == 2) return lin_few<2>(x, ldx, w, ldw, m, k, n, e, s);
        if (m <= 4) return lin_few<4>(x, ldx, w, ldw, m, k, n, e, s);
        return lin_few<8>(x, ldx, w, ldw, m, k, n, e, s);
    }
    const LinTask t = {x, pitch_of(ldx, m, k), 0, w, pitch_of(ldw, k, n), 1, {m, n, k}, e};
    return lin_gemm(&t, 1, plan, sms, true, nullptr, true, workspace, reinterpret_cast<cudaStream_t>(stream));
}

int kge_linear_backward(const void* dout, int64_t ldd, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* slope,
                        int64_t m, int64_t k, int64_t n, int32_t act, void* dx, int64_t lddx, void* dw, void* dbias, void* workspace,
                        size_t workspace_bytes, kge_stream_t stream) {
    const char* fn = "kge_linear_backward";
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    int rc = check_linear(fn, m, k, n, act);
    if (rc) return rc;
    if ((rc = check_rows(fn, "dw", dw, n, k, n, false)) || (rc = check_rows(fn, "dbias", dbias, n, 1, n, false))) return rc;
    if (m == 0) {                           // no rows: the sums over them are zero
        cudaError_t e = dw ? cudaMemsetAsync(dw, 0, 2 * static_cast<size_t>(k) * n, s) : cudaSuccess;
        if (e == cudaSuccess && dbias) e = cudaMemsetAsync(dbias, 0, 2 * static_cast<size_t>(n), s);
        return cuda_status(e, "kge_linear_backward: cudaMemsetAsync");
    }
    if ((rc = check_rows(fn, "dout", dout, ldd, m, n, true)) || (rc = check_rows(fn, "x", x, ldx, m, k, dw != nullptr)) ||
        (rc = check_rows(fn, "w", w, ldw, k, n, dx != nullptr)) || (rc = check_rows(fn, "slope", slope, n, m, n, act != ACT_NONE)) ||
        (rc = check_rows(fn, "dx", dx, lddx, m, k, false))) return rc;
    const int sms = lin_sms(), count = (dx != nullptr) + (dw != nullptr);
    const LinDim both[2] = {{m, k, n}, {k, n, m}}, *dim = dx ? both : both + 1;          // dx and dw, or the one that is wanted
    const LinPlan plan = count > 0 ? lin_plan(dim, count, sms) : LinPlan{{0, 0}, {1, 1}};
    const size_t need = lin_dz_bytes(m, n, act) + lin_col_bytes(m, n) + lin_part_bytes(dim, count, plan);
    if (workspace_bytes < need) { set_error("%s: workspace needs %zu bytes, got %zu", fn, need, workspace_bytes); return KGE_E_WORKSPACE; }
    if ((rc = check_workspace(fn, workspace))) return rc;
    for (const void* p : {dout, x, w, slope})
        if (p && (p == dx || p == dw)) { set_error("%s: a gradient lies over an input", fn); return KGE_E_UNSUPPORTED; }
    char* ws = static_cast<char*>(workspace);
    __nv_bfloat16* dz = nullptr;
    if (act != ACT_NONE) dz = reinterpret_cast<__nv_bfloat16*>(ws);
    ws += lin_dz_bytes(m, n, act);
    const long long blocks = (m + LZ_ROWS - 1) / LZ_ROWS;
    float* colpart = reinterpret_cast<float*>(ws);
    ws += lin_col_bytes(m, n);
    ldd = pitch_of(ldd, m, n);
    if (dz || dbias) {
        const long long strips = (n + 255) / 256;
        if (blocks * strips >= (1LL << 31)) { set_error("%s: m x n too large", fn); return KGE_E_RANGE; }
        linear_dz_kernel<<<static_cast<unsigned>(blocks * strips), 512, 0, s>>>(
            static_cast<const __nv_bfloat16*>(dout), ldd, dz ? static_cast<const __half*>(slope) : nullptr, dz, lin_dz_pitch(n), dbias ? colpart : nullptr, m,
            static_cast<int>(n), static_cast<unsigned>(strips));
        KGE_LAUNCH_CHECK("linear_dz_kernel");
    }
    const void* g = dz ? static_cast<const void*>(dz) : dout;
    const long long ldg = dz ? lin_dz_pitch(n) : ldd;
    LinTask t[2];
    memset(t, 0, sizeof(t));
    int at = 0;
    if (dx) {
        t[at] = {g, ldg, 0, w, pitch_of(ldw, k, n), 0, both[0], {}};
        t[at].e.out = static_cast<__nv_bfloat16*>(dx); t[at].e.ldo = pitch_of(lddx, m, k);
        ++at;
    }
    if (dw) {
        t[at] = {x, pitch_of(ldx, m, k), 1, g, ldg, 1, both[1], {}};
        t[at].e.out = static_cast<__nv_bfloat16*>(dw); t[at].e.ldo = n;
    }
    const LinColumns cols = {colpart, blocks, static_cast<int>(n), static_cast<__nv_bfloat16*>(dbias)};
    if (count > 0 || dbias) return lin_gemm(t, count, plan, sms, false, dbias ? &cols : nullptr, !dz && !dbias, ws, s);
    return 0;
}

}  // extern "C"
