// prompt_attention.cu — causal attention of whole packed prompts on the fifth-generation tensor cores.
//
// 4 · hd flops and one exponential per visible (query, key) pair and head: at hd 128 a tile of 128 × 128 pairs is 1024 clocks of
// tcgen05.mma and 1024 clocks of the SM's 16 exponentials a clock, so neither may wait for the other.  One prompt of 8192 rows with 32 heads:
// 586 µs, 938 TFLOP/s = 59 % of the measured matrix rate, at 990 W (the power cap) and 1.6 GHz: a pair of tiles takes 3070 clocks, its
// chain being scores → maximum 540 → exponentials 1450 → products and scores of the next tile 1070.
//   * A CTA works on two query tiles of 128 rows with the same keys: the same rows of two heads that share a KV head, or — where the
//     heads do not pair up — 256 consecutive rows of one head.
//   * S = Q·Kᵀ (f32) and O (128 × hd f32) live in tensor memory; the probabilities go back over the scores as 16-bit numbers and are
//     the A operand of O += P·V straight from there.  V is the B operand as it lies in memory (rows of keys).
//   * A thread owns a row: its maximum and sum need no exchange between lanes.  O is rescaled only when the running maximum has grown by
//     more than 2^8 — sums are f32 and any reference between is exact — so the rescaling almost never runs.
//   * While the softmax of one query tile runs, the tensor core has the other's products.
//   * K and V tiles of 128 keys come by tiled bulk copies through one ring of shared-memory stages: K0 V0 K1 V1 …
//   * Which sequence and rows a CTA owns it finds in the prefix array itself, late (long) row tiles first: nothing depends on host-side
//     lengths, and a captured call follows the arrays.
//   * A product of 0 and a NaN or infinity in a value row that the query does not see would be NaN: value rows behind the sequence are
//     zeroed in shared memory, and an output row that is not finite is taken again by ax_prompt_row, which reads visible rows only.
//   * Every wait is bounded (two seconds of %globaltimer): on expiry the CTA raises the context's error word, all roles leave, copies
//     in flight are waited for and tensor memory is released.
#include <cuda.h>
#include <type_traits>

#include "prompt_attention.cuh"

namespace {

constexpr int kRows = 128;                        // rows of a query tile, keys of a K / V tile
constexpr int kFirst = 64;                        // keys whose probabilities are handed over first; the rest ends the tile's chain
constexpr int kBoxBytes = kRows * 128;            // one box: 128 rows of 128 bytes
constexpr int kThreads = 384;                     // warps 0..3, 4..7: softmax of tile 0, 1; 8: products; 9: copies; 10: the end of a
                                                  // sequence's last V tile; 11 completes the warpgroup that hands registers over
constexpr int kProduct = 8, kCopy = 9, kCut = 10;
constexpr int kMaxStages = 6;
constexpr unsigned long long kWaitNs = 2000000000ull;

struct PromptDev {
    AxPromptArgs a;
    int pair_heads;                               // 1: two heads of a KV head, 0: 256 rows of one head
    float sc;                                     // |scale| · log2 e
    int negate;                                   // scale < 0
    int* err;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded wait.  false: gave up (this thread's deadline passed, or another role raised the abort flag).
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
    if (mbar_try(bar, parity)) return true;
    unsigned long long t0 = 0;
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 256; i++)                                         // as few instructions as can be: waiting warps share the issue slots
            if (mbar_try(bar, parity)) return true;
        if (*abort_flag) return false;
        const unsigned long long t = ax_globaltimer();
        if (t0 == 0) t0 = t;
        else if (t - t0 > kWaitNs) { *abort_flag = 1; atomicExch(err, code); return false; }
    }
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 :: "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// Shared-memory matrix descriptors, 128-byte swizzle (layout code 2, version 1), groups of eight rows of 128 bytes 1024 bytes apart: the high
// word is always the same, the low word holds the address and, for MN-major operands, how far the next 64 columns lie (one box).
// Advancing is an addition to the low word — the thread that issues the products spent more time on descriptors than the tensor core
// on the products when each was built from its address.
//   K-major (rows hold the contracted index): 16 numbers further are 32 bytes inside the row.
//   MN-major (rows are the contracted index, 64 columns each): 16 numbers further are 16 rows.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) { return (addr >> 4) | ((uint32_t)(kBoxBytes >> 4) << 16); }
template <bool ACC> __device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "r"(b), "r"(idesc), "n"(ACC ? 1 : 0), "n"(kDescHigh) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 y, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHigh) : "memory");
}
// One lane of a converged warp.  The products are issued under this predicate, not under lane == 0: their descriptors live in uniform
// registers, and only here does the compiler know that one thread runs (eight products: 600 clocks instead of 1000).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
#define AX_R32(m) m(0), m(1), m(2), m(3), m(4), m(5), m(6), m(7), m(8), m(9), m(10), m(11), m(12), m(13), m(14), m(15), \
                  m(16), m(17), m(18), m(19), m(20), m(21), m(22), m(23), m(24), m(25), m(26), m(27), m(28), m(29), m(30), m(31)
// Columns of the warp's lane quarter.  The wait is part of the statement: the registers are written asynchronously, and a register that
// the compiler moved or spilled between the load and its wait would be moved too early.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
#define AX_O(i) "=r"(r[i])
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
                 "tcgen05.wait::ld.sync.aligned;" : AX_R32(AX_O) : "r"(addr) : "memory");
#undef AX_O
}
__device__ __forceinline__ void tmem_ld128(uint32_t addr, uint32_t* r) {
#define AX_O(i) "=r"(r[i])
#define AX_P(i) "=r"(r[32 + i])
#define AX_Q(i) "=r"(r[64 + i])
#define AX_S(i) "=r"(r[96 + i])
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x128.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
                 "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63, "
                 "%64, %65, %66, %67, %68, %69, %70, %71, %72, %73, %74, %75, %76, %77, %78, %79, %80, %81, %82, %83, %84, %85, %86, %87, %88, %89, %90, %91, %92, %93, %94, %95, "
                 "%96, %97, %98, %99, %100, %101, %102, %103, %104, %105, %106, %107, %108, %109, %110, %111, %112, %113, %114, %115, %116, %117, %118, %119, %120, %121, %122, %123, %124, %125, %126, %127}, [%128];\n\t"
                 "tcgen05.wait::ld.sync.aligned;" : AX_R32(AX_O), AX_R32(AX_P), AX_R32(AX_Q), AX_R32(AX_S) : "r"(addr) : "memory");
#undef AX_O
#undef AX_P
#undef AX_Q
#undef AX_S
}
#define AX_R16(m) m(0), m(1), m(2), m(3), m(4), m(5), m(6), m(7), m(8), m(9), m(10), m(11), m(12), m(13), m(14), m(15)
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
#define AX_O(i) "=r"(r[i])
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
                 "tcgen05.wait::ld.sync.aligned;" : AX_R16(AX_O) : "r"(addr) : "memory");
#undef AX_O
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
#define AX_I(i) "r"(r[i])
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
                 :: AX_R16(AX_I), "r"(addr) : "memory");
#undef AX_I
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\t"
        "mov.b64 {%0, %1}, w;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// largest of three; NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }
template <bool F16> __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <typename T, int HD>
__device__ __noinline__ void row_again(const AxPromptArgs& a, const AxPromptSeq& s, int h, int i, int lane) {
    ax_prompt_row<T, HD>(a, s, h, i, lane);
}

template <bool F16, int HD>
__global__ void __launch_bounds__(kThreads, 1) ax_prompt_umma_kernel(const __grid_constant__ CUtensorMap map_q,
                                                                     const __grid_constant__ CUtensorMap map_k,
                                                                     const __grid_constant__ CUtensorMap map_v, const PromptDev dv) {
    using T = typename std::conditional<F16, __half, uint16_t>::type;
    constexpr int BOXES = HD / 64, TILE = BOXES * kBoxBytes, NS = HD == 128 ? 5 : 6;
    constexpr uint32_t kS = 0, kO = 256;                                      // columns: scores of tile t at 128 t (its probabilities over the first half), output at 256 + HD t
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t q_full[2], s_full[2], p_ready[2][2], o_done[2], kv_full[kMaxStages], kv_empty[kMaxStages], v_here, v_cut;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_issued, s_seq, s_tile, s_scan[kThreads / 32];
    const int tid = threadIdx.x, warp = __shfl_sync(AX_FULL, tid >> 5, 0), lane = tid & 31;
    const AxPromptArgs& a = dv.a;
    volatile int* abort_flag = &s_abort;
    const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t ring = smem0 + 2 * TILE;

    // ── which rows: tile x of the pack counted from its end ──
    const int tb = dv.pair_heads ? kRows : 2 * kRows;
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(smem_u32(&q_full[i]), 1); mbar_init(smem_u32(&s_full[i]), 1); mbar_init(smem_u32(&o_done[i]), 1);
            for (int b = 0; b < 2; b++) mbar_init(smem_u32(&p_ready[i][b]), kRows);
        }
        for (int i = 0; i < NS; i++) { mbar_init(smem_u32(&kv_full[i]), 1); mbar_init(smem_u32(&kv_empty[i]), 1); }
        mbar_init(smem_u32(&v_here), 1); mbar_init(smem_u32(&v_cut), 1);
        s_abort = 0; s_issued = 0; s_seq = -1; s_tile = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    {
        const int per = (a.batch + kThreads - 1) / kThreads, b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
        int own = 0;
        for (int b = b0; b < b1; b++) own += (ax_prompt_seq(a, b).lq + tb - 1) / tb;
        int inc = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const int x = __shfl_up_sync(AX_FULL, inc, d); if (lane >= d) inc += x; }
        if (lane == 31) s_scan[warp] = inc;
        __syncthreads();
        int at = inc - own, all = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; w++) { if (w < warp) at += s_scan[w]; all += s_scan[w]; }
        const int x = all - 1 - (int)blockIdx.y;
        if (x < 0) return;
        if (x >= at && x < at + own)
            for (int b = b0; b < b1; b++) {
                const int n = (ax_prompt_seq(a, b).lq + tb - 1) / tb;
                if (x < at + n) { s_seq = b; s_tile = x - at; break; }
                at += n;
            }
    }
    if (warp == kProduct) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;
    const AxPromptSeq s = ax_prompt_seq(a, s_seq);
    const int off = s.lk - s.lq;
    const int h0 = dv.pair_heads ? 2 * (int)blockIdx.x : (int)blockIdx.x, kh = h0 / (a.n_heads / a.n_kv);
    int base[2], lo[2], hi[2];                                                // first row and K / V tiles [lo, hi] of both query tiles
    base[0] = s_tile * tb; base[1] = dv.pair_heads ? base[0] : base[0] + kRows;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const int last = min(base[t] + kRows, s.lq) - 1 + off, first = base[t] + off;
        lo[t] = 0; hi[t] = -1;
        if (base[t] < s.lq && last >= 0 && s.lk > 0) {
            lo[t] = a.window > 0 && first - a.window + 1 > 0 ? (first - a.window + 1) / kRows : 0;
            hi[t] = last / kRows;
        }
    }
    const bool on0 = hi[0] >= lo[0], on1 = hi[1] >= lo[1];
    const int j0 = on0 ? (on1 ? min(lo[0], lo[1]) : lo[0]) : lo[1], j1 = max(hi[0], hi[1]);      // j1 < j0: no tile at all
    const bool cut = j1 >= j0 && (j1 + 1) * kRows > s.lk;                     // the last V tile reaches behind the sequence

    // 384 threads start with 168 registers each (64512 in all); a row of scores is 128 of them.  256 · 208 + 128 · 80 = 63488.
    if (warp >= kProduct) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == kCopy) {
        if (elect_one()) {
            for (int t = 0; t < 2; t++)
                if (t ? on1 : on0) {
                    const uint32_t bar = smem_u32(&q_full[t]);
                    mbar_expect_tx(bar, TILE);
                    for (int b = 0; b < BOXES; b++)
                        tma_load_3d(smem0 + t * TILE + b * kBoxBytes, &map_q, b * 64, dv.pair_heads ? h0 + t : h0, s.q0 + base[t], bar);
                }
            const int n = j1 >= j0 ? 2 * (j1 - j0 + 1) : 0;
            int st = 0;
            uint32_t ph = 1;                                                  // a fresh barrier counts as a phase of parity one that is over
            for (int i = 0; i < n; i++) {
                if (!mbar_wait(smem_u32(&kv_empty[st]), ph, abort_flag, dv.err, 721)) break;
                const uint32_t bar = smem_u32(&kv_full[st]);
                mbar_expect_tx(bar, TILE);
                const CUtensorMap* map = i & 1 ? &map_v : &map_k;
                for (int b = 0; b < BOXES; b++) tma_load_3d(ring + st * TILE + b * kBoxBytes, map, b * 64, kh, s.k0 + (j0 + i / 2) * kRows, bar);
                s_issued = i + 1;
                if (++st == NS) { st = 0; ph ^= 1u; }
            }
        }
    } else if (warp == kProduct) {
        constexpr uint32_t fmt = F16 ? 0u : 1u;                               // accumulator f32, A and B f16 or bf16; B of P·V is MN-major
        constexpr uint32_t id_qk = (1u << 4) | (fmt << 7) | (fmt << 10) | ((kRows >> 3) << 17) | ((kRows >> 4) << 24);
        constexpr uint32_t id_pv = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((HD >> 3) << 17) | ((kRows >> 4) << 24);
        // One thread does all of it.  Its loop counts from zero and tensor memory starts at column zero (all of it is ours), so that stages,
        // descriptors and columns are uniform values: with a vector register behind each, issuing a product took longer than the product.
        if (elect_one()) {
            const int n = j1 - j0 + 1, a0 = lo[0] - j0, z0 = on0 ? hi[0] - j0 : -1, a1 = lo[1] - j0, z1 = on1 ? hi[1] - j0 : -1;   // tile t works at i in [a, z]
            bool ok = s_tmem == 0;
            if (!ok) { *abort_flag = 1; atomicExch(dv.err, 728); }
            auto qk = [&](int t, int st) {                                    // scores of query tile t with the K tile in stage st
                const uint32_t k = desc_k(ring) + (uint32_t)st * (TILE >> 4), q = desc_k(smem0) + (uint32_t)t * (TILE >> 4);
                umma_ss<false>(kS + t * 128, q, k, id_qk);
#pragma unroll
                for (int i = 1; i < HD / 16; i++)
                    umma_ss<true>(kS + t * 128, q + (i / 4) * (kBoxBytes >> 4) + (i % 4) * 2, k + (i / 4) * (kBoxBytes >> 4) + (i % 4) * 2, id_qk);
                umma_commit(smem_u32(&s_full[t]));
            };
            int st = 0;                                                       // stages are taken in turn; ph: parity of their phase
            uint32_t ph = 0;
            auto next = [&] { if (++st == NS) { st = 0; ph ^= 1u; } };
            if (n > 0 && ok) {
                ok = mbar_wait(smem_u32(&kv_full[0]), 0, abort_flag, dv.err, 722);
                if (ok && on0) { ok = mbar_wait(smem_u32(&q_full[0]), 0, abort_flag, dv.err, 723); if (ok && a0 == 0) qk(0, 0); }
                if (ok && on1) { ok = mbar_wait(smem_u32(&q_full[1]), 0, abort_flag, dv.err, 723); if (ok && a1 == 0) qk(1, 0); }
                if (ok) umma_commit(smem_u32(&kv_empty[0]));
                next();
            }
            for (int i = 0; i < n && ok; i++) {
                const int sv = st;
                ok = mbar_wait(smem_u32(&kv_full[sv]), ph, abort_flag, dv.err, 722);
                if (ok && i == n - 1 && cut) { mbar_arrive(smem_u32(&v_here)); ok = mbar_wait(smem_u32(&v_cut), 0, abort_flag, dv.err, 729); }
                if (!ok) break;
                next();
                const int sk = st;
                const bool more = i + 1 < n;
                const uint32_t vd = desc_mn(ring) + (uint32_t)sv * (TILE >> 4);
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const int at = t ? a1 : a0, zt = t ? z1 : z0;
                    if (ok && i >= at && i <= zt) {
                        const uint32_t p = (uint32_t)(i - at) & 1u;
#pragma unroll
                        for (int part = 0; part < 2; part++) {                // the product starts with the first probabilities
                            ok = ok && mbar_wait(smem_u32(&p_ready[t][part]), p, abort_flag, dv.err, 724);
                            if (!ok) break;
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                            for (int c = part ? kFirst / 16 : 0; c < (part ? kRows : kFirst) / 16; c++)
                                umma_ts(kO + t * HD, kS + t * 128 + c * 8, vd + c * (2048 >> 4), id_pv, c ? 1u : (uint32_t)(i != at));
                        }
                        if (ok) umma_commit(smem_u32(&o_done[t]));
                    }
                    if (ok && i + 1 >= at && i + 1 <= zt) {                   // over the scores and probabilities just used
                        ok = mbar_wait(smem_u32(&kv_full[sk]), ph, abort_flag, dv.err, 722);
                        if (ok) qk(t, sk);
                    }
                }
                if (!ok) break;
                umma_commit(smem_u32(&kv_empty[sv]));
                if (more) { umma_commit(smem_u32(&kv_empty[sk])); next(); }
            }
        }
        __syncwarp();
    } else if (warp == kCut) {
        // Value rows behind the sequence, in its last tile: zeros, so that whatever lies there meets a probability of zero as a number.
        if (cut) {
            const int vi = 2 * (j1 - j0) + 1, valid = s.lk - j1 * kRows;
            const uint32_t v = ring + (uint32_t)(vi % NS) * TILE;
            const bool ok = mbar_wait(smem_u32(&v_here), 0, abort_flag, dv.err, 730);      // told by the thread that saw it arrive
            if (__all_sync(AX_FULL, ok)) {
                for (int i = lane; i < (kRows - valid) * 8 * BOXES; i += 32) {
                    const int b = i / ((kRows - valid) * 8), r = i % ((kRows - valid) * 8);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" :: "r"(v + b * kBoxBytes + valid * 128 + r * 16), "r"(0) : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&v_cut));
            }
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = warp >> 2;
        const int r = (warp & 3) * 32 + lane, row = base[t] + r, pos = row + off;         // row of the sequence, key at its own position
        const int h = dv.pair_heads ? h0 + t : h0;
        const uint32_t quarter = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t ts = quarter + kS + t * 128, to = quarter + kO + t * HD;
        const float sc = dv.sc;
        const int j_lo = lo[t], j_hi = hi[t];
        const int key_hi = pos, key_lo = a.window > 0 ? pos - a.window : -1;               // visible: key_lo < j <= key_hi
        const int first = base[t] + off, lastp = min(base[t] + kRows, s.lq) - 1 + off;     // positions of the tile's first and last row
        float m = -INFINITY;
        float2 l0 = make_float2(0.f, 0.f), l1 = l0;
        bool ok = true;
        for (int j = j_lo, it = 0; j <= j_hi; j++, it++) {
            ok = mbar_wait(smem_u32(&s_full[t]), (uint32_t)it & 1u, abort_flag, dv.err, 725);
            if (!__all_sync(AX_FULL, ok)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            uint32_t u[kRows];
            tmem_ld128(ts, u);
            float* x = reinterpret_cast<float*>(u);
            if (dv.negate) {
#pragma unroll
                for (int c = 0; c < kRows; c++) x[c] = -x[c];
            }
            const int k0 = j * kRows;
            const bool edge = k0 + kRows - 1 > first || (a.window > 0 && k0 <= lastp - a.window);      // some row of the tile does not see all keys
            if (edge) {
#pragma unroll
                for (int c = 0; c < kRows; c++) if (k0 + c > key_hi || k0 + c <= key_lo) x[c] = -INFINITY;
            }
            float mx[8];
#pragma unroll
            for (int c = 0; c < 8; c++) mx[c] = x[c];
#pragma unroll
            for (int c = 8; c < 120; c += 2) mx[(c >> 1) & 7] = max3(mx[(c >> 1) & 7], x[c], x[c + 1]);
            const float top = max3(max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), max3(mx[6], mx[7], x[120])),
                                   max3(x[121], x[122], x[123]), max3(max3(x[124], x[125], x[126]), x[127], x[127]));
            if (top != top) m = top;                                          // the row is taken again
            const bool grow = top > m && (m == -INFINITY || (top - m) * sc > 8.f);
            if (__any_sync(AX_FULL, grow)) {
                const float f = !grow ? 1.f : m == -INFINITY ? 0.f : ex2((m - top) * sc);
                if (grow) m = top;
                l0.x *= f; l0.y *= f; l1.x *= f; l1.y *= f;
                if (it > 0) {
                    ok = mbar_wait(smem_u32(&o_done[t]), (uint32_t)(it - 1) & 1u, abort_flag, dv.err, 726);
                    if (!__all_sync(AX_FULL, ok)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                    for (int c = 0; c < HD; c += 16) {
                        uint32_t o[16];
                        tmem_ld16(to + c, o);
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st16(to + c, o);
                    }
                }
            }
            const float neg = m == -INFINITY ? 0.f : -m * sc;
            const float2 sc2 = make_float2(sc, sc), neg2 = make_float2(neg, neg);
            auto probs = [&](int c0) {                                        // 32 keys
                uint32_t p[16];
#pragma unroll
                for (int c = 0; c < 16; c++) {
                    float2 y = fma2(make_float2(x[c0 + 2 * c], x[c0 + 2 * c + 1]), sc2, neg2);
                    y.x = ex2(y.x); y.y = ex2(y.y);
                    if (c & 1) l1 = add2(l1, y); else l0 = add2(l0, y);
                    p[c] = pack<F16>(y.x, y.y);
                }
                tmem_st16(ts + c0 / 2, p);
            };
            auto hand_over = [&](int part) {
                tmem_wait_st();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                mbar_arrive(smem_u32(&p_ready[t][part]));
            };
            probs(0); probs(32);
            hand_over(0);
            probs(64); probs(96);
            hand_over(1);
        }
        // ── output ──
        const int tiles = j_hi - j_lo + 1;
        if (ok && tiles > 0) {
            ok = mbar_wait(smem_u32(&o_done[t]), (uint32_t)(tiles - 1) & 1u, abort_flag, dv.err, 727);
            ok = __all_sync(AX_FULL, ok);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        if (ok) {
            const bool live = row < s.lq;
            const float l = (l0.x + l0.y) + (l1.x + l1.y);
            const float inv = l == 0.f ? 0.f : 1.f / l;
            float odd = 0.f;                                                  // becomes NaN with the first output that is not finite
            T* out = (T*)a.out + (long long)(s.q0 + row) * a.o_tok + (long long)h * a.o_head;
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                if (tiles > 0) {
                    tmem_ld32(to + c, o);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = 0u;
                }
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const float x0 = __uint_as_float(o[2 * e]) * inv, x1 = __uint_as_float(o[2 * e + 1]) * inv;
                    odd = fmaf(x0, 0.f, fmaf(x1, 0.f, odd));
                    w[e] = pack<F16>(x0, x1);
                }
                if (live) {
#pragma unroll
                    for (int e = 0; e < 4; e++) *reinterpret_cast<uint4*>(out + c + 8 * e) = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
                }
            }
            const bool sees = key_hi >= 0 && s.lk > 0;
            unsigned again = __ballot_sync(AX_FULL, live && (odd != odd || (sees && !(fabsf(m) <= 3.402823466e38f))));
            __syncwarp();
            while (again) {
                const int i = __ffs(again) - 1;
                again &= again - 1;
                row_again<T, HD>(a, s, h, base[t] + (warp & 3) * 32 + i, lane);
            }
        }
    }

    // ── tail: nothing of this CTA may still be in flight when its shared and tensor memory go away ──
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (s_abort) {
        if (tid == 0) {                                                       // copies issued into stages nobody consumed any more
            const int issued = s_issued;
            for (int i = issued > NS ? issued - NS : 0; i < issued; i++) {
                const unsigned long long t0 = ax_globaltimer();
                while (!mbar_try(smem_u32(&kv_full[i % NS]), (uint32_t)(i / NS) & 1u) && ax_globaltimer() - t0 < kWaitNs) { }
            }
            for (int t = 0; t < 2; t++) {
                const unsigned long long t0 = ax_globaltimer();
                while ((t ? on1 : on0) && !mbar_try(smem_u32(&q_full[t]), 0) && ax_globaltimer() - t0 < kWaitNs) { }
            }
        }
        if (tid == 32) {                                                      // products issued before the failure: time to drain
            const unsigned long long t0 = ax_globaltimer();
            while (ax_globaltimer() - t0 < 2000000ull) { }
        }
        __syncthreads();
    }
    if (warp == kProduct) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem) : "memory");
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) p = nullptr;
        return (EncodeTiledFn)p;
    }();
    return fn;
}
// [rows][heads][hd] seen as boxes of 64 numbers × one head × 128 rows; reads behind the last row give zeros
int make_map(CUtensorMap* map, bool f16, const void* data, int rows, int heads, int hd, long long tok, long long head) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return atlasx_fail(ATLASX_ERR_CUDA, "the driver does not export cuTensorMapEncodeTiled");
    const cuuint64_t dims[3] = { (cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows };
    // a stride that is never used may be anything the caller had; the map wants a multiple of 16 above zero
    const cuuint64_t strides[2] = { (cuuint64_t)(heads > 1 ? head : hd) * 2, (cuuint64_t)(rows > 1 ? tok : (long long)heads * hd) * 2 };
    const cuuint32_t box[3] = { 64, 1, kRows }, step[3] = { 1, 1, 1 };
    const CUresult r = fn(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(data), dims, strides,
                          box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return atlasx_fail(ATLASX_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)r);
    return ATLASX_OK;
}

template <bool F16, int HD>
int launch(atlasx_ctx* ctx, const PromptDev& dv, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v) {
    constexpr int smem = (2 + (HD == 128 ? 5 : 6)) * (HD / 64) * kBoxBytes + 1024;
    static bool ready[64] = {};
    if (ctx->device >= 64 || !ready[ctx->device]) {                           // the limit is per device; asking twice does no harm
        AX_CUDA(cudaFuncSetAttribute(ax_prompt_umma_kernel<F16, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        if (ctx->device < 64) ready[ctx->device] = true;
    }
    const int tb = dv.pair_heads ? kRows : 2 * kRows;
    // at most one unfilled tile per sequence, and no more sequences with rows than rows
    const long long tiles = (long long)dv.a.n_q / tb + (dv.a.batch < dv.a.n_q ? dv.a.batch : dv.a.n_q);
    ax_prompt_umma_kernel<F16, HD><<<dim3((unsigned)(dv.pair_heads ? dv.a.n_heads / 2 : dv.a.n_heads), (unsigned)tiles), kThreads, smem, ctx->stream>>>(q, k, v, dv);
    AX_CHECK_LAUNCH("ax_prompt_umma_kernel");
    return ATLASX_OK;
}

}  // namespace

extern "C" int atlasx_prompt_attention(atlasx_ctx* c, const atlasx_prompt_args* p) {
    AX_ARG(p, "null argument");
    const void *q = p->q, *k = p->k, *v = p->v;
    void* out = p->out;
    const long long q_tok = p->q_token_stride, q_head = p->q_head_stride, k_tok = p->k_token_stride, k_head = p->k_head_stride,
                    v_tok = p->v_token_stride, v_head = p->v_head_stride, o_tok = p->out_token_stride, o_head = p->out_head_stride;
    const int *cu_q = p->cu_q, *cu_k = p->cu_k, dtype = p->dtype, batch = p->batch, n_q = p->n_q, n_k = p->n_k, n_heads = p->n_heads,
              n_kv = p->n_kv_heads, hd = p->head_dim, window = p->window;
    const float scale = p->scale;
    AX_ARG(dtype == ATLASX_BF16 || dtype == ATLASX_F16, "dtype must be bf16 or f16");
    AX_ARG(batch >= 1 && batch <= AX_PAGED_MAX_BATCH, "batch must be in 1..4096");
    AX_ARG(n_q >= 0 && n_k >= 0, "row counts must not be negative");
    AX_ARG(n_q <= 0x3FFFFFFF && n_k <= 0x3FFFFFFF, "too many rows");
    AX_ARG(n_heads >= 1 && n_kv >= 1 && n_heads % n_kv == 0, "n_heads must be a multiple of n_kv_heads");
    AX_ARG(n_heads <= 65535, "too many heads");
    AX_ARG(hd == 64 || hd == 128, "head_dim must be 64 or 128");
    AX_ARG(window >= 0, "window must be non-negative");
    AX_ARG(scale - scale == 0.f, "scale must be finite");
    if (n_q == 0) return ATLASX_OK;
    AX_ARG(q && out && cu_q && cu_k && ((k && v) || n_k == 0), "null argument");
    AX_ARG(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) % 16 == 0 &&
           (q_tok | q_head | k_tok | k_head | v_tok | v_head | o_tok | o_head) % 8 == 0, "rows must start on 16-byte boundaries");
    AX_ARG(q_tok >= 0 && q_head >= 0 && k_tok >= 0 && k_head >= 0 && v_tok >= 0 && v_head >= 0, "strides must not be negative");
    AX_ARG((q_head > 0 || n_heads == 1) && ((k_head > 0 && v_head > 0) || n_kv == 1 || n_k == 0) &&
           (q_tok > 0 || n_q == 1) && ((k_tok > 0 && v_tok > 0) || n_k <= 1), "strides must not be zero");
    AX_ARG((o_head >= hd || n_heads == 1) && (o_tok >= hd || n_q == 1), "rows of out overlap");
    AX_ARG(q_tok < (1ll << 38) && q_head < (1ll << 38) && k_tok < (1ll << 38) && k_head < (1ll << 38) && v_tok < (1ll << 38) && v_head < (1ll << 38),
           "strides must be below 2^38");
    AX_ARG(c, "ctx is null");
    AX_ON_DEVICE(c);
    PromptDev dv = {};
    dv.a = { q, k, v, out, q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head, cu_q, cu_k, batch, n_q, n_k, n_heads, n_kv, hd, window, scale };
    dv.pair_heads = (n_heads / n_kv) % 2 == 0;
    dv.negate = scale < 0.f;
    // a hidden key's score is −inf · sc: a scale of zero must not make it NaN.  Scores below 2^126 / 1e37 of it are still all alike.
    dv.sc = fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-37f);
    dv.err = c->dev_error;
    const bool f16 = dtype == ATLASX_F16;
    CUtensorMap mq, mk, mv;
    int rc = make_map(&mq, f16, q, n_q, n_heads, hd, q_tok, q_head);
    if (!rc && n_k > 0) rc = make_map(&mk, f16, k, n_k, n_kv, hd, k_tok, k_head);
    if (!rc && n_k > 0) rc = make_map(&mv, f16, v, n_k, n_kv, hd, v_tok, v_head);
    if (rc) return rc;
    if (n_k == 0) mk = mv = mq;                                               // never read: no sequence has keys
    if (f16) return hd == 128 ? launch<true, 128>(c, dv, mq, mk, mv) : launch<true, 64>(c, dv, mq, mk, mv);
    return hd == 128 ? launch<false, 128>(c, dv, mq, mk, mv) : launch<false, 64>(c, dv, mq, mk, mv);
}
