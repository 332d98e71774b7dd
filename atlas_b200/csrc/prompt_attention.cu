// prompt_attention.cu — causal attention of whole packed prompts on the fifth-generation tensor cores.
//
// 4 · hd flops and one exponential per visible (query, key) pair and head: at hd 128 a tile of 128 × 128 pairs is 1024 clocks of
// tcgen05.mma and 1024 clocks of the SM's 16 exponentials a clock, so neither may wait for the other.  One prompt of 8192 rows with 32 heads:
// 569 µs, 966 TFLOP/s = 60 % of the measured matrix rate, at 990 W (the power cap) and 1.6 GHz: a pair of tiles takes 3070 clocks, its
// chain being scores → maximum 540 → exponentials 1450 → products and scores of the next tile 1070.  228 pairs an SM are seven eighths of
// the time; the rest is the seven items an SM beside their pairs, 13 to 17 thousand clocks each — both tiles of a CTA come to their end at once,
// and nothing feeds the tensor core while they are read out, stored and the next item is taken.  Of 24 ragged prompts (91 pairs and 13 items
// an SM) that is two fifths.
//   * A CTA works on two query tiles of 128 rows with the same keys: the same rows of two heads that share a KV head, or — where the
//     heads do not pair up — 256 consecutive rows of one head.
//   * S = Q·Kᵀ (f32) and O (128 × hd f32) live in tensor memory; the probabilities go back over the scores as 16-bit numbers and are
//     the A operand of O += P·V straight from there.  V is the B operand as it lies in memory (rows of keys).
//   * A thread owns a row: its maximum and sum need no exchange between lanes.  O is rescaled only when the running maximum has grown by
//     more than 2^8 — sums are f32 and any reference between is exact — so the rescaling almost never runs.
//   * While the softmax of one query tile runs, the tensor core has the other's products.
//   * K and V tiles of 128 keys come by tiled bulk copies through one ring of shared-memory stages: K0 V0 K1 V1 …
//   * An item is one pair of query tiles; there is a CTA for each, late (long) row tiles of all heads first.  A CTA that runs takes over the
//     items of CTAs that have not started (clusterlaunchcontrol: the hardware hands them out, no counter in memory): its copies for
//     the next item run under the end of the one before (a CTA per item spent 5 to 7 µs starting and ending).  A warp of its
//     own finds sequence and rows in the prefix arrays: nothing depends on host-side lengths, and a captured call follows the arrays.
//   * A product of 0 and a NaN or infinity in a value row that the query does not see would be NaN: value rows behind the sequence are
//     zeroed in shared memory, and an output row that is not finite (though its scores are numbers) is taken again by ax_prompt_row, which
//     reads visible rows only.
//   * Every wait is bounded (ten seconds of %globaltimer, in which no row is taken again): on expiry the CTA raises the context's error word,
//     all roles leave, copies in flight are waited for and tensor memory is released.
#include <cuda.h>
#include <atomic>
#include <type_traits>

#include "prompt_attention.cuh"

namespace {

constexpr int kRows = 128;                        // rows of a query tile, keys of a K / V tile
constexpr int kFirst = 64;                        // keys whose probabilities are handed over first; the rest ends the tile's chain
constexpr int kBoxBytes = kRows * 128;            // one box: 128 rows of 128 bytes
constexpr int kThreads = 384;                     // warps 0..3, 4..7: softmax of tile 0, 1; 8: products; 9: copies; 10: the end of a
                                                  // sequence's last V tile; 11: items
constexpr int kProduct = 8, kCopy = 9, kItems = 11;
constexpr int kSlots = 2;                         // items known ahead
constexpr int kReaders = 11;                      // arrivals that free an item's slot: eight softmax warps, products, copies, cut
constexpr int kMaxStages = 6;
// Limit of a wait; the second is for a test that cannot wait that long.  (As an argument of the launch it made the polling loop of waiting warps
// longer: 24 ragged prompts 285 -> 296 µs.)
constexpr int kWaitMs = 10000, kTestWaitMs = 10;
constexpr unsigned long long kAbortNs = 5000000ull;          // after a failure: what is in flight lands within microseconds

struct PromptDev {
    AxPromptArgs a;
    int pair_heads;                               // 1: two heads of a KV head, 0: 256 rows of one head
    float sc;                                     // |scale| · log2 e
    int negate;                                   // scale < 0
    int wide;                                     // rows of out start on 32-byte boundaries
    int lose;                                     // test with short waits: the first CTA's second K tile is never copied
    int* err;
};

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
// Bounded wait.  false: gave up (this thread's deadline passed, or another role raised the abort flag).  flags: [0] abort, [1] warps that take
// rows again — as long as there are any (each row is a loop over its keys, so it ends) the deadline does not run: a long prompt
// with a NaN in its first value has minutes of them.
template <int WAIT_MS> __device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* flags, int* err, int code) {
    if (ax_mbar_try(bar, parity)) return true;
    unsigned long long t0 = 0;
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 256; i++)                                         // as few instructions as can be: waiting warps share the issue slots
            if (ax_mbar_try(bar, parity)) return true;
        if (flags[0]) return false;
        if (flags[1]) t0 = 0;
        const unsigned long long t = ax_globaltimer();
        if (t0 == 0) t0 = t;
        else if (t - t0 > WAIT_MS * 1000000ull) { flags[0] = 1; atomicExch(err, code); return false; }
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

// A pair of query tiles: rows [q0, q0 + lq) and keys [k0, k0 + lk) of its sequence, first row of the pair, first head.  lq < 0: no more.
struct Item { int q0, lq, k0, lk, base, h0; };
// What every role derives from it.
struct Work {
    AxPromptSeq s;
    int off, h0, base0, base1;                    // key at a query's own position = row + off
    int lo0, hi0, lo1, hi1, j0, j1;               // K / V tiles [lo, hi] of both query tiles, and of the pair; hi < lo: none
    bool on0, on1, cut;                           // cut: the last V tile reaches behind the sequence
};
__device__ __forceinline__ Work work_of(const PromptDev& dv, const Item& it) {
    Work w;
    w.s.q0 = it.q0; w.s.lq = it.lq; w.s.k0 = it.k0; w.s.lk = it.lk;
    w.off = it.lk - it.lq; w.h0 = it.h0;
    w.base0 = it.base; w.base1 = dv.pair_heads ? it.base : it.base + kRows;
    auto range = [&](int base, int& lo, int& hi) {
        const int last = min(base + kRows, it.lq) - 1 + w.off, first = base + w.off;
        lo = 0; hi = -1;
        if (base < it.lq && last >= 0 && it.lk > 0) {
            lo = dv.a.window > 0 && first - dv.a.window + 1 > 0 ? (first - dv.a.window + 1) / kRows : 0;
            hi = last / kRows;
        }
    };
    range(w.base0, w.lo0, w.hi0); range(w.base1, w.lo1, w.hi1);
    w.on0 = w.hi0 >= w.lo0; w.on1 = w.hi1 >= w.lo1;
    w.j0 = w.on0 ? (w.on1 ? min(w.lo0, w.lo1) : w.lo0) : w.lo1;
    w.j1 = max(w.hi0, w.hi1);
    if (w.j1 < w.j0) w.j1 = w.j0 - 1;
    w.cut = w.j1 >= w.j0 && (w.j1 + 1) * kRows > it.lk;
    return w;
}

template <bool F16, int HD, int WAIT_MS>
__global__ void __launch_bounds__(kThreads, 1) ax_prompt_umma_kernel(const __grid_constant__ CUtensorMap map_q,
                                                                     const __grid_constant__ CUtensorMap map_k,
                                                                     const __grid_constant__ CUtensorMap map_v, const PromptDev dv) {
    using T = typename std::conditional<F16, __half, uint16_t>::type;
    constexpr int BOXES = HD / 64, TILE = BOXES * kBoxBytes, NS = HD == 128 ? 5 : 6;
    constexpr uint32_t kS = 0, kO = 256;                                      // columns: scores of tile t at 128 t (its probabilities over the first half), output at 256 + HD t
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t q_full[2], q_empty[2], s_full[2], p_ready[2][2], o_done[2], o_free[2], kv_full[kMaxStages], kv_empty[kMaxStages],
        v_here, v_cut, i_full[kSlots], i_empty[kSlots], clc_bar;
    __shared__ __align__(16) uint4 s_clc;
    __shared__ __align__(16) Item s_item[kSlots];
    __shared__ uint32_t s_tmem;
    __shared__ int s_flags[2], s_issued;
    const int tid = threadIdx.x, warp = __shfl_sync(AX_FULL, tid >> 5, 0), lane = tid & 31;
    const AxPromptArgs& a = dv.a;
    volatile int* flags = s_flags;
    const uint32_t smem0 = (ax_smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t ring = smem0 + 2 * TILE;

    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(ax_smem_u32(&q_full[i]), 1); mbar_init(ax_smem_u32(&q_empty[i]), 1); mbar_init(ax_smem_u32(&s_full[i]), 1);
            mbar_init(ax_smem_u32(&o_done[i]), 1); mbar_init(ax_smem_u32(&o_free[i]), kRows);
            for (int b = 0; b < 2; b++) mbar_init(ax_smem_u32(&p_ready[i][b]), kRows);
        }
        for (int i = 0; i < NS; i++) { mbar_init(ax_smem_u32(&kv_full[i]), 1); mbar_init(ax_smem_u32(&kv_empty[i]), 1); }
        for (int i = 0; i < kSlots; i++) { mbar_init(ax_smem_u32(&i_full[i]), 1); mbar_init(ax_smem_u32(&i_empty[i]), kReaders); }
        mbar_init(ax_smem_u32(&v_here), 1); mbar_init(ax_smem_u32(&v_cut), 1); mbar_init(ax_smem_u32(&clc_bar), 1);
        s_flags[0] = s_flags[1] = 0; s_issued = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (tid == kCopy * 32) {
        for (const CUtensorMap* map : { &map_q, &map_k, &map_v }) asm volatile("prefetch.tensormap [%0];" :: "l"(map) : "memory");
    }
    if (warp == kProduct) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(ax_smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;
    // the n-th item of this CTA, for every reader in turn; false: no more
    auto item_at = [&](int n, Item& it) {
        const int slot = n % kSlots;
        if (!mbar_wait<WAIT_MS>(ax_smem_u32(&i_full[slot]), (uint32_t)(n / kSlots) & 1u, flags, dv.err, 731)) return false;
        it = *const_cast<const Item*>(&s_item[slot]);
        return it.lq >= 0;
    };
    auto item_read = [&](int n) { mbar_arrive(ax_smem_u32(&i_empty[n % kSlots])); };

    // 384 threads start with 168 registers each (64512 in all); a row of scores is 128 of them.  256 · 208 + 128 · 80 = 63488.
    if (warp >= kProduct) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == kItems) {
        // Tiles of the sequences before each lane's share of them; then item after item: its tile counted from the pack's end.
        const int tb = dv.pair_heads ? kRows : 2 * kRows, hx = dv.pair_heads ? a.n_heads / 2 : a.n_heads;
        const int per = (a.batch + 31) / 32, b0 = min(lane * per, a.batch), b1 = min(b0 + per, a.batch);
        long long own = 0;                                                    // 64 bits: prefix arrays that overlap may name more rows than there are
        AxPromptSeq held = {};                                                // the lane's sequence where it has one at most
        for (int b = b0; b < b1; b++) { held = ax_prompt_seq(a, b); own += (held.lq + tb - 1) / tb; }
        long long inc = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const long long x = __shfl_up_sync(AX_FULL, inc, d); if (lane >= d) inc += x; }
        const long long before = inc - own, all = __shfl_sync(AX_FULL, inc, 31);
        long long block = blockIdx.x;                                         // the CTA whose item is next
        int n = 0;
        uint32_t clc_phase = 0;
        bool ok = true, more = true;
        while (ok && more) {
            // ask for the next CTA's place while this one's item is looked up
            if (lane == 0) {
                mbar_expect_tx(ax_smem_u32(&clc_bar), 16);
                asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                             :: "r"(ax_smem_u32(&s_clc)), "r"(ax_smem_u32(&clc_bar)) : "memory");
            }
            __syncwarp();
            const long long x = all - 1 - block / hx;
            if (x >= 0) {
                const int g = 31 - __clz((int)__ballot_sync(AX_FULL, x >= before && own > 0));       // the lane in whose share the tile lies
                long long at = __shfl_sync(AX_FULL, before, g);
                const int c0 = min(g * per, a.batch), c1 = min(c0 + per, a.batch);
                Item it = {};
                for (int c = c0; c < c1; c += 32) {
                    const int b = c + lane;
                    AxPromptSeq q = {};
                    if (per == 1) { if (lane == g) q = held; }
                    else if (b < c1) q = ax_prompt_seq(a, b);
                    const int mine = (q.lq + tb - 1) / tb;
                    int up = mine;
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) { const int y = __shfl_up_sync(AX_FULL, up, d); if (lane >= d) up += y; }
                    const unsigned hit = __ballot_sync(AX_FULL, x >= at + up - mine && x < at + up);
                    if (hit) {
                        const int l = __ffs(hit) - 1;
                        it.q0 = __shfl_sync(AX_FULL, q.q0, l); it.lq = __shfl_sync(AX_FULL, q.lq, l);
                        it.k0 = __shfl_sync(AX_FULL, q.k0, l); it.lk = __shfl_sync(AX_FULL, q.lk, l);
                        it.base = (int)(x - __shfl_sync(AX_FULL, at + up - mine, l)) * tb;
                        break;
                    }
                    at += __shfl_sync(AX_FULL, up, 31);
                }
                it.h0 = (int)(block % hx) * (dv.pair_heads ? 2 : 1);
                if (n >= kSlots) ok = mbar_wait<WAIT_MS>(ax_smem_u32(&i_empty[n % kSlots]), (uint32_t)(n / kSlots - 1) & 1u, flags, dv.err, 732);
                ok = __all_sync(AX_FULL, ok);
                if (ok && lane == 0) { s_item[n % kSlots] = it; mbar_arrive(ax_smem_u32(&i_full[n % kSlots])); }
                n++;
            }
            bool got = mbar_wait<WAIT_MS>(ax_smem_u32(&clc_bar), clc_phase, flags, dv.err, 733);
            if (!__all_sync(AX_FULL, got)) { ok = false; break; }
            clc_phase ^= 1u;
            uint32_t took, next;
            asm volatile("{\n\t.reg .b128 r;\n\t.reg .pred p;\n\tld.shared.b128 r, [%2];\n\t"
                         "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
                         "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
                         : "=r"(took), "=r"(next) : "r"(ax_smem_u32(&s_clc)) : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // read before the next answer is written
            __syncwarp();
            more = took != 0;
            block = next;
        }
        if (ok) {
            if (n >= kSlots) ok = mbar_wait<WAIT_MS>(ax_smem_u32(&i_empty[n % kSlots]), (uint32_t)(n / kSlots - 1) & 1u, flags, dv.err, 732);
            if (__all_sync(AX_FULL, ok) && lane == 0) { s_item[n % kSlots].lq = -1; mbar_arrive(ax_smem_u32(&i_full[n % kSlots])); }
        }
        __syncwarp();
    } else if (warp == kCopy) {
        if (elect_one()) {
            Item it;
            int st = 0, nq[2] = { 0, 0 };
            uint32_t ph = 1;                                                  // a fresh barrier counts as a phase of parity one that is over
            bool ok = true;
            for (int n = 0; ok && item_at(n, it); n++) {
                item_read(n);
                const Work w = work_of(dv, it);
                const int kh = w.h0 / (a.n_heads / a.n_kv);
                auto query = [&](int t) {
                    ok = mbar_wait<WAIT_MS>(ax_smem_u32(&q_empty[t]), (uint32_t)(nq[t] + 1) & 1u, flags, dv.err, 734);
                    if (!ok) return;
                    nq[t]++;
                    const uint32_t bar = ax_smem_u32(&q_full[t]);
                    mbar_expect_tx(bar, TILE);
                    for (int b = 0; b < BOXES; b++)
                        tma_load_3d(smem0 + t * TILE + b * kBoxBytes, &map_q, b * 64, dv.pair_heads ? w.h0 + t : w.h0, w.s.q0 + (t ? w.base1 : w.base0), bar);
                };
                // The first K tile goes ahead of the queries: their places are free only when the item before has its last scores.
                const int m = 2 * (w.j1 - w.j0 + 1);
                for (int i = 0; i < m && ok; i++) {
                    ok = mbar_wait<WAIT_MS>(ax_smem_u32(&kv_empty[st]), ph, flags, dv.err, 721);
                    if (!ok) break;
                    const uint32_t bar = ax_smem_u32(&kv_full[st]);
                    mbar_expect_tx(bar, TILE);
                    const CUtensorMap* map = i & 1 ? &map_v : &map_k;
                    const bool lost = WAIT_MS == kTestWaitMs && dv.lose && blockIdx.x == 0 && n == 0 && i == 2;
                    for (int b = 0; b < BOXES && !lost; b++) tma_load_3d(ring + st * TILE + b * kBoxBytes, map, b * 64, kh, w.s.k0 + (w.j0 + i / 2) * kRows, bar);
                    s_issued++;
                    if (++st == NS) { st = 0; ph ^= 1u; }
                    if (i == 0) { if (w.on0) query(0); if (ok && w.on1) query(1); }
                }
            }
        }
        __syncwarp();
    } else if (warp == kProduct) {
        constexpr uint32_t fmt = F16 ? 0u : 1u;                               // accumulator f32, A and B f16 or bf16; B of P·V is MN-major
        constexpr uint32_t id_qk = (1u << 4) | (fmt << 7) | (fmt << 10) | ((kRows >> 3) << 17) | ((kRows >> 4) << 24);
        constexpr uint32_t id_pv = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((HD >> 3) << 17) | ((kRows >> 4) << 24);
        // One thread does all of it.  Its loops count from zero and tensor memory starts at column zero (all of it is ours), so that stages,
        // descriptors and columns are uniform values: with a vector register behind each, issuing a product took longer than the product.
        if (elect_one()) {
            bool ok = s_tmem == 0;
            if (!ok) { flags[0] = 1; atomicExch(dv.err, 728); }
            auto qk = [&](int t, int st) {                                    // scores of query tile t with the K tile in stage st
                const uint32_t k = desc_k(ring) + (uint32_t)st * (TILE >> 4), q = desc_k(smem0) + (uint32_t)t * (TILE >> 4);
                umma_ss<false>(kS + t * 128, q, k, id_qk);
#pragma unroll
                for (int i = 1; i < HD / 16; i++)
                    umma_ss<true>(kS + t * 128, q + (i / 4) * (kBoxBytes >> 4) + (i % 4) * 2, k + (i / 4) * (kBoxBytes >> 4) + (i % 4) * 2, id_qk);
                umma_commit(ax_smem_u32(&s_full[t]));
            };
            int st = 0;                                                       // stages are taken in turn; ph: parity of their phase
            uint32_t ph = 0, pq[2] = { 0, 0 }, pp[2] = { 0, 0 }, cuts = 0;    // parities of a tile's queries and probabilities, of the cuts
            int items[2] = { 0, 0 };                                          // items a tile took part in
            auto next = [&] { if (++st == NS) { st = 0; ph ^= 1u; } };
            Item it;
            for (int ni = 0; ok && item_at(ni, it); ni++) {
                item_read(ni);
                const Work w = work_of(dv, it);
                const int n = w.j1 - w.j0 + 1, a0 = w.lo0 - w.j0, z0 = w.on0 ? w.hi0 - w.j0 : -1, a1 = w.lo1 - w.j0, z1 = w.on1 ? w.hi1 - w.j0 : -1;
                if (n <= 0) continue;
                ok = mbar_wait<WAIT_MS>(ax_smem_u32(&kv_full[st]), ph, flags, dv.err, 722);
#pragma unroll
                for (int t = 0; t < 2; t++)
                    if (ok && (t ? w.on1 : w.on0)) {
                        ok = mbar_wait<WAIT_MS>(ax_smem_u32(&q_full[t]), pq[t], flags, dv.err, 723);
                        pq[t] ^= 1u;
                        if (ok && (t ? a1 : a0) == 0) {
                            qk(t, st);
                            if ((t ? z1 : z0) == 0) umma_commit(ax_smem_u32(&q_empty[t]));
                        }
                    }
                if (!ok) break;
                umma_commit(ax_smem_u32(&kv_empty[st]));
                next();
                for (int i = 0; i < n && ok; i++) {
                    const int sv = st;
                    ok = mbar_wait<WAIT_MS>(ax_smem_u32(&kv_full[sv]), ph, flags, dv.err, 722);
                    if (ok && i == n - 1 && w.cut) {
                        mbar_arrive(ax_smem_u32(&v_here));
                        ok = mbar_wait<WAIT_MS>(ax_smem_u32(&v_cut), cuts & 1u, flags, dv.err, 729);
                        cuts++;
                    }
                    if (!ok) break;
                    next();
                    const int sk = st;
                    const uint32_t vd = desc_mn(ring) + (uint32_t)sv * (TILE >> 4);
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const int at = t ? a1 : a0, zt = t ? z1 : z0;
                        if (ok && i >= at && i <= zt) {
                            // the item before has been read out of the accumulator
                            if (i == at && items[t] > 0) ok = mbar_wait<WAIT_MS>(ax_smem_u32(&o_free[t]), (uint32_t)(items[t] - 1) & 1u, flags, dv.err, 735);
                            if (i == at) items[t]++;
#pragma unroll
                            for (int part = 0; part < 2; part++) {            // the product starts with the first probabilities
                                ok = ok && mbar_wait<WAIT_MS>(ax_smem_u32(&p_ready[t][part]), pp[t], flags, dv.err, 724);
                                if (!ok) break;
                                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                                for (int c = part ? kFirst / 16 : 0; c < (part ? kRows : kFirst) / 16; c++)
                                    umma_ts(kO + t * HD, kS + t * 128 + c * 8, vd + c * (2048 >> 4), id_pv, c ? 1u : (uint32_t)(i != at));
                            }
                            pp[t] ^= 1u;
                            if (ok) umma_commit(ax_smem_u32(&o_done[t]));
                        }
                        if (ok && i + 1 >= at && i + 1 <= zt) {               // over the scores and probabilities just used
                            ok = mbar_wait<WAIT_MS>(ax_smem_u32(&kv_full[sk]), ph, flags, dv.err, 722);
                            if (ok) {
                                qk(t, sk);
                                if (i + 1 == zt) umma_commit(ax_smem_u32(&q_empty[t]));
                            }
                        }
                    }
                    if (!ok) break;
                    umma_commit(ax_smem_u32(&kv_empty[sv]));
                    if (i + 1 < n) { umma_commit(ax_smem_u32(&kv_empty[sk])); next(); }
                }
            }
        }
        __syncwarp();
    } else {
        // Value rows behind the sequence, in its last tile: zeros, so that whatever lies there meets a probability of zero as a number.
        Item it;
        int st = 0;
        uint32_t cuts = 0;
        bool ok = true;
        for (int n = 0; ok; n++) {
            ok = item_at(n, it);
            ok = __all_sync(AX_FULL, ok);
            if (!ok) break;
            __syncwarp();
            if (lane == 0) item_read(n);
            const Work w = work_of(dv, it);
            const int m = 2 * (w.j1 - w.j0 + 1);
            if (w.cut) {
                const int valid = w.s.lk - w.j1 * kRows;
                const uint32_t v = ring + (uint32_t)((st + m - 1) % NS) * TILE;
                ok = mbar_wait<WAIT_MS>(ax_smem_u32(&v_here), cuts & 1u, flags, dv.err, 730);       // told by the thread that saw it arrive
                ok = __all_sync(AX_FULL, ok);
                if (!ok) break;
                cuts++;
#pragma unroll
                for (int b = 0; b < BOXES; b++)
                    for (uint32_t at = valid * 128 + lane * 16; at < kBoxBytes; at += 512)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" :: "r"(v + b * kBoxBytes + at), "r"(0) : "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(ax_smem_u32(&v_cut));
            }
            st = (st + m) % NS;
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = warp >> 2;
        const uint32_t quarter = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t ts = quarter + kS + t * 128, to = quarter + kO + t * HD;
        const float sc = dv.sc;
        uint32_t ps = 0, po = 0;                                              // parities of the tile's scores and of its finished products
        Item item;
        bool ok = true;
        for (int ni = 0; ok; ni++) {
            ok = item_at(ni, item);
            ok = __all_sync(AX_FULL, ok);
            if (!ok) break;
            __syncwarp();
            if (lane == 0) item_read(ni);
            const Work w = work_of(dv, item);
            const int base = t ? w.base1 : w.base0, h = dv.pair_heads ? w.h0 + t : w.h0;
            const int row = base + (warp & 3) * 32 + lane, pos = row + w.off;              // row of the sequence, key at its own position
            const int j_lo = t ? w.lo1 : w.lo0, j_hi = t ? w.hi1 : w.hi0;
            const int key_hi = pos, key_lo = a.window > 0 ? pos - a.window : -1;           // visible: key_lo < j <= key_hi
            const int first = base + w.off, lastp = min(base + kRows, w.s.lq) - 1 + w.off; // positions of the tile's first and last row
            float m = -INFINITY;
            float2 l0 = make_float2(0.f, 0.f), l1 = l0;
            for (int j = j_lo; j <= j_hi; j++) {
                ok = mbar_wait<WAIT_MS>(ax_smem_u32(&s_full[t]), ps, flags, dv.err, 725);
                ok = __all_sync(AX_FULL, ok);
                if (!ok) break;
                ps ^= 1u;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t u[kRows];
                tmem_ld128(ts, u);
                float* x = reinterpret_cast<float*>(u);
                if (dv.negate) {
#pragma unroll
                    for (int c = 0; c < kRows; c++) x[c] = -x[c];
                }
                // What hides keys is looked at in blocks of 32, for the warp's 32 rows: most blocks of a tile on the diagonal are seen by all rows
                // or by none, and those that none sees need no exponentials.  (Two comparisons for each of 128 scores took 3000 clocks.)
                const int k0 = j * kRows;
                unsigned hidden = 0u;                                         // bit q: no row of the warp sees keys 32 q .. 32 q + 31
                if (k0 + kRows - 1 > first || (a.window > 0 && k0 <= lastp - a.window)) {
                    const int p0 = pos - lane, p1 = p0 + 31;
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int kq = k0 + 32 * q;
                        if (kq > p1 || (a.window > 0 && kq + 31 <= p0 - a.window)) {
                            hidden |= 1u << q;
#pragma unroll
                            for (int c = 0; c < 32; c++) x[32 * q + c] = -INFINITY;
                        } else {
                            if (kq + 31 > p0) {
#pragma unroll
                                for (int c = 0; c < 32; c++) if (c > key_hi - kq) x[32 * q + c] = -INFINITY;
                            }
                            if (a.window > 0 && kq <= p1 - a.window) {
#pragma unroll
                                for (int c = 0; c < 32; c++) if (c <= key_lo - kq) x[32 * q + c] = -INFINITY;
                            }
                        }
                    }
                }
                float mx[8];
#pragma unroll
                for (int c = 0; c < 8; c++) mx[c] = x[c];
#pragma unroll
                for (int c = 8; c < 120; c += 2) mx[(c >> 1) & 7] = ax_max3(mx[(c >> 1) & 7], x[c], x[c + 1]);
                const float top = ax_max3(ax_max3(ax_max3(mx[0], mx[1], mx[2]), ax_max3(mx[3], mx[4], mx[5]), ax_max3(mx[6], mx[7], x[120])),
                                       ax_max3(x[121], x[122], x[123]), ax_max3(ax_max3(x[124], x[125], x[126]), x[127], x[127]));
                if (top != top) m = top;                                      // a visible score is NaN: so is every probability from here on
                const bool grow = top > m && (m == -INFINITY || (top - m) * sc > 8.f);
                const bool started = j > j_lo;
                if (__any_sync(AX_FULL, grow)) {
                    const bool moved = grow && m != -INFINITY;                // a row that has seen nothing has sums and outputs of zero
                    const float f = moved ? ax_ex2((m - top) * sc) : 1.f;
                    if (grow) m = top;
                    l0.x *= f; l0.y *= f; l1.x *= f; l1.y *= f;
                    if (started && __any_sync(AX_FULL, moved)) {              // the products of the tile before are in: po is the parity they leave
                        ok = mbar_wait<WAIT_MS>(ax_smem_u32(&o_done[t]), po ^ 1u, flags, dv.err, 726);
                        ok = __all_sync(AX_FULL, ok);
                        if (!ok) break;
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
                // Probabilities are rounded to the type of V, half a step of themselves each, because both operands of a product have one type (hi and
                // lo parts would double the second product); their sum is that of the f32 numbers.  In f16 they are held 2^7 larger (at most 2^15, beside a
                // largest number of 2^16), so that what is lost of the small ones is below 2^-32 of the reference instead of 2^-25.
                const float neg = m == -INFINITY ? 0.f : F16 ? fmaf(-m, sc, 7.f) : -m * sc;
                const float2 sc2 = make_float2(sc, sc), neg2 = make_float2(neg, neg);
                auto probs = [&](int c0, bool some) {                                    // 32 keys
                    uint32_t p[16];
                    if (some && (hidden >> (c0 / 32) & 1u)) {
#pragma unroll
                        for (int c = 0; c < 16; c++) p[c] = 0u;
                    } else
#pragma unroll
                    for (int c = 0; c < 16; c++) {
                        float2 y = ax_fma2(make_float2(x[c0 + 2 * c], x[c0 + 2 * c + 1]), sc2, neg2);
                        y.x = ax_ex2(y.x); y.y = ax_ex2(y.y);
                        if (c & 1) l1 = ax_add2(l1, y); else l0 = ax_add2(l0, y);
                        p[c] = pack<F16>(y.x, y.y);
                    }
                    tmem_st16(ts + c0 / 2, p);
                };
                auto hand_over = [&](int part) {
                    tmem_wait_st();
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    mbar_arrive(ax_smem_u32(&p_ready[t][part]));
                };
                if (hidden) {
                    probs(0, true); probs(32, true);
                    hand_over(0);
                    probs(64, true); probs(96, true);
                    hand_over(1);
                } else {
                    probs(0, false); probs(32, false);
                    hand_over(0);
                    probs(64, false); probs(96, false);
                    hand_over(1);
                }
                po ^= 1u;
            }
            // ── output ──
            const bool any = j_hi >= j_lo;
            if (ok && any) {
                ok = mbar_wait<WAIT_MS>(ax_smem_u32(&o_done[t]), po ^ 1u, flags, dv.err, 727);
                ok = __all_sync(AX_FULL, ok);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            }
            if (!ok) break;
            const bool live = row < w.s.lq;
            const float l = (l0.x + l0.y) + (l1.x + l1.y);
            const float inv = l == 0.f ? 0.f : 1.f / l;
            float odd = 0.f;                                                  // becomes NaN with the first output that is not finite
            T* out = (T*)a.out + (long long)(w.s.q0 + row) * a.o_tok + (long long)h * a.o_head;
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                if (any) {
                    tmem_ld32(to + c, o);
                    if (c + 32 == HD) {                                       // the accumulator may take the next item's products
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        mbar_arrive(ax_smem_u32(&o_free[t]));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = 0u;
                }
                uint32_t pk[16];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const float x0 = __uint_as_float(o[2 * e]) * inv, x1 = __uint_as_float(o[2 * e + 1]) * inv;
                    odd = fmaf(x0, 0.f, fmaf(x1, 0.f, odd));
                    pk[e] = pack<F16>(x0, x1);
                }
                if (live) {
                    if (dv.wide) {                                            // whole sectors
#pragma unroll
                        for (int e = 0; e < 2; e++)
                            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                                         :: "l"(out + c + 16 * e), "r"(pk[8 * e]), "r"(pk[8 * e + 1]), "r"(pk[8 * e + 2]), "r"(pk[8 * e + 3]),
                                            "r"(pk[8 * e + 4]), "r"(pk[8 * e + 5]), "r"(pk[8 * e + 6]), "r"(pk[8 * e + 7]) : "memory");
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) *reinterpret_cast<uint4*>(out + c + 8 * e) = make_uint4(pk[4 * e], pk[4 * e + 1], pk[4 * e + 2], pk[4 * e + 3]);
                    }
                }
            }
            const bool sees = key_hi >= 0 && w.s.lk > 0;
            // a visible score that is NaN makes the row NaN, as it is already
            unsigned again = __ballot_sync(AX_FULL, live && m == m && (odd != odd || (sees && !(fabsf(m) <= 3.402823466e38f))));
            __syncwarp();
            if (again) {
            if (lane == 0) atomicAdd(&s_flags[1], 1);
            while (again) {
                const int i = __ffs(again) - 1;
                again &= again - 1;
                row_again<T, HD>(a, w.s, h, base + (warp & 3) * 32 + i, lane);
            }
            if (lane == 0) atomicAdd(&s_flags[1], -1);
            }
        }
    }

    // ── tail: nothing of this CTA may still be in flight when its shared and tensor memory go away ──
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (s_flags[0]) {
        if (tid == 0) {                                                       // copies issued into stages nobody consumed any more
            const int issued = s_issued;
            for (int i = issued > NS ? issued - NS : 0; i < issued; i++) {
                const unsigned long long t0 = ax_globaltimer();
                while (!ax_mbar_try(ax_smem_u32(&kv_full[i % NS]), (uint32_t)(i / NS) & 1u) && ax_globaltimer() - t0 < kAbortNs) { }
            }
        }
        if (tid == 32) {                                                      // queries, products and an answer asked for before the failure: time to land
            const unsigned long long t0 = ax_globaltimer();
            while (ax_globaltimer() - t0 < kAbortNs) { }
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
    const cuuint64_t strides[2] = { (cuuint64_t)head * 2, (cuuint64_t)tok * 2 };
    const cuuint32_t box[3] = { 64, 1, kRows }, step[3] = { 1, 1, 1 };
    const CUresult r = fn(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(data), dims, strides,
                          box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return atlasx_fail(ATLASX_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)r);
    return ATLASX_OK;
}

template <bool F16, int HD, int WAIT_MS = kWaitMs>
int launch(atlasx_ctx* ctx, const PromptDev& dv, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v) {
    constexpr int smem = (2 + (HD == 128 ? 5 : 6)) * (HD / 64) * kBoxBytes + 1024;
    static std::atomic<bool> ready[64] = {};
    if (ctx->device >= 64 || !ready[ctx->device]) {                           // the limit is per device; asking twice does no harm
        AX_CUDA(cudaFuncSetAttribute(ax_prompt_umma_kernel<F16, HD, WAIT_MS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        if (ctx->device < 64) ready[ctx->device] = true;
    }
    const int tb = dv.pair_heads ? kRows : 2 * kRows;
    // at most one unfilled tile per sequence, and no more sequences with rows than rows
    const long long tiles = (long long)dv.a.n_q / tb + (dv.a.batch < dv.a.n_q ? dv.a.batch : dv.a.n_q);
    const long long items = tiles * (dv.pair_heads ? dv.a.n_heads / 2 : dv.a.n_heads);
    AX_ARG(items <= 0x7FFFFFFFll, "too many rows and heads for one call");
    ax_prompt_umma_kernel<F16, HD, WAIT_MS><<<(unsigned)items, kThreads, smem, ctx->stream>>>(q, k, v, dv);
    AX_CHECK_LAUNCH("ax_prompt_umma_kernel");
    return ATLASX_OK;
}

}  // namespace

extern "C" int atlasx_prompt_attention(atlasx_ctx* c, const atlasx_prompt_args* p) {
    AX_ARG(p, "null argument");
    const void *q = p->q, *k = p->k, *v = p->v;
    void* out = p->out;
    long long q_tok = p->q_token_stride, q_head = p->q_head_stride, k_tok = p->k_token_stride, k_head = p->k_head_stride,
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
    // a stride that is never taken may be anything the caller has: of one row, of one head
    if (n_q == 1) q_tok = o_tok = (long long)n_heads * hd;
    if (n_k <= 1) k_tok = v_tok = (long long)n_kv * hd;
    if (n_heads == 1) q_head = o_head = hd;
    if (n_kv == 1 || n_k == 0) k_head = v_head = hd;
    AX_ARG(q && out && cu_q && cu_k && ((k && v) || n_k == 0), "null argument");
    AX_ARG(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) % 16 == 0 &&
           (q_tok | q_head | k_tok | k_head | v_tok | v_head | o_tok | o_head) % 8 == 0, "rows must start on 16-byte boundaries");
    AX_ARG(q_tok >= 0 && q_head >= 0 && k_tok >= 0 && k_head >= 0 && v_tok >= 0 && v_head >= 0, "strides must not be negative");
    AX_ARG(q_head > 0 && k_head > 0 && v_head > 0 && q_tok > 0 && k_tok > 0 && v_tok > 0, "strides must not be zero");
    // all heads of a row before the next row, or all rows of a head before the next head
    AX_ARG(o_head >= hd && o_tok >= hd && o_tok < (1ll << 38) && o_head < (1ll << 38) &&
           (n_q == 1 || n_heads == 1 || o_tok >= (n_heads - 1) * o_head + hd || o_tok <= (o_head - hd) / (n_q - 1)), "rows of out overlap");
    AX_ARG(q_tok < (1ll << 38) && q_head < (1ll << 38) && k_tok < (1ll << 38) && k_head < (1ll << 38) && v_tok < (1ll << 38) && v_head < (1ll << 38),
           "strides must be below 2^38");
    AX_ARG(c, "ctx is null");
    AX_ON_DEVICE(c);
    PromptDev dv = {};
    dv.a = { q, k, v, out, q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head, cu_q, cu_k, batch, n_q, n_k, n_heads, n_kv, hd,
             window < n_k ? window : 0, scale };                              // no key lies further behind a query, and "position − window" stays within 32 bits
    dv.pair_heads = (n_heads / n_kv) % 2 == 0;
    dv.negate = scale < 0.f;
    dv.wide = (uintptr_t)out % 32 == 0 && o_tok % 16 == 0 && o_head % 16 == 0;
    // a hidden key's score is −inf · sc: a scale of zero must not make it NaN.  Scores below 2^126 / 1e37 of it are still all alike.
    dv.sc = fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-37f);
    dv.err = c->dev_error;
    dv.lose = c->tune.prompt_short_waits == 2;
    const bool f16 = dtype == ATLASX_F16;
    CUtensorMap mq, mk, mv;
    int rc = make_map(&mq, f16, q, n_q, n_heads, hd, q_tok, q_head);
    if (!rc && n_k > 0) rc = make_map(&mk, f16, k, n_k, n_kv, hd, k_tok, k_head);
    if (!rc && n_k > 0) rc = make_map(&mv, f16, v, n_k, n_kv, hd, v_tok, v_head);
    if (rc) return rc;
    if (n_k == 0) mk = mv = mq;                                               // never read: no sequence has keys
    if (c->tune.prompt_short_waits && !f16 && hd == 64) return launch<false, 64, kTestWaitMs>(c, dv, mq, mk, mv);
    if (f16) return hd == 128 ? launch<true, 128>(c, dv, mq, mk, mv) : launch<true, 64>(c, dv, mq, mk, mv);
    return hd == 128 ? launch<false, 128>(c, dv, mq, mk, mv) : launch<false, 64>(c, dv, mq, mk, mv);
}
