// attention_paged.cu — attention of one new token per request over the four-bit paged cache.
//
// What has to move is rows · n_kv · 2 · (hd / 2 + 2 · hd / group) bytes; at the copy bandwidth a tile (16 rows of one KV head,
// 2304 bytes at hd 128, group 32) leaves an SM about 100 clocks.  Unpacking 4096 nibbles, two products with four-times-replicated
// work for f32 accuracy and a softmax in that time is what the kernel is shaped by:
//   * Work is cut evenly: the units (two tiles, 32 rows) of all (request, KV head) segments form one sequence, every warp takes a
//     contiguous piece of it, whatever the lengths are.  Nothing of it is decided on the host, so a captured call follows the lengths.
//   * A unit is one bulk copy (two where its tiles lie in different pages) into the warp's own ring; no barrier of the CTA in the loop.
//   * S = Q·Kᵀ and O = P·V run as mma.m16n8k16 with the (up to eight) query heads of a KV head as rows: rows 0..7 hold the f16
//     hi parts, rows 8..15 the lo parts of the same f32 values, so one instruction gives both and the sum of two accumulators
//     is good to 2^-22 of each value (bf16 halves left 4e-6 of the output, 2^-16 of each value).  The score accumulators are
//     already the operand layout of the second product.  f16 has little range, so a head's query is brought to 2^14 by a power
//     of two, and the softmax reference follows the largest p · scale of V instead of the largest p: what a group of V holds is exact to 2^-32 of
//     the row's largest p · |v|, whatever the size of V is (groups of zeros are stored with the smallest scale; with scales of V
//     above 2^90 rows whose weight is below 2^-133 of the scale are lost, their p being below the range of f32).
//   * A nibble u (the number plus eight) becomes an f16 number by mask-and-or and one exact operation: 1024 + u − 1032, or, four
//     bits up, (1024 + 16u) / 16 − 72: nine instructions for eight numbers.  (A masked nibble of K as the f16 subnormal it
//     is, with −8 · Σq as the accumulators' start, takes 62.5 µs instead of 64.9 for 12 windowed requests and 118 instead of 120 for
//     64 × 8k, but its error against 64 bits is 2.6e-6 instead of 0.4e-6; for V, too, the sum of the numbers over a long context is far
//     smaller than that of their offsets.)  The scale of (row, group) multiplies the group's finished score; the scale of V
//     goes into P.
//   * Segments that end inside a warp's piece are written from registers; the others meet in shared memory, and where they
//     reach over CTAs in the workspace, added up by the last CTA to arrive, in the order of the pieces: no result depends on timing.
#include <atomic>

#include "paged.cuh"

namespace {

constexpr int kWarps = 4;
constexpr int kStages = 2;
constexpr int kCtasPerSm = 3;
constexpr int kUnit = 2;                        // tiles that a warp takes at a time (one where there are not two for each warp: 1 × 700 rows
                                                // take 13 µs so, with two 15.7)
constexpr int kHeads = 8;                       // query heads of one segment
constexpr int kChunk = 64;                      // parts of a segment whose weights are in shared memory at a time
constexpr unsigned long long kWaitNs = 2000000000ull, kSelftestWaitNs = 20000000ull;
constexpr int kErrWait = 741;

struct PagedDev {
    AxP4Shape s;
    const uint8_t* pool;
    AxPagedAttnArgs a;
    int group_heads, head_tiles, nh;            // query heads per KV head, segments per KV head, segments per request
    int hpt;                                    // heads per segment: min(8, group_heads)
    unsigned* tickets;                          // [gridDim] zero between launches
    float* part_ml;                             // [2 · gridDim][hpt][2]
    float* part_o;                              // [2 · gridDim][hpt][hd]
    int *err, *index_err;
    long long lost;                             // self-test: the unit whose copy is never issued
};

struct UnitInfo { int seg, tile, ok, pad; };     // segment, first tile, bit u: tile + u is there


// Bounded, and the same answer for all lanes of the warp: one that saw the copy land just as the others gave up would wait for them for good.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, unsigned long long ns) {
    if (__all_sync(AX_FULL, ax_mbar_try(bar, parity))) return true;
    const unsigned long long t0 = ax_globaltimer();
    for (;;) {
        if (__all_sync(AX_FULL, ax_mbar_try(bar, parity))) return true;
        if (__any_sync(AX_FULL, ax_globaltimer() - t0 > ns)) return false;
    }
}
__device__ __forceinline__ float lg2(float x) { float y; asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {         // round to nearest
    uint32_t r; asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo)); return r;
}
__device__ __forceinline__ float2 unpack_f16(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t r; asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(bits)); return r;
}
// the two numbers whose nibbles lie in the low bits of the halves of a word, or four bits up
__device__ __forceinline__ uint32_t n_low(uint32_t w) {
    uint32_t r; asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(and_or(w, 0x000F000Fu, 0x64006400u)), "r"(0x64086408u)); return r;
}
__device__ __forceinline__ uint32_t n_high(uint32_t w) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(and_or(w, 0x00F000F0u, 0x64006400u)), "r"(0x2C002C00u), "r"(0xD480D480u));
    return r;
}
__device__ __forceinline__ void mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
template <int N> __device__ __forceinline__ void lds(uint32_t (&r)[N], const void* p) {
    if constexpr (N == 4) { const uint4 v = *(const uint4*)p; r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w; }
    else if constexpr (N == 2) { const uint2 v = *(const uint2*)p; r[0] = v.x; r[1] = v.y; }
    else r[0] = *(const uint32_t*)p;
}

// visible rows of a request: [lo, len)
__device__ __forceinline__ void row_range(const PagedDev& dv, int b, int& lo, int& len) {
    len = max(0, (int)min((long long)dv.a.lens[b], (long long)dv.a.table_width * dv.s.page_size));
    lo = dv.a.window > 0 && len > dv.a.window ? len - dv.a.window : 0;
}
__device__ __forceinline__ unsigned tiles_of(int lo, int len) {
    return len > lo ? (unsigned)((len + AX_P4_TILE - 1) / AX_P4_TILE - lo / AX_P4_TILE) : 0u;
}

template <int HD, int GS, bool LOSE = false>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm) ax_paged_attn_kernel(const PagedDev dv) {
    constexpr int W = HD / 32;                  // 32-bit words per lane, row block and plane
    constexpr int NG = HD / GS;                 // groups of a row
    constexpr int WG = GS / 32;                 // words per group
    constexpr int PLANE = AX_P4_TILE * HD / 2, SC = AX_P4_TILE * NG * 2, TILE = 2 * (PLANE + SC);
    constexpr int NT = HD / 8;                  // column blocks of the output
    constexpr unsigned long long kNs = LOSE ? kSelftestWaitNs : kWaitNs;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t s_bar[kWarps][kStages];
    __shared__ __align__(16) UnitInfo s_info[kWarps][kStages];
    __shared__ unsigned s_scan[2][kWarps];
    __shared__ int s_seg[kWarps * 2];
    __shared__ float s_ml[kWarps * 2][kHeads][2];
    __shared__ int s_last, s_gave_up;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int batch = dv.a.batch, hpt = dv.hpt;
    // Shared memory: per warp its ring, its query operand, and the output of a first segment that ends within its piece; the output of the
    // last segment goes over the ring, which is empty by then.  Then [batch + 1] units before each request.
    constexpr int UNIT = kUnit * TILE, RING = kStages * UNIT, QBYTES = W * 2 * 32 * 16;
    const int own = RING + QBYTES + hpt * HD * 4;
    uint8_t* ring = smem + warp * own;
    uint4* s_q = reinterpret_cast<uint4*>(ring + RING);                                     // [step][lane]
    auto s_o = [&](int slot) { return reinterpret_cast<float*>(smem + (slot >> 1) * own + (slot & 1 ? 0 : RING + QBYTES)); };
    unsigned* s_pre = reinterpret_cast<unsigned*>(smem + kWarps * own);

    if (tid < kWarps * kStages) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(ax_smem_u32(&s_bar[tid / kStages][tid % kStages])) : "memory");
    if (tid < kWarps * 2) s_seg[tid] = -1;
    if (tid == 0) s_gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    int us;                                                                   // tiles of a unit: two, or one where that many warps would have none
    {   // exclusive sums of the requests' units
        const int per = (batch + kWarps * 32 - 1) / (kWarps * 32), b0 = min(tid * per, batch), b1 = min(b0 + per, batch);
        unsigned own = 0;
        for (int b = b0; b < b1; b++) { int lo, len; row_range(dv, b, lo, len); own += tiles_of(lo, len); }
        unsigned sum = own;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(AX_FULL, sum, d);
        if (lane == 0) s_scan[0][warp] = sum;
        __syncthreads();
        sum = 0;
#pragma unroll
        for (int w = 0; w < kWarps; w++) sum += s_scan[0][w];
        us = (long long)sum * dv.nh <= (long long)gridDim.x * kWarps ? 1 : kUnit;
        if (us > 1) {
            own = 0;
            for (int b = b0; b < b1; b++) { int lo, len; row_range(dv, b, lo, len); own += (tiles_of(lo, len) + kUnit - 1) / kUnit; }
        }
        unsigned inc = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const unsigned x = __shfl_up_sync(AX_FULL, inc, d); if (lane >= d) inc += x; }
        if (lane == 31) s_scan[1][warp] = inc;
        __syncthreads();
        unsigned at = inc - own;
#pragma unroll
        for (int w = 0; w < kWarps; w++) if (w < warp) at += s_scan[1][w];
        for (int b = b0; b < b1; b++) {
            int lo, len; row_range(dv, b, lo, len);
            s_pre[b] = at; at += (tiles_of(lo, len) + us - 1) / us;
            if (b == batch - 1) s_pre[batch] = at;
        }
        __syncthreads();
    }
    for (int b = blockIdx.x; b < batch; b += gridDim.x)                       // requests without rows
        if (s_pre[b] == s_pre[b + 1])
            for (int i = tid; i < dv.a.n_heads * HD; i += kWarps * 32) dv.a.out[(size_t)b * dv.a.n_heads * HD + i] = 0.f;
    const long long total = (long long)s_pre[batch] * dv.nh;
    const long long want = (total + kWarps - 1) / kWarps;
    const long long C = want < (long long)gridDim.x ? want : (long long)gridDim.x;        // CTAs that share the work
    const long long c = blockIdx.x;
    if (c >= C) return;
    const long long X0 = total * c / C, X1 = total * (c + 1) / C;
    const long long x0 = X0 + (X1 - X0) * warp / kWarps, x1 = X0 + (X1 - X0) * (warp + 1) / kWarps;

    // request, segment of the request and unit of the segment of unit y of the whole
    auto locate = [&](long long y, int& b, int& hh, int& ti) {
        int lo = 0, hi = batch;                                               // last b with s_pre[b] · nh <= y (skipping requests without rows)
        while (hi - lo > 1) { const int m = (lo + hi) >> 1; if ((long long)s_pre[m] * dv.nh <= y) lo = m; else hi = m; }
        const unsigned n = s_pre[lo + 1] - s_pre[lo];
        const long long rem = y - (long long)s_pre[lo] * dv.nh;
        if (total <= 0x7FFFFFFFll) { hh = (int)((unsigned)rem / n); ti = (int)((unsigned)rem % n); }
        else { hh = (int)(rem / n); ti = (int)(rem % n); }
        b = lo;
    };

    // ── the warp's stream of units: 32 positions are resolved at a time, one per lane, and lane i copies unit i of them ──
    const int count = (int)(x1 - x0);
    const uint8_t* src[kUnit] = {};
    UnitInfo mine = {};
    auto fill = [&](int i, int st) {                                          // i uniform over the warp, rising by one; st: its stage
        if (i >= count) return;
        if ((i & 31) == 0) {
            const long long y = x0 + i + lane;
            mine.seg = -1; mine.tile = 0; mine.ok = 0;
            if (y < x1) {
                int lo, hh, ti;
                locate(y, lo, hh, ti);
                int first, len; row_range(dv, lo, first, len);
                mine.seg = lo * dv.nh + hh;
                mine.tile = first / AX_P4_TILE + us * ti;
#pragma unroll
                for (int u = 0; u < kUnit; u++) {
                    const int row = (mine.tile + u) * AX_P4_TILE;
                    if (row >= len || u >= us) continue;
                    const int page = dv.a.table[(size_t)lo * dv.a.table_width + row / dv.s.page_size];
                    if (page >= 0 && page < dv.s.n_pages) {
                        mine.ok |= 1 << u;
                        src[u] = dv.pool + ax_p4_tile_at(dv.s, page, hh / dv.head_tiles, row % dv.s.page_size);
                    } else atomicExch(dv.index_err, AX_DEVERR_PAGE);
                }
            }
        }
        if (lane == (i & 31)) {
            const uint32_t bar = ax_smem_u32(&s_bar[warp][st]);
            s_info[warp][st] = mine;
            auto copy = [&](int u, uint32_t bytes) {
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                             :: "r"(ax_smem_u32(ring + st * UNIT + u * TILE)), "l"(src[u]), "r"(bytes), "r"(bar) : "memory");
            };
            const bool one = mine.ok == 3 && src[1] == src[0] + TILE;          // neighbours in a page
            if (mine.ok) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(mine.ok == 3 ? UNIT : TILE) : "memory");
            else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
            if (LOSE && x0 + i == dv.lost) { }
            else if (one) copy(0, UNIT);
            else {
                if (mine.ok & 1) copy(0, TILE);
                if (mine.ok & 2) copy(1, TILE);
            }
        }
    };
    for (int i = 0; i < kStages; i++) fill(i, i);
    __syncwarp();

    // ── state of the segment at hand ──
    float qback = 1.f;                          // the power of two that the query was divided by
    float o[NT][4], m = -INFINITY;
    float2 l = {};                              // sums of columns 2t and of 2t + 1
    int seg = -1, seg_lo = 0, seg_len = 0;
    auto start = [&](int s) {
        seg = s;
        const int b = s / dv.nh, hh = s % dv.nh, kh = hh / dv.head_tiles, h0 = (hh % dv.head_tiles) * kHeads;
        row_range(dv, b, seg_lo, seg_len);
        const bool live = h0 + g < dv.group_heads;
        const float* q = dv.a.q + ((size_t)b * dv.a.n_heads + (size_t)kh * dv.group_heads + h0 + g) * HD;
        const float f = dv.a.scale * 1.4426950408889634f;
        float x[W][8], big = 0.f;
#pragma unroll
        for (int w = 0; w < W; w++) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[w][i] = 0.f;
            if (live) {
                const float4 u = *(const float4*)(q + (w / WG) * GS + t * (GS / 4) + (w % WG) * 8);
                const float4 v = *(const float4*)(q + (w / WG) * GS + t * (GS / 4) + (w % WG) * 8 + 4);
                x[w][0] = u.x * f; x[w][1] = u.y * f; x[w][2] = u.z * f; x[w][3] = u.w * f;
                x[w][4] = v.x * f; x[w][5] = v.y * f; x[w][6] = v.z * f; x[w][7] = v.w * f;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(x[w][i]));
        }
        big = fmaxf(big, __shfl_xor_sync(AX_FULL, big, 1));
        big = fmaxf(big, __shfl_xor_sync(AX_FULL, big, 2));
        // 2^e brings the largest number into [2^14, 2^15); e stays where 2^e and 2^-e are normal numbers
        const int e = big > 0.f && big <= 3.402823466e38f ? min(max(14 - ((__float_as_int(big) >> 23) - 127), -126), 126) : 0;
        const float up = __int_as_float((e + 127) << 23);
        qback = __int_as_float((127 - e) << 23);
#pragma unroll
        for (int w = 0; w < W; w++)
#pragma unroll
            for (int h = 0; h < 2; h++) {                                      // step 2 · w + h: pairs (p, p + 4) of the word for p = 2h, 2h + 1
                uint32_t q4[4];
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    const float y0 = x[w][2 * h + p] * up, y1 = x[w][2 * h + p + 4] * up;
                    q4[2 * p] = pack_f16(y0, y1);
                    const float2 r = unpack_f16(q4[2 * p]);
                    q4[2 * p + 1] = pack_f16(y0 - r.x, y1 - r.y);
                }
                s_q[(2 * w + h) * 32 + lane] = make_uint4(q4[0], q4[1], q4[2], q4[3]);      // read by this lane alone
            }
#pragma unroll
        for (int i = 0; i < NT; i++) { o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f; }
        m = -INFINITY; l = make_float2(0.f, 0.f);
    };
    // Column n = 2t, 2t + 1 of column block gr · (GS / 8) + i is number gr · GS + n · (GS / 8) + i: a lane holds GS / 4 consecutive numbers
    // of every group.
    auto put = [&](float* dst, float f) {
#pragma unroll
        for (int gr = 0; gr < NG; gr++)
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < GS / 8; i += 4) {
                    float4 v;
                    v.x = (o[gr * (GS / 8) + i][n] + o[gr * (GS / 8) + i][n + 2]) * f;
                    v.y = (o[gr * (GS / 8) + i + 1][n] + o[gr * (GS / 8) + i + 1][n + 2]) * f;
                    v.z = (o[gr * (GS / 8) + i + 2][n] + o[gr * (GS / 8) + i + 2][n + 2]) * f;
                    v.w = (o[gr * (GS / 8) + i + 3][n] + o[gr * (GS / 8) + i + 3][n + 2]) * f;
                    *(float4*)(dst + gr * GS + (2 * t + n) * (GS / 8) + i) = v;
                }
    };
    auto flush = [&]() {
        const int b = seg / dv.nh, hh = seg % dv.nh, kh = hh / dv.head_tiles, h0 = (hh % dv.head_tiles) * kHeads;
        const unsigned n = s_pre[b + 1] - s_pre[b];
        const long long s0 = (long long)s_pre[b] * dv.nh + (long long)hh * n;
        float sum = l.x + l.y;
        sum += __shfl_xor_sync(AX_FULL, sum, 1);
        sum += __shfl_xor_sync(AX_FULL, sum, 2);
        const bool live = h0 + g < dv.group_heads;
        if (s0 >= x0 && s0 + n <= x1) {
            if (live) put(dv.a.out + ((size_t)b * dv.a.n_heads + (size_t)kh * dv.group_heads + h0 + g) * HD, sum == 0.f ? 0.f : 1.f / sum);
        } else {
            const int slot = warp * 2 + (s0 < x0 ? 0 : 1);
            if (lane == 0) s_seg[slot] = seg;
            if (t == 0) { s_ml[slot][g][0] = m; s_ml[slot][g][1] = sum; }
            if (live) put(s_o(slot) + g * HD, 1.f);
        }
    };

    int st = 0, it = 0;
    uint32_t phase = 0;
    for (; it < count; it++) {
        const UnitInfo info = s_info[warp][st];
        // known before the unit is here: a new segment's query comes under its copy
        if (info.seg != seg) { if (seg >= 0) flush(); start(info.seg); }
        if (!mbar_wait(ax_smem_u32(&s_bar[warp][st]), phase, kNs)) break;
        if (info.ok) {
            // Both tiles side by side: their chains — scores, softmax, products — are each other's cover.  (One tile at a time left 54 % of the
            // issue slots and 41 % of the busiest pipe in use.)
            const uint8_t* unit = ring + st * UNIT;
            float2 s[kUnit][2] = {};                                          // columns 2t, 2t + 1 of row block nt
            float2 vs[kUnit][2][NG];                                          // scales of V of the lane's four rows
            {
                uint32_t kw[kUnit][2][W], ks[kUnit][2][NG];
#pragma unroll
                for (int u = 0; u < kUnit; u++)
#pragma unroll
                    for (int nt = 0; nt < 2; nt++) {
                        lds<W>(kw[u][nt], unit + u * TILE + nt * (PLANE / 2) + lane * W * 4);
                        lds<NG>(ks[u][nt], unit + u * TILE + 2 * PLANE + (8 * nt + 2 * t) * NG * 2);
                    }
#pragma unroll
                for (int gr = 0; gr < NG; gr++) {
                    float d[kUnit][2][4] = {};
#pragma unroll
                    for (int i = 0; i < WG; i++) {
                        const uint4 q0 = s_q[(2 * (gr * WG + i)) * 32 + lane], q1 = s_q[(2 * (gr * WG + i) + 1) * 32 + lane];
#pragma unroll
                        for (int u = 0; u < kUnit; u++)
#pragma unroll
                            for (int nt = 0; nt < 2; nt++) mma(d[u][nt], q0, n_low(kw[u][nt][gr * WG + i]), n_high(kw[u][nt][gr * WG + i]));
#pragma unroll
                        for (int u = 0; u < kUnit; u++)
#pragma unroll
                            for (int nt = 0; nt < 2; nt++) {
                                const uint32_t v = kw[u][nt][gr * WG + i] >> 8;
                                mma(d[u][nt], q1, n_low(v), n_high(v));
                            }
                    }
#pragma unroll
                    for (int u = 0; u < kUnit; u++)
#pragma unroll
                        for (int nt = 0; nt < 2; nt++) {                       // scales of columns 2t and 2t + 1, NG numbers each
                            const float k0 = gr & 1 ? ax_bf16_hi(ks[u][nt][gr / 2]) : ax_bf16_lo(ks[u][nt][gr / 2]);
                            const float k1 = (NG + gr) & 1 ? ax_bf16_hi(ks[u][nt][(NG + gr) / 2]) : ax_bf16_lo(ks[u][nt][(NG + gr) / 2]);
                            s[u][nt] = ax_fma2(make_float2(k0, k1), ax_add2(make_float2(d[u][nt][0], d[u][nt][1]), make_float2(d[u][nt][2], d[u][nt][3])), s[u][nt]);
                        }
                }
            }
#pragma unroll
            for (int u = 0; u < kUnit; u++)
#pragma unroll
                for (int nt = 0; nt < 2; nt++) {
                    uint32_t sw[NG];
                    lds<NG>(sw, unit + u * TILE + 2 * PLANE + SC + (8 * nt + 2 * t) * NG * 2);
#pragma unroll
                    for (int gr = 0; gr < NG; gr++) {
                        vs[u][nt][gr].x = gr & 1 ? ax_bf16_hi(sw[gr / 2]) : ax_bf16_lo(sw[gr / 2]);
                        vs[u][nt][gr].y = (NG + gr) & 1 ? ax_bf16_hi(sw[(NG + gr) / 2]) : ax_bf16_lo(sw[(NG + gr) / 2]);
                    }
                    s[u][nt] = ax_mul2(s[u][nt], make_float2(qback, qback));
                }
            const int row = info.tile * AX_P4_TILE;
            if (row < seg_lo || row + kUnit * AX_P4_TILE > seg_len || info.ok != 3) {      // rows out of sight have no score and no scale
#pragma unroll
                for (int u = 0; u < kUnit; u++)
#pragma unroll
                    for (int nt = 0; nt < 2; nt++) {                           // column 8·nt + 2t + b is row 8·nt + 4b + t
                        const int r0 = row + u * AX_P4_TILE + nt * 8 + t, r1 = r0 + 4;
                        const bool here = info.ok >> u & 1;
                        if (!here || r0 < seg_lo || r0 >= seg_len) {
                            s[u][nt].x = -INFINITY;
#pragma unroll
                            for (int gr = 0; gr < NG; gr++) vs[u][nt][gr].x = 0.f;
                        }
                        if (!here || r1 < seg_lo || r1 >= seg_len) {
                            s[u][nt].y = -INFINITY;
#pragma unroll
                            for (int gr = 0; gr < NG; gr++) vs[u][nt][gr].y = 0.f;
                        }
                    }
            }
            // A probability is at most 2^15 over the smallest scale that counts: 2^95, and 2^31 of them stay below 2^127.  Values under
            // that scale are exact to 2^-112 instead of to 2^-32 of the largest.
            constexpr float kSmallest = -80.f;
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < kUnit; u++)
#pragma unroll
                for (int nt = 0; nt < 2; nt++) {
                    float2 big = vs[u][nt][0];
#pragma unroll
                    for (int gr = 1; gr < NG; gr++) { big.x = fmaxf(big.x, vs[u][nt][gr].x); big.y = fmaxf(big.y, vs[u][nt][gr].y); }
                    const float2 z = ax_add2(s[u][nt], make_float2(fmaxf(lg2(big.x), kSmallest), fmaxf(lg2(big.y), kSmallest)));
                    top = fmaxf(top, fmaxf(z.x, z.y));
                }
            top = fmaxf(top, __shfl_xor_sync(AX_FULL, top, 1));
            top = fmaxf(top, __shfl_xor_sync(AX_FULL, top, 2));
            // The reference is moved only where a p · scale would pass 2^15; then the largest becomes 2^7, so what is lost of the small
            // ones (half a step of f16's subnormals, 2^-25) is at most 2^-32 of the largest.
            if (__any_sync(AX_FULL, top > m + 15.f)) {
                const float mn = fmaxf(m, top - 7.f), f = m == -INFINITY ? 0.f : ax_ex2(m - mn);
                l.x *= f; l.y *= f;
#pragma unroll
                for (int i = 0; i < NT; i++) { o[i][0] *= f; o[i][1] *= f; o[i][2] *= f; o[i][3] *= f; }
                m = mn;
            }
            const float mr = m == -INFINITY ? 0.f : -m;
#pragma unroll
            for (int u = 0; u < kUnit; u++)
#pragma unroll
                for (int nt = 0; nt < 2; nt++) {                               // scores become probabilities
                    s[u][nt] = ax_add2(s[u][nt], make_float2(mr, mr));
                    s[u][nt].x = ax_ex2(s[u][nt].x); s[u][nt].y = ax_ex2(s[u][nt].y);
                    l = ax_add2(l, s[u][nt]);
                }
            uint32_t vw[kUnit][2][W];
#pragma unroll
            for (int u = 0; u < kUnit; u++)
#pragma unroll
                for (int nt = 0; nt < 2; nt++) lds<W>(vw[u][nt], unit + u * TILE + PLANE + nt * (PLANE / 2) + lane * W * 4);
#pragma unroll
            for (int gr = 0; gr < NG; gr++) {
                uint4 a[kUnit];
#pragma unroll
                for (int u = 0; u < kUnit; u++) {
                    uint32_t hl[4];
#pragma unroll
                    for (int nt = 0; nt < 2; nt++) {
                        const float2 y = ax_mul2(s[u][nt], vs[u][nt][gr]);
                        hl[2 * nt] = pack_f16(y.x, y.y);
                        const float2 r = ax_fma2(unpack_f16(hl[2 * nt]), make_float2(-1.f, -1.f), y);
                        hl[2 * nt + 1] = pack_f16(r.x, r.y);
                    }
                    a[u] = make_uint4(hl[0], hl[1], hl[2], hl[3]);
                }
#pragma unroll
                for (int i = 0; i < WG; i++) {
                    const int cw = gr * WG + i;
#pragma unroll
                    for (int u = 0; u < kUnit; u++) {
                        const uint32_t u0 = vw[u][0][cw], u1 = vw[u][1][cw];
                        mma(o[cw * 4], a[u], n_low(u0), n_low(u1));
                        mma(o[cw * 4 + 1], a[u], n_high(u0), n_high(u1));
                        mma(o[cw * 4 + 2], a[u], n_low(u0 >> 8), n_low(u1 >> 8));
                        mma(o[cw * 4 + 3], a[u], n_high(u0 >> 8), n_high(u1 >> 8));
                    }
                }
            }
        }
        __syncwarp();                                                          // every lane has read the stage
        fill(it + kStages, st);
        __syncwarp();
        if (++st == kStages) { st = 0; phase ^= 1u; }
    }
    if (it < count) {                                                          // gave up
        if (lane == 0) { atomicExch(dv.err, kErrWait); s_gave_up = 1; }
        for (int y = it; y < count && y < it + kStages; y++)                  // what is in flight lands before the CTA goes
            mbar_wait(ax_smem_u32(&s_bar[warp][y % kStages]), (uint32_t)(y / kStages) & 1u, kNs);
    }
    __syncwarp();                                                              // the ring is read by all lanes before the last output goes over it
    if (seg >= 0) flush();
    __syncthreads();
    if (s_gave_up) {
        // The segment that goes on in the next CTA is entered all the same, with a sum of zero: every CTA of a segment has to arrive at
        // its ticket, or the count is ahead in all later launches.  (The one that began in a CTA before is the first that a warp takes.)
        if (tid == 0) {
            int b, hh, ti;
            locate(X1 - 1, b, hh, ti);
            const int last = b * dv.nh + hh;
            const unsigned n = s_pre[b + 1] - s_pre[b];
            bool entered = (long long)s_pre[b] * dv.nh + (long long)(hh + 1) * n <= X1;
            for (int i = 0; i < kWarps * 2; i++) entered = entered || s_seg[i] == last;
            if (!entered) {
                s_seg[kWarps * 2 - 1] = last;                                 // free: the last warp enters nothing else there
                for (int h = 0; h < kHeads; h++) { s_ml[kWarps * 2 - 1][h][0] = -INFINITY; s_ml[kWarps * 2 - 1][h][1] = 0.f; }
            }
        }
        __syncthreads();
    }

    // ── segments that no warp holds alone ──
    for (int i = 0; i < kWarps * 2;) {
        const int sg = s_seg[i];
        int j = i + 1;
        if (sg < 0) { i = j; continue; }
        while (j < kWarps * 2 && (s_seg[j] == sg || s_seg[j] < 0)) j++;
        const int b = sg / dv.nh, hh = sg % dv.nh, kh = hh / dv.head_tiles, h0 = (hh % dv.head_tiles) * kHeads;
        const int heads = min(kHeads, dv.group_heads - h0);
        const unsigned n = s_pre[b + 1] - s_pre[b];
        const long long s0 = (long long)s_pre[b] * dv.nh + (long long)hh * n;
        const bool whole = s0 >= X0 && s0 + n <= X1;
        float* out = dv.a.out + ((size_t)b * dv.a.n_heads + (size_t)kh * dv.group_heads + h0) * HD;
        const size_t slot = 2 * (size_t)c + (s0 < X0 ? 0 : 1);
        for (int e = tid; e < heads * (HD / 4); e += kWarps * 32) {
            const int h = e / (HD / 4), d = (e % (HD / 4)) * 4;
            float M = -INFINITY, L = 0.f;
            for (int k = i; k < j; k++) if (s_seg[k] == sg) M = fmaxf(M, s_ml[k][h][0]);
            float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k = i; k < j; k++)
                if (s_seg[k] == sg && s_ml[k][h][1] != 0.f) {
                    const float f = s_ml[k][h][0] == M ? 1.f : ax_ex2(s_ml[k][h][0] - M);
                    const float4 v = *(const float4*)(s_o(k) + h * HD + d);
                    L = fmaf(f, s_ml[k][h][1], L);
                    A.x = fmaf(f, v.x, A.x); A.y = fmaf(f, v.y, A.y); A.z = fmaf(f, v.z, A.z); A.w = fmaf(f, v.w, A.w);
                }
            if (whole) {
                const float f = L == 0.f ? 0.f : 1.f / L;
                *(float4*)(out + (size_t)h * HD + d) = make_float4(A.x * f, A.y * f, A.z * f, A.w * f);
            } else {
                __stcg((float4*)(dv.part_o + (slot * hpt + h) * HD + d), A);
                if (d == 0) __stcg((float2*)(dv.part_ml + (slot * hpt + h) * 2), make_float2(M, L));
            }
        }
        if (!whole) {
            const long long cf = ((s0 + 1) * C - 1) / total, cl = ((s0 + n) * C - 1) / total;     // first and last CTA of the segment
            __syncthreads();                                                                      // the CTA's stores come before thread 0's
            if (tid == 0) {                                                                       // release, and through it before the count
                unsigned before;
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(dv.tickets + cf) : "memory");
                s_last = before == (unsigned)(cl - cf);
            }
            __syncthreads();
            if (s_last) {
                // part k is the tail of CTA cf (k = 0) or the head of CTA cf + k
                const int cnt = (int)(cl - cf) + 1;
                const float* ml = dv.part_ml + 2 * (size_t)cf * hpt * 2;
                const float* po = dv.part_o + 2 * (size_t)cf * hpt * HD;
                auto part = [&](int k) { return (size_t)(2 * k + (k == 0)) * hpt; };
                float* wt = reinterpret_cast<float*>(smem + RING);                                // weights of kChunk parts per head, over the first warp's query
                static_assert(kHeads * kChunk * 4 <= QBYTES, "weights do not fit");
                // maxima of the parts; those of the first chunk stay in registers with their sums
                constexpr int HW = kHeads / kWarps;                                               // heads of a warp: warp, warp + kWarps
                float2 own[HW][kChunk / 32];
                float M[HW], L[HW] = {};
#pragma unroll
                for (int i = 0; i < HW; i++) {
                    const int h = warp + i * kWarps;
                    M[i] = -INFINITY;
                    if (h >= heads) continue;
#pragma unroll
                    for (int r = 0; r < kChunk / 32; r++) {
                        const int k = lane + 32 * r;
                        own[i][r] = k < cnt ? __ldcg((const float2*)(ml + (part(k) + h) * 2)) : make_float2(-INFINITY, 0.f);
                        M[i] = fmaxf(M[i], own[i][r].x);
                    }
                    for (int k = lane + kChunk; k < cnt; k += 32) M[i] = fmaxf(M[i], __ldcg(ml + (part(k) + h) * 2));
                    M[i] = ax_warp_max(M[i]);
                }
                constexpr int E = (kHeads * HD / 4 + kWarps * 32 - 1) / (kWarps * 32);            // float4 outputs of a thread
                float4 A[E];
#pragma unroll
                for (int e = 0; e < E; e++) A[e] = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int k0 = 0; k0 < cnt; k0 += kChunk) {
                    const int kn = min(kChunk, cnt - k0);
                    if (k0) __syncthreads();
#pragma unroll
                    for (int i = 0; i < HW; i++) {
                        const int h = warp + i * kWarps;
                        if (h >= heads) continue;
                        float sum = 0.f;
#pragma unroll
                        for (int r = 0; r < kChunk / 32; r++) {
                            const int k = lane + 32 * r;
                            if (k >= kn) continue;
                            const float2 v = k0 ? __ldcg((const float2*)(ml + (part(k0 + k) + h) * 2)) : own[i][r];
                            const float f = v.y == 0.f ? 0.f : v.x == M[i] ? 1.f : ax_ex2(v.x - M[i]);
                            wt[h * kChunk + k] = f;
                            sum += f * v.y;
                        }
                        L[i] += ax_warp_sum(sum);
                    }
                    __syncthreads();
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const int at = tid + e * kWarps * 32, h = at / (HD / 4), d = (at % (HD / 4)) * 4;
                        if (h < heads) {
#pragma unroll 8
                            for (int k = 0; k < kn; k++) {                                        // loads of eight parts under way
                                const float4 v = __ldcg((const float4*)(po + (part(k0 + k) + h) * HD + d));
                                const float f = wt[h * kChunk + k];
                                A[e].x = fmaf(f, v.x, A[e].x); A[e].y = fmaf(f, v.y, A[e].y); A[e].z = fmaf(f, v.z, A[e].z); A[e].w = fmaf(f, v.w, A[e].w);
                            }
                        }
                    }
                }
                if (lane == 0)
                    for (int i = 0; i < HW; i++) if (warp + i * kWarps < heads) s_ml[0][warp + i * kWarps][1] = L[i];
                __syncthreads();
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const int at = tid + e * kWarps * 32, h = at / (HD / 4), d = (at % (HD / 4)) * 4;
                    if (h < heads) {
                        const float f = s_ml[0][h][1] == 0.f ? 0.f : 1.f / s_ml[0][h][1];
                        *(float4*)(out + (size_t)h * HD + d) = make_float4(A[e].x * f, A[e].y * f, A[e].z * f, A[e].w * f);
                    }
                }
                if (tid == 0) dv.tickets[cf] = 0u;                                                // ready for the next launch
            }
            __syncthreads();
        }
        i = j;
    }
}

constexpr int kMaxGrid = 1024;

template <int HD, int GS, bool LOSE = false>
int launch(atlasx_ctx* ctx, const PagedDev& dv, int grid, size_t smem) {
    static std::atomic<bool> ready[64] = {};
    if (ctx->device >= 64 || !ready[ctx->device]) {                           // the limit is per device; asking twice does no harm
        AX_CUDA(cudaFuncSetAttribute(ax_paged_attn_kernel<HD, GS, LOSE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if (ctx->device < 64) ready[ctx->device] = true;
    }
    ax_paged_attn_kernel<HD, GS, LOSE><<<grid, kWarps * 32, smem, ctx->stream>>>(dv);
    AX_CHECK_LAUNCH("ax_paged_attn_kernel");
    return ATLASX_OK;
}

int grid_of(const atlasx_ctx* ctx) { return min(ctx->sm_count * kCtasPerSm, kMaxGrid); }
size_t ticket_bytes(int grid) { return ((size_t)grid * 4 + 15) / 16 * 16; }

}  // namespace

size_t ax_paged_attn_workspace_bytes(const atlasx_ctx* ctx, const AxP4Shape& s) {
    const int grid = grid_of(ctx);
    return ticket_bytes(grid) + (size_t)2 * grid * kHeads * (s.hd + 2) * 4;
}

int ax_paged_attn_launch(atlasx_ctx* ctx, const atlasx_pagedkv* kv, const AxPagedAttnArgs& a, long long lost) {
    PagedDev dv = {};
    dv.s = kv->s; dv.pool = kv->pool; dv.a = a; dv.err = ctx->dev_error; dv.index_err = ctx->index_error();
    dv.lost = lost;
    dv.group_heads = a.n_heads / kv->s.n_kv;
    dv.head_tiles = (dv.group_heads + kHeads - 1) / kHeads;
    dv.hpt = min(kHeads, dv.group_heads);
    if ((long long)kv->s.n_kv * dv.head_tiles * a.batch > 0x7FFFFFFFll)
        return atlasx_fail(ATLASX_ERR_ARG, "batch · heads is too large");
    dv.nh = kv->s.n_kv * dv.head_tiles;
    const int grid = grid_of(ctx);
    uint8_t* w = (uint8_t*)a.workspace;
    dv.tickets = (unsigned*)w;
    dv.part_ml = (float*)(w + ticket_bytes(grid));
    dv.part_o = dv.part_ml + (size_t)2 * grid * kHeads * 2;
    const int tile = ax_p4_tile_bytes(kv->s);
    const size_t smem = (size_t)kWarps * (kStages * kUnit * tile + kv->s.hd / 32 * 2 * 32 * 16 + dv.hpt * kv->s.hd * 4) + (size_t)(a.batch + 1) * 4;
    if (lost >= 0) return launch<64, 32, true>(ctx, dv, grid, smem);
    if (kv->s.hd == 128) return kv->s.group == 32 ? launch<128, 32>(ctx, dv, grid, smem) : launch<128, 64>(ctx, dv, grid, smem);
    return kv->s.group == 32 ? launch<64, 32>(ctx, dv, grid, smem) : launch<64, 64>(ctx, dv, grid, smem);
}
