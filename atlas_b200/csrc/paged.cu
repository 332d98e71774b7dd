// paged.cu — bookkeeping of a packed serving step and the four-bit paged KV cache: block tables, slots and positions from request
// lengths (ax_page_plan_kernel), rows rounded to four bits into their slots (ax_p4_append_kernel) and back (ax_p4_read_kernel).
// The reference keeps one linear f32 cache per sequence (GpuKvCache, crates/atlas-tensor/src/lib.rs:701-785); the number format is
// that of its Int4Tensor (crates/atlas-quant/src/lib.rs:113-145) with the scale held as bf16.
#include <new>

#include "paged.cuh"

namespace {

constexpr int kPlanThreads = 256;
constexpr int kAppendThreads = 64, kReadThreads = 256, kReadRows = 2;
constexpr int kPlanItems = 512;      // tokens (and pages taken) per CTA

struct PlanArgs {
    const int *cached, *fresh, *free;
    int batch, n_free, page_size, n_pages, table_width, n_tokens;
    int *table, *cu, *lens, *slots, *pos, *status;
};

// largest b with start[b] <= x, start[0] = 0
__device__ __forceinline__ int find_start(const int* start, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) { const int m = (lo + hi) >> 1; if (start[m] <= x) lo = m; else hi = m; }
    return lo;
}

// One launch, no second pass: every CTA scans the request lengths itself (at most 4096, from L2) and then serves its own range
// of tokens and of pages taken.  What bounds it is the latency of one dependent chain — lengths → scan → search → table entry —
// and the launch, not bandwidth.  Page j of the plan is free[j]; it belongs to the request in whose range of the scan over
// (pages needed − pages held) j falls, so the result does not depend on the order of CTAs.
__global__ void __launch_bounds__(kPlanThreads) ax_page_plan_kernel(const PlanArgs a) {
    extern __shared__ int sh[];
    int* s_cu = sh;                               // [batch + 1] first token of each request
    int* s_first = sh + a.batch + 1;              // [batch + 1] first page taken
    __shared__ unsigned long long s_tok[kPlanThreads / 32], s_pg[kPlanThreads / 32];
    __shared__ int s_bad;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    const int per = (a.batch + kPlanThreads - 1) / kPlanThreads;
    const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
    unsigned long long tok = 0, pg = 0;
    int bad = 0;
    for (int b = b0; b < b1; b++) {
        const int c = a.cached[b], n = a.fresh[b];
        const long long need = ((long long)c + n + a.page_size - 1) / a.page_size;
        if (c < 0 || n < 0 || need > a.table_width || (long long)c + n > 0x7FFFFFFFll) { bad++; continue; }
        tok += n;
        pg += need - (c + (long long)a.page_size - 1) / a.page_size;
    }
    if (bad) atomicAdd(&s_bad, bad);
    unsigned long long it = tok, ip = pg;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long xt = __shfl_up_sync(AX_FULL, it, d), xp = __shfl_up_sync(AX_FULL, ip, d);
        if (lane >= d) { it += xt; ip += xp; }
    }
    if (lane == 31) { s_tok[warp] = it; s_pg[warp] = ip; }
    __syncthreads();
    unsigned long long bt = 0, bp = 0, all_t = 0, all_p = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; w++) {
        if (w < warp) { bt += s_tok[w]; bp += s_pg[w]; }
        all_t += s_tok[w]; all_p += s_pg[w];
    }
    const int n_bad = s_bad + (all_t > (unsigned long long)a.n_tokens ? 1 : 0);
    const bool short_of = all_p > (unsigned long long)a.n_free;
    const bool refused = n_bad > 0 || short_of;
    if (blockIdx.x == 0 && tid == 0) {
        a.status[0] = refused ? 0 : (int)all_p;
        const unsigned long long miss = all_p - (unsigned long long)a.n_free;
        a.status[1] = !n_bad && short_of ? (int)(miss > 0x7FFFFFFFull ? 0x7FFFFFFFull : miss) : 0;
        a.status[2] = n_bad;
    }
    if (refused) {                                // nothing is planned: the calls that follow see empty requests and absent rows
        for (int i = blockIdx.x * kPlanThreads + tid; i < max(a.batch + 1, a.n_tokens); i += gridDim.x * kPlanThreads) {
            if (i < a.batch + 1) a.cu[i] = 0;
            if (i < a.batch) a.lens[i] = 0;
            if (i < a.n_tokens) { a.slots[i] = -1; a.pos[i] = -1; }
        }
        return;
    }
    int t = (int)(bt + it - tok), p = (int)(bp + ip - pg);
    for (int b = b0; b < b1; b++) {
        const int c = a.cached[b], n = a.fresh[b];
        s_cu[b] = t; s_first[b] = p;
        if (blockIdx.x == 0) { a.cu[b] = t; a.lens[b] = c + n; }
        t += n;
        p += (int)(((long long)c + n + a.page_size - 1) / a.page_size - (c + (long long)a.page_size - 1) / a.page_size);
    }
    if (tid == 0) {
        s_cu[a.batch] = (int)all_t; s_first[a.batch] = (int)all_p;
        if (blockIdx.x == 0) a.cu[a.batch] = (int)all_t;
    }
    __syncthreads();
    const int n_tok = (int)all_t, n_pg = (int)all_p;
    const int base = blockIdx.x * kPlanItems;
    for (int i = base + tid; i < min(base + kPlanItems, n_pg); i += kPlanThreads) {
        const int b = find_start(s_first, a.batch + 1, i);
        const int had = (int)((a.cached[b] + (long long)a.page_size - 1) / a.page_size);
        a.table[(size_t)b * a.table_width + had + (i - s_first[b])] = a.free[i];
    }
    // A thread's tokens side by side: the loads of one step are under way together.
    constexpr int N = kPlanItems / kPlanThreads;
    int b[N], at[N], page[N];
#pragma unroll
    for (int u = 0; u < N; u++) {
        const int i = base + tid + u * kPlanThreads;
        b[u] = i < n_tok ? find_start(s_cu, a.batch + 1, i) : -1;
    }
#pragma unroll
    for (int u = 0; u < N; u++) at[u] = b[u] >= 0 ? a.cached[b[u]] : 0;
#pragma unroll
    for (int u = 0; u < N; u++) {
        page[u] = -1;
        if (b[u] < 0) continue;
        const int c = at[u], had = (int)(((unsigned)c + (unsigned)a.page_size - 1u) / (unsigned)a.page_size);
        at[u] = c + (base + tid + u * kPlanThreads - s_cu[b[u]]);
        const int col = at[u] / a.page_size;
        page[u] = col < had ? a.table[(size_t)b[u] * a.table_width + col] : a.free[s_first[b[u]] + (col - had)];
    }
#pragma unroll
    for (int u = 0; u < N; u++) {
        const int i = base + tid + u * kPlanThreads;
        if (i >= a.n_tokens) continue;                                // rows behind the last request: −1 in both
        a.slots[i] = page[u] >= 0 && page[u] < a.n_pages ? page[u] * a.page_size + at[u] % a.page_size : -1;
        a.pos[i] = b[u] >= 0 ? at[u] : -1;
    }
}

// ── rows to four bits ────────────────────────────────────────────────────────────
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <> __device__ __forceinline__ void load8<uint16_t>(const uint16_t* p, float (&x)[8]) {      // bf16 bits
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = { a.x, a.y, a.z, a.w };
#pragma unroll
    for (int i = 0; i < 4; i++) { x[2 * i] = ax_bf16_lo(w[i]); x[2 * i + 1] = ax_bf16_hi(w[i]); }
}
template <> __device__ __forceinline__ void load8<__half>(const __half* p, float (&x)[8]) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = { a.x, a.y, a.z, a.w };
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
}

struct RowArgs {
    AxP4Shape s;
    unsigned long long inv_page;  // ax_p4_page_inverse
    uint8_t* pool;
    const void *k, *v;            // append: [token][head][hd], token and head strides in elements
    long long k_tok, k_head, v_tok, v_head;
    void *k_out, *v_out;          // read: contiguous [token][head][hd]
    const int* slots;
    int n;
    int* err;
};

// a slot's page and row within it
__device__ __forceinline__ void slot_place(const RowArgs& a, int slot, int& page, int& off) {
    page = ax_p4_page_of(slot, a.inv_page);
    off = slot - page * a.s.page_size;
}
template <int HD, int GS> __device__ __forceinline__ AxP4Shape fixed_shape(const AxP4Shape& s) { return AxP4Shape{ s.n_pages, s.page_size, s.n_kv, HD, GS }; }

// A lane holds thirty-two consecutive numbers of one row of K or V: a group, or half of one whose largest magnitude two lanes
// find with a shuffle.  scale = bf16(max / 7); the number is x · (1 / scale) rounded half away from zero — the f32 arithmetic of
// Int4Tensor::quantize with a scale of 16 bits: the numbers are rounded against the scale that is stored, so its own rounding (2^-8 of
// itself) costs nothing beyond the half step of the number, and no number passes 7 · (1 + 2^-7) before it is rounded: 7 is the largest.
// A group with a NaN or an infinity gets the scale NaN.
// Bytes: the rows once, 4.25 or 4.5 bits per number out.  A CTA takes 16 (hd 128) or 32 consecutive rows of one head: as a rule a whole
// tile of the pool or two.  What bounds it beside the memory is instructions (70 % of the issue slots): 8191 rows × 32 heads × 128 in bf16 took
// 181 µs with run-time shapes and rows found by division, 76 with eight numbers a lane, 50 with sixteen, 39 with thirty-two, 37 with
// pairs of f32 operations and 64 threads a CTA (256 threads: 40; the copy bandwidth: 26).
template <typename T, int HD, int GS>
__global__ void __launch_bounds__(kAppendThreads) ax_p4_append_kernel(const RowArgs a) {
    constexpr int N = 32, LANES = HD / N, GL = GS / N, TOKENS = kAppendThreads / LANES;        // lanes per row, lanes per group, rows per CTA
    const int li = threadIdx.x % LANES, tok = blockIdx.x * TOKENS + threadIdx.x / LANES, head = blockIdx.y, which = blockIdx.z;
    const AxP4Shape sh = fixed_shape<HD, GS>(a.s);
    const bool live = tok < a.n;
    float x[N] = {};
    float top = 0.f;
    int slot = -1;
    if (live) {
        slot = a.slots[tok];
        const T* src = which ? (const T*)a.v + tok * a.v_tok + head * a.v_head : (const T*)a.k + tok * a.k_tok + head * a.k_head;
#pragma unroll
        for (int i = 0; i < N; i += 8) load8<T>(src + N * li + i, reinterpret_cast<float (&)[8]>(x[i]));
#pragma unroll
        for (int i = 0; i < N; i += 2) top = ax_max3(top, fabsf(x[i]), fabsf(x[i + 1]));
    }
#pragma unroll
    for (int d = 1; d < GL; d <<= 1) { const float o = __shfl_xor_sync(AX_FULL, top, d); top = ax_max3(top, o, o); }
    if (!live || slot < 0) return;                                   // a negative slot marks an absent row
    if (slot >= sh.n_pages * sh.page_size) { if (li == 0) atomicExch(a.err, AX_DEVERR_SLOT); return; }
    const bool odd = !(top <= 3.402823466e38f);
    uint16_t sb = ax_f32_to_bf16_rne(__fdiv_rn(top, 7.0f));
    float sc = ax_bf16_to_f32(sb);
    // Below the smallest normal number every number of the group is zero (against a scale of 1).  What is stored is that smallest
    // scale: decode attention takes the size of a row's values from its scales, and a row of zeros has none.
    if (sc < 1.17549435e-38f) { sc = 1.0f; sb = 0x0080; }
    if (odd) { sc = 1.0f; sb = 0x7FC0; }
    const float inv = __frcp_rn(sc);
    uint32_t half[N / 4];                                            // four numbers each
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
        // Σ (number + 8) · 16^j
        int w = 0;
#pragma unroll
        for (int j = 2; j >= 0; j -= 2) {
            float2 y = ax_mul2(make_float2(x[4 * i + j], x[4 * i + j + 1]), make_float2(inv, inv));
            y = ax_add2(y, make_float2(ax_p4_half(y.x), ax_p4_half(y.y)));
            w = (w * 16 + __float2int_rz(y.y)) * 16 + __float2int_rz(y.x);
        }
        half[i] = odd ? 0x8888u : (uint32_t)(w + 0x8888) & 0xFFFFu;
    }
    int page, off;
    slot_place(a, slot, page, off);
    const int r = off % AX_P4_TILE;
    uint8_t* tile = a.pool + ax_p4_tile_at(sh, page, head, off);
    const int plane = ax_p4_plane_bytes(sh);
    if (which == 0) {
        uint32_t* kp = reinterpret_cast<uint32_t*>(tile);
#pragma unroll
        for (int i = 0; i < N / 8; i += 2) {
            const uint32_t w0 = half[2 * i] | (half[2 * i + 1] << 16), w1 = half[2 * i + 2] | (half[2 * i + 3] << 16);
            uint32_t* at = kp + ax_p4_k_word(sh, r, N * li + 8 * i);
            if (GS == 64) *reinterpret_cast<uint2*>(at) = make_uint2(w0, w1);                                 // one thread's pair of words
            else { *at = w0; kp[ax_p4_k_word(sh, r, N * li + 8 * i + 8)] = w1; }
        }
    } else {
        uint16_t* vp = reinterpret_cast<uint16_t*>(tile + plane);
#pragma unroll
        for (int i = 0; i < N / 4; i++) vp[ax_p4_v_half(sh, r, N * li + 4 * i)] = (uint16_t)half[i];
    }
    if (li % GL == 0) {
        uint16_t* sp = reinterpret_cast<uint16_t*>(tile + 2 * plane + which * ax_p4_scale_bytes(sh));
        sp[ax_p4_scale(sh, r, li / GL)] = sb;
    }
}

template <typename T> __device__ __forceinline__ void store4(T* p, const float (&x)[4]);
template <> __device__ __forceinline__ void store4<float>(float* p, const float (&x)[4]) { __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3])); }
template <> __device__ __forceinline__ void store4<uint16_t>(uint16_t* p, const float (&x)[4]) {
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(ax_f32_to_bf16_rne(x[0]) | ((uint32_t)ax_f32_to_bf16_rne(x[1]) << 16),
                                                   ax_f32_to_bf16_rne(x[2]) | ((uint32_t)ax_f32_to_bf16_rne(x[3]) << 16)));
}
template <> __device__ __forceinline__ void store4<__half>(__half* p, const float (&x)[4]) {
    const __half2 h0 = __floats2half2_rn(x[0], x[1]), h1 = __floats2half2_rn(x[2], x[3]);
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1)));
}

// Four numbers times their scale.  A nibble u, i nibbles up, under the exponent of 2^23 is 2^23 + 16^i u; times 16^-i and less 2^23 · 16^-i + 8
// it is the number, all of it exact.
__device__ __forceinline__ void four(uint32_t w, float scale, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const float f0 = i ? 1.f / 256.f : 1.f, f1 = f0 / 16.f;
        const float2 n = ax_fma2(make_float2(__int_as_float((w & 15u << (4 * i)) | 0x4B000000u), __int_as_float((w & 15u << (4 * i + 4)) | 0x4B000000u)),
                                 make_float2(f0, f1), make_float2(-8388608.f * f0 - 8.f, -8388608.f * f1 - 8.f));
        const float2 y = ax_mul2(n, make_float2(scale, scale));
        x[i] = y.x; x[i + 1] = y.y;
    }
}

// The values a slot holds: number · scale, exact in f32 (4 + 8 bits), one rounding for the 16-bit types.  Absent rows read as zeros.
// A lane makes four numbers of K and of V, so that a warp's store is one run of bytes, for two rows: their loads, each behind that of its
// slot, are under way together.  8191 rows × 32 heads × 128 in f32: 75 µs with eight numbers a lane, 63 with four, 57 with two rows (59 with
// four rows; 46 at the copy bandwidth: 5.3 TB/s, most of it stores).  CTAs with all heads of the same rows side by side instead of all rows
// of a head: storing and reading together 98.3 µs instead of 96.8.
template <typename T, int HD, int GS>
__global__ void __launch_bounds__(kReadThreads) ax_p4_read_kernel(const RowArgs a) {
    constexpr int LANES = HD / 4, ROWS = kReadThreads / LANES, TOKENS = ROWS * kReadRows;
    const int li = threadIdx.x % LANES, tok = blockIdx.x * TOKENS + threadIdx.x / LANES, head = blockIdx.y;
    const AxP4Shape sh = fixed_shape<HD, GS>(a.s);
    const int plane = ax_p4_plane_bytes(sh), gr = 4 * li / GS;
    int slot[kReadRows];
#pragma unroll
    for (int u = 0; u < kReadRows; u++) slot[u] = tok + u * ROWS < a.n ? a.slots[tok + u * ROWS] : -1;
    uint32_t kw[kReadRows], vw[kReadRows];
    float ks[kReadRows], vs[kReadRows];
#pragma unroll
    for (int u = 0; u < kReadRows; u++) {
        kw[u] = vw[u] = 0x8888u; ks[u] = vs[u] = 0.f;
        if (slot[u] >= 0 && slot[u] < sh.n_pages * sh.page_size) {
            int page, off;
            slot_place(a, slot[u], page, off);
            const int r = off % AX_P4_TILE;
            const uint8_t* tile = a.pool + ax_p4_tile_at(sh, page, head, off);
            // numbers 4 · li .. + 3: the low or high half of a K word, a half word of V
            kw[u] = reinterpret_cast<const uint16_t*>(tile)[2 * ax_p4_k_word(sh, r, 4 * li & ~7) + (li & 1)];
            vw[u] = reinterpret_cast<const uint16_t*>(tile + plane)[ax_p4_v_half(sh, r, 4 * li)];
            const uint16_t* sp = reinterpret_cast<const uint16_t*>(tile + 2 * plane) + ax_p4_scale(sh, r, gr);
            ks[u] = ax_bf16_to_f32(sp[0]); vs[u] = ax_bf16_to_f32(sp[AX_P4_TILE * (HD / GS)]);
        } else if (slot[u] >= 0) atomicExch(a.err, AX_DEVERR_SLOT);
    }
#pragma unroll
    for (int u = 0; u < kReadRows; u++) {
        if (tok + u * ROWS >= a.n) break;
        const size_t o = ((size_t)(tok + u * ROWS) * sh.n_kv + head) * HD + 4 * li;
        float x[4];
        four(kw[u], ks[u], x);
        store4<T>((T*)a.k_out + o, x);
        four(vw[u], vs[u], x);
        store4<T>((T*)a.v_out + o, x);
    }
}

template <typename T, bool READ>
void launch_rows(const RowArgs& a, cudaStream_t stream) {
    const int tokens = READ ? kReadThreads / (a.s.hd / 4) * kReadRows : kAppendThreads / (a.s.hd / 32);
    const dim3 grid((unsigned)((a.n + (long long)tokens - 1) / tokens), (unsigned)a.s.n_kv, READ ? 1u : 2u);
#define AX_ROWS(HD, GS) do { if (READ) ax_p4_read_kernel<T, HD, GS><<<grid, kReadThreads, 0, stream>>>(a); \
                             else ax_p4_append_kernel<T, HD, GS><<<grid, kAppendThreads, 0, stream>>>(a); } while (0)
    if (a.s.hd == 128) { if (a.s.group == 32) AX_ROWS(128, 32); else AX_ROWS(128, 64); }
    else { if (a.s.group == 32) AX_ROWS(64, 32); else AX_ROWS(64, 64); }
#undef AX_ROWS
}
template <bool READ>
void launch_rows(int dtype, const RowArgs& a, cudaStream_t stream) {
    if (dtype == ATLASX_F32) launch_rows<float, READ>(a, stream);
    else if (dtype == ATLASX_BF16) launch_rows<uint16_t, READ>(a, stream);
    else launch_rows<__half, READ>(a, stream);
}

int elem_bytes(int dtype) { return dtype == ATLASX_F32 ? 4 : 2; }

}  // namespace

extern "C" int atlasx_page_plan(atlasx_ctx* c, const atlasx_page_plan_args* p) {
    AX_ARG(p, "null argument");
    const int *cached = p->cached, *fresh = p->fresh, *free_pages = p->free_pages;
    int *table = p->table, *cu = p->cu, *lens = p->lens, *slots = p->slots, *pos = p->pos, *status = p->status;
    const int batch = p->batch, n_free = p->n_free, page_size = p->page_size, n_pages = p->n_pages, table_width = p->table_width, n_tokens = p->n_tokens;
    AX_ARG(cached && fresh && table && cu && lens && status, "null argument");
    AX_ARG(batch >= 1 && batch <= AX_PAGED_MAX_BATCH, "batch must be in 1..4096");
    AX_ARG(page_size >= 1 && n_pages >= 1 && (long long)page_size * n_pages <= 0x7FFFFFFFll, "page_size · n_pages must be in 1..2^31 - 1");
    AX_ARG(table_width >= 1, "the block table needs a column");
    AX_ARG(n_tokens >= 0 && n_free >= 0, "counts must not be negative");
    AX_ARG(n_tokens <= 0x3FFFFFFF, "too many new rows for one call");
    AX_ARG((free_pages || !n_free) && ((slots && pos) || !n_tokens), "null argument");
    AX_ARG(c, "ctx is null");
    // CTAs read the inputs while others write: an output over an input (lens over cached, say) would be read half new
    struct Range {
        const int* at; long long n;
        bool meets(const Range& o) const { return n && o.n && at < o.at + o.n && o.at < at + n; }
    };
    const Range out[] = { { table, (long long)batch * table_width }, { cu, batch + 1ll }, { lens, batch }, { slots, n_tokens },
                                                           { pos, n_tokens }, { status, 3 } }, in[] = { { cached, batch }, { fresh, batch }, { free_pages, n_free } };
    for (const Range& o : out) {
        for (const Range& i : in) AX_ARG(!o.meets(i), "an output overlaps an input");
        for (const Range& other : out) AX_ARG(&o == &other || !o.meets(other), "outputs overlap");
    }
    AX_ON_DEVICE(c);
    PlanArgs a = { cached, fresh, free_pages, batch, n_free, page_size, n_pages, table_width, n_tokens, table, cu, lens, slots, pos, status };
    const int grid = n_tokens ? (n_tokens + kPlanItems - 1) / kPlanItems : 1;      // a page is taken for a new token: never more pages than tokens
    ax_page_plan_kernel<<<grid, kPlanThreads, (size_t)2 * (batch + 1) * sizeof(int), c->stream>>>(a);
    AX_CHECK_LAUNCH("ax_page_plan_kernel");
    return ATLASX_OK;
}

static int check_shape(int n_pages, int page_size, int n_kv, int hd, int group) {
    AX_ARG(n_pages >= 1 && n_kv >= 1, "n_pages and n_kv_heads must be positive");
    AX_ARG(page_size >= AX_P4_TILE && page_size <= 8192 && page_size % AX_P4_TILE == 0, "page_size must be a multiple of 16, at most 8192");
    AX_ARG((long long)n_pages * page_size <= 0x7FFFFFFFll, "n_pages · page_size must be below 2^31: slots are 32-bit");
    AX_ARG(hd == 64 || hd == 128, "head_dim must be 64 or 128");
    AX_ARG(group == 32 || group == 64, "group must be 32 or 64");
    AX_ARG(n_kv <= 65535, "too many KV heads");
    return ATLASX_OK;
}
extern "C" size_t atlasx_pagedkv_bytes(int n_pages, int page_size, int n_kv, int hd, int group) {
    if (check_shape(n_pages, page_size, n_kv, hd, group)) return 0;
    const AxP4Shape s = { n_pages, page_size, n_kv, hd, group };
    return ax_p4_pool_bytes(s);
}
extern "C" int atlasx_pagedkv_create(atlasx_ctx* c, int n_pages, int page_size, int n_kv, int hd, int group, atlasx_pagedkv** out) {
    AX_ARG(out, "null argument");
    int rc = check_shape(n_pages, page_size, n_kv, hd, group);
    if (rc) return rc;
    AX_ARG(c, "ctx is null");
    AX_ON_DEVICE(c);
    atlasx_pagedkv* kv = new (std::nothrow) atlasx_pagedkv();
    if (!kv) return atlasx_fail(ATLASX_ERR_STATE, "out of host memory");
    kv->ctx = c;
    kv->s = { n_pages, page_size, n_kv, hd, group };
    kv->workspace_bytes = ax_paged_attn_workspace_bytes(c, kv->s);
    const size_t bytes = ax_p4_pool_bytes(kv->s);
    cudaError_t e = cudaMalloc((void**)&kv->pool, bytes);
    if (e == cudaSuccess) e = cudaMalloc(&kv->workspace, kv->workspace_bytes);
    if (e == cudaSuccess) e = cudaMemsetAsync(kv->pool, 0, bytes, c->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(kv->workspace, 0, kv->workspace_bytes, c->stream);
    if (e != cudaSuccess) {
        cudaFree(kv->pool); cudaFree(kv->workspace); delete kv;
        cudaGetLastError();
        return atlasx_fail(ATLASX_ERR_CUDA, "paged cache of %zu bytes: %s", bytes, cudaGetErrorString(e));
    }
    *out = kv;
    return ATLASX_OK;
}
extern "C" int atlasx_pagedkv_free(atlasx_pagedkv* kv) {
    if (!kv || ax_ctx_defer(kv->ctx, [kv] { atlasx_pagedkv_free(kv); })) return ATLASX_OK;
    AX_ON_DEVICE(kv->ctx);
    AxRelaxedCapture relaxed;
    cudaStreamSynchronize(kv->ctx->stream);
    cudaFree(kv->pool); cudaFree(kv->workspace);
    delete kv;
    return ATLASX_OK;
}
extern "C" int atlasx_pagedkv_ptrs(atlasx_pagedkv* kv, void** pool, size_t* bytes, size_t* workspace_bytes) {
    AX_ARG(kv, "kv is null");
    if (pool) *pool = kv->pool;
    if (bytes) *bytes = ax_p4_pool_bytes(kv->s);
    if (workspace_bytes) *workspace_bytes = kv->workspace_bytes;
    return ATLASX_OK;
}

extern "C" int atlasx_pagedkv_append(atlasx_ctx* c, atlasx_pagedkv* kv, const atlasx_pagedkv_rows* p) {
    AX_ARG(p, "null argument");
    const int dtype = p->dtype, n = p->n, *slots = p->slots;
    const void *k = p->k, *v = p->v;
    const long long k_token_stride = p->k_token_stride, k_head_stride = p->k_head_stride, v_token_stride = p->v_token_stride, v_head_stride = p->v_head_stride;
    AX_ARG(dtype == ATLASX_F32 || dtype == ATLASX_BF16 || dtype == ATLASX_F16, "dtype must be f32, bf16 or f16");
    AX_ARG(n >= 0, "the number of rows must not be negative");
    AX_ARG(n <= 0x3FFFFFFF, "too many rows for one call");
    if (n == 0) return ATLASX_OK;
    AX_ARG(k && v && slots, "null argument");
    const long long step = 16 / elem_bytes(dtype);
    // a stride that is never taken may be anything: of one row, of one head
    const long long token_strides = n > 1 ? k_token_stride | v_token_stride : 0, head_strides = !kv || kv->s.n_kv > 1 ? k_head_stride | v_head_stride : 0;
    AX_ARG(((uintptr_t)k | (uintptr_t)v) % 16 == 0 && (token_strides | head_strides) % step == 0, "rows must start on 16-byte boundaries");
    AX_ARG(c && kv, "ctx or cache is null");
    AX_ARG(kv->ctx == c, "the cache belongs to another context");
    AX_ON_DEVICE(c);
    RowArgs a = {};
    a.s = kv->s; a.pool = kv->pool; a.k = k; a.v = v;
    a.k_tok = k_token_stride; a.k_head = k_head_stride; a.v_tok = v_token_stride; a.v_head = v_head_stride;
    a.slots = slots; a.n = n; a.err = c->index_error();
    a.inv_page = ax_p4_page_inverse(kv->s.page_size);
    launch_rows<false>(dtype, a, c->stream);
    AX_CHECK_LAUNCH("ax_p4_append_kernel");
    return ATLASX_OK;
}
extern "C" int atlasx_pagedkv_read(atlasx_ctx* c, const atlasx_pagedkv* kv, const int* slots, int n, int dtype, void* k_out, void* v_out) {
    AX_ARG(dtype == ATLASX_F32 || dtype == ATLASX_BF16 || dtype == ATLASX_F16, "dtype must be f32, bf16 or f16");
    AX_ARG(n >= 0, "the number of rows must not be negative");
    AX_ARG(n <= 0x3FFFFFFF, "too many rows for one call");
    if (n == 0) return ATLASX_OK;
    AX_ARG(k_out && v_out && slots, "null argument");
    AX_ARG(((uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0, "outputs must be 16-byte aligned");
    AX_ARG(c && kv, "ctx or cache is null");
    AX_ARG(kv->ctx == c, "the cache belongs to another context");
    AX_ON_DEVICE(c);
    RowArgs a = {};
    a.s = kv->s; a.pool = kv->pool; a.k_out = k_out; a.v_out = v_out; a.slots = slots; a.n = n; a.err = c->index_error();
    a.inv_page = ax_p4_page_inverse(kv->s.page_size);
    launch_rows<true>(dtype, a, c->stream);
    AX_CHECK_LAUNCH("ax_p4_read_kernel");
    return ATLASX_OK;
}

static int decode_attention(atlasx_ctx* c, const atlasx_pagedkv* kv, const atlasx_pagedkv_attn_args* p, long long lost) {
    AX_ARG(p, "null argument");
    const float* q = p->q;
    float* out = p->out;
    const int *table = p->table, *lens = p->lens, n_heads = p->n_heads, table_width = p->table_width, batch = p->batch, window = p->window;
    const float scale = p->scale;
    void* workspace = p->workspace;
    const size_t workspace_bytes = p->workspace_bytes;
    AX_ARG(q && out && table && lens, "null argument");
    AX_ARG(batch >= 1 && batch <= AX_PAGED_MAX_BATCH, "batch must be in 1..4096");
    AX_ARG(n_heads >= 1, "n_heads must be positive");
    AX_ARG(table_width >= 1, "the block table needs a column");
    AX_ARG(window >= 0, "window must be non-negative");
    AX_ARG(scale - scale == 0.f, "scale must be finite");
    AX_ARG(((uintptr_t)q | (uintptr_t)out) % 16 == 0, "q and out must be 16-byte aligned");
    AX_ARG(c && kv, "ctx or cache is null");
    AX_ARG(kv->ctx == c, "the cache belongs to another context");
    AX_ARG(n_heads % kv->s.n_kv == 0, "n_heads must be a multiple of n_kv_heads");
    const long long rows = (long long)table_width * kv->s.page_size;
    AX_ARG(rows <= 0x7FFFFFFFll && (rows / AX_P4_TILE) * batch <= 0x7FFFFFFFll, "the block table spans too many rows");
    AX_ARG(!workspace || (workspace_bytes >= kv->workspace_bytes && (uintptr_t)workspace % 16 == 0),
           "the workspace is too small or not 16-byte aligned");
    AX_ON_DEVICE(c);
    AxPagedAttnArgs a;
    a.q = q; a.out = out; a.table = table; a.lens = lens; a.table_width = table_width; a.batch = batch; a.n_heads = n_heads;
    a.window = window; a.scale = scale; a.workspace = workspace ? workspace : kv->workspace;
    return ax_paged_attn_launch(c, kv, a, lost);
}
extern "C" int atlasx_pagedkv_decode_attention(atlasx_ctx* c, const atlasx_pagedkv* kv, const atlasx_pagedkv_attn_args* p) {
    return decode_attention(c, kv, p, -1);
}
extern "C" int atlasx_pagedkv_selftest_wait_expiry(atlasx_ctx* c, const atlasx_pagedkv* kv, const atlasx_pagedkv_attn_args* p, long long unit) {
    AX_ARG(unit >= 0, "the unit must not be negative");
    AX_ARG(kv && kv->s.hd == 64 && kv->s.group == 32, "the self-test takes head_dim 64 and groups of 32");
    return decode_attention(c, kv, p, unit);
}
