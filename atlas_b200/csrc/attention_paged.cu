// attention_paged.cu — attention of one new token per request over the four-bit paged cache.
#include "paged.cuh"

namespace {

struct PagedDev {
    AxP4Shape s;
    const uint8_t* pool;
    AxPagedAttnArgs a;
    int* err;
};

// One CTA per (query head, request): every warp takes every fourth row, lanes hold hd / 32 numbers each, online softmax.
template <int HD>
__global__ void __launch_bounds__(128) ax_paged_attn_simple_kernel(const PagedDev dv) {
    constexpr int N = HD / 32;
    __shared__ float s_m[4], s_l[4], s_o[4][HD];
    const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const AxP4Shape& s = dv.s;
    const int kh = h / (dv.a.n_heads / s.n_kv);
    const int len = max(0, (int)min((long long)dv.a.lens[b], (long long)dv.a.table_width * s.page_size));
    const int lo = dv.a.window > 0 && len > dv.a.window ? len - dv.a.window : 0;
    float q[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) { q[i] = dv.a.q[((size_t)b * dv.a.n_heads + h) * HD + lane * N + i] * dv.a.scale; o[i] = 0.f; }
    for (int t = lo + warp; t < len; t += 4) {
        const int page = dv.a.table[(size_t)b * dv.a.table_width + t / s.page_size], off = t % s.page_size, r = off % AX_P4_TILE;
        if (page < 0 || page >= s.n_pages) { if (lane == 0) atomicExch(dv.err, AX_DEVERR_PAGE); continue; }
        const uint8_t* tile = dv.pool + ax_p4_tile_at(s, page, kh, off);
        const int plane = ax_p4_plane_bytes(s);
        const uint16_t* sp = reinterpret_cast<const uint16_t*>(tile + 2 * plane);
        float d = 0.f, v[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int e = lane * N + i, gr = e / s.group;
            const uint32_t kw = ax_p4_unrot(reinterpret_cast<const uint32_t*>(tile)[ax_p4_k_word(s, r, e & ~7)]);
            const uint32_t vw = reinterpret_cast<const uint16_t*>(tile + plane)[ax_p4_v_half(s, r, e & ~3)];
            d += q[i] * ((float)((int)((kw >> (4 * (e & 7))) & 15u) - 8) * ax_bf16_to_f32(sp[ax_p4_scale(s, r, gr)]));
            v[i] = (float)((int)((vw >> (4 * (e & 3))) & 15u) - 8) * ax_bf16_to_f32(sp[AX_P4_TILE * ax_p4_groups(s) + ax_p4_scale(s, r, gr)]);
        }
        d = ax_warp_sum(d);
        const float mn = fmaxf(m, d);
        const float c = m == mn ? 1.f : expf(m - mn), p = d == mn ? 1.f : expf(d - mn);
        l = l * c + p; m = mn;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = o[i] * c + p * v[i];
    }
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
    for (int i = 0; i < N; i++) s_o[warp][lane * N + i] = o[i];
    __syncthreads();
    if (threadIdx.x < HD) {
        float M = -INFINITY, L = 0.f, A = 0.f;
        for (int w = 0; w < 4; w++) M = fmaxf(M, s_m[w]);
        for (int w = 0; w < 4; w++) {
            const float c = s_l[w] == 0.f ? 0.f : expf(s_m[w] - M);
            L += c * s_l[w]; A += c == 0.f && s_l[w] == 0.f ? 0.f : c * s_o[w][threadIdx.x];
        }
        dv.a.out[((size_t)b * dv.a.n_heads + h) * HD + threadIdx.x] = len > lo && L != 0.f ? A / L : 0.f;
    }
}

}  // namespace

size_t ax_paged_attn_workspace_bytes(const atlasx_ctx* ctx, const AxP4Shape& s) { (void)ctx; (void)s; return 16; }

int ax_paged_attn_launch(atlasx_ctx* ctx, const atlasx_pagedkv* kv, const AxPagedAttnArgs& a) {
    PagedDev dv = { kv->s, kv->pool, a, ctx->dev_error };
    const dim3 grid((unsigned)a.n_heads, (unsigned)a.batch);
    if (kv->s.hd == 128) ax_paged_attn_simple_kernel<128><<<grid, 128, 0, ctx->stream>>>(dv);
    else ax_paged_attn_simple_kernel<64><<<grid, 128, 0, ctx->stream>>>(dv);
    AX_CHECK_LAUNCH("ax_paged_attn_simple_kernel");
    return ATLASX_OK;
}
