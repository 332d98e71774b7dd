// prompt_attention.cu — causal attention of whole packed prompts.
#include "prompt_attention.cuh"

namespace {

template <typename T, int HD>
__global__ void __launch_bounds__(128) ax_prompt_row_kernel(const AxPromptArgs a) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    int lo = 0, hi = a.batch;                                     // the last sequence that starts at or before the row
    while (hi - lo > 1) { const int m = (lo + hi) >> 1; if (a.cu_q[m] <= row) lo = m; else hi = m; }
    const AxPromptSeq s = ax_prompt_seq(a, lo);
    if (row < s.q0 || row >= s.q0 + s.lq) return;                 // rows outside every sequence are left as they are
    ax_prompt_row<T, HD>(a, s, (int)blockIdx.y, row - s.q0, lane);
}

}  // namespace

extern "C" int atlasx_prompt_attention(atlasx_ctx* c, int dtype, const void* q, long long q_tok, long long q_head,
                                       const void* k, long long k_tok, long long k_head, const void* v, long long v_tok, long long v_head,
                                       void* out, long long o_tok, long long o_head, const int* cu_q, const int* cu_k, int batch,
                                       int n_q, int n_k, int n_heads, int n_kv, int hd, float scale, int window) {
    AX_ARG(dtype == ATLASX_BF16 || dtype == ATLASX_F16, "dtype must be bf16 or f16");
    AX_ARG(batch >= 1 && batch <= AX_PAGED_MAX_BATCH, "batch must be in 1..4096");
    AX_ARG(n_q >= 0 && n_k >= 0, "row counts must not be negative");
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
    AX_ARG((o_head >= hd || n_heads == 1) && (o_tok >= hd || n_q == 1), "rows of out overlap");
    AX_ARG(c, "ctx is null");
    AX_ON_DEVICE(c);
    AxPromptArgs a = { q, k, v, out, q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head, cu_q, cu_k, batch, n_q, n_k,
                       n_heads, n_kv, hd, window, scale };
    const dim3 grid((unsigned)((n_q + 3) / 4), (unsigned)n_heads);
    if (dtype == ATLASX_BF16) {
        if (hd == 128) ax_prompt_row_kernel<uint16_t, 128><<<grid, 128, 0, c->stream>>>(a);
        else ax_prompt_row_kernel<uint16_t, 64><<<grid, 128, 0, c->stream>>>(a);
    } else {
        if (hd == 128) ax_prompt_row_kernel<__half, 128><<<grid, 128, 0, c->stream>>>(a);
        else ax_prompt_row_kernel<__half, 64><<<grid, 128, 0, c->stream>>>(a);
    }
    AX_CHECK_LAUNCH("ax_prompt_row_kernel");
    return ATLASX_OK;
}
