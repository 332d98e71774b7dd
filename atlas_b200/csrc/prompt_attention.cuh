// prompt_attention.cuh — arguments of the packed prompt attention and the form of a single row, for rows that are taken again.
#pragma once
#include "paged.cuh"

struct AxPromptArgs {
    const void *q, *k, *v;
    void* out;
    long long q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;      // strides in elements
    const int *cu_q, *cu_k;          // [batch + 1] first row of each sequence in q / out and in k / v
    int batch, n_q, n_k;             // sequences, rows of q and out, rows of k and v
    int n_heads, n_kv, hd, window;
    float scale;
};

// One sequence as the kernels see it: the row ranges the two prefix arrays name, cut to the buffers.
struct AxPromptSeq { int q0, lq, k0, lk; };
__device__ __forceinline__ AxPromptSeq ax_prompt_seq(const AxPromptArgs& a, int b) {
    AxPromptSeq s;
    s.q0 = min(max(a.cu_q[b], 0), a.n_q); s.lq = max(min(max(a.cu_q[b + 1], 0), a.n_q) - s.q0, 0);
    s.k0 = min(max(a.cu_k[b], 0), a.n_k); s.lk = max(min(max(a.cu_k[b + 1], 0), a.n_k) - s.k0, 0);
    return s;
}

template <typename T> __device__ __forceinline__ float ax_to_f32(T x);
template <> __device__ __forceinline__ float ax_to_f32<uint16_t>(uint16_t x) { return ax_bf16_to_f32(x); }
template <> __device__ __forceinline__ float ax_to_f32<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T ax_from_f32(float x);
template <> __device__ __forceinline__ uint16_t ax_from_f32<uint16_t>(float x) { return ax_f32_to_bf16_rne(x); }
template <> __device__ __forceinline__ __half ax_from_f32<__half>(float x) { return __float2half_rn(x); }

// One query row of one head by one warp: only visible keys and values are read, everything in f32.  i: row within the sequence.
template <typename T, int HD>
__device__ __forceinline__ void ax_prompt_row(const AxPromptArgs& a, const AxPromptSeq& s, int h, int i, int lane) {
    constexpr int N = HD / 32;
    const int kh = h / (a.n_heads / a.n_kv);
    const long long at = (long long)i + s.lk - s.lq;                  // the key at the query's own position
    const long long hi = at + 1 < s.lk ? at + 1 : s.lk, lo = a.window > 0 && at + 1 > a.window ? at + 1 - a.window : 0;
    const T* qp = (const T*)a.q + (long long)(s.q0 + i) * a.q_tok + h * a.q_head + lane * N;
    float q[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < N; e++) { q[e] = ax_to_f32<T>(qp[e]) * a.scale; o[e] = 0.f; }
    for (long long j = lo; j < hi; j++) {
        const T* kp = (const T*)a.k + (s.k0 + j) * a.k_tok + kh * a.k_head + lane * N;
        const T* vp = (const T*)a.v + (s.k0 + j) * a.v_tok + kh * a.v_head + lane * N;
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < N; e++) d += q[e] * ax_to_f32<T>(kp[e]);
        d = ax_warp_sum(d);
        const float mn = fmaxf(m, d);
        const float c = l == 0.f ? 0.f : expf(m - mn), p = d == -INFINITY ? 0.f : expf(d - mn);      // d − mn is NaN while all scores are −inf
        l = l * c + p; m = mn;
#pragma unroll
        for (int e = 0; e < N; e++) o[e] = o[e] * c + p * ax_to_f32<T>(vp[e]);
    }
    T* op = (T*)a.out + (long long)(s.q0 + i) * a.o_tok + h * a.o_head + lane * N;
#pragma unroll
    for (int e = 0; e < N; e++) op[e] = ax_from_f32<T>(lo < hi ? o[e] / l : 0.f);
}
