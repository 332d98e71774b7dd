// paged.cuh — object and launch declarations of the packed serving step: four-bit paged cache and prompt attention.
#pragma once
#include "common.cuh"
#include "paged_index.h"

#define AX_PAGED_MAX_BATCH 4096

// codes of the context's second device error word: what an index array holds was wrong
#define AX_DEVERR_PAGE 801      // a block table names a page outside the pool
#define AX_DEVERR_SLOT 802      // a slot lies behind the pool

struct atlasx_pagedkv {
    atlasx_ctx* ctx = nullptr;
    AxP4Shape s = {};
    uint8_t* pool = nullptr;
    void* workspace = nullptr;       // of the calls that bring none
    size_t workspace_bytes = 0;
};

// Makes the context's device current for the duration of a call and puts the caller's back.
struct AxDeviceGuard {
    int prev = -1;
    cudaError_t err = cudaSuccess;
    explicit AxDeviceGuard(int device) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != device) err = cudaSetDevice(device);
        else prev = -1;
    }
    ~AxDeviceGuard() { if (prev >= 0) cudaSetDevice(prev); }
};
#define AX_ON_DEVICE(ctx)                                                                  \
    AxDeviceGuard _guard((ctx)->device);                                                   \
    if (_guard.err != cudaSuccess)                                                         \
        return atlasx_fail(ATLASX_ERR_CUDA, "device %d: %s", (ctx)->device, cudaGetErrorString(_guard.err))

struct AxPagedAttnArgs {
    const float* q;                  // [batch][n_heads][hd]
    float* out;
    const int* table;                // [batch][table_width] page numbers
    const int* lens;                 // [batch] cached rows
    int table_width, batch, n_heads, window;
    float scale;
    void* workspace;                 // of ax_paged_attn_workspace_bytes()
};
size_t ax_paged_attn_workspace_bytes(const atlasx_ctx* ctx, const AxP4Shape& s);
// lost >= 0: self-test, the copy of that unit is not issued
int ax_paged_attn_launch(atlasx_ctx* ctx, const atlasx_pagedkv* kv, const AxPagedAttnArgs& a, long long lost = -1);

// two f32 operations in one instruction
__device__ __forceinline__ float2 ax_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\t"
        "mov.b64 {%0, %1}, w;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 ax_add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 ax_mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// largest of three; NaN if one is
__device__ __forceinline__ float ax_max3(float a, float b, float c) { float d; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }
__device__ __forceinline__ float ax_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

__device__ __forceinline__ uint32_t ax_smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool ax_mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
