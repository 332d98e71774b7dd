// paged_index.h — where a number of the four-bit paged cache lies.  Plain C++ (host and device), so that the arithmetic can be
// checked without a GPU.
//
// The pool is an array of tiles.  A tile holds 16 consecutive rows of one KV head — the K nibbles, the V nibbles, then the
// bf16 scales of K and of V — and is contiguous, so one bulk copy of a warp brings everything that 16 cached tokens need:
//
//     tile(page, head, r / 16) = ((page · n_kv + head) · (page_size / 16) + r / 16) · tile_bytes
//
// Inside a tile the nibbles lie in the order in which the lanes of mma.m16n8k16 want them (attention_paged.cu): lane 4·g + t
// reads its share of eight rows as one 16-byte word group (hd / 32 words of 32 bits), no bank conflicts and no shuffles.
//   K: the B operand of S = Q·Kᵀ.  Column g of row block nt is row 8·nt + 4·(g & 1) + (g >> 1); thread t owns GS / 4
//      consecutive numbers of every group of GS numbers.
//   V: the B operand of O = P·V.  A 32-bit word holds four numbers of row 8·nt + t in its low half and the same four of row
//      8·nt + 4 + t in its high half (the k pair 2t, 2t + 1 of the product), column g owning GS / 8 consecutive numbers of a group.
// A nibble is the number plus eight.
#pragma once
#include <math.h>
#include <stdint.h>
#include <stddef.h>
#ifdef __CUDACC__
#define AX_HD __host__ __device__ __forceinline__
#else
#define AX_HD static inline
#endif

#define AX_P4_TILE 16           // rows of a tile

struct AxP4Shape {
    int n_pages, page_size, n_kv, hd, group;
};

AX_HD int ax_p4_groups(const AxP4Shape& s) { return s.hd / s.group; }
AX_HD int ax_p4_plane_bytes(const AxP4Shape& s) { return AX_P4_TILE * s.hd / 2; }              // nibbles of K (and of V)
AX_HD int ax_p4_scale_bytes(const AxP4Shape& s) { return AX_P4_TILE * ax_p4_groups(s) * 2; }   // scales of K (and of V)
AX_HD int ax_p4_tile_bytes(const AxP4Shape& s) { return 2 * (ax_p4_plane_bytes(s) + ax_p4_scale_bytes(s)); }
AX_HD size_t ax_p4_pool_bytes(const AxP4Shape& s) {
    return (size_t)s.n_pages * s.n_kv * (s.page_size / AX_P4_TILE) * (size_t)ax_p4_tile_bytes(s);
}
// byte offset of the tile that holds row `off` of `page` for KV head `head`; the caller has checked the ranges
AX_HD size_t ax_p4_tile_at(const AxP4Shape& s, int page, int head, int off) {
    return (((size_t)page * s.n_kv + head) * (s.page_size / AX_P4_TILE) + off / AX_P4_TILE) * (size_t)ax_p4_tile_bytes(s);
}
// row r (0..15) of a tile → the column index that the product gives it (8·nt + g)
AX_HD int ax_p4_col(int r) { return (r & 8) | ((r & 3) << 1) | ((r >> 2) & 1); }
// K: 32-bit word (within the K plane) of the eight numbers d8 = 8·i .. 8·i + 7 of row r; number j of them is nibble j
AX_HD int ax_p4_k_word(const AxP4Shape& s, int r, int d8) {
    const int dg = d8 % s.group, t = dg / (s.group / 4), sub = (dg % (s.group / 4)) / 8;
    return (ax_p4_col(r) * 4 + t) * (s.hd / 32) + (d8 / s.group) * (s.group / 32) + sub;
}
// V: 16-bit half word (within the V plane) of the four numbers d4 = 4·i .. 4·i + 3 of row r; number j of them is nibble j
AX_HD int ax_p4_v_half(const AxP4Shape& s, int r, int d4) {
    const int dg = d4 % s.group, g = dg / (s.group / 8), c = (d4 / s.group) * (s.group / 32) + (dg % (s.group / 8)) / 4;
    return ((((r >> 3) * 8 + g) * 4 + (r & 3)) * (s.hd / 32) + c) * 2 + ((r >> 2) & 1);
}
// scale (within the K or V scales) of group gr of row r
AX_HD int ax_p4_scale(const AxP4Shape& s, int r, int gr) { return ax_p4_col(r) * ax_p4_groups(s) + gr; }
// What is added to a scaled value |y| < 8 before it is cut off to a whole number: rounds half away from zero (1/2 − 2^-25, so that the number
// below 1/2 stays below 1).
AX_HD float ax_p4_half(float y) { return copysignf(0.49999997f, y); }
// slot / page_size without a division: (slot / 16) · ceil(2^36 / (page_size / 16)) >> 36.  slot / 16 < 2^27 and page_size / 16 ≤ 2^9, so it is exact.
AX_HD unsigned long long ax_p4_page_inverse(int page_size) {
    const unsigned long long d = (unsigned long long)page_size / AX_P4_TILE;
    return ((1ull << 36) + d - 1) / d;
}
AX_HD int ax_p4_page_of(int slot, unsigned long long inverse) { return (int)(((unsigned long long)(unsigned)(slot >> 4) * inverse) >> 36); }
