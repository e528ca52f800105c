// The paged key/value cache: its device view, its tiles' order, and which rows
// of a call belong to which tokens.
#pragma once

#include "qlinear_dev.h"

namespace vq {

constexpr int KV_TILE = VIPER_KV_TILE;

// What every kernel over a cache takes (by value).
struct KvArgs {
    const int32_t* table;  // [batch][width]
    const int32_t* lens;   // [batch]
    const int32_t* offs;   // [batch + 1] or null
    void* k;
    void* v;
    float* ks;  // (FP4: bytes)
    float* vs;
    int batch, max_rows, total_rows, width;
    int kvh, pages, tpl;  // tiles of a page: 1 << tpl
};

// Element of (token t of the tile, octet c of the row: dims 8c .. 8c + 7) in a
// K tile.  Octets are contiguous there.  A wave's load of one chunk (kb, s) is
// the A operand of a 16x16x32 product: row m = 4a + i of it is token 8a + 4s +
// i, so the products of s = 0 and 1 leave each lane with the scores of the 8
// consecutive tokens 8g .. 8g + 7 (g = lane / 16), the k-slots of the second
// product's operand.
template <bool I8>
__device__ __forceinline__ int k_place(int t, int c) {
    const int s = (t >> 2) & 1, m = 4 * (t >> 3) + (t & 3), lane = 16 * (c & 3) + m;
    return I8 ? 1024 * (2 * (c >> 3) + s) + 16 * lane + 8 * ((c >> 2) & 1) : 512 * (2 * (c >> 2) + s) + 8 * lane;
}
// Element of (token t, dim d) in a V tile: 8 consecutive tokens of a dim are
// contiguous; a chunk is the A operand with dims as its rows.
template <bool I8>
__device__ __forceinline__ int v_place(int t, int d) {
    const int lane = 16 * (t >> 3) + (d & 15);
    return I8 ? 1024 * (d >> 5) + 16 * lane + 8 * ((d >> 4) & 1) + (t & 7) : 512 * (d >> 4) + 8 * lane + (t & 7);
}

// FP4 tiles, in bytes: octet c of token t of a K tile is one word, and so are 8
// tokens of dim d of a V tile.  A lane's 16 bytes of K are 32 (head_dim 64: 16)
// consecutive dims of its token, so that they share a power of two.  The first
// product's k-slots are then dims q4_dim() and not kb * 32 + 8 g, for Q as well.
template <int D>
__device__ __forceinline__ int k4_place(int t, int c) {
    const int s = (t >> 2) & 1, m = 4 * (t >> 3) + (t & 3);
    return D == 64 ? 16 * (16 * (c >> 1) + m) + 8 * s + 4 * (c & 1)
                   : 1024 * (2 * (c >> 4) + s) + 16 * (16 * ((c >> 2) & 3) + m) + 4 * (c & 3);
}
__device__ __forceinline__ int v4_place(int t, int d) {
    return 1024 * (d >> 6) + 16 * (16 * (t >> 3) + (d & 15)) + 4 * ((d >> 4) & 3);
}
// Byte of block c (of 32 dims) of token t in a tile's powers of two
template <int D>
__device__ __forceinline__ int k4_exp_place(int t, int c) {
    const int s = (t >> 2) & 1, m = 4 * (t >> 3) + (t & 3);
    return D == 64 ? 2 * (16 * c + m) + s : (16 * (c & 3) + m) * (D / 64) + 2 * (c >> 2) + s;
}
template <int D>
__device__ __forceinline__ int q4_dim(int kb, int g) {
    return D == 64 ? 16 * g + 8 * kb : 128 * (kb >> 2) + 32 * g + 8 * (kb & 3);
}
// 8 codes of a word times the power of two of `scale` (only its exponent counts,
// NaN's makes NaN), one instruction for two of them; exact
__device__ __forceinline__ u32x4 fp4_bf16(uint32_t w, float scale) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
}
__device__ __forceinline__ void fp4_f32(uint32_t w, float scale, float* f) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1),
               c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
    f[0] = a[0], f[1] = a[1], f[2] = b[0], f[3] = b[1], f[4] = c[0], f[5] = c[1], f[6] = d[0], f[7] = d[1];
}
// The power of two that a byte of k_scales stands for
__device__ __forceinline__ float fp4_power(uint32_t byte) { return __uint_as_float(byte << 23); }

// Wave-uniform reads of the arrays through the scalar cache (read-only within a
// launch), so that a page's number is in scalar registers and its wait does not
// count the vector loads in flight.
typedef const __attribute__((address_space(4))) int32_t* kv_cptr;
__device__ __forceinline__ int kv_sload(const int32_t* p, size_t i) { return ((kv_cptr)(uintptr_t)p)[i]; }

// Sum over the lanes of a wave up to the lane's own
__device__ __forceinline__ unsigned wave_upto(unsigned v) {
    v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);  // from 1, 2, 4, 8 lanes back in the row
    v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
    v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
    v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
    v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);  // a row's last lane to the row behind it
    v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);  // the lower half's to the upper half
    return v;
}

// Sequence b's rows: the first, their count (0 where the offsets do not fit)
// and the sequence's length.
struct KvSeq {
    int row0, n, len;
};
__device__ __forceinline__ KvSeq kv_seq(const KvArgs& a, int b) {
    KvSeq q;
    q.len = kv_sload(a.lens, b);
    if (a.offs != nullptr) {
        const int o = kv_sload(a.offs, b), e = kv_sload(a.offs, b + 1);
        const bool fits = o >= 0 && o <= e && e <= a.total_rows && e - o <= a.max_rows;
        q.row0 = fits ? o : 0;
        q.n = fits ? e - o : 0;
    } else {
        q.row0 = b * a.max_rows;
        q.n = a.max_rows;
    }
    return q;
}

// Page of tile `tile` of sequence b, -1 where the table has none in the pool.
__device__ __forceinline__ int kv_page(const KvArgs& a, int b, int tile) {
    const int col = tile >> a.tpl;
    if (col >= a.width) return -1;
    const int p = a.table[(size_t)b * a.width + col];
    return (unsigned)p < (unsigned)a.pages ? p : -1;
}
__device__ __forceinline__ int kv_page_uniform(const KvArgs& a, int b, int tile) {
    const int col = tile >> a.tpl;
    if (col >= a.width) return -1;
    const int p = kv_sload(a.table, (size_t)b * a.width + col);
    return (unsigned)p < (unsigned)a.pages ? p : -1;
}
// Tile number in the pool (times 32 * D elements; times 32 for the scales).
__device__ __forceinline__ size_t kv_tile_at(const KvArgs& a, int page, int head, int tile) {
    return (((size_t)page * a.kvh + head) << a.tpl) + (tile & ((1 << a.tpl) - 1));
}

}  // namespace vq
