// Host side of the cache operators: argument checks and the kernels' view.
#pragma once

#include "kv_dev.h"
#include "qlinear_host.h"

namespace vq {

inline int kv_check(const viper_kv_cache* c, const viper_kv_batch* b) {
    if (c == nullptr || b == nullptr) return VIPER_INVALID_ARGUMENT;
    if (c->kv_type != VIPER_KV_BF16 && c->kv_type != VIPER_KV_INT8) return VIPER_INVALID_ARGUMENT;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return VIPER_INVALID_ARGUMENT;
    if (c->page_size != 32 && c->page_size != 64 && c->page_size != 128 && c->page_size != 256)
        return VIPER_INVALID_ARGUMENT;
    if (c->kv_heads <= 0 || c->kv_heads > 1024 || c->num_pages <= 0) return VIPER_INVALID_ARGUMENT;
    if (c->k == nullptr || c->v == nullptr || misaligned(c->k, 16) || misaligned(c->v, 16)) return VIPER_INVALID_ARGUMENT;
    const bool scales = c->k_scales != nullptr && c->v_scales != nullptr;
    if (c->kv_type == VIPER_KV_INT8) {
        if (!scales || misaligned(c->k_scales, 16) || misaligned(c->v_scales, 16)) return VIPER_INVALID_ARGUMENT;
    } else if (c->k_scales != nullptr || c->v_scales != nullptr) {
        return VIPER_INVALID_ARGUMENT;
    }
    if (b->batch <= 0 || b->max_rows <= 0 || b->total_rows < 0 || b->table_width <= 0) return VIPER_INVALID_ARGUMENT;
    if (b->batch > 65535 || (int64_t)b->table_width * c->page_size > INT32_MAX) return VIPER_INVALID_ARGUMENT;
    if (b->block_table == nullptr || b->seq_lens == nullptr || misaligned(b->block_table, 4) ||
        misaligned(b->seq_lens, 4) || misaligned(b->row_offsets, 4))
        return VIPER_INVALID_ARGUMENT;
    if (b->row_offsets == nullptr && (int64_t)b->batch * b->max_rows != b->total_rows) return VIPER_INVALID_ARGUMENT;
    return VIPER_OK;
}

inline KvArgs kv_args(const viper_kv_cache* c, const viper_kv_batch* b) {
    KvArgs a;
    a.table = b->block_table;
    a.lens = b->seq_lens;
    a.offs = b->row_offsets;
    a.k = c->k;
    a.v = c->v;
    a.ks = c->k_scales;
    a.vs = c->v_scales;
    a.batch = b->batch;
    a.max_rows = b->max_rows;
    a.total_rows = b->total_rows;
    a.width = b->table_width;
    a.kvh = c->kv_heads;
    a.pages = c->num_pages;
    a.tpl = c->page_size == 32 ? 0 : c->page_size == 64 ? 1 : c->page_size == 128 ? 2 : 3;
    return a;
}

// Rows of a bf16 row tensor: dense values, rows 16-byte aligned.
inline bool bad_rows(const void* p, int64_t stride, int64_t width) {
    return p == nullptr || misaligned(p, 16) || stride < width || stride % 8 != 0 || stride > (int64_t)1 << 40;
}

// Whether two tensors of n rows (dense rows of pw and ow bf16 values, their strides
// in elements) have a value in common, or reach further than any memory.  Columns of
// one wider matrix have one stride and need no walk.
inline bool rows_meet(const void* p, int64_t ps, int64_t pw, const void* o, int64_t os, int64_t ow, int64_t n) {
    if (ps > ((int64_t)1 << 48) / n || os > ((int64_t)1 << 48) / n) return true;
    // the second begins d elements past the first
    const int64_t d = ((int64_t)(uintptr_t)o - (int64_t)(uintptr_t)p) / 2;
    if (d >= (n - 1) * ps + pw || -d >= (n - 1) * os + ow) return false;
    auto below = [](int64_t a, int64_t b) { return a >= 0 ? a / b : -((-a + b - 1) / b); };  // floor(a / b)
    if (ps == os) {  // row i + k of the second begins d + k s past row i: from -ow + 1 to pw - 1 they meet
        const int64_t k0 = below(-ow - d, os) + 1, k1 = below(pw - 1 - d, os);
        return (k0 > 1 - n ? k0 : 1 - n) <= (k1 < n - 1 ? k1 : n - 1);
    }
    for (int64_t i = 0; i < n; ++i) {
        const int64_t e = i * ps - d, j0 = below(e - ow, os) + 1, j1 = below(e + pw - 1, os);
        if ((j0 > 0 ? j0 : 0) <= (j1 < n - 1 ? j1 : n - 1)) return true;
    }
    return false;
}

}  // namespace vq
