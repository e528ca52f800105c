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

}  // namespace vq
