// Launch of the paged attention kernels (attention.h).
#include "attention.h"
#include "kv_host.h"

namespace vq {

const void* attn_kernel_bf16(int D, int qt);
const void* attn_kernel_int8(int D, int qt);

struct AttnPlan {
    int qt, qgroups, splits, min_tiles;
    size_t bytes;  // of workspace; 0: one part
};

static AttnPlan attn_plan(const viper_kv_cache* c, const viper_kv_batch* b, int heads) {
    AttnPlan p;
    const int gqa = heads / c->kv_heads, most = at_qt_max(c->head_dim);
    const int t16 = (b->max_rows * gqa + 15) / 16;
    p.qgroups = (t16 + most - 1) / most;
    p.qt = (t16 + p.qgroups - 1) / p.qgroups;
    p.min_tiles = AT_W;  // one per wave
    const int64_t base = (int64_t)b->batch * c->kv_heads * p.qgroups;
    const int64_t tiles = (int64_t)b->table_width * (c->page_size / KV_TILE);
    int64_t s = 1;
    if (base <= AT_CNT) {
        s = (2 * (int64_t)device_cus() + base - 1) / base;
        const int64_t fit = (tiles + p.min_tiles - 1) / p.min_tiles;
        if (s > fit) s = fit;
    }
    p.splits = (int)s;
    p.bytes = s > 1 ? AT_CNT * 4 + (size_t)base * s * at_part_floats(c->head_dim, p.qt) * 4 : 0;
    return p;
}

static int attn_check(const viper_kv_cache* c, const viper_kv_batch* b, int heads) {
    const int rc = kv_check(c, b);
    if (rc != VIPER_OK) return rc;
    if (b->max_rows > VIPER_QLINEAR_MAX_M) return VIPER_INVALID_ARGUMENT;
    if (heads <= 0 || heads % c->kv_heads != 0 || heads / c->kv_heads > 64) return VIPER_INVALID_ARGUMENT;
    return VIPER_OK;
}

}  // namespace vq

extern "C" size_t viper_hip_attention_workspace_bytes(const viper_kv_cache* cache, const viper_kv_batch* batch, int heads) {
    if (vq::attn_check(cache, batch, heads) != VIPER_OK) return 0;
    return vq::attn_plan(cache, batch, heads).bytes;
}

extern "C" int viper_hip_attention_paged(const viper_kv_cache* cache, const viper_kv_batch* batch, const void* q_bf16,
                                         int64_t q_stride, int heads, float scale, int window, int sinks, void* out_bf16,
                                         int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace vq;
    const int rc = attn_check(cache, batch, heads);
    if (rc != VIPER_OK) return rc;
    const int64_t width = (int64_t)heads * cache->head_dim;
    if (bad_rows(q_bf16, q_stride, width) || bad_rows(out_bf16, out_stride, width)) return VIPER_INVALID_ARGUMENT;
    if (!(scale > 0.0f) || scale > 1e30f || window < 0 || sinks < 0) return VIPER_INVALID_ARGUMENT;
    AttnPlan p = attn_plan(cache, batch, heads);
    if (workspace == nullptr) {
        p.splits = 1;
    } else if (misaligned(workspace, 16) || workspace_bytes < p.bytes) {
        return VIPER_INVALID_ARGUMENT;
    }
    if (batch->total_rows == 0) return VIPER_OK;
    AttnArgs a;
    a.c = kv_args(cache, batch);
    a.q = (const uint16_t*)q_bf16;
    a.out = (uint16_t*)out_bf16;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.cnt = (unsigned*)workspace;
    a.part = (float*)workspace + AT_CNT;
    a.gqa = heads / cache->kv_heads;
    a.qgroups = p.qgroups;
    a.splits = p.splits;
    a.min_tiles = p.min_tiles;
    // a window longer than any sequence hides nothing (and p - window stays in 32 bits)
    a.window = window > INT32_MAX - VIPER_QLINEAR_MAX_M ? 0 : window;
    a.sinks = sinks;
    a.scale = scale * 1.44269504088896340736f;
    const int64_t grid = (int64_t)batch->batch * cache->kv_heads * p.qgroups * p.splits;
    if (grid > (1 << 24) - 1) return VIPER_INVALID_ARGUMENT;
    const int D = cache->head_dim;
    const void* fn = cache->kv_type == VIPER_KV_INT8 ? attn_kernel_int8(D, p.qt) : attn_kernel_bf16(D, p.qt);
    if (fn == nullptr) return VIPER_INTERNAL;
    void* args[] = {&a};
    launch(fn, (unsigned)grid, AT_NT, at_lds_bytes(D, p.qt), (hipStream_t)stream, args);
    return status_of(hipGetLastError());
}
