// Launch of the paged attention kernels (attention.h).
#include "attention.h"
#include "kv_host.h"

namespace vq {

AttnFn attn_kernels_bf16(int D, int qt, int W);
AttnFn attn_kernels_int8(int D, int qt, int W);

// One row of 20 heads over 4 key heads, 128 dims:
//  * 8 waves a CU (one workgroup, each wave a tile in use and one in flight): 131072
//    tokens 47.2 us, with 4 waves 52.3, 16 (in two workgroups) 49.5;
//  * up to 4096 tokens in the table workgroups of 4 waves, one tile each, over more
//    CUs (a CU reads 0.1 TB/s): 512 tokens 7.1 us, in eights 7.7;
//  * 80 KB of parts or more of a group of rows are joined by a launch of their own,
//    below by the workgroup that counts last: 16384 tokens in 64 parts 13.3 us
//    against 16.1, 512 in 4 parts 8.5 against 7.1 (2 x 16 rows of 8000: 20 against 37).
// Both limits lie between measured sizes, and both count what the table could hold (the
// host does not know the lengths): 611 tokens take 6.4 us in a table of 640, 7.5 in one
// of 4096 (a join launch for 5 parts), 7.0 of 4160 and 8.1 of 32768 (3 parts of 8 waves).
// Parts of equal steps dealt out over all sequences of a batch, whatever their
// lengths, were slower (32 x 8192 tokens 92.9 us against 85.7, 256 x 600 76 against
// 36): a part that ends one sequence and begins another waits at both.
constexpr int AT_WAVES = 8, AT_PARTS = 64, AT_SHORT = 4096 / KV_TILE, AT_APART = 80000;

struct AttnPlan {
    int qt, qgroups, waves, splits, lrows;
    size_t bytes;  // of workspace; 0: one part
};

static AttnPlan attn_plan(const viper_kv_cache* c, const viper_kv_batch* b, int heads) {
    AttnPlan p;
    const int gqa = heads / c->kv_heads, most = at_qt_max(c->head_dim);
    const int t16 = (b->max_rows * gqa + 15) / 16;
    p.qgroups = (t16 + most - 1) / most;
    p.qt = (t16 + p.qgroups - 1) / p.qgroups;
    p.lrows = b->max_rows * gqa < p.qt * 16 ? b->max_rows * gqa : p.qt * 16;
    const int64_t base = (int64_t)b->batch * c->kv_heads * p.qgroups;
    const int64_t tiles = (int64_t)b->table_width * (c->page_size / KV_TILE);
    p.waves = at_waves(c->head_dim, p.qt);
    if (tiles <= AT_SHORT) p.waves = 4;
    int64_t s = 1;
    if (base <= AT_CNT) {
        const bool two = b->batch > 1 && at_two(c->head_dim, c->kv_type == VIPER_KV_INT8, p.qt);
        const int64_t wgs = (int64_t)device_cus() * AT_WAVES * (two ? 2 : 1) / p.waves;
        s = (wgs + base - 1) / base;
        const int64_t fit = (tiles + p.waves - 1) / p.waves;
        if (s > fit) s = fit;
        if (s > AT_PARTS) s = AT_PARTS;
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
    // (rows may be read again after others are written)
    if (rows_meet(q_bf16, q_stride, width, out_bf16, out_stride, width, batch->total_rows)) return VIPER_INVALID_ARGUMENT;
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
    a.lrows = p.lrows;
    // a window longer than any sequence hides nothing (and p - window stays in 32 bits)
    a.window = window > INT32_MAX - VIPER_QLINEAR_MAX_M ? 0 : window;
    a.sinks = sinks;
    a.scale = scale * 1.44269504088896340736f;
    const int D = cache->head_dim;
    const AttnFn fn = cache->kv_type == VIPER_KV_INT8 ? attn_kernels_int8(D, p.qt, p.waves) : attn_kernels_bf16(D, p.qt, p.waves);
    if (fn.attn == nullptr) return VIPER_INTERNAL;
    a.by_gqa = (65536u + (unsigned)a.gqa - 1) / (unsigned)a.gqa;
    a.apart = p.splits > 1 && (int64_t)p.splits * p.lrows * D * 4 >= AT_APART;
    void* args[] = {&a};
    const dim3 grid((unsigned)p.splits, (unsigned)(cache->kv_heads * p.qgroups), (unsigned)batch->batch);
    (void)hipLaunchKernel(fn.attn, grid, dim3((unsigned)p.waves * 64), args, at_lds_bytes(D, p.qt, p.waves, p.lrows),
                          (hipStream_t)stream);
    if (a.apart) {
        const int rc2 = status_of(hipGetLastError());
        if (rc2 != VIPER_OK) return rc2;
        (void)hipLaunchKernel(fn.join, dim3((unsigned)p.lrows, grid.y, grid.z), dim3(AT_JNT), args, 0, (hipStream_t)stream);
    }
    return status_of(hipGetLastError());
}
