// Launch of the paged attention kernels (attention.h).
#include "attention.h"
#include "kv_host.h"

namespace vq {

AttnFn attn_kernels_bf16(int D, int qt, int W);
AttnFn attn_kernels_int8(int D, int qt, int W);
AttnFn attn_kernels_fp4(int D, int qt, int W);
AttnFn attn_selected_bf16(int D, int qt, int W);
AttnFn attn_selected_int8(int D, int qt, int W);
AttnFn attn_selected_fp4(int D, int qt, int W);

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
constexpr int AT_WAVES = 8, AT_SHORT = 4096 / KV_TILE, AT_APART = 80000;

struct AttnPlan {
    int qt, qgroups, waves, splits, lrows;
    int shared;  // parts of all sequences together where they are shared out by length, 0: not
    bool two;      // workgroups of 8 waves to a CU
    size_t bytes;  // of workspace; 0: one part
};

// `units` sequences of `rows` rows that look at up to `tiles` tiles each
static AttnPlan attn_plan(const viper_kv_cache* c, int rows, int64_t units, int64_t tiles, int heads, bool share) {
    AttnPlan p;
    const int gqa = heads / c->kv_heads, most = at_qt_max(c->head_dim);
    const int t16 = (rows * gqa + 15) / 16;
    p.qgroups = (t16 + most - 1) / most;
    p.qt = (t16 + p.qgroups - 1) / p.qgroups;
    p.lrows = rows * gqa < p.qt * 16 ? rows * gqa : p.qt * 16;
    const int64_t base = units * c->kv_heads * p.qgroups;
    p.waves = at_waves(c->head_dim, p.qt);
    if (tiles <= AT_SHORT) p.waves = 4;
    int64_t s = 1;
    p.shared = 0;
    p.two = false;
    if (base <= AT_CNT) {
        p.two = units > 1 && at_two(c->head_dim, c->kv_type != VIPER_KV_BF16, p.qt);
        const int64_t wgs = (int64_t)device_cus() * AT_WAVES * (p.two ? 2 : 1) / p.waves;
        s = (wgs + base - 1) / base;
        const int64_t fit = (tiles + p.waves - 1) / p.waves;
        if (share && units > 1 && units <= 64 && s > 1 && fit > 1) {
            const int64_t all = wgs / (c->kv_heads * p.qgroups);  // (at least one to a sequence)
            p.shared = (int)(all < units * fit ? all : units * fit);
        }
        if (s > fit) s = fit;
        if (s > AT_PARTS) s = AT_PARTS;
    }
    p.splits = (int)s;
    const int64_t parts = base * s, shared = (int64_t)p.shared * c->kv_heads * p.qgroups;
    p.bytes = s > 1 ? AT_CNT * 4 + (size_t)(parts > shared ? parts : shared) * at_part_floats(c->head_dim, p.qt) * 4 : 0;
    return p;
}
static AttnPlan attn_plan(const viper_kv_cache* c, const viper_kv_batch* b, int heads) {
    return attn_plan(c, b->max_rows, b->batch, (int64_t)b->table_width * (c->page_size / KV_TILE), heads,
                     c->kv_type == VIPER_KV_FP4);
}
// (over lists, every row is a sequence of its own)
static AttnPlan attn_plan_selected(const viper_kv_cache* c, const viper_kv_batch* b, int heads, int count) {
    return attn_plan(c, 1, (int64_t)b->batch * b->max_rows, (int64_t)count * (c->page_size / KV_TILE), heads, false);
}

static int attn_check(const viper_kv_cache* c, const viper_kv_batch* b, int heads) {
    const int rc = kv_check(c, b);
    if (rc != VIPER_OK) return rc;
    if (b->max_rows > VIPER_QLINEAR_MAX_M) return VIPER_INVALID_ARGUMENT;
    if (heads <= 0 || heads % c->kv_heads != 0 || heads / c->kv_heads > 64) return VIPER_INVALID_ARGUMENT;
    return VIPER_OK;
}

static int selected_check(const viper_kv_cache* c, const viper_kv_batch* b, int heads, int count) {
    const int rc = attn_check(c, b, heads);
    if (rc != VIPER_OK) return rc;
    return count > 0 && (int64_t)count * c->page_size <= INT32_MAX ? VIPER_OK : VIPER_INVALID_ARGUMENT;
}

// One call: over the whole sequences, or over the pages of lists (sel)
static int attn_call(const viper_kv_cache* cache, const viper_kv_batch* batch, const void* q_bf16, int64_t q_stride, int heads,
                     float scale, int window, int sinks, const int32_t* sel, int count, void* out_bf16, int64_t out_stride,
                     void* workspace, size_t workspace_bytes, AttnPlan p, void* stream) {
    const int64_t width = (int64_t)heads * cache->head_dim;
    if (bad_rows(q_bf16, q_stride, width) || bad_rows(out_bf16, out_stride, width)) return VIPER_INVALID_ARGUMENT;
    if (!(scale > 0.0f) || scale > 1e30f || window < 0 || sinks < 0) return VIPER_INVALID_ARGUMENT;
    if (workspace == nullptr) {
        p.splits = 1;
    } else if (misaligned(workspace, 16) || workspace_bytes < p.bytes) {
        return VIPER_INVALID_ARGUMENT;
    }
    if (batch->total_rows == 0) return VIPER_OK;
    // (rows may be read again after others are written)
    if (rows_meet(q_bf16, q_stride, width, out_bf16, out_stride, width, batch->total_rows)) return VIPER_INVALID_ARGUMENT;
    if (sel != nullptr && ranges_meet(out_bf16, ((size_t)(batch->total_rows - 1) * out_stride + width) * 2, sel,
                                      (size_t)batch->total_rows * cache->kv_heads * count * 4))
        return VIPER_INVALID_ARGUMENT;
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
    a.sel = sel;
    a.count = count;
    a.share = p.splits > 1 && p.shared > 0 && a.window == 0;
    if (a.share) a.splits = p.shared;
    const int D = cache->head_dim, rows = sel != nullptr ? batch->max_rows : 1;
    const int kind = (cache->kv_type == VIPER_KV_INT8 ? 1 : cache->kv_type == VIPER_KV_FP4 ? 2 : 0) + (sel != nullptr ? 3 : 0);
    static AttnFn (*const of[])(int, int, int) = {attn_kernels_bf16,  attn_kernels_int8,  attn_kernels_fp4,
                                                  attn_selected_bf16, attn_selected_int8, attn_selected_fp4};
    const AttnFn fn = of[kind](D, p.qt, p.waves);
    if (fn.attn == nullptr) return VIPER_INTERNAL;
    a.by_gqa = (65536u + (unsigned)a.gqa - 1) / (unsigned)a.gqa;
    a.apart = p.splits > 1 && (int64_t)p.splits * p.lrows * D * 4 >= AT_APART;
    // Over lists, and over FP4 caches where parts are not shared out: from 16 parts on, from 8 where two
    // workgroups share a CU and 128 join.  FP4, 20 heads over 4 of 128 dims, lists of 64 tiles (16 parts) of
    // 1 / 4 / 16 rows 7.7 / 9.9 / 15.3 us joined below and 7.4 / 7.7 / 10.4 apart, of 32 tiles (8 parts) 6.9 / 8.0 / 9.6
    // and 7.3 / 7.5 / 8.3, of 16 tiles (4 parts) 6.4 / 6.9 / 7.5 and 7.1 / 7.3 / 7.4 (bf16, 8 parts of 16
    // rows over 128 tiles 24.6 and 25.1); shared out parts of 4 sequences of 1024 tokens 7.7 and 8.9.
    if (sel != nullptr || (cache->kv_type == VIPER_KV_FP4 && !a.share)) {
        const int64_t joined = (int64_t)p.splits * batch->batch * rows * cache->kv_heads * p.qgroups;
        a.apart |= p.splits >= 16 || (p.two && p.splits >= 8 && joined >= 128);
    }
    void* args[] = {&a};
    const dim3 grid((unsigned)(a.splits * rows), (unsigned)(cache->kv_heads * p.qgroups), a.share ? 1u : (unsigned)batch->batch);
    (void)hipLaunchKernel(fn.attn, grid, dim3((unsigned)p.waves * 64), args, at_lds_bytes(D, p.qt, p.waves, p.lrows),
                          (hipStream_t)stream);
    if (a.apart) {
        const int rc2 = status_of(hipGetLastError());
        if (rc2 != VIPER_OK) return rc2;
        (void)hipLaunchKernel(fn.join, dim3((unsigned)(p.lrows * rows), grid.y, (unsigned)batch->batch), dim3(AT_JNT), args, 0, (hipStream_t)stream);
    }
    return status_of(hipGetLastError());
}

}  // namespace vq

extern "C" size_t viper_hip_attention_workspace_bytes(const viper_kv_cache* cache, const viper_kv_batch* batch, int heads) {
    if (vq::attn_check(cache, batch, heads) != VIPER_OK) return 0;
    return vq::attn_plan(cache, batch, heads).bytes;
}

extern "C" int viper_hip_attention_paged(const viper_kv_cache* cache, const viper_kv_batch* batch, const void* q_bf16,
                                         int64_t q_stride, int heads, float scale, int window, int sinks, void* out_bf16,
                                         int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = vq::attn_check(cache, batch, heads);
    if (rc != VIPER_OK) return rc;
    return vq::attn_call(cache, batch, q_bf16, q_stride, heads, scale, window, sinks, nullptr, 0, out_bf16, out_stride, workspace,
                         workspace_bytes, vq::attn_plan(cache, batch, heads), stream);
}

extern "C" size_t viper_hip_attention_selected_workspace_bytes(const viper_kv_cache* cache, const viper_kv_batch* batch, int heads,
                                                               int count) {
    if (vq::selected_check(cache, batch, heads, count) != VIPER_OK) return 0;
    return vq::attn_plan_selected(cache, batch, heads, count).bytes;
}

extern "C" int viper_hip_attention_selected(const viper_kv_cache* cache, const viper_kv_batch* batch, const void* q_bf16,
                                            int64_t q_stride, int heads, float scale, const int32_t* selected, int count,
                                            void* out_bf16, int64_t out_stride, void* workspace, size_t workspace_bytes,
                                            void* stream) {
    const int rc = vq::selected_check(cache, batch, heads, count);
    if (rc != VIPER_OK) return rc;
    if (selected == nullptr || vq::misaligned(selected, 4)) return VIPER_INVALID_ARGUMENT;
    return vq::attn_call(cache, batch, q_bf16, q_stride, heads, scale, 0, 0, selected, count, out_bf16, out_stride, workspace,
                         workspace_bytes, vq::attn_plan_selected(cache, batch, heads, count), stream);
}
