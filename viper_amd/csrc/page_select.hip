// Which pages of a long sequence a row is to look at.
//
// bounds: per page and key head the least and largest value of every dimension over the
// keys held.  bf16 patterns are compared as 16-bit integers in the values' order, two at
// a time, where NaN lies past the infinities and so is not lost.
//
// selection: q . k of any key of a page is at most sum_d max(q_d lo_d, q_d hi_d), the page's
// score for a query head; the largest over the heads of a key head counts.  A page at the
// border is in or out, so products (exact in 32 bits) are summed in 64.  Scores become
// integers in their order; the smallest that is in is found bit by bit, by counting.

#include "kv_host.h"

namespace vq {

constexpr int PB_NT = 256;

// ----------------------------------------------------------------- bounds

struct BoundsArgs {
    KvArgs c;
    uint16_t* out;
    int span;  // pages that a sequence's rows can touch
};

typedef short pb_i16x2 __attribute__((ext_vector_type(2)));
// bf16 patterns <-> integers in the values' order (its own inverse)
__device__ __forceinline__ uint32_t pb_order(uint32_t w) {
    const pb_i16x2 v = __builtin_bit_cast(pb_i16x2, w);
    return w ^ (__builtin_bit_cast(uint32_t, v >> 15) & 0x7fff7fffu);
}
__device__ __forceinline__ uint32_t pb_min(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(pb_i16x2, a), __builtin_bit_cast(pb_i16x2, b)));
}
__device__ __forceinline__ uint32_t pb_max(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pb_i16x2, a), __builtin_bit_cast(pb_i16x2, b)));
}
template <int CTRL>
__device__ __forceinline__ void pb_step(uint32_t* lo, uint32_t* hi) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo[i] = pb_min(lo[i], (uint32_t)dpp_i<CTRL>((int)lo[i]));
        hi[i] = pb_max(hi[i], (uint32_t)dpp_i<CTRL>((int)hi[i]));
    }
}

// A workgroup per page and head; a wave takes chunks of 32 dims of all tiles, a lane the
// octet of the token that the tile's order gives it.
template <int D, int KT>
__global__ void __launch_bounds__(PB_NT)
page_bounds_kernel(BoundsArgs a) {
    constexpr int NKB = D / 32, W = NKB < 4 ? NKB : 4;
    const int tid = (int)threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = (int)blockIdx.x;
    const int head = id % a.c.kvh;
    id /= a.c.kvh;
    const int b = id / a.span;
    const KvSeq s = kv_seq(a.c, b);
    if (s.n == 0 || s.len <= 0) return;
    const int from = max(0, s.len - s.n), shift = a.c.tpl + 5;
    const int64_t page64 = (int64_t)(from >> shift) + id % a.span;
    if (page64 << shift >= s.len) return;
    const int tile0 = (int)(page64 << a.c.tpl), tiles = min(1 << a.c.tpl, (s.len - 1) / KV_TILE - tile0 + 1);
    const int page = kv_page_uniform(a.c, b, tile0);
    if (page < 0) return;
    for (int kb = wave; kb < NKB; kb += W) {
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lo[i] = 0x7fff7fffu;
            hi[i] = 0x80008000u;
        }
#pragma unroll 2
        for (int tl = 0; tl < tiles; ++tl) {
            const size_t at = kv_tile_at(a.c, page, head, tl);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int t = 8 * (m >> 2) + 4 * h + (m & 3), c = 4 * kb + g;
                u32x4 x;
                if constexpr (KT == VIPER_KV_BF16) {
                    x = *(const u32x4*)((const uint16_t*)a.c.k + at * (KV_TILE * D) + k_place<false>(t, c));
                } else if constexpr (KT == VIPER_KV_INT8) {
                    const u32x2 w = *(const u32x2*)((const int8_t*)a.c.k + at * (KV_TILE * D) + k_place<true>(t, c));
                    const float sc = a.c.ks[at * KV_TILE + t];
                    float y[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[j] = (float)(int8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3))) * sc;
                    x = u32x4{f2bf2(y[0], y[1]), f2bf2(y[2], y[3]), f2bf2(y[4], y[5]), f2bf2(y[6], y[7])};
                } else {
                    const uint32_t w = *(const uint32_t*)((const uint8_t*)a.c.k + at * (KV_TILE * D / 2) + k4_place<D>(t, c));
                    x = fp4_bf16(w, fp4_power(((const uint8_t*)a.c.ks)[at * D + k4_exp_place<D>(t, kb)]));
                }
                const bool held = (tile0 + tl) * KV_TILE + t < s.len;
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t v = pb_order(w[i]);
                    lo[i] = pb_min(lo[i], held ? v : 0x7fff7fffu);
                    hi[i] = pb_max(hi[i], held ? v : 0x80008000u);
                }
            }
        }
        pb_step<DPP_SWAP1>(lo, hi);
        pb_step<DPP_SWAP2>(lo, hi);
        pb_step<DPP_HALF_MIRROR>(lo, hi);
        pb_step<DPP_MIRROR>(lo, hi);
        if (m < 2) {  // one lane stores the least, one the largest values
            u32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t l = pb_order(lo[i]), u = pb_order(hi[i]);
                v[i] = m == 0 ? l : u;
                // a NaN key makes both NaN
                const uint32_t n0 = (l & 0x7fffu) > 0x7f80u || (u & 0x7fffu) > 0x7f80u ? 0x7fc0u : 0u;
                const uint32_t n1 = (l >> 16 & 0x7fffu) > 0x7f80u || (u >> 16 & 0x7fffu) > 0x7f80u ? 0x7fc00000u : 0u;
                v[i] = n0 != 0u ? (v[i] & 0xffff0000u) | n0 : v[i];
                v[i] = n1 != 0u ? (v[i] & 0xffffu) | n1 : v[i];
            }
            *(u32x4*)(a.out + (((size_t)page * a.c.kvh + head) * 2 + m) * D + 32 * kb + 8 * g) = v;
        }
    }
}

// ----------------------------------------------------------------- scores

constexpr int PS_NT = 256;
constexpr int PS_LDS = 32768;  // bytes of q that a workgroup keeps at a time

struct SelectArgs {
    KvArgs c;
    const uint16_t* q;
    int64_t q_stride;
    const uint16_t* bounds;
    int32_t* out;
    uint32_t* keys;  // [batch * max_rows][key head][width]
    int gqa, count, first, last, chunks;
};

// Pages of the row at position p (0: no token)
__device__ __forceinline__ int ps_pages(const KvArgs& c, int64_t p) {
    return p < 0 ? 0 : (int)min((int64_t)c.width, (p >> (c.tpl + 5)) + 1);
}
// A score as an integer in its order, above 0; NaN as +inf
__device__ __forceinline__ uint32_t ps_key(float v) {
    if (v != v) v = __builtin_inff();
    const uint32_t u = __float_as_uint(v);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
template <int L>
__device__ __forceinline__ double ps_sum(double v) {
    auto step = [&](auto dpp) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)dpp((int)(uint32_t)u), hi = (uint32_t)dpp((int)(u >> 32));
        v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    };
    step([](int x) { return dpp_i<DPP_SWAP1>(x); });
    step([](int x) { return dpp_i<DPP_SWAP2>(x); });
    step([](int x) { return dpp_i<DPP_HALF_MIRROR>(x); });
    if constexpr (L >= 16) step([](int x) { return dpp_i<DPP_MIRROR>(x); });
    if constexpr (L >= 32) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const auto l = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false);
        const auto h = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
        v = __builtin_bit_cast(double, (uint64_t)h[0] << 32 | l[0]) + __builtin_bit_cast(double, (uint64_t)h[1] << 32 | l[1]);
    }
    return v;
}

// D / 8 lanes to a page, each with 8 dims of it; the rows' queries come from LDS
template <int D>
__global__ void __launch_bounds__(PS_NT)
page_score_kernel(SelectArgs a) {
    constexpr int L = D / 8, PP = PS_NT / L;
    extern __shared__ __align__(16) uint16_t lq[];  // [rows of a turn][gqa][D]
    const int tid = (int)threadIdx.x, l = tid % L;
    const int head = (int)blockIdx.y, b = (int)blockIdx.z;
    const KvSeq s = kv_seq(a.c, b);
    const int64_t pos0 = (int64_t)s.len - s.n;
    const int all = ps_pages(a.c, (int64_t)s.len - 1), p = (int)blockIdx.x * PP + tid / L;
    if (s.n == 0 || (int)blockIdx.x * PP >= all) return;
    const int page = p < all ? a.c.table[(size_t)b * a.c.width + p] : -1;
    const bool there = (unsigned)page < (unsigned)a.c.pages;
    float lo[8], hi[8];
    {
        u32x4 x = {0u, 0u, 0u, 0u}, y = x;
        if (there) {
            const uint16_t* at = a.bounds + ((size_t)page * a.c.kvh + head) * (2 * D) + 8 * l;
            x = *(const u32x4*)at;
            y = *(const u32x4*)(at + D);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lo[i] = bf16f(x[i >> 1] >> (16 * (i & 1)) & 0xffffu);
            hi[i] = bf16f(y[i >> 1] >> (16 * (i & 1)) & 0xffffu);
        }
    }
    const int turn = max(1, PS_LDS / (a.gqa * D * 2));  // (64 heads of 256 dims: one row)
    for (int r0 = 0; r0 < s.n; r0 += turn) {
        const int rows = min(turn, s.n - r0);
        if (r0) __syncthreads();
        for (int i = tid; i < rows * a.gqa * L; i += PS_NT) {
            const int r = i / (a.gqa * L), x = i % (a.gqa * L);
            *(u32x4*)(lq + (size_t)i * 8) =
                *(const u32x4*)(a.q + (size_t)(s.row0 + r0 + r) * a.q_stride + (size_t)head * a.gqa * D + 8 * x);
        }
        __syncthreads();
        for (int r = 0; r < rows; ++r) {
            if (p >= ps_pages(a.c, pos0 + r0 + r)) continue;
            double best = -__builtin_inf();
            bool nan = false;
            for (int h = 0; h < a.gqa; ++h) {
                const u32x4 w = *(const u32x4*)(lq + (size_t)(r * a.gqa + h) * D + 8 * l);
                double sum = 0.0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = bf16f(w[i >> 1] >> (16 * (i & 1)) & 0xffffu);
                    // (NaN where either product is: an infinite bound under a zero)
                    const float u = x * lo[i], v = x * hi[i];
                    sum += (double)(u != u || v != v ? __builtin_nanf("") : fmaxf(u, v));
                }
                sum = ps_sum<L>(sum);
                nan |= sum != sum;
                best = fmax(best, sum);
            }
            if (l == 0)
                a.keys[((size_t)(b * a.c.max_rows + r0 + r) * a.c.kvh + head) * a.c.width + p] =
                    there ? ps_key(nan ? __builtin_inff() : (float)best) : 0u;
        }
    }
}

// ----------------------------------------------------------------- selection

constexpr int PK_NT = 512, PK_KPT = 8, PK_W = PK_NT / 64;

// A workgroup per row and key head; a thread holds PK_KPT consecutive pages (rows of more
// pages than that are walked again at each step).
__global__ void __launch_bounds__(PK_NT)
page_pick_kernel(SelectArgs a) {
    __shared__ unsigned part[2][PK_W];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = (int)blockIdx.x, head = (int)blockIdx.y, b = (int)blockIdx.z;
    const KvSeq s = kv_seq(a.c, b);
    if (r >= s.n) return;
    const int64_t p = (int64_t)s.len - s.n + r;
    const int n = ps_pages(a.c, p);
    const int first = min(a.first, n), last = max(first, n - a.last);  // first and last are in, [first, last) is ranked
    int32_t* const out = a.out + ((size_t)(s.row0 + r) * a.c.kvh + head) * a.count;
    const uint32_t* const keys = a.keys + ((size_t)(b * a.c.max_rows + r) * a.c.kvh + head) * a.c.width;
    const unsigned want = (unsigned)(a.count - (n - (last - first)));  // of the ranked ones (first + last <= count)
    const int turns = (n + PK_NT * PK_KPT - 1) / (PK_NT * PK_KPT);
    uint32_t key[PK_KPT];
    auto load = [&](int turn) {
#pragma unroll
        for (int k = 0; k < PK_KPT; ++k) {
            const int at = (turn * PK_NT + tid) * PK_KPT + k;
            key[k] = at >= first && at < last ? keys[at] : 0u;
        }
    };
    int side = 0;
    auto total = [&](unsigned mine) {  // (of the waves' counts)
        if (lane == 0) part[side][wave] = mine;
        __syncthreads();
        unsigned t = 0;
#pragma unroll
        for (int w = 0; w < PK_W; ++w) t += part[side][w];
        side ^= 1;
        return t;
    };
    if (turns == 1) load(0);
    auto count_from = [&](uint32_t t) {
        unsigned c = 0;
        for (int turn = 0; turn < turns; ++turn) {
            if (turns > 1) load(turn);
#pragma unroll
            for (int k = 0; k < PK_KPT; ++k) c += (unsigned)__popcll(__ballot(key[k] >= t));
        }
        return total(c);
    };
    // the largest t that `want` keys reach; 0: there are not so many
    uint32_t t = 0;
    for (int bit = 31; bit >= 0; --bit)
        if (count_from(t | 1u << bit) >= want) t |= 1u << bit;
    const unsigned ties = t == 0u || t == 0xffffffffu ? 0u : want - count_from(t + 1);  // of the keys that are t
    // their numbers in order: what is in for certain and how many ties come before a thread's
    unsigned sure0 = 0, tie0 = 0;
    for (int turn = 0; turn < turns; ++turn) {
        if (turns > 1) load(turn);
        const int at0 = (turn * PK_NT + tid) * PK_KPT;
        unsigned mine = 0;  // sure ones, and ties in the upper half
#pragma unroll
        for (int k = 0; k < PK_KPT; ++k) {
            const int at = at0 + k;
            const bool in = at < n && (at < first || at >= last || key[k] > t);
            mine += in ? 1u : at < n && t != 0u && key[k] == t ? 1u << 16 : 0u;
        }
        unsigned before = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const unsigned v = (unsigned)__shfl_up((int)before, d);
            if (lane >= d) before += v;
        }
        const unsigned wave_sum = (unsigned)__shfl((int)before, 63);
        before -= mine;
        if (lane == 0) part[side][wave] = wave_sum;
        __syncthreads();
        unsigned sum = 0;
#pragma unroll
        for (int w = 0; w < PK_W; ++w) {
            if (w < wave) before += part[side][w];
            sum += part[side][w];
        }
        side ^= 1;
        unsigned sure = sure0 + (before & 0xffffu), tie = tie0 + (before >> 16);
#pragma unroll
        for (int k = 0; k < PK_KPT; ++k) {
            const int at = at0 + k;
            const bool in = at < n && (at < first || at >= last || key[k] > t);
            const bool eq = !in && at < n && t != 0u && key[k] == t;
            if (in || (eq && tie < ties)) out[sure + min(tie, ties)] = at;
            sure += in;
            tie += eq;
        }
        sure0 += sum & 0xffffu;
        tie0 += sum >> 16;
    }
    for (unsigned i = sure0 + min(tie0, ties) + tid; i < (unsigned)a.count; i += PK_NT) out[i] = -1;
}

template <int D>
static const void* bounds_fn(int kv) {
    return kv == VIPER_KV_INT8  ? (const void*)page_bounds_kernel<D, VIPER_KV_INT8>
           : kv == VIPER_KV_FP4 ? (const void*)page_bounds_kernel<D, VIPER_KV_FP4>
                                : (const void*)page_bounds_kernel<D, VIPER_KV_BF16>;
}

static size_t bounds_bytes(const viper_kv_cache* c) { return (size_t)c->num_pages * c->kv_heads * c->head_dim * 4; }
static bool ranges_meet(const void* p, size_t n, const void* o, size_t m) {
    return n != 0 && m != 0 && (uintptr_t)p < (uintptr_t)o + m && (uintptr_t)o < (uintptr_t)p + n;
}

static int select_check(const viper_kv_cache* c, const viper_kv_batch* b, int heads, int count) {
    const int rc = kv_check(c, b);
    if (rc != VIPER_OK) return rc;
    if (b->max_rows > VIPER_QLINEAR_MAX_M) return VIPER_INVALID_ARGUMENT;
    if (heads <= 0 || heads % c->kv_heads != 0 || heads / c->kv_heads > 64) return VIPER_INVALID_ARGUMENT;
    return count > 0 && (int64_t)count * c->page_size <= INT32_MAX ? VIPER_OK : VIPER_INVALID_ARGUMENT;
}
static size_t select_bytes(const viper_kv_cache* c, const viper_kv_batch* b) {
    return (size_t)b->batch * b->max_rows * c->kv_heads * b->table_width * 4;
}

}  // namespace vq

extern "C" int viper_hip_kv_page_bounds(const viper_kv_cache* cache, const viper_kv_batch* batch, void* bounds_bf16, void* stream) {
    using namespace vq;
    const int rc = kv_check(cache, batch);
    if (rc != VIPER_OK) return rc;
    if (bounds_bf16 == nullptr || misaligned(bounds_bf16, 16)) return VIPER_INVALID_ARGUMENT;
    const size_t keys = bounds_bytes(cache) / 4 * cache->page_size * (cache->kv_type == VIPER_KV_BF16 ? 2 : 1) /
                        (cache->kv_type == VIPER_KV_FP4 ? 2 : 1);
    if (ranges_meet(bounds_bf16, bounds_bytes(cache), cache->k, keys)) return VIPER_INVALID_ARGUMENT;
    if (batch->total_rows == 0) return VIPER_OK;
    BoundsArgs a;
    a.c = kv_args(cache, batch);
    a.c.max_rows = batch->max_rows < batch->total_rows ? batch->max_rows : batch->total_rows;
    a.out = (uint16_t*)bounds_bf16;
    a.span = (int)(((int64_t)a.c.max_rows + cache->page_size - 2) / cache->page_size + 1);
    const int64_t grid = (int64_t)batch->batch * a.span * cache->kv_heads;
    if (grid >= 1 << 24) return VIPER_INVALID_ARGUMENT;
    const int D = cache->head_dim, kv = cache->kv_type;
    void* args[] = {&a};
    launch(D == 64 ? bounds_fn<64>(kv) : D == 128 ? bounds_fn<128>(kv) : bounds_fn<256>(kv), (unsigned)grid, D == 64 ? 128 : 256, 0,
           (hipStream_t)stream, args);
    return status_of(hipGetLastError());
}

extern "C" size_t viper_hip_select_pages_workspace_bytes(const viper_kv_cache* cache, const viper_kv_batch* batch, int heads, int count) {
    return vq::select_check(cache, batch, heads, count) == VIPER_OK ? vq::select_bytes(cache, batch) : 0;
}

extern "C" int viper_hip_select_pages(const viper_kv_cache* cache, const viper_kv_batch* batch, const void* q_bf16, int64_t q_stride,
                                      int heads, const void* bounds_bf16, int first, int last, int32_t* selected, int count,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    using namespace vq;
    int rc = select_check(cache, batch, heads, count);
    if (rc != VIPER_OK) return rc;
    const int D = cache->head_dim;
    const int64_t width = (int64_t)heads * D;
    if (bad_rows(q_bf16, q_stride, width) || bounds_bf16 == nullptr || misaligned(bounds_bf16, 16)) return VIPER_INVALID_ARGUMENT;
    if (first < 0 || last < 1 || (int64_t)first + last > count || selected == nullptr || misaligned(selected, 4))
        return VIPER_INVALID_ARGUMENT;
    const size_t need = select_bytes(cache, batch);
    if (workspace == nullptr || misaligned(workspace, 16) || workspace_bytes < need) return VIPER_INVALID_ARGUMENT;
    if (batch->total_rows == 0) return VIPER_OK;
    const size_t n = (size_t)batch->total_rows, lists = n * cache->kv_heads * count * 4, rows = ((n - 1) * q_stride + width) * 2;
    if (ranges_meet(selected, lists, q_bf16, rows) || ranges_meet(selected, lists, bounds_bf16, bounds_bytes(cache)) ||
        ranges_meet(selected, lists, workspace, need) || ranges_meet(workspace, need, q_bf16, rows) ||
        ranges_meet(workspace, need, bounds_bf16, bounds_bytes(cache)))
        return VIPER_INVALID_ARGUMENT;
    SelectArgs a;
    a.c = kv_args(cache, batch);
    a.q = (const uint16_t*)q_bf16;
    a.q_stride = q_stride;
    a.bounds = (const uint16_t*)bounds_bf16;
    a.out = selected;
    a.keys = (uint32_t*)workspace;
    a.gqa = heads / cache->kv_heads;
    a.count = count;
    a.first = first;
    a.last = last;
    const int pp = PS_NT / (D / 8), turn = PS_LDS / (a.gqa * D * 2) > 1 ? PS_LDS / (a.gqa * D * 2) : 1;
    const int held = turn < batch->max_rows ? turn : batch->max_rows;
    void* args[] = {&a};
    const dim3 grid((unsigned)((batch->table_width + pp - 1) / pp), (unsigned)cache->kv_heads, (unsigned)batch->batch);
    if ((int64_t)grid.x * grid.y * grid.z >= 1 << 24) return VIPER_INVALID_ARGUMENT;
    const void* fn = D == 64 ? (const void*)page_score_kernel<64> : D == 128 ? (const void*)page_score_kernel<128> : (const void*)page_score_kernel<256>;
    (void)hipLaunchKernel(fn, grid, dim3(PS_NT), args, (size_t)held * a.gqa * D * 2, (hipStream_t)stream);
    rc = status_of(hipGetLastError());
    if (rc != VIPER_OK) return rc;
    (void)hipLaunchKernel((const void*)page_pick_kernel, dim3((unsigned)batch->max_rows, grid.y, grid.z), dim3(PK_NT), args, 0,
                          (hipStream_t)stream);
    return status_of(hipGetLastError());
}
