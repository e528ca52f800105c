// Which pages of a long sequence a row is to look at.
//
// bounds: per page and key head the least and largest value of every dimension over the
// keys held.  bf16 patterns are compared as 16-bit integers in the values' order, two at
// a time, where NaN lies past the infinities and so is not lost.
//
// selection: q . k of any key of a page is at most sum_d max(q_d lo_d, q_d hi_d), the page's
// score for a query head; the largest over the heads of a key head counts.  (Keys as kv_read
// gives them: int8 keys are bounded after their rounding to bf16, which attention does not
// make, so there q . k may be larger by 2^-8 sum_d |q_d k_d|: a page that close to the border
// may be taken for a lesser one, and what is listed is the same on every run.)  A page at the
// border is in or out, so a score is that of the sum in 64 bits.  One launch has all scores
// as matrix products in 32 bits, with a limit to how far they may be off; a second finds the
// border among them and computes in 64 bits only the pages too near to it.
//
// Measured (20 heads over 4 key heads of 128 dims): 64 of 2048 pages for one row 8.6 us
// (scores 4.4, selection 5.2: latency); 128 of up to 2032 for 4 rows of 16 sequences 21.2
// (13.0 and 8.4; 38 MB of bounds, 5.7 us at 6.7 TB/s); all scores in 64 bits took 48.  A row
// and key head with a score that is no finite number (a NaN key), or with more than 64 pages
// in doubt (equal ones), has all pages scored in 64 bits by its one workgroup: 1.05 ms and 1.15.

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
constexpr int DPP_ROR8 = 0x128;  // lane i <- i ^ 8 within 16

// A wave takes a page of a key head (of pages of several tiles two or four waves, which
// meet in LDS) with the tile's 16-byte loads.  The least and, complemented, the largest of a
// lane's token are R registers; each step of the way over the 16 lanes of other tokens
// halves them, a lane keeping the half that one bit of its number says.  3 prompts of
// 20000 tokens in pages of 32, int8, take 9.1 us (16.5 MB, 2.5 us at 6.7 TB/s: 820 VALU
// instructions in each of the 3500 waves that have a page are 5 us of issue), one decode row
// of 16 sequences 3.3; 4 pages to a workgroup of one wave for each 32 dims took 11.5.
template <int D, int KT>
__global__ void __launch_bounds__(PB_NT)
page_bounds_kernel(BoundsArgs a) {
    constexpr int NKB = D / 32, R = 8 * NKB, N = R / 16;
    __shared__ uint32_t lv[PB_NT / 64][64][N];
    const int tid = (int)threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wl = min(a.c.tpl, 2), part = wave & ((1 << wl) - 1);
    int64_t id = ((int64_t)blockIdx.x * (PB_NT / 64) + wave) >> wl;
    const int head = (int)(id % a.c.kvh);
    id /= a.c.kvh;
    const int b = (int)(id / a.span);
    const KvSeq s = b < a.c.batch ? kv_seq(a.c, b) : KvSeq{0, 0, 0};
    const int from = max(0, s.len - s.n), shift = a.c.tpl + 5;
    const int64_t page64 = (int64_t)(from >> shift) + id % a.span;
    const bool live = s.n > 0 && page64 << shift < s.len;
    const int tile0 = live ? (int)(page64 << a.c.tpl) : 0;
    const int tiles = live ? min(1 << a.c.tpl, (s.len - 1) / KV_TILE - tile0 + 1) : 0;
    const int page = live ? kv_page_uniform(a.c, b, tile0) : -1;
    // words [side][32 dims][pair of dims], of the largest the complement: all are made smaller
    uint32_t v[R];
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = 0x7fff7fffu;
    for (int tl = part; tl < tiles && page >= 0; tl += 1 << wl) {
        const size_t at = kv_tile_at(a.c, page, head, tl);
        u32x4 x[NKB][2];
        if constexpr (KT == VIPER_KV_BF16) {
            const u32x4* const p = (const u32x4*)((const uint16_t*)a.c.k + at * (KV_TILE * D)) + lane;
#pragma unroll
            for (int i = 0; i < 2 * NKB; ++i) x[i >> 1][i & 1] = p[64 * i];
        } else if constexpr (KT == VIPER_KV_INT8) {
            const u32x4* const p = (const u32x4*)((const int8_t*)a.c.k + at * (KV_TILE * D)) + lane;
            u32x4 w[NKB];
#pragma unroll
            for (int i = 0; i < NKB; ++i) w[i] = p[64 * i];
            float sc[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) sc[h] = a.c.ks[at * KV_TILE + 8 * (m >> 2) + 4 * h + (m & 3)];
#pragma unroll
            for (int i = 0; i < NKB; ++i) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {  // dims 64 (i / 2) + 32 k + 8 g ..
                    float y[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[j] = (float)(int8_t)(w[i][2 * k + (j >> 2)] >> (8 * (j & 3))) * sc[i & 1];
                    x[2 * (i >> 1) + k][i & 1] = u32x4{f2bf2(y[0], y[1]), f2bf2(y[2], y[3]), f2bf2(y[4], y[5]), f2bf2(y[6], y[7])};
                }
            }
        } else {
            const u32x4* const p = (const u32x4*)((const uint8_t*)a.c.k + at * (KV_TILE * D / 2)) + lane;
            const uint8_t* const e = (const uint8_t*)a.c.ks + at * D;
            u32x4 w[D / 64];
#pragma unroll
            for (int i = 0; i < D / 64; ++i) w[i] = p[64 * i];
            const uint32_t ex = D == 256 ? *(const uint32_t*)(e + 4 * lane) : *(const uint16_t*)(e + (D == 64 ? 2 * (16 * (g >> 1) + m) : 2 * lane));
#pragma unroll
            for (int kb = 0; kb < NKB; ++kb) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    x[kb][h] = fp4_bf16(D == 64 ? w[0][2 * h + kb] : w[2 * (kb >> 2) + h][kb & 3],
                                        fp4_power((ex >> (8 * (2 * (kb >> 2) + h))) & 0xffu));
            }
        }
        const bool whole = (tile0 + tl + 1) * KV_TILE <= s.len;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool held = whole || (tile0 + tl) * KV_TILE + 8 * (m >> 2) + 4 * h + (m & 3) < s.len;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t u = pb_order(x[kb][h][i]);
                    v[4 * kb + i] = pb_min(v[4 * kb + i], held ? u : 0x7fff7fffu);
                    v[4 * (NKB + kb) + i] = pb_min(v[4 * (NKB + kb) + i], held ? ~u : 0x7fff7fffu);
                }
            }
        }
    }
    auto halve = [&](auto dpp, bool upper, int half) {
#pragma unroll
        for (int i = 0; i < R / 2; ++i) {
            if (i >= half) continue;
            const uint32_t keep = upper ? v[i + half] : v[i], send = upper ? v[i] : v[i + half];
            v[i] = pb_min(keep, (uint32_t)dpp((int)send));
        }
    };
    // (the half mirror turns the lower bits too: it comes before they choose)
    halve([](int x) { return dpp_i<DPP_ROR8>(x); }, m & 8, R / 2);
    halve([](int x) { return dpp_i<DPP_HALF_MIRROR>(x); }, m & 4, R / 4);
    halve([](int x) { return dpp_i<DPP_SWAP2>(x); }, m & 2, R / 8);
    halve([](int x) { return dpp_i<DPP_SWAP1>(x); }, m & 1, R / 16);
    if (wl > 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) lv[wave][lane][i] = v[i];
        __syncthreads();
        if (part != 0) return;
        for (int w = 1; w < 1 << wl; ++w) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = pb_min(v[i], lv[wave + w][lane][i]);
        }
    }
    if (page < 0) return;
    // word `first` of the lane's N: its side, 32 dims and pair
    const int first = (m >> 2 & 1) * (R / 4) + (m >> 1 & 1) * (R / 8) + (m & 1) * (R / 16), kb = first / 4;
    const int dim = (KT == VIPER_KV_FP4 ? q4_dim<D>(kb, g) : 32 * kb + 8 * g) + 2 * (first & 3);
    uint32_t* const out = (uint32_t*)(a.out + (((size_t)page * a.c.kvh + head) * 2 + (m >> 3)) * D + dim);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t mine = pb_order(m & 8 ? ~v[i] : v[i]), other = (uint32_t)dpp_i<DPP_ROR8>((int)mine);
        // a NaN key makes both NaN
        auto nan = [](uint32_t w) { return (w & 0x7fffu) > 0x7f80u; };
        uint32_t w = mine;
        if (nan(mine) || nan(other)) w = (w & 0xffff0000u) | 0x7fc0u;
        if (nan(mine >> 16) || nan(other >> 16)) w = (w & 0xffffu) | 0x7fc00000u;
        out[i] = w;
    }
}

// ----------------------------------------------------------------- scores

struct SelectArgs {
    KvArgs c;
    const uint16_t* q;
    int64_t q_stride;
    const uint16_t* bounds;
    int32_t* out;
    uint32_t* keys;  // [batch * max_rows][key head][width]
    uint32_t* off;   // [batch * max_rows][key head][tiles]: how far the scores of 16 pages may be off (fp32 patterns)
    int gqa, count, first, last;
    int cols, shift;  // a row's gqa queries, padded to 2^shift from 4 (shift 5: to a multiple of 16)
    int tiles;  // of 16 pages
};

// Pages of the row at position p (0: no token)
__device__ __forceinline__ int ps_pages(const KvArgs& c, int64_t p) {
    return p < 0 ? 0 : (int)min((int64_t)c.width, (p >> (c.tpl + 5)) + 1);
}
// A score as an integer in its order, above 0; NaN as +inf
constexpr uint32_t PS_INF = 0xff800000u, PS_NINF = 0x007fffffu;
__device__ __forceinline__ uint32_t ps_key(float v) {
    if (v != v) v = __builtin_inff();
    const uint32_t u = __float_as_uint(v);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float ps_score(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }
__device__ __forceinline__ size_t ps_row(const SelectArgs& a, int b, int r, int head) {
    return (size_t)(b * a.c.max_rows + r) * a.c.kvh + head;
}

// Scores in 32 bits, sum_d max(q_d, 0) hi_d + min(q_d, 0) lo_d, as products of 16 pages and
// 16 queries over 32 dims at a time whose sums are added one after the other.  In whatever
// order a product adds its 32 terms, and if it truncates, a sum is off by at most 32 2^-23 of
// the sum of its terms' magnitudes; the 2 D / 32 <= 16 additions add 16 2^-24 of all.
// PS_OFF is above these 40 2^-23 by a fifth, which covers the rounding of the magnitudes' sum
// and of what a score is compared with.  Values and products under 2^-126 may count as zero:
// magnitudes are taken as 2^-100 at least, and 2^-117 is added.  page_pick_kernel computes
// the few pages that are too near to the border for that in 64 bits.
constexpr float PS_OFF = 48 * 0x1p-23f, PS_OFF_MIN = 0x1p-117f;
typedef __bf16 ps_bf16x8 __attribute__((ext_vector_type(8)));
typedef float ps_f32x4 __attribute__((ext_vector_type(4)));
constexpr int PS_NT = 256;

// A wave takes 16 pages and all rows of its sequence.  Queries are the rows of the products, so
// that the heads of a row meet in a lane's registers (as columns 2.5 us longer in the batch above).
// Bounds are read in whole rows of 4 D bytes and turned in LDS, its 16 bytes in an order by
// page that spreads the banks (operands loaded as they are, 64 bytes of 16 pages at a time, take
// 2.4 us longer over 38 MB), and queries are read once for the four waves.  Of the batch's 13
// us 2.3 are an empty dispatch, 5.5 the loads and 5 the products' and sums' issue, which few
// loads cover, as all waves start together (two tiles to a wave, or fewer waves that go on to
// further tiles, were no faster).
template <int D>
__global__ void __launch_bounds__(PS_NT)
page_score_kernel(SelectArgs a) {
    constexpr int NKB = D / 32, PC = D / 4, QC = D / 8, NL = 16 * PC / 64, QX = QC < 16 ? QC - 1 : 15;  // PC, QC: 16 bytes of a page, a query
    constexpr int NQ = 16 * QC < PS_NT ? 1 : 16 * QC / PS_NT;
    __shared__ u32x4 lb[PS_NT / 64][16 * PC];
    __shared__ u32x4 lq[2][16 * QC];
    const int tid = (int)threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int chunk = (int)blockIdx.x / a.c.kvh, head = (int)blockIdx.x - chunk * a.c.kvh, b = (int)blockIdx.z;
    const int tile = chunk * (PS_NT / 64) + wave;
    const int entry = tile * 16 + m < a.c.width ? a.c.table[(size_t)b * a.c.width + tile * 16 + m] : -1;
    const KvSeq s = kv_seq(a.c, b);
    const int64_t pos0 = (int64_t)s.len - s.n;
    const int last = s.n == 0 ? 0 : ps_pages(a.c, (int64_t)s.len - 1);
    if (chunk * (PS_NT / 64) * 16 >= last) return;
    const bool live = tile * 16 < last;
    // a row's queries, padded with its last one, are the rows of the products, 16 to a turn
    const int shift = min(a.shift, 4), per = 1 << shift;
    int r0 = 0, h0 = 0;  // of a turn: query i is head h0 + i % per of row r0 + i / per
    auto advance = [&] {
        h0 += 16;
        if (h0 < a.cols) return;
        h0 = 0;
        r0 += 16 >> shift;
    };
    u32x4 next[NQ];
    auto load_q = [&] {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int at = tid + i * PS_NT;
            if (16 * QC < PS_NT && at >= 16 * QC) continue;
            const int r = min(r0 + (at / QC >> shift), s.n - 1), h = min(h0 + (at / QC & (per - 1)), a.gqa - 1);
            next[i] = *(const u32x4*)(a.q + (size_t)(s.row0 + r) * a.q_stride + (head * a.gqa + h) * D + 8 * (at % QC));
        }
    };
    auto store_q = [&](u32x4* to) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int at = tid + i * PS_NT, n = at / QC;
            if (16 * QC < PS_NT && at >= 16 * QC) continue;
            to[n * QC + (at % QC ^ (n & QX))] = next[i];
        }
    };
    load_q();
    const bool there = (unsigned)entry < (unsigned)a.c.pages;
    u32x4 lo[NKB], hi[NKB], rows[NL];
    if (live) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int n = (i * 64 + lane) / PC, c = (i * 64 + lane) % PC;
            const int e = __shfl(there ? entry : 0, n);
            rows[i] = *(const u32x4*)(a.bounds + ((size_t)e * a.c.kvh + head) * (2 * D) + 8 * c);
        }
    }
    store_q(lq[0]);
    __syncthreads();
    if (live) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int n = (i * 64 + lane) / PC, c = (i * 64 + lane) % PC;
            lb[wave][n * PC + (c ^ n)] = rows[i];
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
            lo[kb] = lb[wave][m * PC + ((4 * kb + g) ^ m)];
            hi[kb] = lb[wave][m * PC + ((QC + 4 * kb + g) ^ m)];
        }
    }
    constexpr uint32_t LEAST = 0x0d800d80u;  // 2^-100
    auto of = [](const u32x4& v) { return __builtin_bit_cast(ps_bf16x8, v); };
    float best = 0.0f;
    uint32_t off = 0;
#pragma unroll 1
    for (int turn = 0;; turn ^= 1) {
        const int r = r0 + (4 * g >> shift), h = h0 + (4 * g & (per - 1));
        advance();
        const bool more = r0 < s.n;
        if (more) load_q();
        if (live) {
            const ps_f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
            ps_f32x4 S = zero, Q = zero;
#pragma unroll
            for (int kb = 0; kb < NKB; ++kb) {
                const u32x4 q = lq[turn][m * QC + ((4 * kb + g) ^ (m & QX))];
                u32x4 up, dn, mag, most;  // most: the larger magnitude of either bound
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // (as integers, values with a sign are under 0)
                    up[i] = pb_max(q[i], 0u);
                    dn[i] = pb_min(q[i], 0u);
                    mag[i] = pb_max(q[i] & 0x7fff7fffu, LEAST);
                    most[i] = pb_max(pb_max(lo[kb][i] & 0x7fff7fffu, hi[kb][i] & 0x7fff7fffu), LEAST);
                }
                S += __builtin_amdgcn_mfma_f32_16x16x32_bf16(of(up), of(hi[kb]), zero, 0, 0, 0);
                S += __builtin_amdgcn_mfma_f32_16x16x32_bf16(of(dn), of(lo[kb]), zero, 0, 0, 0);
                Q = __builtin_amdgcn_mfma_f32_16x16x32_bf16(of(mag), of(most), Q, 0, 0, 0);
            }
            // The lane's four queries are of one row, whose others lie 16 and 32 lanes further and in
            // further turns.  A score that is no number has a Q that is not finite, and as
            // patterns NaN and infinity are the largest of these: pages in 64 bits then.
            float v = fmaxf(fmaxf(S[0], S[1]), fmaxf(S[2], S[3]));
            uint32_t e = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) e = max(e, __float_as_uint(Q[i]) & 0x7fffffffu);
            if (shift >= 3) {
                auto w = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
                v = fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
                w = __builtin_amdgcn_permlane16_swap(e, e, false, false);
                e = max(w[0], w[1]);
            }
            if (shift >= 4) {
                auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
                v = fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
                w = __builtin_amdgcn_permlane32_swap(e, e, false, false);
                e = max(w[0], w[1]);
            }
            if (h >= 16) {
                v = fmaxf(v, best);
                e = max(e, off);
            }
            best = v;
            off = e;
            e = there ? e : 0u;  // over the tile's pages
            e = max(e, (uint32_t)dpp_i<DPP_SWAP1>((int)e));
            e = max(e, (uint32_t)dpp_i<DPP_SWAP2>((int)e));
            e = max(e, (uint32_t)dpp_i<DPP_HALF_MIRROR>((int)e));
            e = max(e, (uint32_t)dpp_i<DPP_MIRROR>((int)e));
            const int p = tile * 16 + m, pages = ps_pages(a.c, pos0 + r);
            if ((h & 15) == 0 && (h + 16 >= a.cols) && r < s.n && tile * 16 < pages) {
                const size_t row = ps_row(a, b, r, head);
                if (p < pages) a.keys[row * a.c.width + p] = there ? ps_key(v) : 0u;
                if (m == 0) a.off[row * a.tiles + tile] = __float_as_uint(__uint_as_float(e) * PS_OFF + PS_OFF_MIN);
            }
        }
        if (!more) break;
        store_q(lq[turn ^ 1]);
        __syncthreads();
    }
}

// ----------------------------------------------------------------- selection

constexpr int PK_NT = 512, PK_W = PK_NT / 64, PK_BINS = 1024, PK_LIST = 64;

__device__ __forceinline__ double wave_sum(double v) {
    auto step = [&](auto f) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        uint32_t a[2], b[2];
        f((uint32_t)u, a);
        f((uint32_t)(u >> 32), b);
        v = __builtin_bit_cast(double, (uint64_t)b[0] << 32 | a[0]) + __builtin_bit_cast(double, (uint64_t)b[1] << 32 | a[1]);
    };
    auto dpp = [&](auto f) { step([&](uint32_t x, uint32_t* y) { y[0] = x; y[1] = (uint32_t)f((int)x); }); };
    dpp([](int x) { return dpp_i<DPP_SWAP1>(x); });
    dpp([](int x) { return dpp_i<DPP_SWAP2>(x); });
    dpp([](int x) { return dpp_i<DPP_HALF_MIRROR>(x); });
    dpp([](int x) { return dpp_i<DPP_MIRROR>(x); });
    step([](uint32_t x, uint32_t* y) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        y[0] = r[0], y[1] = r[1];
    });
    step([](uint32_t x, uint32_t* y) {
        const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        y[0] = r[0], y[1] = r[1];
    });
    return v;
}
// The score of a page for one query head by a wave: products are exact in 32 bits, sums in 64
__device__ __forceinline__ uint32_t page_exact(const uint16_t* at, const uint16_t* q, int D) {
    const int lane = (int)threadIdx.x & 63;
    uint32_t x[4], lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + 64 * i;
        x[i] = lo[i] = hi[i] = 0u;
        if (d < D) {
            x[i] = q[d];
            lo[i] = at[d];
            hi[i] = at[D + d];
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double y = (double)bf16f(x[i]), u = y * (double)bf16f(lo[i]), v = y * (double)bf16f(hi[i]);
        sum += u != u || v != v ? __builtin_nan("") : fmax(u, v);
    }
    return ps_key((float)wave_sum(sum));
}

// Least / largest over a wave
template <bool MAX>
__device__ __forceinline__ uint32_t wave_most(uint32_t v) {
    auto of = [](uint32_t x, uint32_t y) { return MAX ? max(x, y) : min(x, y); };
    v = of(v, (uint32_t)dpp_i<DPP_SWAP1>((int)v));
    v = of(v, (uint32_t)dpp_i<DPP_SWAP2>((int)v));
    v = of(v, (uint32_t)dpp_i<DPP_HALF_MIRROR>((int)v));
    v = of(v, (uint32_t)dpp_i<DPP_MIRROR>((int)v));
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = of(r[0], r[1]);
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return of(r[0], r[1]);
}

// A workgroup per row and key head.  A wave holds KPT 64 consecutive pages, a lane every
// 64th of them, so that ballots count and number them in order (MULTI: there are more
// pages than the workgroup holds, and keys are read again at each step).  The border is
// found through a histogram of the keys between the least and the largest, then within
// the bin that holds it; once few keys are left they are ranked.  Every wave does so for
// itself from what is in LDS: each step costs one barrier.  Bound by the latency of its
// steps; run once and straight on, also by that of its own code: hence small variants.
template <int KPT, bool MULTI>
__global__ void __launch_bounds__(PK_NT)
page_pick_kernel(SelectArgs a, int D) {
    __shared__ __align__(16) unsigned hist[3][PK_BINS];  // (one is cleared while another may still be read)
    __shared__ uint32_t part[2][4][PK_W];
    __shared__ uint32_t list_key[PK_LIST];
    __shared__ int list_page[PK_LIST];
    __shared__ unsigned listed;
    constexpr int ALL = PK_NT * KPT;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = (int)blockIdx.x, head = (int)blockIdx.y, b = (int)blockIdx.z;
    uint32_t* const keys = a.keys + ps_row(a, b, r, head) * a.c.width;
    const auto kbuf = buf(keys, (uint32_t)a.c.width * 4);  // (past the end: 0)
    const uint32_t* const offs = a.off + ps_row(a, b, r, head) * a.tiles;
    // the first keys are asked for before the sequence's length is known
    uint32_t key[KPT];
    const int at0 = wave * (KPT * 64) + lane;
#pragma unroll
    for (int k = 0; k < KPT; ++k) key[k] = bload4(kbuf, (at0 + 64 * k) * 4);
    uint32_t err = bload4(buf(offs, (uint32_t)a.tiles * 4), tid * 4);
    const KvSeq s = kv_seq(a.c, b);
    if (r >= s.n) return;
    const int n = ps_pages(a.c, (int64_t)s.len - s.n + r);
    const int first = min(a.first, n), last = max(first, n - a.last);  // [first, last) is ranked, the others are in
    const size_t row = (size_t)s.row0 + r;
    int32_t* const out = a.out + (row * a.c.kvh + head) * a.count;
    const unsigned want = (unsigned)(a.count - (n - (last - first)));  // of the ranked ones (first + last <= count)
    const int turns = MULTI ? (n + ALL - 1) / ALL : 1;
    auto ranked = [&](int at) { return (unsigned)(at - first) < (unsigned)(last - first); };
#pragma unroll
    for (int k = 0; k < KPT; ++k) key[k] = ranked(at0 + 64 * k) ? key[k] : 0u;
    // (patterns of values that are not under 0 are in their order, NaN the largest)
    err = tid * 16 < n ? err : 0u;
    if (MULTI)
        for (int i = PK_NT + tid; i * 16 < n; i += PK_NT) err = max(err, offs[i]);
    auto each = [&](auto f) {  // over the thread's keys of all turns: f(k, page)
        for (int turn = 0; turn < turns; ++turn) {
#pragma unroll
            for (int k = 0; k < KPT; ++k) {
                const int at = turn * ALL + at0 + 64 * k;
                if (MULTI) key[k] = ranked(at) ? bload4(kbuf, at * 4) : 0u;
            }
#pragma unroll
            for (int k = 0; k < KPT; ++k) f(k, turn * ALL + at0 + 64 * k);
        }
    };
    int side = 0;
    // A wave's two counts as all waves': those of the waves before it and of all
    auto meet = [&](unsigned x, unsigned y, unsigned* before, unsigned* all) {
        if (lane == 0) {
            part[side][0][wave] = x;
            part[side][1][wave] = y;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // (a lane to each wave's)
            const unsigned c = part[side][i][lane & (PK_W - 1)], upto = wave_upto(c);
            before[i] = wave == 0 ? 0u : (unsigned)__builtin_amdgcn_readlane((int)upto, (wave - 1) & (PK_W - 1));
            all[i] = (unsigned)__builtin_amdgcn_readlane((int)upto, PK_W - 1);
        }
        side ^= 1;
    };

    const unsigned all_want = want + (unsigned)(n - (last - first));
    // keys over `above` are in, and of those from `from` on so many as to have `want`
    uint32_t above = 0u, from = 1u;
    for (bool exact = false, settled = false;; exact = true) {
        bool fine = true;
        if (!settled) {
            uint32_t least = 0xffffffffu, most = 0;
            unsigned there = 0;
            each([&](int k, int) {
                least = key[k] != 0u ? min(least, key[k]) : least;
                most = max(most, key[k]);
                there += (unsigned)__popcll(__ballot(key[k] != 0u));
            });
            least = wave_most<false>(least);
            most = wave_most<true>(most);
            err = wave_most<true>(err);
            if (lane == 0) {
                part[side][0][wave] = least;
                part[side][1][wave] = most;
                part[side][2][wave] = err;
                part[side][3][wave] = there;
            }
            for (int i = tid; i < PK_BINS; i += PK_NT) hist[0][i] = 0u;
            if (tid == 0) listed = 0u;
            __syncthreads();
            const int w = lane & (PK_W - 1);
            least = wave_most<false>(part[side][0][w]);
            most = wave_most<true>(part[side][1][w]);
            err = wave_most<true>(part[side][2][w]);
            there = (unsigned)__builtin_amdgcn_readlane((int)wave_upto(part[side][3][w]), PK_W - 1);
            side ^= 1;
            const float e2 = 2.0f * __uint_as_float(err);
            if (want == 0u) {
                above = from = 0xffffffffu;
            } else if (there > want) {  // (else all that are there)
                // (sums that are not finite: all pages in 64 bits)
                fine = exact || (least > PS_NINF && most < PS_INF && e2 < 0x1p100f);
                uint32_t lo = least, hi = fine ? most : least;
                unsigned left = want;  // of the keys lo .. hi
                for (int level = 0; lo != hi; ++level) {
                    unsigned* const h = hist[level % 3];
                    const int shift = max(0, 22 - (int)__clz((int)((hi - lo) | 1u)));
                    each([&](int k, int) {
                        if (key[k] >= lo && key[k] <= hi) atomicAdd(&h[(key[k] - lo) >> shift], 1u);
                    });
                    for (int i = tid; i < PK_BINS; i += PK_NT) hist[(level + 1) % 3][i] = 0u;
                    __syncthreads();
                    // the bin of the left-th key from above: 16 bins to a lane, then a lane to each of those
                    constexpr int BPL = PK_BINS / 64;
                    const u32x4* const mine = (const u32x4*)&h[PK_BINS - BPL * (lane + 1)];
                    unsigned sum = 0;
#pragma unroll
                    for (int i = 0; i < BPL / 4; ++i) sum += mine[i].x + mine[i].y + mine[i].z + mine[i].w;
                    unsigned upto = wave_upto(sum);
                    int src = __ffsll((long long)__ballot(upto >= left)) - 1;
                    left -= (unsigned)__builtin_amdgcn_readlane((int)(upto - sum), src);
                    const int top = PK_BINS - 1 - BPL * src;
                    const unsigned one = lane < BPL ? h[top - lane] : 0u;
                    upto = wave_upto(one);
                    src = __ffsll((long long)__ballot(upto >= left)) - 1;
                    const unsigned held = (unsigned)__builtin_amdgcn_readlane((int)one, src);
                    left -= (unsigned)__builtin_amdgcn_readlane((int)upto, src) - held;
                    lo += (uint32_t)(top - src) << shift;
                    hi = shift == 0 ? lo : min(hi, lo + (1u << shift) - 1u);
                    if (lo != hi && held <= PK_LIST) {
                        each([&](int k, int) {
                            if (key[k] >= lo && key[k] <= hi) list_key[atomicAdd(&listed, 1u)] = key[k];
                        });
                        __syncthreads();
                        const uint32_t v = lane < (int)held ? list_key[lane] : 0u;
                        unsigned higher = 0, same = 0;
                        for (unsigned i = 0; i < held; ++i) {
                            const uint32_t x = (uint32_t)__builtin_amdgcn_readlane((int)v, i);
                            higher += x > v;
                            same += x == v;
                        }
                        const uint64_t is = __ballot(lane < (int)held && higher < left && higher + same >= left);
                        lo = hi = (uint32_t)__builtin_amdgcn_readlane((int)v, __ffsll((long long)is) - 1);
                    }
                }
                // lo is the want-th key, and the want-th score differs from it by e2 / 2 at most
                above = exact ? lo : ps_key(ps_score(lo) + e2);
                from = exact ? lo : ps_key(ps_score(lo) - e2);
            }
        }
        auto is_in = [&](int k, int at) { return at < n && (!ranked(at) || key[k] > above); };
        auto may_be = [&](int k) { return key[k] >= from && key[k] <= above; };
        unsigned sure = 0, may = 0, before[2], all[2];
        auto count = [&](int k, int at) {
            sure += (unsigned)__popcll(__ballot(is_in(k, at)));
            may += (unsigned)__popcll(__ballot(may_be(k)));
        };
        each(count);
        meet(sure, may, before, all);
        const unsigned need = min(all[1], all_want - all[0]), doubt = all[1];
        if (fine && (exact || need == doubt)) {  // numbers in order; of equal scores the first
            unsigned in0 = 0, may0 = 0, turn_all[2] = {0, 0};
            for (int turn = 0; turn < turns; ++turn) {
                if (MULTI) {
#pragma unroll
                    for (int k = 0; k < KPT; ++k) {
                        const int at = turn * ALL + at0 + 64 * k;
                        key[k] = ranked(at) ? bload4(kbuf, at * 4) : 0u;
                    }
                    sure = may = 0;
#pragma unroll
                    for (int k = 0; k < KPT; ++k) count(k, turn * ALL + at0 + 64 * k);
                    meet(sure, may, before, turn_all);
                }
                unsigned x = in0 + before[0], y = may0 + before[1];
#pragma unroll
                for (int k = 0; k < KPT; ++k) {
                    const int at = turn * ALL + at0 + 64 * k;
                    const bool i = is_in(k, at), e = may_be(k);
                    const uint64_t bi = __ballot(i), be = __ballot(e), under = (1ull << lane) - 1;
                    const unsigned xi = x + (unsigned)__popcll(bi & under), yi = y + (unsigned)__popcll(be & under);
                    if (i || (e && yi < need)) out[xi + min(yi, need)] = at;
                    x += (unsigned)__popcll(bi);
                    y += (unsigned)__popcll(be);
                }
                in0 += turn_all[0];
                may0 += turn_all[1];
            }
            for (unsigned i = all[0] + need + tid; i < (unsigned)a.count; i += PK_NT) out[i] = -1;
            return;
        }
        // scores in 64 bits, of the pages in doubt or, where those are too many, of all; a wave takes
        // a page for one head at a time, and the largest counts
        settled = fine && doubt <= PK_LIST;
        const int items = settled ? (int)doubt : last - first;
        if (settled) {
            if (tid == 0) listed = 0u;
            if (tid < PK_LIST) list_key[tid] = 0u;
            __syncthreads();
            each([&](int k, int at) {
                if (may_be(k)) list_page[atomicAdd(&listed, 1u)] = at;
            });
        } else {
            for (int i = tid; i < items; i += PK_NT) keys[first + i] = 0u;
        }
        __syncthreads();
        for (int i = 0, h = wave;; h += PK_W) {
            for (; h >= a.gqa; h -= a.gqa) ++i;
            if (i >= items) break;
            const int c = settled ? list_page[i] : first + i;
            const int page = a.c.table[(size_t)b * a.c.width + c];
            if ((unsigned)page >= (unsigned)a.c.pages) continue;
            const uint32_t v = page_exact(a.bounds + ((size_t)page * a.c.kvh + head) * (2 * D),
                                          a.q + row * a.q_stride + (size_t)(head * a.gqa + h) * D, D);
            if (lane != 0) continue;
            if (settled) atomicMax(&list_key[i], v);
            else atomicMax(&keys[c], v);
        }
        if (!settled) __threadfence();  // (keys are read back past the atomics)
        __syncthreads();
        if (settled) {  // in or out, by score and number
            const uint32_t v = lane < (int)doubt ? list_key[lane] : 0u;
            const int p = lane < (int)doubt ? list_page[lane] : 0x7fffffff;
            unsigned higher = 0;
            for (unsigned i = 0; i < doubt; ++i) {
                const uint32_t x = (uint32_t)__builtin_amdgcn_readlane((int)v, i);
                const int o = __builtin_amdgcn_readlane(p, i);
                higher += x > v || (x == v && o < p);
            }
            const uint64_t chosen = __ballot(lane < (int)doubt && higher < need);
            for (unsigned i = 0; i < doubt; ++i) {
                const int o = __builtin_amdgcn_readlane(p, i);
                const uint32_t x = (chosen >> i) & 1ull ? 0xffffffffu : 0u;
                if (MULTI) {
                    if (tid == 0) keys[o] = x;
                } else {
#pragma unroll
                    for (int k = 0; k < KPT; ++k) key[k] = at0 + 64 * k == o ? x : key[k];
                }
            }
            from = 0xffffffffu;
            above = min(above, 0xfffffffeu);
        }
        if (MULTI) {
            __syncthreads();
        } else if (!settled) {
#pragma unroll
            for (int k = 0; k < KPT; ++k) key[k] = ranked(at0 + 64 * k) ? bload4(kbuf, (at0 + 64 * k) * 4) : 0u;
        }
    }
}

template <int D>
static const void* bounds_fn(int kv) {
    return kv == VIPER_KV_INT8  ? (const void*)page_bounds_kernel<D, VIPER_KV_INT8>
           : kv == VIPER_KV_FP4 ? (const void*)page_bounds_kernel<D, VIPER_KV_FP4>
                                : (const void*)page_bounds_kernel<D, VIPER_KV_BF16>;
}

static size_t bounds_bytes(const viper_kv_cache* c) { return (size_t)c->num_pages * c->kv_heads * c->head_dim * 4; }
static int select_check(const viper_kv_cache* c, const viper_kv_batch* b, int heads, int count) {
    const int rc = kv_check(c, b);
    if (rc != VIPER_OK) return rc;
    if (b->max_rows > VIPER_QLINEAR_MAX_M) return VIPER_INVALID_ARGUMENT;
    if (heads <= 0 || heads % c->kv_heads != 0 || heads / c->kv_heads > 64) return VIPER_INVALID_ARGUMENT;
    return count > 0 && (int64_t)count * c->page_size <= INT32_MAX ? VIPER_OK : VIPER_INVALID_ARGUMENT;
}
static size_t select_bytes(const viper_kv_cache* c, const viper_kv_batch* b) {
    return (size_t)b->batch * b->max_rows * c->kv_heads * (b->table_width + ((size_t)b->table_width + 15) / 16) * 4;
}

}  // namespace vq

extern "C" int viper_hip_kv_page_bounds(const viper_kv_cache* cache, const viper_kv_batch* batch, void* bounds_bf16, void* stream) {
    using namespace vq;
    const int rc = kv_check(cache, batch);
    if (rc != VIPER_OK) return rc;
    if (bounds_bf16 == nullptr || misaligned(bounds_bf16, 16)) return VIPER_INVALID_ARGUMENT;
    const size_t keys = bounds_bytes(cache) / 4 * cache->page_size * (cache->kv_type == VIPER_KV_BF16 ? 2 : 1) /
                        (cache->kv_type == VIPER_KV_FP4 ? 2 : 1);
    const size_t rows = (size_t)cache->num_pages * cache->kv_heads * cache->page_size;
    const size_t scales = cache->kv_type == VIPER_KV_FP4 ? rows * (cache->head_dim / 32) : rows * 4;
    auto over = [&](const void* p, size_t n) { return p != nullptr && ranges_meet(bounds_bf16, bounds_bytes(cache), p, n); };
    if (over(cache->k, keys) || over(cache->v, keys) || over(cache->k_scales, scales) || over(cache->v_scales, rows * 4))
        return VIPER_INVALID_ARGUMENT;
    if (batch->total_rows == 0) return VIPER_OK;
    BoundsArgs a;
    a.c = kv_args(cache, batch);
    a.c.max_rows = batch->max_rows < batch->total_rows ? batch->max_rows : batch->total_rows;
    a.out = (uint16_t*)bounds_bf16;
    a.span = (int)(((int64_t)a.c.max_rows + cache->page_size - 2) / cache->page_size + 1);
    const int64_t units = (int64_t)batch->batch * a.span * cache->kv_heads;
    if (units >= 1 << 24) return VIPER_INVALID_ARGUMENT;
    const int waves = PB_NT / 64, per = waves >> (a.c.tpl < 2 ? a.c.tpl : 2);
    const int D = cache->head_dim, kv = cache->kv_type;
    void* args[] = {&a};
    launch(D == 64 ? bounds_fn<64>(kv) : D == 128 ? bounds_fn<128>(kv) : bounds_fn<256>(kv), (unsigned)((units + per - 1) / per), PB_NT, 0,
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
    if (q_stride > ((int64_t)1 << 48) / batch->total_rows) return VIPER_INVALID_ARGUMENT;  // (further than any memory)
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
    a.off = a.keys + (size_t)batch->batch * batch->max_rows * cache->kv_heads * batch->table_width;
    a.tiles = (batch->table_width + 15) / 16;
    a.gqa = heads / cache->kv_heads;
    a.count = count;
    a.first = first;
    a.last = last;
    a.shift = 2;
    while (a.shift <= 4 && 1 << a.shift < a.gqa) ++a.shift;
    a.cols = a.shift <= 4 ? 1 << a.shift : (a.gqa + 15) / 16 * 16;
    int d = D;
    void* args[] = {&a, &d};
    const int64_t chunks = (a.tiles + PS_NT / 64 - 1) / (PS_NT / 64);
    if (chunks * cache->kv_heads * batch->batch >= 1 << 24) return VIPER_INVALID_ARGUMENT;
    const dim3 grid((unsigned)(chunks * cache->kv_heads), 1, (unsigned)batch->batch);
    const void* score = D == 64 ? (const void*)page_score_kernel<64> : D == 128 ? (const void*)page_score_kernel<128> : (const void*)page_score_kernel<256>;
    (void)hipLaunchKernel(score, grid, dim3(PS_NT), args, 0, (hipStream_t)stream);
    rc = status_of(hipGetLastError());
    if (rc != VIPER_OK) return rc;
    const int w = batch->table_width;
    const void* pick = w <= PK_NT       ? (const void*)page_pick_kernel<1, false>
                       : w <= 2 * PK_NT ? (const void*)page_pick_kernel<2, false>
                       : w <= 4 * PK_NT ? (const void*)page_pick_kernel<4, false>
                       : w <= 8 * PK_NT ? (const void*)page_pick_kernel<8, false>
                                        : (const void*)page_pick_kernel<8, true>;
    (void)hipLaunchKernel(pick, dim3((unsigned)batch->max_rows, (unsigned)cache->kv_heads, grid.z), dim3(PK_NT), args, 0, (hipStream_t)stream);
    return status_of(hipGetLastError());
}
